"""Refusals of the calls over a cache in 8 bits or with a window, and the reference's own rounding,
on any machine."""
import os

import pytest

from omegalax_amd import _lib
from test_attn_host import BAD_CACHE, BIG, DECODE, PAGED, WRITE, _run

needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH),
                               reason="libomx_gdn.so not built (python -m omegalax_amd.build)")


def _put(args, after, before_ws=(), **more):
    """The arguments with `more` behind `after`, and `before_ws` before the workspace."""
    out = {}
    for name, x in args.items():
        if name == "ws":
            out.update(before_ws)
        out[name] = x
        if name == after:
            out.update(more)
    return out


SIGHT = dict(window=40, sinks=4)
WRITE8 = _put(WRITE, "v_pages", k_exps=16, v_exps=16)
PAGEDW = _put(PAGED, "v_pages", SIGHT, k_exps=16, v_exps=16)
DECODEW = _put(DECODE, "v_pages", SIGHT, k_exps=16, v_exps=16)
BAD_SIGHT = [(dict(window=-1), _lib.EINVAL, "window"), (dict(sinks=-1), _lib.EINVAL, "sinks"),
             (dict(window=0, sinks=3), _lib.EINVAL, "sinks")]
EXPS = [(dict(k_exps=None), _lib.EINVAL, "k_exps"), (dict(v_exps=None), _lib.EINVAL, "k_exps")]


@needs_lib
@pytest.mark.parametrize("over,code,msg", BAD_CACHE + [
    (dict(k=None), _lib.EINVAL, "NULL"), (dict(k=8), _lib.EINVAL, "aligned"), (dict(v_ld=128), _lib.EINVAL, "v_ld"),
    (dict(N=1), _lib.EINVAL, "N must equal B"), (dict(k_exps=None), _lib.EINVAL, "NULL"), (dict(v_exps=None), _lib.EINVAL, "NULL"),
    (dict(B=1 << 27, N=1 << 27, T=1, Hkv=32, k_ld=4096, v_ld=4096), _lib.EINVAL, "grid too large"),
])
def test_append_refuses(over, code, msg):
    rc, err = _run("omx_gdn_kv_write8", WRITE8, over)
    assert rc == code and msg in err


@needs_lib
@pytest.mark.parametrize("over,code,msg", BAD_CACHE + BAD_SIGHT + EXPS + [
    (dict(q=None), _lib.EINVAL, "NULL"), (dict(o=8), _lib.EINVAL, "aligned"), (dict(scale=0.0), _lib.EINVAL, "scale"),
    (dict(width=100, page=64, window=0, sinks=0), _lib.EINVAL, "workspace"),
    (dict(width=100, page=64, window=5000), _lib.EINVAL, "workspace")])
def test_paged_attention_refuses(over, code, msg):
    rc, err = _run("omx_gdn_attn_paged_window", PAGEDW, over)
    assert rc == code and msg in err


@needs_lib
@pytest.mark.parametrize("over,code,msg", BAD_CACHE + BAD_SIGHT + EXPS + [
    (dict(q=None), _lib.EINVAL, "NULL"), (dict(out=8), _lib.EINVAL, "aligned"), (dict(k_ld=128), _lib.EINVAL, "k_ld"),
    (dict(width=100, page=64, window=0, sinks=0), _lib.EINVAL, "workspace")])
def test_decode_refuses(over, code, msg):
    rc, err = _run("omx_gdn_attn_decode_window", DECODEW, over)
    assert rc == code and msg in err


@needs_lib
@pytest.mark.parametrize("fn,good", [("paged", [1, 40, 4, 2, 128, 1, 0, 64, 100]), ("decode", [3, 4, 2, 128, 64, 100])])
def test_workspace_sizes(fn, good):
    """Impossible shapes have none; a window of everything asks for what the call without asks for, and
    a small one for no more."""
    size = getattr(_lib.lib(), f"omx_gdn_attn_{fn}_window_workspace_size")
    whole = getattr(_lib.lib(), f"omx_gdn_attn_{fn}_workspace_size")(*good)
    assert size(*good, 0, 0) == size(*good, 1 << 62, 0) == size(*good, 10, 1 << 62) == whole > 0
    assert size(*good, 1, 0) <= whole and size(*good, 3000, 4) <= whole
    assert size(*good, -1, 0) == 0 and size(*good, 5, -1) == 0
    for i in range(len(good)):
        for x in BIG[2:]:
            if fn == "paged" and i == 6:  # a flag, not a number
                continue
            assert size(*good[:i], x, *good[i + 1:], 100, 4) == 0


@needs_lib
def test_empty_calls_are_no_ops():
    assert _run("omx_gdn_kv_write8", WRITE8, dict(T=0, k=None))[0] == _lib.OK
    assert _run("omx_gdn_attn_paged_window", PAGEDW, dict(T=0, q=None))[0] == _lib.OK
    assert _run("omx_gdn_attn_decode_window", DECODEW, dict(B=0, q=None))[0] == _lib.OK


def test_the_reference_rounds_as_the_type_does():
    """Every bf16 of a size up to 448, against torch's own conversion, and every code against itself."""
    torch = pytest.importorskip("torch")
    from cache8_reference import E4M3, asked, nearest
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    x = x[x.isfinite() & (x.abs() <= 448)]
    assert torch.equal(nearest(x.double()), x.to(E4M3).double())
    c = torch.arange(256, dtype=torch.uint8).view(E4M3).double()
    assert torch.equal(nearest(c[c.isfinite()]), c[c.isfinite()])
    for most, e in ((0.0, -100), (448.0, 0), (449.0, 1), (3.5, -7), (3.51, -6), (3.3e38, 120), (1e-38, -100)):
        assert float(asked(torch.tensor(most, dtype=torch.float64).view(1, 1, 1))) == e


def test_python_checks_before_the_library():
    torch = pytest.importorskip("torch")
    import omegalax_amd as om
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for bad in (dict(window=0), dict(window=5, sinks=-1), dict(sinks=2)):
        with pytest.raises(ValueError, match="window|sinks"):
            om.attention_prefill_paged(q, q, q, table, lengths, **bad)
        with pytest.raises(ValueError, match="window|sinks"):
            om.attention_decode_step(q[0], q[0], q[0], q, q, table, lengths, **bad)
