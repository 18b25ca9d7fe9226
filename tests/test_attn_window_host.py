"""Refusals of the windowed attention entry points and of their arguments, on any machine."""
import os

import pytest

from omegalax_amd import _lib
from test_attn_host import BIG, BWD, FWD, SHAPES, _run

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH),
                                reason="libomx_gdn.so not built (python -m omegalax_amd.build)")


def _with(args, **more):
    """The arguments with `more` before the workspace."""
    out = {}
    for name, x in args.items():
        if name == "ws":
            out.update(more)
        out[name] = x
    return out


SIGHT = [(dict(window=0), "window"), (dict(window=-1), "window"), (dict(sinks=-1), "sinks")]


@pytest.mark.parametrize("over,code,msg", SHAPES + [(o, _lib.EINVAL, m) for o, m in SIGHT])
def test_forward_refuses(over, code, msg):
    rc, err = _run("omx_gdn_attn_window_fwd", _with(FWD, window=10, sinks=2), over)
    assert rc == code and msg in err


@pytest.mark.parametrize("over,code,msg", SHAPES + [(o, _lib.EINVAL, m) for o, m in SIGHT] + [
    (dict(lse=None), _lib.EINVAL, "NULL"), (dict(ws=None), _lib.EINVAL, "workspace"), (dict(ws_bytes=100), _lib.EINVAL, "workspace")])
def test_backward_refuses(over, code, msg):
    rc, err = _run("omx_gdn_attn_window_bwd", _with(BWD, window=10, sinks=2), over)
    assert rc == code and msg in err


def test_workspace_sizes_of_impossible_shapes():
    size = _lib.lib().omx_gdn_attn_window_bwd_workspace_size
    good = [2, 5000, 4, 2, 128, 0, 100, 4]
    assert size(*good) > 0
    for i in range(6):
        for x in BIG[2:]:
            assert size(*good[:i], x, *good[i + 1:]) == 0
    assert size(*good[:6], 0, 4) == 0 and size(*good[:7], -1) == 0
    # a window or sinks of everything ask for what the attention without does
    whole = _lib.lib().omx_gdn_attn_bwd_workspace_size(*good[:6])
    assert size(*good[:6], 1 << 62, 0) == whole and size(*good[:6], 10, 1 << 62) == whole and size(*good[:6], 5000, 0) == whole


def test_empty_calls_are_no_ops():
    assert _run("omx_gdn_attn_window_fwd", _with(FWD, window=10, sinks=2), dict(T=0, q=None, o=None))[0] == _lib.OK
    assert _run("omx_gdn_attn_window_bwd", _with(BWD, window=10, sinks=2), dict(B=0, N=0, q=None))[0] == _lib.OK


def test_python_checks_before_the_library():
    torch = pytest.importorskip("torch")
    import omegalax_amd as om
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    lse = torch.zeros(1, 4, 2)
    for bad in (dict(window=0), dict(window=-3), dict(window=5, sinks=-1), dict(sinks=2)):
        with pytest.raises(ValueError, match="window|sinks"):
            om.attention_prefill(q, q, q, **bad)
        with pytest.raises(ValueError, match="window|sinks"):
            om.attention_prefill_bwd(q, q, q, q, lse, q, **bad)
    with pytest.raises(TypeError):
        om.attention_prefill(q, q, q, window=2.5)
    with pytest.raises(ValueError, match="GPU"):
        om.attention_prefill(q, q, q, window=5, sinks=1)


@pytest.mark.parametrize("B,T,N", [(0, 100, 1), (0, 100, 64), (0, 100, 65), (0, 0, 3), (3, 0, 0), (1, 0, 2), (0, 100, 0), (0, 0, 0)])
@pytest.mark.parametrize("window,sinks", [(10, 0), (10, 4), (1, 0)])
def test_workspace_sizes_of_no_tokens(B, T, N, window, sinks):
    """None of a batch's or a packed call's tokens: nothing to share, so what the attention without a window asks for."""
    L = _lib.lib()
    shape = [B, T, 8, 2, 64, N]
    assert L.omx_gdn_attn_window_bwd_workspace_size(*shape, window, sinks) == L.omx_gdn_attn_bwd_workspace_size(*shape)
