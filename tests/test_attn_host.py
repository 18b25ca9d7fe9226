"""Refusals of the attention entry points, on any machine: every bad argument is turned into an
error before the first HIP call."""
import os

import pytest

from omegalax_amd import _lib

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH),
                                reason="libomx_gdn.so not built (python -m omegalax_amd.build)")


def _run(fn, args, over):
    a = dict(args, **over)
    L = _lib.lib()
    rc = getattr(L, fn)(*a.values())
    return rc, L.omx_gdn_last_error().decode()


FWD = dict(q=16, k=16, v=16, q_ld=512, k_ld=256, v_ld=256, cu=None, N=2, o=16, lse=None, o_rest=None, B=2, T=100, Hq=4,
           Hkv=2, D=128, scale=0.1, ws=None, ws_bytes=0, stream=None)
BWD = dict(q=16, k=16, v=16, q_ld=512, k_ld=256, v_ld=256, cu=None, N=2, o=16, lse=16, o_rest=None, do=16, dq=16, dk=16,
           dv=16,
           B=2, T=100, Hq=4, Hkv=2, D=128, scale=0.1, ws=256, ws_bytes=1 << 20, stream=None)
SHAPES = [
    (dict(Hq=5), _lib.EINVAL, "multiple of key heads"), (dict(Hkv=0), _lib.EINVAL, "positive"),
    (dict(D=12), _lib.EINVAL, "multiple of 8"), (dict(D=0), _lib.EINVAL, "multiple of 8"),
    (dict(D=264, q_ld=2048, k_ld=2048, v_ld=2048), _lib.EUNSUPPORTED, "above 256"),
    (dict(Hq=66, q_ld=66 * 128), _lib.EUNSUPPORTED, "above 32"), (dict(B=-1, N=-1), _lib.EINVAL, "negative"),
    (dict(T=1 << 31), _lib.EINVAL, "too many tokens"), (dict(N=3), _lib.EINVAL, "N must equal B"),
    (dict(cu=16), _lib.EINVAL, "batch 1"), (dict(cu=16, B=1, N=0), _lib.EINVAL, "sequence count"),
    (dict(q_ld=504), _lib.EINVAL, "q_ld"), (dict(k_ld=260), _lib.EINVAL, "k_ld"), (dict(v_ld=1 << 23), _lib.EINVAL, "v_ld"),
    (dict(scale=0.0), _lib.EINVAL, "scale"), (dict(scale=float("nan")), _lib.EINVAL, "scale"),
    (dict(scale=-1.0), _lib.EINVAL, "scale"), (dict(scale=2e6), _lib.EINVAL, "scale"), (dict(q=None), _lib.EINVAL, "NULL"), (dict(o=None), _lib.EINVAL, "NULL"),
    (dict(v=24), _lib.EINVAL, "aligned"),
]


@pytest.mark.parametrize("over,code,msg", SHAPES)
def test_forward_refuses(over, code, msg):
    rc, err = _run("omx_gdn_attn_fwd", FWD, over)
    assert rc == code and msg in err


@pytest.mark.parametrize("over,code,msg", SHAPES + [
    (dict(lse=None), _lib.EINVAL, "NULL"), (dict(dv=None), _lib.EINVAL, "NULL"), (dict(dk=8), _lib.EINVAL, "aligned"),
    (dict(ws=None), _lib.EINVAL, "workspace"), (dict(ws=8), _lib.EINVAL, "aligned"), (dict(ws_bytes=100), _lib.EINVAL, "workspace"),
])
def test_backward_refuses(over, code, msg):
    rc, err = _run("omx_gdn_attn_bwd", BWD, over)
    assert rc == code and msg in err


@pytest.mark.parametrize("fn,args,over", [
    ("omx_gdn_attn_fwd", "FWD", dict(B=1 << 24, N=1 << 24, T=1)), ("omx_gdn_attn_fwd", "FWD", dict(B=1, N=1, T=1 << 29)),
    ("omx_gdn_attn_fwd", "FWD", dict(B=1 << 22, N=1 << 22, T=300, Hq=2)), ("omx_gdn_attn_bwd", "BWD", dict(B=1 << 24, N=1 << 24, T=1)),
    ("omx_gdn_attn_paged", "PAGED", dict(B=1 << 24, N=1 << 24, T=1)), ("omx_gdn_kv_write", "WRITE", dict(B=1 << 28, N=1 << 28, T=1)),
    ("omx_gdn_attn_decode_step", "DECODE", dict(B=1 << 19, Hq=32, Hkv=32, q_ld=4096, k_ld=4096, v_ld=4096)),
])
def test_launches_of_too_many_threads_are_refused(fn, args, over):
    """A launch holds less than 2^32 threads, 256 of them a workgroup: one more is an error of the
    arguments, before anything is launched."""
    rc, err = _run(fn, globals()[args], dict(over, ws=256, ws_bytes=1 << 50))
    assert rc == _lib.EINVAL and ("grid too large" in err or "out of range" in err)


def test_a_million_sequences_of_few_tokens_are_no_large_grid():
    """Most of them are empty: the launch is as large as the tokens ask for."""
    many = dict(B=1, N=1 << 20, cu=16, Hq=32, Hkv=32, q_ld=4096, k_ld=4096, v_ld=4096)
    assert _run("omx_gdn_attn_fwd", FWD, dict(many, T=0, ws=256, ws_bytes=1 << 30))[0] == _lib.OK
    rc, err = _run("omx_gdn_attn_fwd", FWD, dict(many, T=1000))
    assert rc == _lib.EINVAL and "workspace" in err  # the next check: the tile list's room


def test_many_packed_sequences_need_their_plan():
    L = _lib.lib()
    assert L.omx_gdn_attn_fwd_workspace_size(5000, 4, 2, 64) == 0
    need = L.omx_gdn_attn_fwd_workspace_size(5000, 4, 2, 65)
    assert need > 0
    for ws, n in ((256, need - 1), (None, need), (8, need)):
        rc, err = _run("omx_gdn_attn_fwd", FWD, dict(cu=16, B=1, T=5000, N=65, ws=ws, ws_bytes=n))
        assert rc == _lib.EINVAL and "workspace" in err


CACHE = dict(k_pages=16, v_pages=16, n_pages=10, page=16, table=16, width=10, lengths=16)
WRITE = dict(k=16, v=16, k_ld=256, v_ld=256, cu=None, N=2, **CACHE, B=2, T=3, Hkv=2, D=128, ws=None, ws_bytes=0, stream=None)
PAGED = dict(q=16, q_ld=512, cu=None, N=2, **CACHE, o=16, B=2, T=3, Hq=4, Hkv=2, D=128, scale=0.1, ws=None, ws_bytes=0,
             stream=None)
DECODE = dict(q=16, k=16, v=16, q_ld=512, k_ld=256, v_ld=256, **CACHE, out=16, B=2, Hq=4, Hkv=2, D=128, scale=0.1, ws=None,
              ws_bytes=0, stream=None)
BAD_CACHE = [
    (dict(page=8), _lib.EINVAL, "page size"), (dict(page=24), _lib.EINVAL, "page size"), (dict(page=1 << 17), _lib.EINVAL, "page size"),
    (dict(n_pages=-1), _lib.EINVAL, "page count"), (dict(width=-1), _lib.EINVAL, "block table"),
    (dict(width=1 << 30), _lib.EINVAL, "block table"), (dict(k_pages=None), _lib.EINVAL, "NULL"),
    (dict(table=None), _lib.EINVAL, "NULL"), (dict(lengths=None), _lib.EINVAL, "NULL"), (dict(v_pages=8), _lib.EINVAL, "aligned"),
    (dict(D=96), _lib.EUNSUPPORTED, "not compiled"), (dict(D=100), _lib.EINVAL, "multiple of 8"),
]


@pytest.mark.parametrize("over,code,msg", BAD_CACHE + [
    (dict(k=None), _lib.EINVAL, "NULL"), (dict(k=8), _lib.EINVAL, "aligned"), (dict(v_ld=128), _lib.EINVAL, "v_ld"),
    (dict(N=1), _lib.EINVAL, "N must equal B"),
])
def test_append_refuses(over, code, msg):
    rc, err = _run("omx_gdn_kv_write", WRITE, over)
    assert rc == code and msg in err


@pytest.mark.parametrize("over,code,msg", BAD_CACHE + [
    (dict(q=None), _lib.EINVAL, "NULL"), (dict(o=8), _lib.EINVAL, "aligned"), (dict(q_ld=128), _lib.EINVAL, "q_ld"),
    (dict(scale=0.0), _lib.EINVAL, "scale"), (dict(Hq=3), _lib.EINVAL, "multiple of key heads"),
    (dict(width=100, page=64), _lib.EINVAL, "workspace"),
])
def test_paged_attention_refuses(over, code, msg):
    rc, err = _run("omx_gdn_attn_paged", PAGED, over)
    assert rc == code and msg in err


@pytest.mark.parametrize("over,code,msg", BAD_CACHE + [
    (dict(q=None), _lib.EINVAL, "NULL"), (dict(out=8), _lib.EINVAL, "aligned"), (dict(k_ld=128), _lib.EINVAL, "k_ld"),
    (dict(scale=float("inf")), _lib.EINVAL, "scale"), (dict(B=-1), _lib.EINVAL, "negative"),
    (dict(width=100, page=64), _lib.EINVAL, "workspace"),
])
def test_decode_refuses(over, code, msg):
    rc, err = _run("omx_gdn_attn_decode_step", DECODE, over)
    assert rc == code and msg in err


@pytest.mark.parametrize("B,T,Hq,Hkv,D,page,width", [(8, 512, 32, 8, 128, 64, 128), (16, 512, 16, 2, 256, 64, 128),
                                                     (16, 256, 16, 2, 256, 16, 1000), (1000, 1, 8, 1, 64, 16, 2000)])
def test_a_batch_that_fills_the_chip_reads_its_cache_whole(B, T, Hq, Hkv, D, page, width):
    """Every row has its own tiles: 512 of them leave nothing to share, packed or not, and no
    partial sums are kept."""
    size = _lib.lib().omx_gdn_attn_paged_workspace_size
    assert B * -(-T // (128 // (Hq // Hkv))) * Hkv >= 512
    assert size(B, T, Hq, Hkv, D, B, 0, page, width) == 0


@pytest.mark.parametrize("B,T,Hq,Hkv,D,page,width,shares", [
    (2, 40, 4, 1, 128, 64, 100, 32), (4, 100, 8, 2, 64, 16, 250, 16), (3, 130, 2, 2, 256, 48, 50, 18), (2, 1, 8, 8, 64, 16, 20, 2)])
def test_rows_that_leave_the_chip_idle_share_their_keys(B, T, Hq, Hkv, D, page, width, shares):
    """Shares of 512 workgroups, 32 at most, none of less than 128 keys."""
    size = _lib.lib().omx_gdn_attn_paged_workspace_size
    tiles = B * -(-T // (128 // (Hq // Hkv))) * Hkv
    assert shares == min(512 // tiles, 32, page * width // 128)
    up = lambda x: -(-x // 256) * 256
    assert size(B, T, Hq, Hkv, D, B, 0, page, width) == up(shares * B * T * Hq * D * 4) + up(shares * B * T * Hq * 8)


@pytest.mark.parametrize("B,Hq,Hkv,D,page,width,ranges", [
    (64, 32, 8, 128, 64, 70, 32), (128, 32, 8, 128, 64, 70, 32), (1024, 8, 1, 64, 16, 200, 256), (512, 16, 2, 256, 64, 10, 128),
    (7, 8, 1, 256, 65536, 32767, 256), (11, 8, 1, 256, 65536, 32767, 0),  # 2^30 stages of 16 keys: they are counted in 32 bits
    (1025, 8, 1, 64, 16, 200, 0), (64, 32, 8, 128, 64, 16, 0), (1, 16, 4, 128, 16, 64, 0), (1, 16, 4, 128, 16, 65, 64)])
def test_decode_batches_share_the_keys_in_equal_ranges(B, Hq, Hkv, D, page, width, ranges):
    """One workgroup for each compute unit, whatever the number of sequences, up to 1,024 and but for
    the shortest tables; their partial sums are a sequence's segments."""
    size = _lib.lib().omx_gdn_attn_decode_workspace_size
    rows, up = (ranges + B) * Hq if ranges else 0, lambda x: -(-x // 256) * 256
    assert size(B, Hq, Hkv, D, page, width) == up(rows * D * 4) + up(rows * 8)


BIG = [-1, 0, 1 << 31, 1 << 40, (1 << 63) - 1, -(1 << 63)]


@pytest.mark.parametrize("fn,good", [
    ("fwd", [5000, 4, 2, 65]), ("bwd", [2, 5000, 4, 2, 128, 0]), ("paged", [1, 40, 4, 2, 128, 1, 0, 64, 100]),
    ("decode", [3, 4, 2, 128, 64, 100])])
def test_workspace_sizes_of_impossible_shapes(fn, good):
    """Any numbers get an answer: those that no entry point takes have no size."""
    size = getattr(_lib.lib(), f"omx_gdn_attn_{fn}_workspace_size")
    assert size(*good) > 0
    for i in range(len(good)):
        for j in range(len(good)):
            for x in BIG[2:]:
                for y in BIG:
                    if fn == "paged" and 6 in (i, j):  # a flag, not a number
                        continue
                    args = list(good)
                    args[j], args[i] = y, x
                    assert size(*args) == 0


def test_workspace_size_of_an_impossible_append():
    size = _lib.lib().omx_gdn_kv_write_workspace_size
    assert size(5000, 65) > 0
    assert not any(size(x, y) for x in BIG[2:] for y in (65, *BIG)) and not any(size(5000, x) for x in BIG[2:])


def test_empty_calls_are_no_ops():
    assert _run("omx_gdn_attn_fwd", FWD, dict(T=0, q=None, o=None))[0] == _lib.OK
    assert _run("omx_gdn_attn_bwd", BWD, dict(B=0, N=0, q=None))[0] == _lib.OK
    assert _run("omx_gdn_kv_write", WRITE, dict(T=0, k=None))[0] == _lib.OK
    assert _run("omx_gdn_attn_paged", PAGED, dict(T=0, q=None))[0] == _lib.OK
    assert _run("omx_gdn_attn_decode_step", DECODE, dict(B=0, q=None))[0] == _lib.OK


def test_python_checks_before_the_library():
    torch = pytest.importorskip("torch")
    import omegalax_amd as om
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        om.attention_prefill(q, q, q)
    with pytest.raises(ValueError, match="GPU"):
        om.attention_decode_step(q[0], q[0], q[0], q, q, torch.zeros(4, 1, dtype=torch.int32),
                                 torch.zeros(4, dtype=torch.int32))


@pytest.mark.parametrize("dual", range(5))
def test_forward_mode_derivatives_are_refused(dual):
    """A dual tensor's tangent would be lost: no entry point takes one, with or without no_grad."""
    torch = pytest.importorskip("torch")
    from torch.autograd import forward_ad
    import omegalax_amd as om
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    lse, table, lengths = torch.zeros(1, 4, 2), torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    calls = [(lambda *x: om.attention_prefill(*x), [q] * 3), (lambda *x: om.attention_prefill_bwd(*x[:4], lse, x[4]), [q] * 5),
             (lambda *x: om.kv_pages_write(*x, table, lengths), [q] * 4),
             (lambda *x: om.attention_prefill_paged(*x, table, lengths), [q] * 3),
             (lambda *x: om.attention_decode_step(*x, table, lengths), [q[0]] * 3 + [q] * 2)]
    for call, args in calls:
        if dual >= len(args):
            continue
        with forward_ad.dual_level():
            x = [forward_ad.make_dual(t, torch.ones_like(t)) if i == dual else t for i, t in enumerate(args)]
            with pytest.raises(ValueError, match="forward-mode"):
                call(*x)
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                call(*x)
            with pytest.raises(ValueError, match="GPU"):  # a level alone changes nothing
                call(*args)
    with pytest.raises(ValueError, match="forward-mode"):
        torch.func.jvp(lambda t: om.attention_prefill(t, q, q), (q,), (q,))
