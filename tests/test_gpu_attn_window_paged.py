"""Attention with a window and sinks over a paged cache of bf16: new tokens and the decode step."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import omegalax_amd as om
from attn_reference import check
from sight_reference import one_sequence, seen
from test_gpu_attn import draw, offsets, say
from test_gpu_attn_paged import CASES, DECODE, Cache, NAN

SIGHTS = [(1, 0), (17, 3), (64, 0), (200, 70), (500, 1)]


@pytest.mark.parametrize("held,new,page,Hq,Hkv,D", CASES + [([3000, 50], [20, 9], 64, 4, 1, 128), ([900, 2500], [70, 1], 16, 8, 2, 64),
                                                            ([4000], [130], 128, 8, 1, 256)], ids=lambda x: str(x)[:12])
@pytest.mark.parametrize("window,sinks", SIGHTS)
def test_turns(held, new, page, Hq, Hkv, D, window, sinks):
    say(f"windowed turn held={held[:6]} new={new[:6]} page={page} Hq={Hq} Hkv={Hkv} D={D} window={window} sinks={sinks}")
    c = Cache(held, new, page, Hkv, D, seed=len(held))
    T = sum(new)
    q, k, v = draw(7, 1, T, Hq, D, scale=1.5), draw(8, 1, T, Hkv, D), draw(9, 1, T, Hkv, D)
    cu = offsets(new)
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
    om.kv_pages_write(k, v, *c.args(), cu_seqlens=cu_t)
    o = om.attention_prefill_paged(q, *c.args(), cu_seqlens=cu_t, window=window, sinks=sinks)
    for n, (a, b) in enumerate(zip(cu, cu[1:])):
        if b > a:
            val, tol = one_sequence(q[0, a:b].double(), torch.cat([c.keys[n], k[0, a:b]]).double(),
                                    torch.cat([c.values[n], v[0, a:b]]).double(),
                                    seen(b - a, held[n] + b - a, held[n], window, sinks))
            check(f"o of sequence {n}", o[0, a:b], val["o"], tol["o"])


@pytest.mark.parametrize("held,page,Hq,Hkv,D,width", DECODE + [([5, 900, -1] * 30, 16, 8, 2, 64, 80), ([20000, 7], 64, 8, 1, 128, 0)],
                         ids=lambda x: str(x)[:12])
@pytest.mark.parametrize("window,sinks", SIGHTS)
def test_steps(held, page, Hq, Hkv, D, width, window, sinks):
    say(f"windowed step held={held[:6]} page={page} Hq={Hq} Hkv={Hkv} D={D} window={window} sinks={sinks}")
    c = Cache(held, [1 if h >= 0 else 0 for h in held], page, Hkv, D, seed=3, width=width)
    B = len(held)
    q, k, v = draw(1, B, Hq, D, scale=1.5), draw(2, B, Hkv, D), draw(3, B, Hkv, D)
    o = om.attention_decode_step(q, k, v, *c.args(), window=window, sinks=sinks)
    for n, h in enumerate(held):
        if h < 0:
            assert not bool(o[n].any())
            continue
        val, tol = one_sequence(q[n:n + 1].double(), torch.cat([c.keys[n], k[n:n + 1]]).double(),
                                torch.cat([c.values[n], v[n:n + 1]]).double(), seen(1, h + 1, h, window, sinks))
        check(f"sequence {n}", o[n:n + 1], val["o"], tol["o"])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_pages_behind_the_window_are_not_needed(D):
    """Dropped from the table, and filled with NaN by whoever holds them now."""
    held, page, window, sinks = [1000, 333], 16, 100, 20
    c = Cache(held, [1, 1], page, 2, D)
    q, k, v = draw(1, 2, 8, D), draw(2, 2, 2, D), draw(3, 2, 2, D)
    sight = dict(window=window, sinks=sinks)
    want = om.attention_decode_step(q, k, v, *c.args(), **sight)
    want2 = om.attention_prefill_paged(q[:, None], *c.args(), **sight)
    for n, h in enumerate(held):
        for j in range(-(-sinks // page), (h + 1 - window) // page):
            c.k_pages[int(c.table[n, j])] = NAN
            c.v_pages[int(c.table[n, j])] = NAN
    assert torch.equal(want, om.attention_decode_step(q, k, v, *c.args(), **sight))
    assert torch.equal(want2, om.attention_prefill_paged(q[:, None], *c.args(), **sight))
    for n, h in enumerate(held):
        c.table[n, -(-sinks // page):(h + 1 - window) // page] = -1
    c.block_table.copy_(c.table)
    assert torch.equal(want, om.attention_decode_step(q, k, v, *c.args(), **sight))
    # tiles of 64 keys part of whose pages are gone are masked, which changes no weight
    assert torch.equal(want2, om.attention_prefill_paged(q[:, None], *c.args(), **sight))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sinks", [1, 15, 16, 17, 63, 64, 65, 100])
def test_nothing_between_the_sinks_and_the_window_counts(D, sinks):
    held, new, window = 500, 30, 60
    c = Cache([held], [new], 32, 2, D)
    bad = draw(5, 1, held - window + 1 - sinks, 2, D) * NAN
    om.kv_pages_write(bad, bad, c.args()[0], c.args()[1], c.args()[2], torch.tensor([sinks], dtype=torch.int32, device="cuda"))
    q, k, v = draw(7, 1, new, 6, D), draw(8, 1, new, 2, D), draw(9, 1, new, 2, D)
    om.kv_pages_write(k, v, *c.args())
    o = om.attention_prefill_paged(q, *c.args(), window=window, sinks=sinks)
    val, tol = one_sequence(q[0].double(), torch.cat([c.keys[0], k[0]]).double(), torch.cat([c.values[0], v[0]]).double(),
                            seen(new, held + new, held, window, sinks))
    check("o", o[0], val["o"], tol["o"])


def test_a_window_of_everything_is_no_window():
    c = Cache([300, 20], [5, 5], 16, 2, 128)
    q, k = draw(1, 2, 5, 8, 128), draw(2, 2, 5, 2, 128)
    om.kv_pages_write(k, k, *c.args())
    want = om.attention_prefill_paged(q, *c.args())
    for sight in (dict(window=400), dict(window=1 << 40), dict(window=300, sinks=100), dict(window=1, sinks=1 << 40)):
        assert torch.equal(want, om.attention_prefill_paged(q, *c.args(), **sight))
