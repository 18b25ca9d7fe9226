"""Attention with a window and sinks on the GPU, against 64 bits: prompts and their gradient."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import omegalax_amd as om
from attn_reference import check
from sight_reference import one_sequence, seen
from test_gpu_attn import BF, draw, offsets, say, spans_of

NAN = float("nan")


def check_prompts(q, k, v, spans, window, sinks, *, cu=None, do=None, scale=None, only=None):
    x = [t.detach().requires_grad_(do is not None) for t in (q, k, v)]
    o, lse = om.attention_prefill(*x, cu_seqlens=cu, scale=scale, output_lse=True, window=window, sinks=sinks)
    grads = torch.autograd.grad(o, x, do) if do is not None else ()
    flat = lambda t: t.detach().flatten(0, 1)
    got = dict(o=flat(o), **{n: flat(t) for n, t in zip(("dq", "dk", "dv"), grads)})
    for n, (a, b) in enumerate(spans):
        if a == b or (only is not None and n not in only):
            continue
        val, tol = one_sequence(*(flat(t)[a:b].double() for t in (q, k, v)), seen(b - a, b - a, 0, window, sinks),
                                do=None if do is None else flat(do)[a:b].double(), scale=scale)
        for name, t in got.items():
            check(f"{name} of sequence {n}", t[a:b], val[name], tol[name])
        # fp32 scores of size |s| <= 20 and a sum of up to 2^13 weights: below 2e-5
        assert float((flat(lse)[a:b].double() - val["lse"]).abs().max()) < 5e-5
    return o


@pytest.mark.parametrize("B,T,Hq,Hkv,D,window,sinks", [
    (1, 1, 1, 1, 64, 1, 0), (2, 2, 4, 1, 128, 1, 0), (1, 5, 2, 1, 64, 1, 1), (1, 31, 8, 2, 256, 7, 3), (3, 64, 2, 2, 64, 63, 0),
    (1, 65, 16, 4, 128, 64, 0), (1, 130, 4, 1, 72, 65, 64), (2, 333, 32, 1, 128, 100, 4), (1, 517, 4, 4, 256, 33, 70),
    (1, 700, 3, 1, 64, 1, 130), (1, 1030, 16, 8, 128, 128, 1), (2, 400, 7, 1, 256, 129, 200), (1, 300, 6, 2, 96, 299, 0),
    (1, 2500, 8, 2, 128, 500, 4), (1, 1900, 16, 2, 256, 200, 16), (1, 3000, 2, 2, 64, 31, 2), (5, 258, 3, 1, 64, 40, 33),
])
def test_batches_and_their_gradients(B, T, Hq, Hkv, D, window, sinks):
    say(f"window B={B} T={T} Hq={Hq} Hkv={Hkv} D={D} window={window} sinks={sinks}")
    q, k, v, do = (draw(T + i, B, T, h, D, scale=s) for i, (h, s) in
                   enumerate(((Hq, 1.5), (Hkv, 1.0), (Hkv, 1.0), (Hq, 1.0))))
    check_prompts(q, k, v, spans_of(B, T, None), window, sinks, do=do)


PACKS = [[1, 1, 1], [5, 0, 0, 130, 1, 64], [63, 64, 65, 127, 128, 129, 2], [700, 3, 90], [0, 1500, 0, 33],
         [1800, 20, 50, 7, 300], [17] * 64, [9, 0, 40] * 30, [2000, 1] + [33] * 70]


@pytest.mark.parametrize("lens", PACKS, ids=lambda l: f"{len(l)}x{sum(l)}")
@pytest.mark.parametrize("Hq,Hkv,D,window,sinks", [(8, 2, 128, 50, 4), (3, 3, 64, 200, 0), (8, 1, 256, 30, 140)])
def test_packed_sequences_and_their_gradients(lens, Hq, Hkv, D, window, sinks):
    say(f"packed window {len(lens)} sequences, {sum(lens)} tokens, Hq={Hq} Hkv={Hkv} D={D} window={window} sinks={sinks}")
    T = sum(lens)
    q, k, v, do = (draw(T + i, 1, T, h, D) for i, h in enumerate((Hq, Hkv, Hkv, Hq)))
    cu = offsets(lens)
    check_prompts(q, k, v, spans_of(1, T, cu), window, sinks, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), do=do)


@pytest.mark.parametrize("window,sinks", [(300, 0), (1 << 40, 0), (200, 100), (299, 1), (10, 1 << 40)])
def test_a_window_of_everything_is_no_window(window, sinks):
    x = [draw(i, 2, 300, h, 128).requires_grad_(True) for i, h in enumerate((8, 2, 2))]
    do = draw(5, 2, 300, 8, 128)
    a = om.attention_prefill(*x)
    b = om.attention_prefill(*x, window=window, sinks=sinks)
    assert torch.equal(a, b)
    for s, t in zip(torch.autograd.grad(a, x, do), torch.autograd.grad(b, x, do)):
        assert torch.equal(s, t)


def test_a_window_of_one_is_the_value():
    q, k, v = draw(1, 1, 200, 4, 64), draw(2, 1, 200, 2, 64), draw(3, 1, 200, 2, 64)
    assert torch.equal(om.attention_prefill(q, k, v, window=1), v.repeat_interleave(2, 2))


@pytest.mark.parametrize("Hq,Hkv,D,T,window,sinks,bad_at", [
    (4, 2, 128, 600, 100, 0, 250), (2, 2, 64, 400, 64, 10, 130), (8, 1, 256, 500, 33, 3, 70), (3, 1, 80, 700, 1, 1, 300)])
@pytest.mark.parametrize("bad", [NAN, float("inf")])
def test_rows_do_not_see_infinities_behind_their_window(Hq, Hkv, D, T, window, sinks, bad_at, bad):
    """One token's key and value are not finite: rows before it and rows past its window are as if it
    were any other, those that see it are not finite."""
    say(f"window {window}, token {bad_at} not finite, D={D}, {bad}")
    q, k, v = draw(1, 1, T, Hq, D), draw(2, 1, T, Hkv, D), draw(3, 1, T, Hkv, D)
    kb, vb = k.clone(), v.clone()
    kb[:, bad_at], vb[:, bad_at] = NAN, bad
    o = om.attention_prefill(q, kb, vb, window=window, sinks=sinks)
    val, tol = one_sequence(*(t[0].double() for t in (q, k, v)), seen(T, T, 0, window, sinks))
    check("before", o[0, :bad_at], val["o"][:bad_at], tol["o"][:bad_at])
    past = bad_at + window
    check("past", o[0, past:], val["o"][past:], tol["o"][past:])
    assert bool(o[0, bad_at:past].isnan().all())


@pytest.mark.parametrize("D", [64, 72, 128, 256])
@pytest.mark.parametrize("sinks", [1, 31, 63, 64, 65, 100])
def test_nothing_between_the_sinks_and_the_window_counts(D, sinks):
    """Rows whose tile holds the sinks and the window's first keys, with no number between."""
    T, first, window = 500, 300, 60
    q, k, v = draw(1, 1, T, 6, D), draw(2, 1, T, 2, D), draw(3, 1, T, 2, D)
    k[:, sinks:first - window + 1], v[:, sinks:first - window + 1] = NAN, float("inf")
    o = om.attention_prefill(q, k, v, window=window, sinks=sinks)
    val, tol = one_sequence(*(t[0].double() for t in (q[:, first:], k, v)), seen(T - first, T, first, window, sinks))
    check("rows past them", o[0, first:], val["o"], tol["o"])


def test_columns_of_one_projection():
    B, T, Hq, Hkv, D = 2, 190, 8, 2, 128
    qkv = draw(4, B, T, Hq + 2 * Hkv, D).requires_grad_(True)
    q, k, v = qkv.split([Hq, Hkv, Hkv], 2)
    o = om.attention_prefill(q, k, v, window=50, sinks=3)
    dense = [t.detach().contiguous().requires_grad_(True) for t in (q, k, v)]
    o2 = om.attention_prefill(*dense, window=50, sinks=3)
    assert torch.equal(o, o2)
    do = draw(5, B, T, Hq, D)
    g, = torch.autograd.grad(o, qkv, do)
    assert torch.equal(g, torch.cat(torch.autograd.grad(o2, dense, do), 2))


def test_gradients_against_differences():
    """The directional derivative of sum(o * do) in 64 bits by central differences of the definition,
    against the kernels' gradients along the same direction."""
    T, Hq, Hkv, D, window, sinks = 90, 4, 2, 64, 20, 3
    x = [draw(i, 1, T, h, D) for i, h in enumerate((Hq, Hkv, Hkv))]
    do = draw(3, 1, T, Hq, D)
    u = [draw(10 + i, *t.shape[1:]).double() for i, t in enumerate(x)]
    leaves = [t.clone().requires_grad_(True) for t in x]
    grads = torch.autograd.grad(om.attention_prefill(*leaves, window=window, sinks=sinks), leaves, do)
    see = seen(T, T, 0, window, sinks)
    f = lambda e: ((one_sequence(*(t[0].double() + e * d for t, d in zip(x, u)), see)[0]["o"]) * do[0].double()).sum()
    h = 1e-4
    want = float((f(h) - f(-h)) / (2 * h))
    got = sum(float((g[0].double() * d).sum()) for g, d in zip(grads, u))
    _, tol = one_sequence(*(t[0].double() for t in x), see, do=do[0].double())
    bound = sum(float((tol[n] * d.abs()).sum()) for n, d in zip(("dq", "dk", "dv"), u))
    # errors of either sign: the bound of their sum's size is the root of the sum of squares
    root = sum(float(((tol[n] * d) ** 2).sum()) for n, d in zip(("dq", "dk", "dv"), u)) ** 0.5
    assert abs(got - want) <= min(bound, 6 * root) + 1e-6 * abs(want)


def test_packed_rows_equal_separate_ones():
    lens = [(37 * n) % 300 for n in range(80)]
    T = sum(lens)
    q, k, v = draw(1, 1, T, 8, 128), draw(2, 1, T, 2, 128), draw(3, 1, T, 2, 128)
    cu = offsets(lens)
    o = om.attention_prefill(q, k, v, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), window=60, sinks=2)
    for a, b in zip(cu, cu[1:]):
        if b - a > 62:  # one that fits its window is the attention without
            assert torch.equal(o[:, a:b], om.attention_prefill(q[:, a:b], k[:, a:b], v[:, a:b], window=60, sinks=2))


@pytest.mark.parametrize("T,D", [(260, 64), (900, 128), (1700, 256)])
def test_captured_forward_and_backward(T, D):
    x = [draw(i, 1, T, h, D) for i, h in enumerate((4, 2, 2))]
    do = draw(5, 1, T, 4, D)
    cu = torch.tensor([0, 100, 100, T], dtype=torch.int32, device="cuda")
    sight = dict(window=90, sinks=5)

    def both():
        o, lse = om.attention_prefill(*x, cu_seqlens=cu, output_lse=True, **sight)
        return [o, *om.attention_prefill_bwd(*x, o, lse, do, cu_seqlens=cu, **sight)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = both()
    for r in range(3):
        for i, t in enumerate((*x, do)):
            t.copy_(draw(20 + 5 * r + i, *t.shape))
        cu.copy_(torch.tensor([0, 30 * r, 100 + r, T], dtype=torch.int32))
        want = both()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_streams_at_once():
    sets = [[draw(10 * i + j, 1, 1200, h, D) for j, h in enumerate((8, 2, 2, 8))] for i, D in enumerate((128, 256))]
    sight = dict(window=130, sinks=4)
    run = lambda q, k, v, do: [*(r := om.attention_prefill(q, k, v, output_lse=True, **sight)),
                               *om.attention_prefill_bwd(q, k, v, *r, do, **sight)]
    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(*sets[i]))
    torch.cuda.synchronize()
    for w, rs in zip(want, got):
        for r in rs:
            assert all(torch.equal(a, b) for a, b in zip(w, r))


def test_one_token_of_a_long_prompt_by_itself():
    """Rows far into a long prompt, whose first key tile lies a hundred tiles on: 64 bits of a few."""
    T, Hq, Hkv, D, window, sinks = 20000, 4, 1, 128, 300, 4
    q, k, v = draw(1, 1, T, Hq, D, scale=1.5), draw(2, 1, T, Hkv, D), draw(3, 1, T, Hkv, D)
    o = om.attention_prefill(q, k, v, window=window, sinks=sinks)
    for a in (5000, 12345, 19990):
        see = seen(10, a + 10, a, window, sinks)
        val, tol = one_sequence(q[0, a:a + 10].double(), k[0, :a + 10].double(), v[0, :a + 10].double(), see)
        check(f"rows from {a}", o[0, a:a + 10], val["o"], tol["o"])
