"""Causal softmax attention of packed prompts and its gradient on the GPU, against 64 bits."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import omegalax_amd as om
from attn_reference import check, one_sequence

BF = torch.bfloat16


def say(msg):
    print(msg, flush=True)


def draw(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(BF).cuda()


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def spans_of(B, T, cu):
    return list(zip(cu, cu[1:])) if cu is not None else [(b * T, (b + 1) * T) for b in range(B)]


def check_prefill(q, k, v, spans, *, cu=None, do=None, scale=None, only=None):
    """Forward, and with `do` backward, of q [B,T,Hq,D] against each sequence by itself."""
    x = [t.detach().requires_grad_(do is not None) for t in (q, k, v)]
    o, lse = om.attention_prefill(*x, cu_seqlens=cu, scale=scale, output_lse=True)
    grads = torch.autograd.grad(o, x, do) if do is not None else ()
    flat = lambda t: t.detach().flatten(0, 1)
    got = dict(o=flat(o), **{n: flat(t) for n, t in zip(("dq", "dk", "dv"), grads)})
    for n, (a, b) in enumerate(spans):
        if a == b or (only is not None and n not in only):
            continue
        val, tol = one_sequence(*(flat(t)[a:b].double() for t in (q, k, v)), 0,
                                do=None if do is None else flat(do)[a:b].double(), scale=scale)
        for name, t in got.items():
            check(f"{name} of sequence {n}", t[a:b], val[name], tol[name])
        # fp32 scores of size |s| <= 20 and a sum of up to 2^13 weights: below 2e-5
        assert float((flat(lse)[a:b].double() - val["lse"]).abs().max()) < 5e-5
    return o


@pytest.mark.parametrize("B,T,Hq,Hkv,D", [
    (1, 1, 1, 1, 64), (2, 2, 4, 1, 128), (1, 31, 8, 2, 256), (3, 64, 2, 2, 64), (1, 65, 16, 4, 128),
    (1, 2000, 3, 1, 72), (2, 127, 6, 2, 128), (1, 129, 10, 2, 64), (1, 200, 7, 1, 256), (2, 333, 32, 1, 128),
    (1, 517, 4, 4, 256), (5, 258, 3, 1, 64), (1, 1030, 16, 8, 128),
])
def test_batches_and_their_gradients(B, T, Hq, Hkv, D):
    say(f"attention B={B} T={T} Hq={Hq} Hkv={Hkv} D={D}")
    q, k, v, do = (draw(T + i, B, T, h, D, scale=s) for i, (h, s) in
                   enumerate(((Hq, 1.5), (Hkv, 1.0), (Hkv, 1.0), (Hq, 1.0))))
    check_prefill(q, k, v, spans_of(B, T, None), do=do)


@pytest.mark.parametrize("B,T,Hq,Hkv,D", [(1, 900, 7, 1, 128), (1, 700, 32, 1, 256), (1, 1500, 5, 1, 64),
                                          (3, 600, 3, 1, 256), (1, 1300, 2, 2, 200)])
def test_few_tiles_of_keys_share_their_rows(B, T, Hq, Hkv, D):
    say(f"shares of rows B={B} T={T} Hq={Hq} Hkv={Hkv} D={D}")
    q, k, v, do = (draw(2 * T + i, B, T, h, D) for i, h in enumerate((Hq, Hkv, Hkv, Hq)))
    check_prefill(q, k, v, spans_of(B, T, None), do=do)


def test_packed_rows_past_32_bit_offsets():
    """2.5 billion elements of q: short sequences at the end, by themselves bit for bit."""
    N, L, Hq, Hkv, D = 6000, 101, 32, 8, 128
    T = N * L
    say(f"{T} tokens of {Hq} heads of {D}")
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, do = (torch.randn((1, T, h, D), generator=g, device="cuda", dtype=BF) for h in (Hq, Hkv, Hkv, Hq))
    cu = torch.arange(0, T + 1, L, dtype=torch.int32, device="cuda")
    run = lambda q, k, v, do, cu: [*(r := om.attention_prefill(q, k, v, cu_seqlens=cu, output_lse=True)),
                                   *om.attention_prefill_bwd(q, k, v, *r, do, cu_seqlens=cu)]
    got = run(q, k, v, do, cu)
    for n in (0, 3000, N - 1):
        part = [t[:, n * L:(n + 1) * L] for t in (q, k, v, do)]
        for a, b in zip(got, run(*part, None)):
            assert torch.equal(a[:, n * L:(n + 1) * L], b)


@pytest.mark.parametrize("D", [8, 24, 80, 96, 136, 200, 248])
def test_head_dims_between_the_compiled_ones(D):
    say(f"attention D={D}")
    q, k, v, do = (draw(D + i, 1, 150, h, D) for i, h in enumerate((6, 3, 3, 6)))
    check_prefill(q, k, v, [(0, 150)], do=do)


PACKS = [
    [1, 1, 1], [5, 0, 0, 130, 1, 64], [0, 0, 300, 0], [63, 64, 65, 127, 128, 129, 2],
    [700, 3, 90], [796, 842, 265], [0, 1500, 0, 33], [1800, 20, 50, 7, 300], [17] * 64, [9, 0, 40] * 30, [1] * 200, [2000, 1] + [33] * 70,
]


@pytest.mark.parametrize("lens", PACKS, ids=lambda l: f"{len(l)}x{sum(l)}")
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (3, 3, 64), (8, 1, 256)])
def test_packed_sequences_and_their_gradients(lens, Hq, Hkv, D):
    say(f"packed attention {len(lens)} sequences, {sum(lens)} tokens, Hq={Hq} Hkv={Hkv} D={D}")
    T = sum(lens)
    q, k, v, do = (draw(T + i, 1, T, h, D) for i, h in enumerate((Hq, Hkv, Hkv, Hq)))
    cu = offsets(lens)
    check_prefill(q, k, v, spans_of(1, T, cu), cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), do=do)


@pytest.mark.parametrize("N", [5, 80])
def test_packed_rows_equal_separate_ones(N):
    """Tiles start at each sequence, so packing changes no bit."""
    lens = [(37 * n) % 300 for n in range(N)]
    T = sum(lens)
    q, k, v = draw(1, 1, T, 8, 128), draw(2, 1, T, 2, 128), draw(3, 1, T, 2, 128)
    cu = offsets(lens)
    o = om.attention_prefill(q, k, v, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    for a, b in zip(cu, cu[1:]):
        if b > a:
            alone = om.attention_prefill(q[:, a:b], k[:, a:b], v[:, a:b])
            assert torch.equal(o[:, a:b], alone)


@pytest.mark.parametrize("N", [6, 70])
def test_invalid_offsets_read_as_their_repair(N):
    T = 500
    g = torch.Generator().manual_seed(N)
    raw = torch.randint(-100, 900, (N + 1,), generator=g)
    fixed, top = [0], 0
    for x in raw[1:-1].tolist():
        top = max(top, min(max(x, 0), T))
        fixed.append(top)
    fixed.append(T)
    x = [draw(i, 1, T, h, 64) for i, h in enumerate((4, 2, 2))]
    dev = lambda t: torch.as_tensor(t, dtype=torch.int32).cuda()
    x = [t.requires_grad_(True) for t in x]
    a = om.attention_prefill(*x, cu_seqlens=dev(raw))
    b = om.attention_prefill(*x, cu_seqlens=dev(fixed))
    assert torch.equal(a, b)
    do = draw(9, 1, T, 4, 64)
    for s, t in zip(torch.autograd.grad(a, x, do), torch.autograd.grad(b, x, do)):
        assert torch.equal(s, t)


def test_columns_of_one_projection():
    """q, k and v as views into one [B, T, (Hq + 2 Hkv) D] tensor, read where they lie."""
    B, T, Hq, Hkv, D = 2, 190, 8, 2, 128
    qkv = draw(4, B, T, Hq + 2 * Hkv, D).requires_grad_(True)
    q, k, v = qkv.split([Hq, Hkv, Hkv], 2)
    assert not q.is_contiguous()
    o = om.attention_prefill(q, k, v)
    dense = [t.detach().contiguous().requires_grad_(True) for t in (q, k, v)]
    o2 = om.attention_prefill(*dense)
    assert torch.equal(o, o2)
    do = draw(5, B, T, Hq, D)
    g, = torch.autograd.grad(o, qkv, do)
    assert torch.equal(g, torch.cat(torch.autograd.grad(o2, dense, do), 2))


def test_other_layouts_are_copied():
    T, D = 70, 64
    q, k, v = draw(1, 4, T, D), draw(2, 2, T, D), draw(3, 2, T, D)  # heads before tokens
    o = om.attention_prefill(*(t.transpose(0, 1)[None] for t in (q, k, v)))
    o2 = om.attention_prefill(*(t.transpose(0, 1).contiguous()[None] for t in (q, k, v)))
    assert torch.equal(o, o2)
    odd = torch.empty(T * 4 * D + 1, dtype=BF, device="cuda")[1:].view(1, T, 4, D)  # 2-byte aligned
    odd.copy_(q.transpose(0, 1)[None])
    assert torch.equal(om.attention_prefill(odd, *(t.transpose(0, 1)[None] for t in (k, v))), o)


def test_a_sequence_keeps_its_infinities_to_itself():
    lens = [70, 90, 33, 100]
    T = sum(lens)
    cu = offsets(lens)
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
    x = [draw(i, 1, T, h, 128) for i, h in enumerate((4, 2, 2))]
    do = draw(7, 1, T, 4, 128)
    bad = [t.clone() for t in x]
    for t in bad:
        t[:, cu[1]:cu[2]] = float("nan")
        t[:, cu[3]:] = float("inf")
    outs = []
    for t in (x, bad):
        t = [u.requires_grad_(True) for u in t]
        o = om.attention_prefill(*t, cu_seqlens=cu_t)
        outs.append([o, *torch.autograd.grad(o, t, do)])
    for a, b in zip(*outs):
        for n in (0, 2):
            assert torch.equal(a[:, cu[n]:cu[n + 1]], b[:, cu[n]:cu[n + 1]])
    assert bool(outs[1][0][:, cu[1]:cu[2]].isnan().all())


@pytest.mark.parametrize("Hq,Hkv,D,T,at", [(4, 2, 128, 300, 170), (2, 2, 64, 130, 64), (8, 1, 256, 90, 33),
                                           (3, 1, 80, 200, 199), (6, 2, 128, 70, 1),
                                           (4, 2, 128, 700, 300), (8, 1, 200, 600, 513)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_before_a_token_do_not_see_its_infinities(Hq, Hkv, D, T, at, bad):
    """Keys and values that are not finite, from one token on (a padded row's, say): the rows before
    are those of the sequence cut off there, and the rows from there on are not finite where a
    value is not."""
    say(f"not finite from {at} of {T}, Hq={Hq} D={D}, {bad}")
    q, k, v = draw(1, 1, T, Hq, D), draw(2, 1, T, Hkv, D), draw(3, 1, T, Hkv, D)
    for keys in (False, True):
        kb, vb = k.clone(), v.clone()
        if keys:
            kb[:, at:] = float("nan")
            vb[:, at:] = bad
        else:
            vb[:, at:, :, 1::3] = bad  # some columns only: the others stay as they are
        o = om.attention_prefill(q, kb, vb)
        val, tol = one_sequence(*(t[0, :at].double() for t in (q, k, v)), 0)
        check("rows before", o[0, :at], val["o"], tol["o"])
        if keys:
            assert bool(o[:, at:].isnan().all())
        else:
            assert not bool(o[:, at:, :, 1::3].isfinite().any())
            val, tol = one_sequence(*(t[0].double() for t in (q, k, v)), 0)
            for c in (0, 2):
                check("other columns", o[0, at:, :, c::3], val["o"][at:, :, c::3], tol["o"][at:, :, c::3])


def test_large_scores_and_scale():
    """Scores far from zero in both directions, so that the running maximum moves by a lot."""
    T, D = 300, 64
    q, k, v, do = (draw(i, 1, T, 2, D, scale=4.0 if i < 2 else 1.0) for i in range(4))
    k = k * torch.linspace(0.1, 3, T, device="cuda").to(BF)[None, :, None, None]
    x = [t.clone() for t in (q, k, v)]
    o = om.attention_prefill(*x, scale=0.5)
    val, tol = one_sequence(*(t[0].double() for t in x), 0, scale=0.5)
    # scores up to 2,000: fp32 products of 64 terms are off by 64 * 2^-24 * 2000 = 0.008 at most, and
    # each weight by that factor twice (numerator and sum)
    _, wide = one_sequence(x[0][0].double(), x[1][0].double(), x[2][0].double().abs(), 0, scale=0.5)
    mass = wide["o"] / 2.0 / 2.0 ** -8 / 1.05
    check("o", o[0], val["o"], tol["o"] + 0.016 * mass)


def test_empty_calls():
    for B, T in ((0, 5), (3, 0)):
        q = torch.zeros((B, T, 4, 64), dtype=BF, device="cuda", requires_grad=True)
        k = torch.zeros((B, T, 2, 64), dtype=BF, device="cuda")
        o = om.attention_prefill(q, k, k)
        assert o.shape == q.shape
        assert torch.autograd.grad(o.float().sum(), q)[0].shape == q.shape


def test_gradients_against_differences():
    """The directional derivative of sum(o * do) in 64 bits by central differences of the
    definition, against the kernels' gradients along the same direction."""
    T, Hq, Hkv, D = 90, 4, 2, 64
    x = [draw(i, 1, T, h, D) for i, h in enumerate((Hq, Hkv, Hkv))]
    do = draw(3, 1, T, Hq, D)
    u = [draw(10 + i, *t.shape[1:]).double() for i, t in enumerate(x)]
    leaves = [t.clone().requires_grad_(True) for t in x]
    grads = torch.autograd.grad(om.attention_prefill(*leaves), leaves, do)
    f = lambda e: sum((one_sequence(*(t[0].double() + e * d for t, d in zip(x, u)), 0)[0]["o"] * do[0].double()).flatten())
    h = 1e-4
    want = float((f(h) - f(-h)) / (2 * h))
    got = sum(float((g[0].double() * d).sum()) for g, d in zip(grads, u))
    val, tol = one_sequence(*(t[0].double() for t in x), 0, do=do[0].double())
    bound = sum(float((tol[n] * d.abs()).sum()) for n, d in zip(("dq", "dk", "dv"), u))
    # errors of either sign: the bound of their sum's size is the root of the sum of squares
    root = sum(float(((tol[n] * d) ** 2).sum()) for n, d in zip(("dq", "dk", "dv"), u)) ** 0.5
    assert abs(got - want) <= min(bound, 6 * root) + 1e-6 * abs(want)


def test_repeated_calls_are_equal_and_other_streams_too():
    T = 700
    x = [draw(i, 2, T, h, 128).requires_grad_(True) for i, h in enumerate((8, 2, 2))]
    do = draw(5, 2, T, 8, 128)
    run = lambda: [o := om.attention_prefill(*x), *torch.autograd.grad(o, x, do)]
    first = run()
    for a, b in zip(first, run()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_streams_at_once():
    """Two streams' forward and backward calls of their own, at the same time."""
    sets = [[draw(10 * i + j, 1, 1200, h, D) for j, h in enumerate((8, 2, 2, 8))] for i, D in enumerate((128, 256))]
    run = lambda q, k, v, do: [*(r := om.attention_prefill(q, k, v, output_lse=True)),
                               *om.attention_prefill_bwd(q, k, v, *r, do)]
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


def test_cotangents_of_any_layout_and_one_derivative():
    q, k, v = (draw(i, 2, 90, h, 64).requires_grad_(True) for i, h in enumerate((4, 2, 2)))
    one = torch.ones(2, 90, 4, 64, dtype=BF, device="cuda")
    want = torch.autograd.grad(om.attention_prefill(q, k, v), (q, k, v), one)
    got = torch.autograd.grad(om.attention_prefill(q, k, v).sum(), (q, k, v))  # an expanded cotangent
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = torch.autograd.grad(om.attention_prefill(q, k, v).transpose(1, 2), (q, k, v),
                              one.transpose(1, 2).contiguous())
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    dq, = torch.autograd.grad(om.attention_prefill(q, k, v).float().pow(2).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.float().sum(), k)


@pytest.mark.parametrize("T,D", [(260, 64), (900, 128), (700, 256)])
def test_captured_forward_and_backward(T, D):
    x = [draw(i, 1, T, h, D) for i, h in enumerate((4, 2, 2))]
    do = draw(5, 1, T, 4, D)
    cu = torch.tensor([0, 100, 100, T], dtype=torch.int32, device="cuda")

    def both():
        o, lse = om.attention_prefill(*x, cu_seqlens=cu, output_lse=True)
        return [o, *om.attention_prefill_bwd(*x, o, lse, do, cu_seqlens=cu)]

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
