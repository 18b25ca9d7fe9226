"""The paged cache in 8 bits on the GPU: append, attention of new tokens, decode step, with and without
a window, against the definition in 64 bits."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import omegalax_amd as om
from attn_reference import check
from cache8_reference import E4M3, Cache8
from sight_reference import one_sequence, seen
from test_gpu_attn import BF, draw, offsets, say

NAN, INF = float("nan"), float("inf")


def new_rows(c, new, seed=9):
    """Packed new tokens of every sequence, [1, T, Hkv, D] each of k and v, larger than what the blocks hold."""
    x = [torch.cat([c.rows(n, 2.0) for n in new])[None] for _ in range(2)]
    return [t.cuda() for t in x]


def put_all(c, new, k, v):
    for n, (a, b) in enumerate(zip(offsets(new), offsets(new)[1:])):
        if c.held[n] >= 0:
            c.put(n, c.held[n], k[0, a:b], v[0, a:b])


CASES = [  # held, new, page, Hq, Hkv, D
    ([0], [1], 16, 1, 1, 64), ([0, 0], [5, 70], 16, 4, 2, 128), ([1, 15, 16, 17], [1, 1, 16, 40], 16, 8, 2, 64),
    ([100, 0, 333], [64, 130, 1], 48, 8, 1, 128), ([63, 64, 65, 200], [3, 3, 3, 3], 64, 16, 2, 256),
    ([500], [77], 16, 6, 2, 128), ([1000, 10], [200, 350], 128, 7, 1, 256), ([40] * 70, [3] * 70, 32, 4, 4, 64),
    ([0, 5, 0], [0, 9, 0], 16, 2, 1, 128), ([7, -1, 30], [20, 5, 1], 32, 4, 2, 64), ([3] * 100, [1, 0] * 50, 16, 2, 2, 256),
    ([2500, 9], [33, 2], 64, 8, 2, 128),
]
SIGHTS = [(None, 0), (1, 0), (50, 4), (300, 70)]


@pytest.mark.parametrize("held,new,page,Hq,Hkv,D", CASES, ids=lambda x: str(x)[:12])
def test_append_and_turn(held, new, page, Hq, Hkv, D):
    say(f"turn of 8 bits held={held[:6]} new={new[:6]} page={page} Hq={Hq} Hkv={Hkv} D={D}")
    c = Cache8(held, [n if h >= 0 else 0 for n, h in zip(new, held)], page, Hkv, D, seed=len(held))
    T = sum(new)
    q = draw(7, 1, T, Hq, D, scale=1.5)
    k, v = new_rows(c, new)
    cu = offsets(new)
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
    om.kv_pages_write(k, v, *c.args(), cu_seqlens=cu_t, **c.exps())
    put_all(c, new, k, v)
    c.same()
    for window, sinks in SIGHTS:
        o = om.attention_prefill_paged(q, *c.args(), cu_seqlens=cu_t, window=window, sinks=sinks, **c.exps())
        for n, (a, b) in enumerate(zip(cu, cu[1:])):
            if held[n] < 0:
                assert not bool(o[0, a:b].any())
            elif b > a:
                keys, values, there = c.seq(n, held[n] + b - a)
                see = seen(b - a, held[n] + b - a, held[n], window, sinks, there)
                val, tol = one_sequence(q[0, a:b].double(), keys, values, see)
                check(f"o of sequence {n}, window {window}", o[0, a:b], val["o"], tol["o"])
    c.same()


@pytest.mark.parametrize("N", [1, 3, 63, 64, 65, 100])
@pytest.mark.parametrize("pads", [1, 70])
def test_rows_behind_the_last_offset_are_left_out(N, pads):
    """Large and infinite ones, which would raise the exponents of the last sequence's tokens."""
    held, new = [5 * n % 37 for n in range(N)], [1 + n % 3 for n in range(N)]
    c = Cache8(held, [80] * N, 16, 2, 64)
    k, v = new_rows(c, new)
    cu = torch.tensor(offsets(new), dtype=torch.int32, device="cuda")
    more = torch.full((1, pads, 2, 64), 1e30, dtype=BF, device="cuda")
    more[:, ::3] = INF
    om.kv_pages_write(*(torch.cat([t, more], 1) for t in (k, v)), *c.args(), cu_seqlens=cu, **c.exps())
    put_all(c, new, k, v)
    c.same()
    # offsets that are not in order count as their running maximum
    bad = cu.clone()
    bad[-1] = 0
    om.kv_pages_write(*(torch.cat([t, more], 1) for t in (k, v)), *c.args(), cu_seqlens=bad, **c.exps())
    put_all(c, new[:-1] + [0], k, v)
    c.same()


@pytest.mark.parametrize("held,T,page,Hkv,D", [([20, 0, 131], 50, 16, 2, 64), ([5, 16], 1, 32, 1, 256), ([0, 40, 9, 33], 17, 48, 3, 128)])
def test_unpacked_rows(held, T, page, Hkv, D):
    B = len(held)
    c = Cache8(held, [T] * B, page, Hkv, D)
    q = draw(1, B, T, 2 * Hkv, D)
    k, v = (t.view(B, T, Hkv, D) for t in new_rows(c, [T] * B))
    om.kv_pages_write(k, v, *c.args(), **c.exps())
    put_all(c, [T] * B, k.reshape(1, B * T, Hkv, D), v.reshape(1, B * T, Hkv, D))
    c.same()
    o = om.attention_prefill_paged(q, *c.args(), **c.exps())
    for n in range(B):
        keys, values, there = c.seq(n, held[n] + T)
        val, tol = one_sequence(q[n].double(), keys, values, seen(T, held[n] + T, held[n]))
        check(f"o of row {n}", o[n], val["o"], tol["o"])


def step_and_check(c, Hq, sight=(None, 0), seed=1, size=2.0):
    B = len(c.held)
    q = draw(seed, B, Hq, c.D, scale=1.5)
    k, v = (c.rows(B, size).cuda() for _ in range(2))
    out = om.attention_decode_step(q, k, v, *c.args(), window=sight[0], sinks=sight[1], **c.exps())
    for n, h in enumerate(c.held):
        if h >= 0:
            c.put(n, h, k[n:n + 1], v[n:n + 1])
    c.same()
    cap = c.table.shape[1] * c.page
    for n, h in enumerate(c.held):
        if h < 0:
            assert not bool(out[n].any())
            continue
        h = min(h, cap)
        keys, values, there = c.seq(n, min(h + 1, cap))
        see = seen(1, h + 1, h, *sight)[:, :keys.shape[0]] & there
        val, tol = one_sequence(q[n:n + 1].double(), keys, values, see)
        check(f"sequence {n}, window {sight}", out[n:n + 1], val["o"], tol["o"])


DECODE = [  # held, page, Hq, Hkv, D, least table width
    ([0], 16, 1, 1, 64, 0), ([0, 1, 15, 16, 17, 31, 32, 33], 16, 8, 2, 128, 0), ([63, 64, 65], 64, 4, 4, 64, 0),
    ([611], 16, 16, 4, 128, 0), ([100, 4000, 3], 48, 8, 1, 256, 0), ([250], 128, 32, 1, 128, 100), ([700, -1, 90], 32, 20, 1, 64, 200),
    ([3000, 47], 16, 24, 1, 256, 0), ([5, 900] * 40, 16, 8, 2, 64, 80), ([1300, 20], 64, 6, 2, 128, 300),
]


@pytest.mark.parametrize("held,page,Hq,Hkv,D,width", DECODE, ids=lambda x: str(x)[:12])
@pytest.mark.parametrize("sight", SIGHTS)
def test_decode_steps(held, page, Hq, Hkv, D, width, sight):
    say(f"decode of 8 bits held={held[:6]} page={page} Hq={Hq} Hkv={Hkv} D={D} window={sight}")
    c = Cache8(held, [1 if h >= 0 else 0 for h in held], page, Hkv, D, seed=3, width=width)
    step_and_check(c, Hq, sight)


def test_steps_behind_each_other_grow_a_block():
    """Tokens of growing size, one by one through three blocks: every exponent grows many times."""
    c = Cache8([5, 0], [40, 40], 16, 2, 64)
    for i in range(36):
        step_and_check(c, 4, (None, 0) if i % 2 else (20, 2), seed=i, size=1.4 ** i)
        c.held = [h + 1 for h in c.held]
        c.lengths += 1


SIZES = [0.0, 2.0 ** -120, 2.0 ** -90, 1e-30, 1.0, 447.0, 449.0, 1e30, 3.3e38]


@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_sizes_from_zero_to_the_types_largest(decode, D):
    """Blocks whose new token is of another order than the older ones; values that are not finite."""
    for first in SIZES:
        B = len(SIZES)
        c = Cache8([3] * B, [1] * B, 16, 1, D, size=first)
        k, v = (torch.cat([c.rows(1, 1.0).clamp(-1, 1).float().mul(s) for s in SIZES]).clamp(-3.3895e38, 3.3895e38).to(BF).cuda()
                for _ in range(2))
        k[0, 0, 5], v[4, 0, 0], k[8, 0, 3], v[2, 0, D - 1] = NAN, INF, -INF, NAN
        if decode:
            om.attention_decode_step(draw(1, B, 2, D), k, v, *c.args(), **c.exps())
        else:
            om.kv_pages_write(k[:, None], v[:, None], *c.args(), **c.exps())
        for n in range(B):
            c.put(n, 3, k[n:n + 1], v[n:n + 1])
        c.same()


@pytest.mark.parametrize("decode", [False, True])
def test_missing_pages_and_full_tables(decode):
    """A page missing in the middle, at the new token, and a table without room: nothing is written
    there, and what has no page is left out of the softmax."""
    D, page, Hkv, Hq = 64, 16, 1, 2
    held = [40, 47, 32, 30, 48, 48]
    c = Cache8(held, [1, 1, 1, 1, 0, 0], page, Hkv, D, seed=5)
    c.table = torch.cat([c.table, torch.full((6, 1), -1, dtype=torch.int32)], 1)[:, :3]
    c.table[0, 1], c.table[1, 2], c.table[3, 0] = -1, 1 << 20, -7
    c.block_table = c.table.cuda().contiguous()
    c.lengths[5] = 2 ** 31 - 5
    c.held[5] = 2 ** 31 - 5
    if decode:
        step_and_check(c, Hq)
        return
    k, v = (c.rows(6, 1.0).cuda() for _ in range(2))
    om.kv_pages_write(k[:, None], v[:, None], *c.args(), **c.exps())
    for n, h in enumerate(held):
        c.put(n, h, k[n:n + 1], v[n:n + 1])
    c.same()


@pytest.mark.parametrize("held,new,page,Hq,Hkv,D,sight", [
    ([3000], [20], 64, 4, 1, 128, (None, 0)), ([2000, 900], [70, 3], 16, 8, 2, 64, (700, 4)), ([5000], [130], 64, 8, 1, 256, (900, 20)),
    ([6000, 100], [40, 1], 32, 2, 2, 128, (2500, 0))])
def test_few_rows_over_a_long_cache(held, new, page, Hq, Hkv, D, sight):
    """The cache is read in shares, which a second kernel joins."""
    say(f"long cache of 8 bits held={held} new={new} Hq={Hq} D={D} window={sight}")
    c = Cache8(held, new, page, Hkv, D)
    T = sum(new)
    q = draw(1, 1, T, Hq, D)
    k, v = new_rows(c, new)
    cu = torch.tensor(offsets(new), dtype=torch.int32, device="cuda")
    om.kv_pages_write(k, v, *c.args(), cu_seqlens=cu, **c.exps())
    put_all(c, new, k, v)
    o = om.attention_prefill_paged(q, *c.args(), cu_seqlens=cu, window=sight[0], sinks=sight[1], **c.exps())
    for n, (a, b) in enumerate(zip(offsets(new), offsets(new)[1:])):
        keys, values, there = c.seq(n, held[n] + b - a)
        val, tol = one_sequence(q[0, a:b].double(), keys, values, seen(b - a, held[n] + b - a, held[n], *sight))
        check(f"o of sequence {n}", o[0, a:b], val["o"], tol["o"])


def test_conversation_through_a_cache_of_8_bits():
    """Prompts, a turn and single tokens with a window whose pages are dropped behind it: what one
    pass over the cache's numbers gives."""
    Hq, Hkv, D, page, window, sinks = 8, 2, 128, 16, 100, 5
    new = [[130, 61], [70, 45], [1, 1], [1, 1], [1, 1]]
    total = [sum(x) for x in zip(*new)]
    c = Cache8([0, 0], total, page, Hkv, D)
    for step, lens in enumerate(new):
        for n in range(2):  # pages wholly behind the window, but for the sinks'
            first = max(0, c.held[n] + 1 - window)
            for j in range(-(-sinks // page), first // page):
                old = int(c.table[n, j])
                c.table[n, j] = -1
                if old >= 0:
                    c.want[0][old], c.want[1][old] = NAN, NAN
                    c.k_pages[old] = c.v_pages[old] = torch.full((), NAN).to(E4M3).cuda()
        c.block_table.copy_(c.table)
        cu = offsets(lens)
        q = draw(20 + step, 1, cu[-1], Hq, D, scale=1.5)
        k, v = new_rows(c, lens)
        if step < 2:
            cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
            om.kv_pages_write(k, v, *c.args(), cu_seqlens=cu_t, **c.exps())
            o = om.attention_prefill_paged(q, *c.args(), cu_seqlens=cu_t, window=window, sinks=sinks, **c.exps())
        else:
            o = om.attention_decode_step(q[0], k[0], v[0], *c.args(), window=window, sinks=sinks, **c.exps())[None]
        put_all(c, lens, k, v)
        c.same()
        for n, (a, b) in enumerate(zip(cu, cu[1:])):
            keys, values, there = c.seq(n, c.held[n] + b - a)
            see = seen(b - a, c.held[n] + b - a, c.held[n], window, sinks)
            assert bool(there[see.any(0)].all())
            val, tol = one_sequence(q[0, a:b].double(), keys, values, see)
            check(f"step {step}, sequence {n}", o[0, a:b], val["o"], tol["o"])
        c.held = [h + m for h, m in zip(c.held, lens)]
        c.lengths += torch.tensor(lens, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("held,new,D,sight", [(0, 90, 128, (None, 0)), (3000, 30, 64, (None, 0)), (300, 70, 256, (20, 2)), (0, 200, 64, (33, 0))])
def test_queries_do_not_see_infinities_elsewhere(held, new, D, sight, bad):
    c = Cache8([held], [new], 16, 2, D)
    q = draw(1, 1, new, 4, D)
    k, v = new_rows(c, [new])
    cut = new // 2
    k[:, cut, 0], v[:, cut] = NAN, bad
    om.kv_pages_write(k, v, *c.args(), **c.exps())
    put_all(c, [new], k, v)
    c.same()
    o = om.attention_prefill_paged(q, *c.args(), window=sight[0], sinks=sight[1], **c.exps())
    keys, values, _ = c.seq(0, held + new)
    keys[held + cut], values[held + cut] = 0.0, 0.0
    val, tol = one_sequence(q[0].double(), keys, values, seen(new, held + new, held, *sight))
    past = new if sight[0] is None else min(new, cut + sight[0])
    for a, b in ((0, cut), (past, new)):
        check(f"queries {a} to {b}", o[0, a:b], val["o"][a:b], tol["o"][a:b])
    assert bool(o[0, cut:past].isnan().all())


def test_pools_larger_than_32_bit_offsets():
    """Pages past 2^32 bytes of each pool."""
    Hkv, D, page = 8, 256, 64
    pool = (1 << 32) // (page * Hkv * D) + 40
    c = Cache8([100], [60], page, Hkv, D, extra=0)
    n = c.k_pages.shape[0]
    zeros = lambda *s, t: torch.zeros(s, dtype=torch.uint8, device="cuda").view(t)
    big = [zeros(pool, page, Hkv, D, t=E4M3) for _ in range(2)]
    bige = [zeros(pool, page // 16, Hkv, t=torch.int8) for _ in range(2)]
    for t, s in zip((*big, *bige), (c.k_pages, c.v_pages, c.k_exps, c.v_exps)):
        t[pool - n:] = s
    table = (c.block_table + (pool - n)).to(torch.int32)
    exps = dict(k_exps=bige[0], v_exps=bige[1])
    T = 50
    q = draw(1, 1, T, 16, D)
    k, v = new_rows(c, [T])
    om.kv_pages_write(k, v, *big, table, c.lengths, **exps)
    c.put(0, 100, k[0], v[0])
    o = om.attention_prefill_paged(q, *big, table, c.lengths, **exps)
    keys, values, _ = c.seq(0, 150)
    val, tol = one_sequence(q[0].double(), keys, values, seen(T, 150, 100))
    check("turn", o[0], val["o"], tol["o"])
    q1, k1, v1 = draw(4, 1, 16, D), c.rows(1).cuda(), c.rows(1).cuda()
    o = om.attention_decode_step(q1, k1, v1, *big, table, c.lengths + T, **exps)
    c.put(0, 150, k1, v1)
    keys, values, _ = c.seq(0, 151)
    val, tol = one_sequence(q1.double(), keys, values, seen(1, 151, 150))
    check("decode", o, val["o"], tol["o"])
    c.k_pages, c.v_pages, c.k_exps, c.v_exps = (t[pool - n:] for t in (*big, *bige))
    c.same()
    assert not bool(big[0][:pool - n].view(torch.uint8).any())


def test_shared_pages():
    """Two sequences with the same first pages, each with a block of its own behind them."""
    c = Cache8([64, 64], [5, 5], 32, 2, 64)
    c.table[1, :2] = c.table[0, :2]
    c.block_table.copy_(c.table)
    step_and_check(c, 4)


@pytest.mark.parametrize("N,room", [(3, 40), (70, 5)])
def test_captured_turns_and_steps(N, room):
    """An append, its attention and a step captured once, replayed with other lengths, offsets and pages."""
    Hq, Hkv, D, page, T = 8, 2, 128, 16, 60 if N == 3 else 150
    held = [37 * n % 900 for n in range(N)]
    c, e = (Cache8(held, [page + room] * N, page, Hkv, D) for _ in range(2))
    for x in (c, e):  # every slot a number: lengths change below
        for t in (x.k_pages, x.v_pages):
            t.copy_(torch.where(t.float().isnan(), 0.5, t.float()).to(E4M3))
        for t in (x.k_exps, x.v_exps):
            t.copy_(t.clamp(-9, -5))
    q, k, v = draw(1, 1, T, Hq, D), draw(2, 1, T, Hkv, D), draw(3, 1, T, Hkv, D)
    q1, k1, v1 = draw(4, N, Hq, D), draw(5, N, Hkv, D), draw(6, N, Hkv, D)
    cu = torch.tensor([n * T // N for n in range(N + 1)], dtype=torch.int32, device="cuda")

    def turn(c):
        om.kv_pages_write(k, v, *c.args(), cu_seqlens=cu, **c.exps())
        o = om.attention_prefill_paged(q, *c.args(), cu_seqlens=cu, window=200, sinks=3, **c.exps())
        return o, om.attention_decode_step(q1, k1, v1, *c.args(), window=150, **c.exps()), \
            om.attention_decode_step(q1, k1, v1, *c.args(), **c.exps())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    state = [t.clone() for t in (c.k_pages, c.v_pages, c.k_exps, c.v_exps)]
    with torch.cuda.stream(side):
        turn(c)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = turn(c)
    for t, s in zip((c.k_pages, c.v_pages, c.k_exps, c.v_exps), state):
        t.copy_(s)
    for r in range(3):
        for i, t in enumerate((q, k, v, q1, k1, v1)):
            t.copy_(draw(50 + 6 * r + i, *t.shape, scale=2.0 ** r))
        lens = torch.tensor([max(0, h - 5 * r) if n % 7 != 3 else -1 for n, h in enumerate(held)], dtype=torch.int32)
        order = torch.randperm(N, generator=torch.Generator().manual_seed(r))  # whole tables change hands
        for x in (c, e):
            x.lengths.copy_(lens[order] if r else lens)
            x.block_table.copy_(x.table[order] if r else x.table)
        want = turn(e)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(o, want):
            assert torch.equal(a, b) and bool(a.isfinite().all())
        for a, b in zip((c.k_pages, c.v_pages, c.k_exps, c.v_exps), (e.k_pages, e.v_pages, e.k_exps, e.v_exps)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_streams_at_once():
    """Turns and steps of two caches on two streams at the same time, each as by itself."""
    shapes = [([900, 40, 2000], 30, 64, 8, 2, 128), ([700] * 40 + [3] * 30, 2, 64, 16, 8, 64)]
    sets = []
    for i, (held, T, page, Hq, Hkv, D) in enumerate(shapes):
        c = Cache8(held, [T + 1] * len(held), page, Hkv, D, seed=i, width=40)
        B = len(held)
        sets.append((c, draw(1, B, T, Hq, D), draw(2, B, T, Hkv, D), draw(3, B, T, Hkv, D), draw(4, B, Hq, D),
                     draw(5, B, Hkv, D), draw(6, B, Hkv, D), c.lengths + T))

    def run(c, q, k, v, q1, k1, v1, longer):
        om.kv_pages_write(k, v, *c.args(), **c.exps())
        o = om.attention_prefill_paged(q, *c.args(), **c.exps())
        return o, om.attention_decode_step(q1, k1, v1, *c.args()[:3], longer, **c.exps())

    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(*sets[i]))
    torch.cuda.synchronize()
    for w, rs in zip(want, got):
        assert all(bool(t.isfinite().all()) for t in w)
        for r in rs:
            assert all(torch.equal(a, b) for a, b in zip(w, r))


@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("kept", [16, 20])
def test_a_draft_that_is_turned_down(decode, kept):
    """Large tokens appended and taken back by a shorter length, then small ones in their place: the block that the
    kept tokens end in stays as the draft left it, a block that begins anew forgets it."""
    c = Cache8([kept], [20], 16, 2, 64)
    for size, n in ((500.0, 3), (1.0, 2), (1e-3, 1)):
        for i in range(n if decode else 1):
            k, v = (c.rows(1 if decode else n, size).cuda() for _ in range(2))
            if decode:
                om.attention_decode_step(draw(i, 1, 4, 64), k, v, *c.args()[:3], c.lengths + i, **c.exps())
            else:
                om.kv_pages_write(k[None], v[None], *c.args(), **c.exps())
            c.put(0, kept + i, k, v)
        c.same()


def test_refused_caches():
    c = Cache8([20], [5], 16, 2, 64)
    q, k = draw(1, 1, 5, 4, 64), draw(2, 1, 5, 2, 64)
    with pytest.raises(ValueError, match="go together"):
        om.kv_pages_write(k, k, *c.args(), k_exps=c.k_exps)
    with pytest.raises(ValueError, match="bf16"):
        om.kv_pages_write(k, k, *c.args())
    with pytest.raises(ValueError, match="k_exps must be int8"):
        om.attention_prefill_paged(q, *c.args(), k_exps=c.k_exps.float(), v_exps=c.v_exps)
    with pytest.raises(ValueError, match="v_exps must be int8"):
        om.attention_decode_step(q[0, :1], k[0, :1], k[0, :1], *c.args(), k_exps=c.k_exps, v_exps=c.v_exps[:1])
    b = c.k_pages.to(BF)
    with pytest.raises(ValueError, match="float8"):
        om.kv_pages_write(k, k, b, b, c.block_table, c.lengths, **c.exps())
