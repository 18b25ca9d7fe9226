"""Pages of a cache, dealt and returned on the GPU: whole numbers, equal to those of the host."""
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import omegalax_amd as om
from attn_reference import check
from cache8_reference import Cache8
from pages_reference import assign, release
from sight_reference import one_sequence, seen
from test_gpu_attn import draw, say

ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")


class Pool:
    """Tables whose first pages hold `held` tokens, and the other pages on the stack, on both sides."""

    def __init__(self, held, n_pages, width, page, seed=0):
        r = random.Random(seed)
        order = list(range(n_pages))
        r.shuffle(order)
        self.page, self.width = page, width
        self.table = [[-1] * width for _ in held]
        for row, h in zip(self.table, held):
            for i in range(min(width, -(-max(h, 0) // page))):
                row[i] = order.pop() if order else -1
        self.count = len(order)
        self.free = order + [r.randrange(-5, n_pages + 5) for _ in range(n_pages - len(order))]
        self.on_gpu()

    def on_gpu(self):
        self.t = ints(self.table).view(len(self.table), self.width)
        self.f, self.c = ints(self.free), ints([self.count])

    def same(self):
        assert self.t.tolist() == self.table
        assert int(self.c) == self.count
        assert self.f.tolist() == self.free

    def assign(self, lengths, new, T):
        got = om.kv_pages_assign(self.t, ints(lengths), ints(new), self.f, self.c, page_size=self.page, tokens=T)
        cu, positions, slots, missing, self.count = assign(self.table, lengths, new, self.free, self.count, self.page, T)
        for name, a, b in zip(("cu_seqlens", "positions", "slots", "missing"), got, (cu, positions, slots, [missing])):
            assert a.tolist() == b, name
        self.same()
        return got

    def release(self, lengths, **sight):
        om.kv_pages_release(self.t, ints(lengths), self.f, self.c, page_size=self.page, **sight)
        self.count = release(self.table, lengths, self.free, self.count, self.page, **sight)
        self.same()


@pytest.mark.parametrize("N,most_held,most_new,page,width,spare", [
    (0, 0, 0, 16, 4, 3), (1, 0, 1, 16, 1, 1), (1, 100, 50, 16, 12, 20), (7, 100, 3, 16, 9, 10), (64, 4000, 1, 16, 440, 70),
    (64, 300, 200, 64, 10, 400), (300, 50, 70, 32, 5, 300), (1500, 40, 3, 16, 4, 900), (5000, 30, 4, 16, 3, 4000),
    (3, 10, 20000, 16, 1300, 5000), (2, 70000, 100, 65536, 3, 4), (5, 200, 300, 16, 20, 11), (40, 100, 90, 16, 0, 5),
    (700, 20, 30, 48, 60, 900),
])
def test_dealt_and_returned(N, most_held, most_new, page, width, spare):
    """Room for new tokens, given back; then some of them stay and others end, with and without a window."""
    say(f"pages of {N} sequences, page {page}, width {width}, {spare} free")
    r = random.Random(N + width)
    held = [r.choice([-1, 0, r.randrange(most_held + 1), r.randrange(most_held + 1)]) for _ in range(N)]
    new = [r.choice([0, -3, r.randrange(most_new + 1), r.randrange(most_new + 1)]) for _ in range(N)]
    used = sum(min(width, -(-max(h, 0) // page)) for h in held)
    p = Pool(held, used + spare, width, page, seed=N)
    total = sum(n for n, h in zip(new, held) if n > 0 and h >= 0)
    before = [row[:] for row in p.table], list(p.free), p.count
    p.assign(held, new, total)
    dealt = [row[:] for row in p.table]
    p.assign(held, new, total + 5)  # a second time: whatever has its page keeps it, and what is short stays so
    assert p.table == dealt
    p.release(held)
    assert p.table == before[0] and p.count == before[2]
    assert p.free[:p.count] == before[1][:p.count]
    p.assign(held, new, max(0, total - 7))  # without room for the last ones
    keep = [h if h < 0 else r.choice([0, -1, h, h + max(0, n), h + max(0, n) // 2]) for h, n in zip(held, new)]
    p.release(keep)
    held = [max(0, k) for k in keep]
    for sight in (dict(window=40, sinks=5), dict(window=17), dict(window=1 << 40, sinks=1 << 41)):
        p.release(held, **sight)


@pytest.mark.parametrize("width", [1, 3])
@pytest.mark.parametrize("N", [8191, 8192, 8193])
def test_more_rows_than_one_workgroup_returns(N, width):
    """Tables of few entries and many rows: the return's rows lie in LDS up to 8,192 of them."""
    say(f"pages of {N} sequences, width {width}")
    r = random.Random(N + width)
    held = [r.choice([-1, 0, r.randrange(16 * width + 1)]) for _ in range(N)]
    used = sum(-(-max(h, 0) // 16) for h in held)
    for sight in (dict(), dict(window=9, sinks=3), dict(window=1)):
        p = Pool(held, used + 40, width, 16, seed=N)
        p.release([h if h < 0 else r.choice([h, 0, h // 2, -1]) for h in held], **sight)
        p.release([0] * N, **sight)


@pytest.mark.parametrize("count", [-4, 0, 3, 50, 1 << 30])
def test_a_count_out_of_range_is_read_as_the_nearest(count):
    for what in ("assign", "release"):
        p = Pool([40, 0, 3], 50, 6, 16)
        p.count = count
        p.on_gpu()
        if what == "assign":
            p.assign([40, 0, 3], [30, 16, 1], 60)
        else:
            p.release([0, 0, 1])


def test_entries_that_are_no_page_are_replaced():
    p = Pool([0, 0], 20, 4, 16)
    p.table = [[-7, 25, 20, 3], [1 << 30, -1, 5, -(1 << 31)]]
    p.on_gpu()
    p.assign([0, 16], [64, 48], 112)
    p.release([16, 16])


def test_lengths_far_past_the_table():
    p = Pool([0, 0, 5], 9, 3, 16)
    p.assign([2 ** 31 - 3, 47, 5], [10, 5, 2], 17)
    p.release([2 ** 31 - 1, 48, 7], window=2 ** 31 - 1)


def test_sinks_past_every_position():
    """More sinks than there are positions: nothing is behind the window, whatever the page's size."""
    p = Pool([150000], 6, 4, 65536)
    p.release([150000], window=10, sinks=2 ** 31 - 1)
    p.release([150000], window=10, sinks=2)


def test_more_tokens_than_the_others_sum():
    """Numbers whose sum passes 32 bits: the room decides."""
    p = Pool([0, 3, 9], 40, 10, 16)
    p.assign([0, 3, 9], [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], 100)


def test_a_captured_step_of_pages():
    """Dealt and returned in one graph, replayed with other lengths and eager calls between."""
    a, b = (Pool([20 * n % 70 for n in range(90)], 900, 400, 16, seed=1) for _ in range(2))
    lengths, new, keep = ints([20 * n % 70 for n in range(90)]), ints([n % 3 for n in range(90)]), ints([-1] * 90)

    def step(p):
        made = om.kv_pages_assign(p.t, lengths, new, p.f, p.c, page_size=16, tokens=6000)
        om.kv_pages_release(p.t, keep, p.f, p.c, page_size=16, window=30)
        return made

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        made = step(a)
    a.on_gpu_again = [x.copy_(y) for x, y in ((a.t, b.t), (a.f, b.f), (a.c, b.c))]
    for i in range(4):
        r = random.Random(i)
        new.copy_(ints([r.randrange(-1, 60) for _ in range(90)]))
        keep.copy_(ints([r.choice([-1, 0, 30, 100]) for _ in range(90)]))
        want = step(b)
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip((*made, a.t, a.f, a.c), (*want, b.t, b.f, b.c)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("eight", [False, True])
def test_a_serving_loop_without_a_length_on_the_host(eight):
    """Prompts come, tokens follow, pages behind the window go back and one request ends: appends and
    attention by what is dealt, against 64 bits of each sequence's own tokens."""
    Hq, Hkv, D, page, window, sinks, width, pool = 8, 2, 64, 16, 50, 3, 40, 60
    lens = [130, 7, 64]
    sight = dict(window=window, sinks=sinks)
    dtype = torch.float8_e4m3fn if eight else torch.bfloat16
    kp, vp = (torch.full((pool, page, Hkv, D), float("nan"), device="cuda").to(dtype) for _ in range(2))
    exps = dict(k_exps=torch.zeros((pool, 1, Hkv), dtype=torch.int8, device="cuda"),
                v_exps=torch.zeros((pool, 1, Hkv), dtype=torch.int8, device="cuda")) if eight else {}
    table, lengths = torch.full((3, width), -1, dtype=torch.int32, device="cuda"), ints([0, 0, 0])
    free, count = ints(list(range(pool))), ints([pool])
    past = [[torch.empty(0, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(3)]
    host = [0, 0, 0]
    # the 8-bit cache's own rounding is in its tests: here its values are read back through the table
    for step in range(30):
        new = lens if step == 0 else [1, 1, 1] if step < 20 else [1, -1, 1]
        T = sum(max(0, n) for n in new)
        if step == 20:  # the second request has ended
            lengths[1] = 0
            om.kv_pages_release(table, lengths, free, count, page_size=page, **sight)
            assert not bool((table[1] >= 0).any())
            lengths[1] = -1
        cu, positions, slots, missing = om.kv_pages_assign(table, lengths, ints(new), free, count, page_size=page, tokens=T)
        assert int(missing) == 0 and bool((slots >= 0).all())
        q, k, v = draw(step, 1, T, Hq, D), draw(100 + step, 1, T, Hkv, D), draw(200 + step, 1, T, Hkv, D)
        cache = (kp, vp, table, lengths)
        om.kv_pages_write(k, v, *cache, cu_seqlens=cu, **exps)
        o = om.attention_prefill_paged(q, *cache, cu_seqlens=cu, **exps, **sight)
        if not eight:  # the slots are where the append put the tokens
            assert torch.equal(kp.flatten(0, 1)[slots], k[0])
        at = 0
        for n, m in enumerate(new):
            if m <= 0:
                continue
            assert positions[at:at + m].tolist() == list(range(host[n], host[n] + m))
            past[n] = [torch.cat([p, x[0, at:at + m]]) for p, x in zip(past[n], (k, v))]
            if eight:
                rows = torch.arange(host[n] + m, device="cuda")
                page_of = table[n].long()[rows // page]
                scale = lambda e: torch.exp2(e[page_of.clamp(min=0), 0].double())[..., None]
                back = lambda t, e: t[page_of.clamp(min=0), rows % page].double() * scale(e)
                keys, values = back(kp, exps["k_exps"]), back(vp, exps["v_exps"])
            else:
                keys, values = (x.double() for x in past[n])
            see = seen(m, host[n] + m, host[n], window, sinks)
            val, tol = one_sequence(q[0, at:at + m].double(), keys, values, see)
            check(f"step {step}, sequence {n}", o[0, at:at + m], val["o"], tol["o"])
            if eight:  # off by half a step of the block's largest, 2^-4 of a value or 2^-10 of 2^e
                live = see.any(0)
                for got, x, e in ((keys, past[n][0], "k_exps"), (values, past[n][1], "v_exps")):
                    x = x.double()
                    # a block grows a few times at most, each growth half a step again
                    far = (got - x).abs() - 4 * (x.abs() * 2.0 ** -4 + scale(exps[e]) * 2.0 ** -10)
                    assert float(far[live].max()) <= 0
            at += m
            host[n] += m
        lengths += ints([max(0, m) for m in new])
        om.kv_pages_release(table, lengths, free, count, page_size=page, **sight)
        if step > 3:  # the window's pages, those of the sinks, and no others
            assert int((table[0] >= 0).sum()) <= window // page + 3


@pytest.mark.parametrize("eight", [False, True])
def test_a_padded_batch(eight):
    """Room for more tokens than there are, whose rows a last row of the table takes: what the batch without them gives."""
    Hq, Hkv, D, page, held, new, T = 4, 2, 64, 16, [20, 0, 45, -1], [7, 30, 1, 0], 60
    pools = []
    for tokens in (T, sum(new)):
        p = Pool(held, 40, 6, page)
        cache = [torch.zeros((40, page, Hkv, D), device="cuda").to(torch.float8_e4m3fn if eight else torch.bfloat16) for _ in range(2)]
        exps = dict(zip(("k_exps", "v_exps"), torch.zeros((2, 40, 1, Hkv), dtype=torch.int8, device="cuda"))) if eight else {}
        cu = p.assign(held, new, tokens)[0]
        q, k, v = (draw(i, 1, T, h, D) for i, h in enumerate((Hq, Hkv, Hkv)))
        k[:, sum(new):], v[:, sum(new):] = float("nan"), float("inf")
        at = (*cache, p.t, ints(held))
        om.kv_pages_write(k[:, :tokens], v[:, :tokens], *at, cu_seqlens=cu, **exps)
        o = om.attention_prefill_paged(q[:, :tokens], *at, cu_seqlens=cu, window=30, sinks=2, **exps)
        pools.append((cache, exps, o))
    (a, ea, oa), (b, eb, ob) = pools
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))
    assert all(torch.equal(ea[n], eb[n]) for n in ea)
    assert torch.equal(oa[:, :sum(new)], ob) and not bool(oa[:, sum(new):].any())


def test_refusals():
    p = Pool([40, 0], 20, 6, 16)
    l, n = ints([40, 0]), ints([1, 1])
    good = dict(page_size=16, tokens=2)
    with pytest.raises(ValueError, match="block_table"):
        om.kv_pages_assign(p.t[:1], l, n, p.f, p.c, **good)
    with pytest.raises(ValueError, match="contiguous"):
        om.kv_pages_assign(p.t[:, ::2], l, n, p.f, p.c, **good)
    with pytest.raises(ValueError, match="new_tokens"):
        om.kv_pages_assign(p.t, l, n[:1], p.f, p.c, **good)
    with pytest.raises(ValueError, match="free_count"):
        om.kv_pages_release(p.t, l, p.f, p.f, page_size=16)
    with pytest.raises(ValueError, match="tokens"):
        om.kv_pages_assign(p.t, l, n, p.f, p.c, page_size=16, tokens=-1)
    with pytest.raises(ValueError, match="window"):
        om.kv_pages_release(p.t, l, p.f, p.c, page_size=16, window=0)
    with pytest.raises(om.GDNError, match="page size"):
        om.kv_pages_release(p.t, l, p.f, p.c, page_size=24)
    p.same()
