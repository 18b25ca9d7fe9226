"""The paged key-value cache on the GPU: append, attention of new tokens, decode step."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import omegalax_amd as om
from attn_reference import check, one_sequence
from test_gpu_attn import BF, draw, offsets, say

NAN = float("nan")


class Cache:
    """Sequences of given lengths in shuffled pages, every unused slot a NaN; `width` is the least
    number of table columns.  keys[n], values[n]: what the sequence holds, in order."""

    def __init__(self, held, room, page, Hkv, D, seed=0, extra=3, width=0):
        n_pages = [-(-(max(h, 0) + r) // page) for h, r in zip(held, room)]
        pool = sum(n_pages) + extra
        self.page, self.Hkv, self.D = page, Hkv, D
        self.k_pages = torch.full((pool, page, Hkv, D), NAN, dtype=BF, device="cuda")
        self.v_pages = torch.full_like(self.k_pages, NAN)
        order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = torch.full((len(held), max(width, *n_pages)), -1, dtype=torch.int32)
        at = 0
        for n, p in enumerate(n_pages):
            self.table[n, :p] = torch.tensor(order[at:at + p], dtype=torch.int32)
            at += p
        self.held = list(held)
        self.keys, self.values = [], []
        for n, h in enumerate(held):
            h = max(h, 0)
            self.keys.append(draw(seed + 2 * n + 1, h, Hkv, D))
            self.values.append(draw(seed + 2 * n + 2, h, Hkv, D))
            self.put(n, 0, self.keys[n], self.values[n])
        self.block_table = self.table.cuda()
        self.lengths = torch.tensor(held, dtype=torch.int32, device="cuda")

    def put(self, n, pos, k, v, pools=None):
        kp, vp = pools or (self.k_pages, self.v_pages)
        for i in range(k.shape[0]):
            page = int(self.table[n, (pos + i) // self.page]) if (pos + i) // self.page < self.table.shape[1] else -1
            if 0 <= page < kp.shape[0]:
                kp[page, (pos + i) % self.page] = k[i]
                vp[page, (pos + i) % self.page] = v[i]

    def args(self):
        return self.k_pages, self.v_pages, self.block_table, self.lengths


def equal(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def same_pools(c, want):
    assert equal(c.k_pages, want[0]) and equal(c.v_pages, want[1])


CASES = [  # held, new, page, Hq, Hkv, D
    ([0], [1], 16, 1, 1, 64), ([0, 0], [5, 70], 16, 4, 2, 128), ([1, 15, 16, 17], [1, 1, 16, 40], 16, 8, 2, 64),
    ([100, 0, 333], [64, 130, 1], 48, 8, 1, 128), ([63, 64, 65, 200], [3, 3, 3, 3], 64, 16, 2, 256),
    ([500], [77], 16, 6, 2, 128), ([1000, 10], [200, 350], 128, 7, 1, 256), ([40] * 70, [3] * 70, 32, 4, 4, 64),
    ([0, 5, 0], [0, 9, 0], 16, 2, 1, 128),
]


@pytest.mark.parametrize("held,new,page,Hq,Hkv,D", CASES, ids=lambda x: str(x)[:12])
def test_append_and_turn(held, new, page, Hq, Hkv, D):
    say(f"turn held={held[:6]} new={new[:6]} page={page} Hq={Hq} Hkv={Hkv} D={D}")
    c = Cache(held, new, page, Hkv, D, seed=len(held))
    T = sum(new)
    q, k, v = draw(7, 1, T, Hq, D, scale=1.5), draw(8, 1, T, Hkv, D), draw(9, 1, T, Hkv, D)
    cu = offsets(new)
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
    want = c.k_pages.clone(), c.v_pages.clone()
    for n, (a, b) in enumerate(zip(cu, cu[1:])):
        c.put(n, held[n], k[0, a:b], v[0, a:b], want)
    om.kv_pages_write(k, v, *c.args(), cu_seqlens=cu_t)
    same_pools(c, want)
    o = om.attention_prefill_paged(q, *c.args(), cu_seqlens=cu_t)
    for n, (a, b) in enumerate(zip(cu, cu[1:])):
        if b > a:
            val, tol = one_sequence(q[0, a:b].double(), torch.cat([c.keys[n], k[0, a:b]]).double(),
                                    torch.cat([c.values[n], v[0, a:b]]).double(), held[n])
            check(f"o of sequence {n}", o[0, a:b], val["o"], tol["o"])
    same_pools(c, want)


@pytest.mark.parametrize("B,T", [(3, 1), (2, 50)])
def test_unpacked_rows(B, T):
    held = [20, 0, 131][:B]
    c = Cache(held, [T] * B, 16, 2, 64)
    q, k, v = draw(1, B, T, 4, 64), draw(2, B, T, 2, 64), draw(3, B, T, 2, 64)
    om.kv_pages_write(k, v, *c.args())
    o = om.attention_prefill_paged(q, *c.args())
    for n in range(B):
        val, tol = one_sequence(q[n].double(), torch.cat([c.keys[n], k[n]]).double(),
                                torch.cat([c.values[n], v[n]]).double(), held[n])
        check(f"o of row {n}", o[n], val["o"], tol["o"])


def shares(B, T, Hq, Hkv, D, c, packed=False):
    """Of a turn's keys, by the workspace for their partial sums."""
    size = om._lib.lib().omx_gdn_attn_paged_workspace_size(B, T, Hq, Hkv, D, len(c.held), packed, c.page, c.table.shape[1])
    return max(1, size // (B * T * Hq * (D + 2) * 4))


@pytest.mark.parametrize("held,T,page,Hq,Hkv,D,split", [
    ([3000, 0, 1111], 20, 64, 4, 1, 128, True), ([2000, 900], 70, 16, 8, 2, 64, True), ([1500, 2222, 5, 640], 33, 48, 8, 1, 256, True),
    ([700, -1, 2500], 1, 64, 32, 1, 128, True), ([600, 900, 0, 300, 1100, 20, 450, 800], 300, 64, 16, 8, 64, False),
])
def test_rows_of_a_batch_over_long_caches(held, T, page, Hq, Hkv, D, split):
    """Rows that are not packed, few of them with their keys in shares and enough without."""
    say(f"batch over long caches held={held} T={T} Hq={Hq} Hkv={Hkv} D={D}")
    B = len(held)
    c = Cache(held, [T] * B, page, Hkv, D, seed=B)
    assert (shares(B, T, Hq, Hkv, D, c) > 1) == split
    q, k, v = draw(1, B, T, Hq, D, scale=1.5), draw(2, B, T, Hkv, D), draw(3, B, T, Hkv, D)
    om.kv_pages_write(k, v, *c.args())
    o = om.attention_prefill_paged(q, *c.args())
    for n in range(B):
        if held[n] < 0:
            assert not bool(o[n].any())
            continue
        val, tol = one_sequence(q[n].double(), torch.cat([c.keys[n], k[n]]).double(),
                                torch.cat([c.values[n], v[n]]).double(), held[n])
        check(f"o of row {n}", o[n], val["o"], tol["o"])


@pytest.mark.parametrize("new,held", [(2, 4000), (40, 3000), (130, 5000)])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 1, 128), (2, 2, 64), (8, 1, 256)])
def test_few_rows_over_a_long_cache(new, held, Hq, Hkv, D):
    """The cache is read in shares, which a second kernel joins."""
    say(f"long cache new={new} held={held} Hq={Hq} D={D}")
    c = Cache([held, 100], [new, 1], 64, Hkv, D)
    T = new + 1
    q, k, v = draw(1, 1, T, Hq, D), draw(2, 1, T, Hkv, D), draw(3, 1, T, Hkv, D)
    cu = torch.tensor([0, new, T], dtype=torch.int32, device="cuda")
    om.kv_pages_write(k, v, *c.args(), cu_seqlens=cu)
    o = om.attention_prefill_paged(q, *c.args(), cu_seqlens=cu)
    for n, (a, b) in enumerate(((0, new), (new, T))):
        val, tol = one_sequence(q[0, a:b].double(), torch.cat([c.keys[n], k[0, a:b]]).double(),
                                torch.cat([c.values[n], v[0, a:b]]).double(), c.held[n])
        check(f"o of sequence {n}", o[0, a:b], val["o"], tol["o"])


DECODE = [  # held, page, Hq, Hkv, D, least table width
    ([0], 16, 1, 1, 64, 0), ([0, 1, 15, 16, 17, 31, 32, 33], 16, 8, 2, 128, 0), ([63, 64, 65], 64, 4, 4, 64, 0),
    ([611], 16, 16, 4, 128, 0), ([100, 4000, 3], 48, 8, 1, 256, 0), ([250], 128, 32, 1, 128, 100),
    ([70, 300], 32, 34, 2, 64, 0), ([129, 5], 16, 64, 2, 256, 0), ([5000], 64, 2, 1, 64, 2000), ([40] * 90, 16, 6, 2, 128, 0),
    ([9000, 0, 10, 2500], 64, 10, 2, 128, 0),
]


@pytest.mark.parametrize("held,page,Hq,Hkv,D,width", DECODE, ids=lambda x: str(x)[:12])
def test_decode_steps(held, page, Hq, Hkv, D, width):
    say(f"decode held={held[:8]} page={page} Hq={Hq} Hkv={Hkv} D={D}")
    c = Cache(held, [2] * len(held), page, Hkv, D, seed=5, width=width)
    for step in range(2):
        B = len(held)
        q, k, v = draw(50 + step, B, Hq, D, scale=1.5), draw(60 + step, B, Hkv, D), draw(70 + step, B, Hkv, D)
        want = c.k_pages.clone(), c.v_pages.clone()
        for n in range(B):
            c.put(n, held[n] + step, k[n:n + 1], v[n:n + 1], want)
            c.keys[n], c.values[n] = torch.cat([c.keys[n], k[n:n + 1]]), torch.cat([c.values[n], v[n:n + 1]])
        o = om.attention_decode_step(q, k, v, *c.args())
        same_pools(c, want)
        for n in range(B):
            val, tol = one_sequence(q[n:n + 1].double(), c.keys[n].double(), c.values[n].double(), held[n] + step)
            check(f"step {step}, sequence {n}", o[n:n + 1], val["o"], tol["o"])
        c.lengths += 1


def segments(c, Hq):
    """Room for a decode step's partial sums, in sequences' segments: none in one launch."""
    N, Hkv, D = len(c.held), c.Hkv, c.D
    size = om._lib.lib().omx_gdn_attn_decode_workspace_size(N, Hq, Hkv, D, c.page, c.table.shape[1])
    return size // (Hq * (D + 2) * 4)


def step_and_check(c, Hq, seed=50):
    """One decode step; sequences of negative length take no part."""
    B, Hkv, D, held = len(c.held), c.Hkv, c.D, c.held
    q, k, v = draw(seed, B, Hq, D, scale=1.5), draw(seed + 1, B, Hkv, D), draw(seed + 2, B, Hkv, D)
    want = c.k_pages.clone(), c.v_pages.clone()
    for n in range(B):
        if held[n] >= 0:
            c.put(n, held[n], k[n:n + 1], v[n:n + 1], want)
    o = om.attention_decode_step(q, k, v, *c.args())
    same_pools(c, want)
    for n in range(B):
        if held[n] < 0:
            assert not bool(o[n].any())
            continue
        val, tol = one_sequence(q[n:n + 1].double(), torch.cat([c.keys[n], k[n:n + 1]]).double(),
                                torch.cat([c.values[n], v[n:n + 1]]).double(), held[n])
        check(f"sequence {n}", o[n:n + 1], val["o"], tol["o"])


@pytest.mark.parametrize("held,page,Hq,Hkv,D,width", [
    ([40] * 63 + [2500], 64, 16, 8, 128, 0), ([3000] + [97 * n % 200 for n in range(64)], 16, 8, 8, 64, 0),
    ([31 * n % 300 for n in range(256)] + [-1], 64, 4, 2, 256, 100), ([7] * 512, 16, 2, 1, 128, 80),
], ids=lambda x: str(x)[:12])
def test_decode_steps_of_large_batches(held, page, Hq, Hkv, D, width):
    """At least 512 sequences' key heads, of lengths that differ: equal ranges of the keys, joined."""
    say(f"decode, large batch of {len(held)}, Hq={Hq} Hkv={Hkv} D={D}")
    c = Cache(held, [1] * len(held), page, Hkv, D, seed=9, width=width)
    assert len(held) * Hkv >= 512 and segments(c, Hq) == 256 // Hkv + len(held)
    step_and_check(c, Hq)


@pytest.mark.parametrize("decode", [False, True])
def test_pages_that_are_none_and_sequences_that_take_no_part(decode):
    """Tokens of entries outside the pool are left out; negative lengths give zeros; nothing is
    written outside the pages."""
    D, page, Hq, Hkv = 128, 32, 4, 2
    held = [100, -1, 90, 64, 0]
    c = Cache(held, [1, 0, 1, 1, 1], page, Hkv, D)
    c.table[0, 1] = -1                       # a hole in the middle
    c.table[2, :] = 2 ** 31 - 1              # nothing left
    c.table[3, 2] = c.k_pages.shape[0]       # the new token has no page
    c.block_table.copy_(c.table)
    B = len(held)
    q, k, v = draw(1, B, Hq, D), draw(2, B, Hkv, D), draw(3, B, Hkv, D)
    want = c.k_pages.clone(), c.v_pages.clone()
    for n in (0, 2, 3, 4):
        c.put(n, held[n], k[n:n + 1], v[n:n + 1], want)
    if decode:
        o = om.attention_decode_step(q, k, v, *c.args())
    else:
        om.kv_pages_write(k[:, None], v[:, None], *c.args())
        o = om.attention_prefill_paged(q[:, None], *c.args())[:, 0]
    same_pools(c, want)
    for n in (0, 3, 4):
        keys, values = torch.cat([c.keys[n], k[n:n + 1]]).double(), torch.cat([c.values[n], v[n:n + 1]]).double()
        there = torch.tensor([0 <= int(c.table[n, i // page]) < c.k_pages.shape[0] for i in range(held[n] + 1)]).cuda()
        val, tol = one_sequence(q[n:n + 1].double(), keys, values, held[n], allowed=there)
        check(f"sequence {n}", o[n:n + 1], val["o"], tol["o"])
    assert not bool(o[1].any()) and not bool(o[2].any())


@pytest.mark.parametrize("decode", [False, True])
def test_a_full_table_takes_no_more(decode):
    D, page = 64, 16
    c = Cache([32, 40], [0, 1], page, 1, D)
    c.table[1, 2] = -1
    c.block_table.copy_(c.table)
    c.lengths.copy_(torch.tensor([48, 2 ** 31 - 5], dtype=torch.int32))
    c.block_table = c.block_table[:, :2].contiguous()  # room for 32 tokens each
    q, k, v = draw(1, 2, 2, D), draw(2, 2, 1, D), draw(3, 2, 1, D)
    want = c.k_pages.clone(), c.v_pages.clone()
    if decode:
        o = om.attention_decode_step(q, k, v, *c.args())
    else:
        om.kv_pages_write(k[:, None], v[:, None], *c.args())
        o = om.attention_prefill_paged(q[:, None], *c.args())[:, 0]
    same_pools(c, want)
    for n in range(2):
        val, tol = one_sequence(q[n:n + 1].double(), c.keys[n][:32].double(), c.values[n][:32].double(), 100)
        check(f"sequence {n}", o[n:n + 1], val["o"], tol["o"])


def test_prompt_then_turn_then_tokens():
    """A conversation through the cache gives what one whole prompt gives."""
    Hq, Hkv, D, page = 8, 2, 128, 16
    lens, turn, steps = [130, 61], [20, 45], 3
    total = [a + b + steps for a, b in zip(lens, turn)]
    q, k, v = ([draw(10 * i + n, t, h, D) for n, t in enumerate(total)] for i, h in enumerate((Hq, Hkv, Hkv)))
    c = Cache([0, 0], total, page, Hkv, D)
    pack = lambda ts, at, n: torch.cat([t[a:a + m] for t, a, m in zip(ts, at, n)])[None]
    got = [[], []]
    at = [0, 0]
    for new in (lens, turn):
        cu = torch.tensor(offsets(new), dtype=torch.int32, device="cuda")
        x = [pack(t, at, new) for t in (q, k, v)]
        om.kv_pages_write(*x[1:], *c.args(), cu_seqlens=cu)
        o = om.attention_prefill(*x, cu_seqlens=cu) if at == [0, 0] else \
            om.attention_prefill_paged(x[0], *c.args(), cu_seqlens=cu)
        for n in range(2):
            got[n].append(o[0, offsets(new)[n]:offsets(new)[n + 1]])
        at = [a + m for a, m in zip(at, new)]
        c.lengths += torch.tensor(new, dtype=torch.int32, device="cuda")
    for _ in range(steps):
        o = om.attention_decode_step(*(torch.stack([t[n][at[n]] for n in range(2)]) for t in (q, k, v)), *c.args())
        for n in range(2):
            got[n].append(o[n:n + 1])
        at = [a + 1 for a in at]
        c.lengths += 1
    for n in range(2):
        val, tol = one_sequence(q[n].double(), k[n].double(), v[n].double(), 0)
        check(f"sequence {n}", torch.cat(got[n]), val["o"], tol["o"])


def test_pools_larger_than_32_bit_offsets():
    """Pages past 2^31 elements (4 GiB) of each pool."""
    Hkv, D, page = 8, 256, 64
    pool = (1 << 31) // (page * Hkv * D) + 40
    c = Cache([100], [60], page, Hkv, D, extra=0)
    big = [torch.zeros((pool, page, Hkv, D), dtype=BF, device="cuda") for _ in range(2)]
    n = c.k_pages.shape[0]
    for t, s in zip(big, (c.k_pages, c.v_pages)):
        t[pool - n:] = s
    table = (c.block_table + (pool - n)).to(torch.int32)
    T = 50
    q, k, v = draw(1, 1, T, 16, D), draw(2, 1, T, Hkv, D), draw(3, 1, T, Hkv, D)
    om.kv_pages_write(k, v, *big, table, c.lengths)
    o = om.attention_prefill_paged(q, *big, table, c.lengths)
    val, tol = one_sequence(q[0].double(), torch.cat([c.keys[0], k[0]]).double(), torch.cat([c.values[0], v[0]]).double(), 100)
    check("turn", o[0], val["o"], tol["o"])
    q1, k1, v1 = draw(4, 1, 16, D), draw(5, 1, Hkv, D), draw(6, 1, Hkv, D)
    o = om.attention_decode_step(q1, k1, v1, *big, table, c.lengths + T)
    val, tol = one_sequence(q1.double(), torch.cat([c.keys[0], k[0], k1]).double(),
                            torch.cat([c.values[0], v[0], v1]).double(), 150)
    check("decode", o, val["o"], tol["o"])
    assert not bool(big[0][:pool - n].any())


@pytest.mark.parametrize("held,new,D", [(0, 70, 128), (3000, 20, 64), (200, 90, 256)])
def test_queries_before_a_token_do_not_see_its_infinities(held, new, D):
    """The last new tokens' values are not finite; the queries before them are unharmed, over a
    cache read at once and one read in shares."""
    c = Cache([held], [new], 16, 2, D)
    q, k, v = draw(1, 1, new, 4, D), draw(2, 1, new, 2, D), draw(3, 1, new, 2, D)
    cut = new - 5
    k[:, cut:], v[:, cut:] = NAN, float("inf")
    om.kv_pages_write(k, v, *c.args())
    o = om.attention_prefill_paged(q, *c.args())
    val, tol = one_sequence(q[0, :cut].double(), torch.cat([c.keys[0], k[0, :cut]]).double(),
                            torch.cat([c.values[0], v[0, :cut]]).double(), held)
    check("queries before", o[0, :cut], val["o"], tol["o"])
    assert bool(o[:, cut:].isnan().all())


def test_shared_pages():
    """Two sequences with the same first pages."""
    c = Cache([64, 64], [5, 5], 32, 2, 64)
    c.block_table[1, :2] = c.block_table[0, :2]
    q, k, v = draw(1, 2, 4, 64), draw(2, 2, 2, 64), draw(3, 2, 2, 64)
    o = om.attention_decode_step(q, k, v, *c.args())
    for n in range(2):
        val, tol = one_sequence(q[n:n + 1].double(), torch.cat([c.keys[0], k[n:n + 1]]).double(),
                                torch.cat([c.values[0], v[n:n + 1]]).double(), 64)
        check(f"sequence {n}", o[n:n + 1], val["o"], tol["o"])


@pytest.mark.parametrize("N,room", [(3, 40), (70, 5)])
def test_captured_turns(N, room):
    """An append and its attention captured once, replayed with other lengths, offsets and pages."""
    Hq, Hkv, D, page, T = 8, 2, 128, 16, 60 if N == 3 else 150
    held = [37 * n % 900 for n in range(N)]
    c, e = (Cache(held, [page + room] * N, page, Hkv, D) for _ in range(2))
    q, k, v = draw(1, 1, T, Hq, D), draw(2, 1, T, Hkv, D), draw(3, 1, T, Hkv, D)
    cu = torch.tensor([n * T // N for n in range(N + 1)], dtype=torch.int32, device="cuda")

    def turn(c):
        om.kv_pages_write(k, v, *c.args(), cu_seqlens=cu)
        return om.attention_prefill_paged(q, *c.args(), cu_seqlens=cu)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    pools = c.k_pages.clone(), c.v_pages.clone()
    with torch.cuda.stream(side):
        turn(c)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = turn(c)
    c.k_pages.copy_(pools[0])
    c.v_pages.copy_(pools[1])
    for r in range(3):
        for i, t in enumerate((q, k, v)):
            t.copy_(draw(50 + 3 * r + i, *t.shape))
        lens = torch.tensor([max(0, h - 5 * r) if n % 7 != 3 else -1 for n, h in enumerate(held)], dtype=torch.int32)
        order = torch.randperm(N, generator=torch.Generator().manual_seed(r))  # whole tables change hands
        for x in (c, e):
            x.lengths.copy_(lens[order] if r else lens)
            x.block_table.copy_(x.table[order] if r else x.table)
        want = turn(e)
        g.replay()
        torch.cuda.synchronize()
        assert equal(o, want) and bool(o.isfinite().all())
        same_pools(c, (e.k_pages, e.v_pages))


@pytest.mark.parametrize("width", [0, 200])
def test_captured_decode_steps(width):
    """One captured step, replayed as the lengths grow, with eager steps of another cache between."""
    Hq, Hkv, D, page = 8, 2, 128, 16
    c, e = (Cache([500, 30, 700], [8] * 3, page, Hkv, D, width=width) for _ in range(2))
    q, k, v = draw(1, 3, Hq, D), draw(2, 3, Hkv, D), draw(3, 3, Hkv, D)
    c0 = c.k_pages.clone(), c.v_pages.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        om.attention_decode_step(q, k, v, *c.args())
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = om.attention_decode_step(q, k, v, *c.args())
        c.lengths += 1
    c.k_pages.copy_(c0[0])
    c.v_pages.copy_(c0[1])
    for r in range(4):
        for i, t in enumerate((q, k, v)):
            t.copy_(draw(30 + 3 * r + i, *t.shape))
        want = om.attention_decode_step(q, k, v, *e.args())
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)
        same_pools(c, (e.k_pages, e.v_pages))
        e.lengths += 1


def ragged(N, most, seed):
    """Lengths up to `most`, some of them zero, some negative."""
    g = torch.Generator().manual_seed(seed)
    held = torch.randint(0, most, (N,), generator=g).tolist()
    return [(-1 if n % 11 == 7 else 0 if n % 13 == 5 else h) for n, h in enumerate(held)]


@pytest.mark.parametrize("held,page,Hq,Hkv,D,width", [
    (ragged(90, 300, 1), 64, 16, 2, 64, 40), (ragged(90, 250, 2), 16, 8, 2, 128, 70), (ragged(90, 200, 3), 48, 12, 1, 256, 12),
    (ragged(200, 150, 4), 32, 34, 2, 128, 40), ([-1] * 70 + [2000] + [-1, 0, 3], 64, 8, 1, 64, 40),
], ids=lambda x: str(x)[:12])
def test_decode_ranges_of_more_than_64_sequences(held, page, Hq, Hkv, D, width):
    """Ranges found past the first 64 sequences, joined with a wavefront a row."""
    say(f"decode, ranges of {len(held)} sequences, Hq={Hq} Hkv={Hkv} D={D}")
    c = Cache(held, [1 if h >= 0 else 0 for h in held], page, Hkv, D, seed=3, width=width)
    assert len(held) > 64 and len(held) * Hq > 512 and segments(c, Hq) > len(held)
    step_and_check(c, Hq)


@pytest.mark.parametrize("held,page,Hq,Hkv,D", [
    ([10300], 64, 4, 1, 256), ([5, 9000, 0], 128, 8, 2, 256), ([21000], 256, 2, 1, 128), ([0, 20000] + [3] * 70, 64, 8, 1, 128)])
def test_decode_rows_of_more_than_64_segments(held, page, Hq, Hkv, D):
    """A sequence whose keys are so many ranges that its join passes over their sums in turns of 64."""
    say(f"decode, many segments held={held[:4]} Hq={Hq} Hkv={Hkv} D={D}")
    c = Cache(held, [1] * len(held), page, Hkv, D, seed=4)
    stages = [-(-(h + 1) * D // 4096) for h in held]
    ranges = segments(c, Hq) - len(held)
    assert ranges == 256 // Hkv and max(stages) // max(8, -(-sum(stages) // ranges)) > 64
    step_and_check(c, Hq)


def test_captured_steps_of_a_large_batch():
    """A step of 70 sequences in equal ranges, captured once: replays with other lengths (none, long,
    past the table, taking no part), eager steps and other allocations between them."""
    N, Hq, Hkv, D, page, width = 70, 16, 8, 64, 16, 160
    c, e = (Cache([300] * N, [1] * N, page, Hkv, D, width=width) for _ in range(2))
    assert segments(c, Hq) == 256 // Hkv + N
    for x in (c, e):  # tables without holes, over pages that hold numbers
        g = torch.Generator().manual_seed(3)
        x.k_pages = torch.randn((N * width, page, Hkv, D), generator=g).to(BF).cuda()
        x.v_pages = torch.randn((N * width, page, Hkv, D), generator=g).to(BF).cuda()
        x.block_table = torch.randperm(N * width, generator=g).to(torch.int32).view(N, width).cuda()
    q, k, v = draw(1, N, Hq, D), draw(2, N, Hkv, D), draw(3, N, Hkv, D)
    first = c.k_pages.clone(), c.v_pages.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        om.attention_decode_step(q, k, v, *c.args())
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = om.attention_decode_step(q, k, v, *c.args())
    c.k_pages.copy_(first[0])
    c.v_pages.copy_(first[1])
    for r in range(4):
        lens = torch.randint(0, (40, 2600, 300, 3000)[r], (N,), generator=torch.Generator().manual_seed(r))
        lens[r::9] = -1
        for x in (c, e):
            x.lengths.copy_(lens.to(torch.int32))
        for i, t in enumerate((q, k, v)):
            t.copy_(draw(80 + 3 * r + i, *t.shape))
        want = om.attention_decode_step(q, k, v, *e.args())
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and bool(o.isfinite().all())
        same_pools(c, (e.k_pages, e.v_pages))


def test_streams_at_once_over_caches():
    """Turns and decode steps of two caches on two streams at the same time, each as by itself."""
    shapes = [([900, 40, 2000], 30, 64, 8, 2, 128), ([700] * 40 + [3] * 30, 2, 64, 16, 8, 64)]
    sets = []
    for i, (held, T, page, Hq, Hkv, D) in enumerate(shapes):
        c = Cache(held, [T + 1] * len(held), page, Hkv, D, seed=i, width=40)
        B = len(held)
        sets.append((c, draw(1, B, T, Hq, D), draw(2, B, T, Hkv, D), draw(3, B, T, Hkv, D), draw(4, B, Hq, D),
                     draw(5, B, Hkv, D), draw(6, B, Hkv, D), c.lengths + T))

    def run(c, q, k, v, q1, k1, v1, longer):
        om.kv_pages_write(k, v, *c.args())
        o = om.attention_prefill_paged(q, *c.args())
        return o, om.attention_decode_step(q1, k1, v1, *c.args()[:3], longer)

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
