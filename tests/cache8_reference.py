"""The paged cache in 8 bits, restated: e4m3 numbers and an exponent for each 16 tokens of a head.

The append rounds each value once to the nearest number, so codes and exponents are equal, not near.
"""
import torch

BLOCK = 16
E4M3 = torch.float8_e4m3fn
LARGEST = 1.875 * 2.0 ** 127


def nearest(x):
    """The nearest e4m3 numbers of x in 64 bits, |x| <= 448, ties to even; NaN for what is not finite."""
    size = torch.where(x.isfinite(), x.abs(), 1.0).clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    return torch.where(x.isfinite(), torch.round(x / step) * step, float("nan"))


def asked(x):
    """Exponents [Hkv] that rows x [n, Hkv, D] ask for."""
    most = torch.where(x.isfinite(), x.abs(), 0.0).amax((0, 2))
    e = torch.ceil(torch.log2(most.clamp(min=2.0 ** -300) / 448))
    return torch.where(most > 448 * torch.exp2(e), e + 1, e).clamp(-100, 120)


def append(codes, exps, h, x):
    """One sequence's codes [m, Hkv, D] and exponents [m / 16, Hkv] in 64 bits, in place: x [n, Hkv, D]
    behind its h tokens."""
    x = torch.where(x.isfinite(), x.clamp(-LARGEST, LARGEST), x)
    end = h + x.shape[0]
    for b in range(h // BLOCK, -(-end // BLOCK)):
        lo, hi = max(h, b * BLOCK), min(end, (b + 1) * BLOCK)
        e = asked(x[lo - h:hi - h])
        if lo > b * BLOCK:
            e = torch.maximum(e, exps[b])
            codes[b * BLOCK:lo] = nearest(codes[b * BLOCK:lo] * torch.exp2(exps[b] - e)[:, None])
        exps[b] = e
        codes[lo:hi] = nearest(x[lo - h:hi - h] * torch.exp2(-e)[:, None])


def same_codes(got, want):
    """Equal numbers (zeros of either sign), NaN where NaN."""
    a, b = got.view(torch.uint8), want.view(torch.uint8)
    a, b = (torch.where(x == 0x80, 0, torch.where((x & 0x7f) == 0x7f, 0x7f, x)) for x in (a, b))
    return torch.equal(a, b)


class Cache8:
    """Sequences of given lengths in shuffled pages; every unused slot a NaN, unused exponents anything.
    `want`: what the pools should hold, in 64 bits; `seqs(n, m)`: keys and values of sequence n, [m, Hkv, D]."""

    def __init__(self, held, room, page, Hkv, D, seed=0, extra=3, width=0, size=1.0):
        self.gen = torch.Generator().manual_seed(seed)
        n_pages = [-(-(max(h, 0) + r) // page) for h, r in zip(held, room)]
        pool = sum(n_pages) + extra
        self.page, self.Hkv, self.D, self.held = page, Hkv, D, list(held)
        order = torch.randperm(pool, generator=self.gen).tolist()
        self.table = torch.full((len(held), max(width, *n_pages)), -1, dtype=torch.int32)
        at = 0
        for n, p in enumerate(n_pages):
            self.table[n, :p] = torch.tensor(order[at:at + p], dtype=torch.int32)
            at += p
        self.want = [torch.full((pool, page, Hkv, D), float("nan"), dtype=torch.float64) for _ in range(2)]
        self.want_e = [torch.randint(-128, 128, (pool, page // BLOCK, Hkv), generator=self.gen).double() for _ in range(2)]
        for n, h in enumerate(held):
            if h > 0:
                self.put(n, 0, *(self.rows(h, size) for _ in range(2)))
        self.k_pages, self.v_pages = (w.to(torch.float32).to(E4M3).cuda() for w in self.want)
        self.k_exps, self.v_exps = (e.to(torch.int8).cuda() for e in self.want_e)
        self.block_table = self.table.cuda()
        self.lengths = torch.tensor(held, dtype=torch.int32, device="cuda")

    def rows(self, n, size=1.0):
        """Tokens whose sizes differ by head and token."""
        x = torch.randn((n, self.Hkv, self.D), generator=self.gen)
        x = x * torch.exp(torch.randn((n, self.Hkv, 1), generator=self.gen)) * size
        return x.to(torch.bfloat16)

    def put(self, n, pos, k, v):
        """Appends to what should be there, block by block where a page is."""
        room = self.table.shape[1] * self.page
        k, v = k[:max(0, room - pos)], v[:max(0, room - pos)]
        if k.shape[0] == 0:
            return
        first, last = pos // BLOCK, (pos + k.shape[0] - 1) // BLOCK
        per = self.page // BLOCK
        for i, x in enumerate((k, v)):
            for b in range(first, last + 1):
                page = int(self.table[n, b // per])
                if not 0 <= page < self.want[i].shape[0]:
                    continue
                lo, hi = max(pos, b * BLOCK), min(pos + x.shape[0], (b + 1) * BLOCK)
                rows = slice(b % per * BLOCK, b % per * BLOCK + BLOCK)
                append(self.want[i][page, rows], self.want_e[i][page, b % per:b % per + 1], lo - b * BLOCK,
                       x[lo - pos:hi - pos].double().cpu())

    def seq(self, n, m):
        """What positions 0 .. m of sequence n should hold, zeros where there is no page, and which are there."""
        out, there = [], torch.zeros(m, dtype=torch.bool)
        for w, e in zip(self.want, self.want_e):
            x = torch.zeros((m, self.Hkv, self.D), dtype=torch.float64)
            for j in range(-(-m // self.page)):
                page = int(self.table[n, j]) if j < self.table.shape[1] else -1
                if 0 <= page < w.shape[0]:
                    a, b = j * self.page, min(m, (j + 1) * self.page)
                    x[a:b] = (w[page] * torch.exp2(e[page]).repeat_interleave(BLOCK, 0)[..., None])[:b - a]
                    there[a:b] = True
            out.append(x.cuda())
        return (*out, there.cuda())

    def same(self):
        for got, w in zip((self.k_pages, self.v_pages), self.want):
            assert same_codes(got.cpu(), w.to(torch.float32).to(E4M3))
        for got, w in zip((self.k_exps, self.v_exps), self.want_e):
            assert torch.equal(got.cpu(), w.to(torch.int8))

    def args(self):
        return self.k_pages, self.v_pages, self.block_table, self.lengths

    def exps(self):
        return dict(k_exps=self.k_exps, v_exps=self.v_exps)
