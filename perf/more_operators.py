"""Attention that sees a window of its keys, a cache held in 8 bits, and the pages that a batch gets.

A hybrid decoder serves long conversations from a paged cache.  The operators bound what that
costs: attention over the last ``window`` keys and a few first ones that stay visible
(``sinks``), for prompts with its gradient, for new tokens over a cache and for single tokens;
a cache of e4m3 numbers with a power of two for each 16 tokens of a head, its append and the
attention that reads it; and the block tables, positions and slots of new tokens, built on the
GPU from the requests' lengths, with the return of pages.  Tokens are bf16 and token-major;
query head h reads key head h / (hq / hkv).

``run`` computes them in plain torch in 32 bits where ``own`` is false, and calls the
framework's operators where it is true.  ``exact`` restates each from its definition in 64
bits, sequence by sequence.  Pools of 8-bit numbers are returned as float8 tensors, whose values
count, with the exponents that scale them.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16 = torch.bfloat16
E4M3 = torch.float8_e4m3fn
BLOCK = 16            # tokens that share an exponent
LEAST, MOST = -100, 120  # of the exponents
LARGEST = 1.875 * 2.0 ** 127  # what is larger would leave bf16 when it is read back


def listed():
    return [
        # one long document through a layer of few key heads of dim 256
        dict(name="window_prompt", kind="prompt", batch=1, tokens=12000, packed=0, hq=16, hkv=2, d=256,
             window=1024, sinks=4, mix=1),
        # a handful of short requests with small heads and a narrow window
        dict(name="window_prompts", kind="prompt", batch=1, tokens=3001, packed=5, hq=8, hkv=8, d=64,
             window=128, sinks=0, mix=3),
        # a training step at the batch of the benchmark
        dict(name="window_train_batch", kind="train", batch=4, tokens=4096, packed=0, hq=32, hkv=8, d=128,
             window=1024, sinks=16, mix=1),
        # fine-tuning on one row of packed documents of ragged lengths
        dict(name="window_train_packed", kind="train", batch=1, tokens=3001, packed=5, hq=16, hkv=2, d=256,
             window=500, sinks=4, mix=3),
        # a serving batch's next tokens behind long conversations, of which they see the end
        dict(name="window_step", kind="step", seqs=64, held=8000, page=64, hq=32, hkv=8, d=128, bits=16,
             window=1024, sinks=4, mix=5),
        # a short turn's keys and values go into a cache of 8 bits, behind a block that it shares
        dict(name="write_turn", kind="write", seqs=1, new=77, held=5000, page=16, hkv=8, d=64, bits=8, mix=1),
        # those of several prompts at once
        dict(name="write_prompts", kind="write", seqs=8, new=4000, held=0, page=64, hkv=8, d=128, bits=8, mix=6),
        # the next pieces of several long prompts, each over what its cache of 8 bits holds
        dict(name="turn_batch", kind="turn", seqs=6, new=700, held=7000, page=64, hq=32, hkv=8, d=128, bits=8,
             window=0, sinks=0, mix=4),
        # one user's next token: nothing but latency
        dict(name="step_one", kind="step", seqs=1, held=611, page=16, hq=16, hkv=4, d=128, bits=8,
             window=0, sinks=0, mix=1),
        # a serving batch's next tokens over caches of 8 bits and uneven lengths
        dict(name="step_batch", kind="step", seqs=64, held=4000, page=64, hq=16, hkv=2, d=256, bits=8,
             window=0, sinks=0, mix=5),
        # room for one more token of each running request, given back as a turned down draft's is
        dict(name="pages_step", kind="pages", seqs=64, new=1, held=4000, page=16, mix=5),
        # room for a wave of new prompts, all of it given back
        dict(name="pages_prompts", kind="pages", seqs=512, new=300, held=0, page=16, mix=7),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _cost(case):
    """What bounds a drawn case: its work, the cache that it lies over and the pairs of query and key without
    a window."""
    new, held = _shape(case)
    w, most = work(case), max(n + h for n, h in zip(new, held))
    cache = sum(held) * case.get("hkv", 0) * case.get("d", 0) * case.get("bits", 0)
    return w["bytes"], w["flops"], cache, len(new) * max(new) * most * case.get("hq", 0)


def _fits(case):
    """Whether a case costs no more than the dearest listed ones of its kind."""
    cost, others = _cost(case), [_cost(c) for c in listed() if c["kind"] == case["kind"]]
    return all(x <= max(y) for x, y in zip(cost, zip(*others)))


def draw(rng):
    """A case of the listed kinds, made smaller until it is no dearer than the listed ones."""
    kind = rng.choice(["prompt", "prompt", "train", "train", "write", "turn", "turn", "step", "step", "pages"])
    c = dict(kind=kind, mix=rng.randrange(1, 10000))
    if kind != "pages":
        c.update(hkv=rng.choice([1, 2, 4, 8]), d=rng.choice([64, 128, 128, 256]))
    if kind in ("prompt", "train", "turn", "step"):
        c["hq"] = c["hkv"] * rng.choice([1, 2, 4, 4, 8])
        while c["hq"] > 32:
            c["hq"] //= 2
    if kind in ("prompt", "train"):
        c["packed"] = rng.choice([0, 0, 2, 5, 11])
        c["batch"] = 1 if c["packed"] else rng.choice([1, 1, 2, 3, 5])
        c["tokens"] = _log_int(rng, 16, 12000 // c["batch"])
        c["window"] = _log_int(rng, 1, 3000)
    else:
        c["page"] = rng.choice([16, 16, 32, 64, 128])
        c["seqs"] = rng.choice([1, 1, 2, 4, 7]) if kind == "turn" else _log_int(rng, 1, 500 if kind == "pages" else 100)
        c["held"] = _log_int(rng, 1, {"turn": 16000, "step": 130000, "write": 5000, "pages": 8000}[kind])
        if kind != "step":
            c["new"] = _log_int(rng, 1, {"turn": 1500, "write": 8000, "pages": 400}[kind])
        if kind in ("turn", "step"):
            c["bits"] = rng.choice([8, 8, 16])
            c["window"] = _log_int(rng, 1, 4000) if c["bits"] == 16 or rng.random() < 0.4 else 0
        elif kind == "write":
            c["bits"] = 8
    if "window" in c:
        c["sinks"] = rng.choice([0, 0, 1, 4, 16, 100]) if c["window"] else 0
    while not _fits(c):
        for n in ("tokens", "new", "held"):
            if n in c:
                c[n] = max(1, c[n] * 4 // 5)
    return c


# ---------------------------------------------------------------- inputs


def _uneven(total, n, mix):
    """n lengths that sum to the total, at least one token each, the same for one case."""
    n = min(n, total)
    rng = random.Random(mix)
    w = [-math.log(1.0 - rng.random()) + 0.05 for _ in range(n)]
    lens = [1 + int((total - n) * x / sum(w)) for x in w]
    lens[0] += total - sum(lens)
    return lens


def _around(mean, n, mix):
    """n lengths between a quarter and seven quarters of the mean; the mean itself for one."""
    if n == 1:
        return [mean]
    rng = random.Random(mix)
    return [max(0, round(mean * rng.uniform(0.25, 1.75))) for _ in range(n)]


def _shape(case):
    """(new tokens, tokens held before) of each sequence."""
    kind = case["kind"]
    if kind in ("prompt", "train"):
        if case["packed"]:
            new = _uneven(case["tokens"], case["packed"], case["mix"])
            return new, [0] * len(new)
        return [case["tokens"]] * case["batch"], [0] * case["batch"]
    held = _around(case["held"], case["seqs"], case["mix"])
    if kind == "step":
        return [1] * case["seqs"], held
    return [max(1, n) for n in _around(case["new"], case["seqs"], case["mix"] + 1)], held


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


class _Draws:
    """Seeded draws on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape, scale=1.0):
        return (torch.randn(shape, generator=self.gen, device="cuda") * scale).to(BF16)

    def uneven(self, *shape):
        """Normal draws of tokens and heads whose size differs."""
        x = torch.randn(shape, generator=self.gen, device="cuda")
        return (x * torch.exp(torch.randn((*shape[:-1], 1), generator=self.gen, device="cuda"))).to(BF16)

    def codes(self, *shape):
        """e4m3 numbers of a block whose largest is near the type's."""
        x = torch.randn(shape, generator=self.gen, device="cuda") * 64
        return x.clamp_(-448.0, 448.0).to(E4M3)

    def exponents(self, *shape):
        return torch.randint(-8, -4, shape, generator=self.gen, device="cuda").to(torch.int8)


def _dealt(case, seed, new, held):
    """(pool size, the pool's pages in the order dealt, table of the pages that `held` tokens fill)."""
    page = case["page"]
    have = [-(-h // page) for h in held]
    want = [-(-(n + h) // page) for n, h in zip(new, held)]
    pool = sum(want) + 3
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    fill = have if case["kind"] == "pages" else want
    table, at = torch.full((len(new), max(want)), -1, dtype=torch.int32), 0
    for row, n in enumerate(fill):
        table[row, :n] = order[at:at + n]
        at += n
    return pool, order[at:], table


def prepare(case, seed):
    r = _Draws(seed)
    kind = case["kind"]
    new, held = _shape(case)
    s = dict(kind=kind, new=new, held=held, window=case.get("window", 0) or None, sinks=case.get("sinks", 0))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    if kind not in ("prompt", "train"):
        s["lengths"] = ints(held)
        pool, spare, table = _dealt(case, seed, new, held)
        s["table"] = table.cuda()
    if kind == "pages":
        # the free pages lie at the stack's bottom, what was dealt is above its top
        s["page"], s["new_tokens"], s["tokens"] = case["page"], ints(new), sum(new)
        s["free"] = torch.full((pool,), -1, dtype=torch.int32)
        s["free"][:len(spare)] = spare
        s["free"], s["count"] = s["free"].cuda(), ints([len(spare)])
        return s
    hkv, d = case["hkv"], case["d"]
    if kind in ("prompt", "train"):
        lead = (case["batch"], case["tokens"])
    elif kind == "step":
        lead = (case["seqs"],)
    else:
        lead = (1, sum(new))
    if kind != "write":
        # normalised queries times a learned weight: scores with a standard deviation of 1.5
        s["q"] = r.normal(*lead, case["hq"], d, scale=1.5)
    eight = case.get("bits") == 8
    tokens = r.uneven if eight else r.normal
    s["k"], s["v"] = tokens(*lead, hkv, d), tokens(*lead, hkv, d)
    s["cu"] = None
    if case.get("packed") or kind in ("turn", "write"):
        s["cu"] = ints(_offsets(new))
    if kind == "train":
        s["do"] = r.normal(*lead, case["hq"], d)
        for n in "qkv":
            s[n].requires_grad_(True)
    if kind in ("turn", "step", "write"):
        page = case["page"]
        rows = r.codes if eight else r.normal
        s["k_pages"], s["v_pages"] = rows(pool, page, hkv, d), rows(pool, page, hkv, d)
        s["k_exps"] = s["v_exps"] = None
        if eight:
            s["k_exps"], s["v_exps"] = (r.exponents(pool, page // BLOCK, hkv) for _ in range(2))
    return s


# ---------------------------------------------------------------- one pass


def _weights(q, k, allowed):
    """Softmax weights [N, hkv, g, Tq, Tk] of q [N, Tq, hq, d] over k [N, Tk, hkv, d], in 32
    bits; rows that nothing is allowed for are zero."""
    N, Tq, hq, d = q.shape
    Tk, hkv = k.shape[1], k.shape[2]
    g = hq // hkv
    qf = q.float().permute(0, 2, 1, 3).reshape(N, hkv, g * Tq, d)
    kf = k.float().permute(0, 2, 3, 1).contiguous()
    s = (torch.matmul(qf, kf) * d ** -0.5).view(N, hkv, g, Tq, Tk)
    s = s.masked_fill_(~allowed, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    p = torch.exp_(s.sub_(top))
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total > 0, total, 1.0))


def _mixed(p, v):
    """[N, Tq, hq, d] in 32 bits: the weighted sums of v [N, Tk, hkv, d]."""
    N, hkv, g, Tq, Tk = p.shape
    vf = v.float().permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(p.view(N, hkv, g * Tq, Tk), vf)
    return o.view(N, hkv * g, Tq, -1).permute(0, 2, 1, 3)


def _seen(s, pos, key):
    """Whether the query at a position sees a key: in its window, or one of the first."""
    seen = key <= pos
    if s["window"]:
        seen = seen & ((key > pos - s["window"]) | (key < s["sinks"]))
    return seen


def _allowed(s, tokens):
    """[1, 1, 1, T, T] of whole prompts."""
    at = torch.arange(tokens, device="cuda")
    if s["cu"] is None:
        return _seen(s, at[:, None], at)[None, None, None]
    cu = s["cu"].long()
    seq = torch.bucketize(at, cu[1:], right=True)
    pos = at - cu[seq]
    return (_seen(s, pos[:, None], pos) & (seq[:, None] == seq))[None, None, None]


def _plain_train(s):
    q, k, v = (s[n].detach() for n in "qkv")
    N, T, hq, d = q.shape
    hkv = k.shape[2]
    g = hq // hkv
    p = _weights(q, k, _allowed(s, T))
    o = _mixed(p, v)
    do = s["do"].float()
    delta = (do * o).sum(-1).permute(0, 2, 1).reshape(N, hkv, g, T, 1)
    rows = lambda t: t.float().permute(0, 2, 1, 3).reshape(N, hkv, g * T, d)
    heads = lambda t: t.float().permute(0, 2, 1, 3).contiguous()
    back = lambda t: t.permute(0, 2, 1, 3).to(BF16)
    do_r, q_r = rows(do), rows(q)
    p_r = p.view(N, hkv, g * T, T)
    dv = torch.matmul(p_r.transpose(2, 3), do_r)
    dp = torch.matmul(do_r, heads(v).transpose(2, 3)).view(N, hkv, g, T, T)
    ds = dp.sub_(delta).mul_(p).mul_(d ** -0.5).view(N, hkv, g * T, T)
    dq = torch.matmul(ds, heads(k)).view(N, hq, T, d)
    dk = torch.matmul(ds.transpose(2, 3), q_r)
    return [o.to(BF16), back(dq), back(dk), back(dv)]


def _append8(s, pages, exps, x, pos, row):
    """New rows x [n, hkv, d] at flat rows `row` of a pool of 8 bits: a block's exponent is the
    largest that its new tokens ask for, or its older tokens have, which are rounded again."""
    hkv, d = x.shape[1:]
    x = x.float().clamp(-LARGEST, LARGEST)
    top, exponent = torch.frexp(x.abs().amax(-1))
    ask = (exponent - 9 + (top > 0.875)).clamp_(LEAST, MOST).float()
    codes, flat = pages.view(torch.uint8).view(-1, hkv, d), exps.view(-1, hkv)
    block = row // BLOCK
    # a block that begins with one of these tokens forgets what its exponent was
    first = torch.zeros(flat.shape[0], device="cuda").scatter_reduce_(0, block, (pos % BLOCK == 0).float(), "amax")
    before = flat.float()
    after = torch.where(first[:, None] > 0, float(LEAST), before)
    after.scatter_reduce_(0, block[:, None].expand(-1, hkv), ask, "amax")
    new = (x * torch.exp2(-after[block])[..., None]).to(E4M3).view(torch.uint8)
    # the older tokens of each sequence's first block
    lengths = s["lengths"].long()
    into = (lengths // BLOCK * BLOCK)[:, None] + torch.arange(BLOCK, device="cuda")
    page = pages.shape[1]
    slot = (into // page).clamp_(max=s["table"].shape[1] - 1)
    old = s["table"].long().gather(1, slot) * page + into % page
    keep = (into < lengths[:, None]).flatten()
    old = torch.where(keep, old.flatten(), row[0])
    shift = torch.exp2(before[old // BLOCK] - after[old // BLOCK])[..., None]
    again = (codes[old].view(E4M3).float() * shift).to(E4M3).view(torch.uint8)
    codes[old] = torch.where(keep[:, None, None], again, new[:1])
    codes[row] = new
    flat.copy_(after)


def _plain_write(s, k, v):
    """New tokens' keys and values into their pages, behind what the sequence holds."""
    page = s["k_pages"].shape[1]
    at = torch.arange(k.shape[0], device="cuda")
    if s["cu"] is None:
        seq, pos = at, s["lengths"].long()
    else:
        seq = torch.bucketize(at, s["cu"][1:].long(), right=True)
        pos = s["lengths"].long()[seq] + at - s["cu"].long()[seq]
    into = s["table"].long()[seq, pos // page]
    if s["k_exps"] is None:
        s["k_pages"][into, pos % page] = k
        s["v_pages"][into, pos % page] = v
    else:
        for n, x in (("k", k), ("v", v)):
            _append8(s, s[n + "_pages"], s[n + "_exps"], x, pos, into * page + pos % page)


def _gathered(s):
    """(k, v) [N, capacity, hkv, d] as the tables lay them out."""
    table = s["table"].long().clamp(min=0)
    if s["k_exps"] is None:
        return [s[n][table].flatten(1, 2) for n in ("k_pages", "v_pages")]
    scale = lambda e: torch.exp2(e[table].flatten(1, 2).float()).repeat_interleave(BLOCK, 1)[..., None]
    bits = lambda t: t.view(torch.uint8)[table].view(E4M3).flatten(1, 2)
    return [bits(s[n + "_pages"]).float() * scale(s[n + "_exps"]) for n in "kv"]


def _cache(s):
    return [s[n] for n in ("k_pages", "v_pages", "k_exps", "v_exps") if s[n] is not None]


def _plain_turn(s):
    q = s["q"][0]
    _plain_write(s, s["k"][0], s["v"][0])
    cu = s["cu"].long()
    most = max(s["new"])
    i = torch.arange(most, device="cuda")
    token = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)      # [N, most], rows past the last idle
    k, v = _gathered(s)
    key = torch.arange(k.shape[1], device="cuda")
    allowed = _seen(s, (s["lengths"].long()[:, None] + i)[..., None], key)
    o = _mixed(_weights(q[token], k, allowed[:, None, None]), v).to(BF16)
    seq = torch.bucketize(torch.arange(q.shape[0], device="cuda"), cu[1:], right=True)
    return [o[seq, torch.arange(q.shape[0], device="cuda") - cu[seq]][None], *_cache(s)]


def _plain_step(s):
    _plain_write(s, s["k"], s["v"])
    k, v = _gathered(s)
    allowed = _seen(s, s["lengths"].long()[:, None], torch.arange(k.shape[1], device="cuda"))
    p = _weights(s["q"][:, None], k, allowed[:, None, None, None])
    return [_mixed(p, v)[:, 0].to(BF16), *_cache(s)]


def _plain_pages(s):
    """Pages for the new tokens from the stack's top, the tokens' places, and the pages back."""
    page, table, free, count = s["page"], s["table"], s["free"], s["count"]
    h, m = s["lengths"].long(), s["new_tokens"].long()
    cu = torch.cat([torch.zeros_like(m[:1]), m.cumsum(0)])
    first = torch.arange(table.shape[1], device="cuda") * page
    need = (first + page > h[:, None]) & (first < (h + m)[:, None]) & (m > 0)[:, None]
    need &= (table < 0) | (table >= free.shape[0])
    rank = (need.flatten().cumsum(0) - 1).view_as(need)
    total, c = need.sum(), count[0].long()
    got = need & (rank < c)
    table.copy_(torch.where(got, free[(c - 1 - rank).clamp(0, free.shape[0] - 1)], table))
    missing = (total - c).clamp(min=0)
    count.copy_(count - (total - missing))
    at = torch.arange(s["tokens"], device="cuda")
    seq = torch.bucketize(at, cu[1:], right=True).clamp_(max=len(h) - 1)
    pos = h[seq] + at - cu[seq]
    slot = pos // page
    into = table.long()[seq, slot.clamp(max=table.shape[1] - 1)]
    there = (into >= 0) & (into < free.shape[0]) & (slot < table.shape[1])
    slots = torch.where(there, into * page + pos % page, -1)
    # what lies wholly past the tokens that are kept goes back in the order that it came
    back = (first >= h[:, None]) & (table >= 0) & (table < free.shape[0])
    rank = (back.flatten().cumsum(0) - 1).view_as(back)
    n, c = back.sum(), count[0].long()
    to = torch.where(back, c + n - 1 - rank, free.shape[0])
    more = torch.cat([free, free[:1]])
    more[to] = table
    free.copy_(more[:-1])
    table.copy_(torch.where(back, -1, table))
    count.copy_(count + n)
    return [cu.int(), pos.int(), slots, missing.int().view(1), table, free, count]


def _own(s):
    import omegalax_amd as om
    kind = s["kind"]
    sight = dict(window=s["window"], sinks=s["sinks"])
    if kind == "prompt":
        return [om.attention_prefill(s["q"], s["k"], s["v"], cu_seqlens=s["cu"], **sight)]
    if kind == "train":
        x = [s[n] for n in "qkv"]
        o = om.attention_prefill(*x, cu_seqlens=s["cu"], **sight)
        return [o.detach(), *torch.autograd.grad(o, x, s["do"])]
    if kind == "pages":
        stack = (s["free"], s["count"])
        made = om.kv_pages_assign(s["table"], s["lengths"], s["new_tokens"], *stack, page_size=s["page"],
                                  tokens=s["tokens"])
        om.kv_pages_release(s["table"], s["lengths"], *stack, page_size=s["page"])
        return [*made, s["table"], *stack]
    cache = (s["k_pages"], s["v_pages"], s["table"], s["lengths"])
    exps = dict(k_exps=s["k_exps"], v_exps=s["v_exps"])
    if kind == "step":
        return [om.attention_decode_step(s["q"], s["k"], s["v"], *cache, **exps, **sight), *_cache(s)]
    om.kv_pages_write(s["k"], s["v"], *cache, cu_seqlens=s["cu"], **exps)
    if kind == "write":
        return _cache(s)
    return [om.attention_prefill_paged(s["q"], *cache, cu_seqlens=s["cu"], **exps, **sight), *_cache(s)]


def run(s):
    if own:
        return _own(s)
    kind = s["kind"]
    if kind == "prompt":
        return [_mixed(_weights(s["q"], s["k"], _allowed(s, s["q"].shape[1])), s["v"]).to(BF16)]
    if kind == "train":
        return _plain_train(s)
    if kind == "turn":
        return _plain_turn(s)
    if kind == "step":
        return _plain_step(s)
    if kind == "pages":
        return _plain_pages(s)
    _plain_write(s, s["k"][0], s["v"][0])
    return _cache(s)


# ---------------------------------------------------------------- what a pass cannot do without


def _pairs(new, held, window, sinks):
    """(pairs of query and key that see each other, keys held before that some new token sees)."""
    pairs = keys = 0
    for n, h in zip(new, held):
        if not window:
            pairs, keys = pairs + n * h + n * (n + 1) // 2, keys + h
            continue
        # the sum over positions p of min(p + 1, window), and of the sinks behind the window
        upto = lambda x, w: x * (x + 1) // 2 if x < w else w * (w + 1) // 2 + (x - w) * w
        pairs += upto(h + n, window) - upto(h, window)
        past = lambda x: upto(max(0, x - window), sinks) if sinks else 0
        pairs += past(h + n) - past(h)
        lo = max(0, h - window + 1)
        keys += h - lo + min(sinks, lo)
    return pairs, keys


def work(case):
    new, held = _shape(case)
    kind = case["kind"]
    tokens = sum(new)
    if kind == "pages":
        page = case["page"]
        given = sum(-(-(n + h) // page) - -(-h // page) for n, h in zip(new, held))
        # lengths, new tokens and offsets; positions and slots; pages off the stack and back on, and
        # their entries written, cleared
        return dict(bytes=12 * len(new) + 12 * tokens + 16 * given, flops=0)
    hkv, d = case["hkv"], case["d"]
    size = case.get("bits", 16) // 8
    exps = 1 / (BLOCK * d) if size == 1 else 0  # a byte for each block of a head
    row, cached = hkv * d * 2, hkv * d * (size + exps)
    if kind == "write":
        return dict(bytes=round(2 * tokens * (row + cached)), flops=0)
    hq = case["hq"]
    pairs, keys = _pairs(new, held, case["window"], case["sinks"])
    if kind in ("prompt", "train"):
        q = tokens * hq * d * 2
        if kind == "prompt":
            return dict(bytes=2 * q + 2 * tokens * row, flops=4 * hq * d * pairs)
        return dict(bytes=4 * q + 4 * tokens * row, flops=14 * hq * d * pairs)
    # new keys and values read and written, held ones read; queries in, outputs out
    return dict(bytes=round(2 * tokens * (row + cached) + 2 * keys * cached + 4 * tokens * hq * d),
                flops=4 * hq * d * pairs)


# ---------------------------------------------------------------- the definition in 64 bits


def _rows64(q, k, v, first, window, sinks):
    """Attention of one head: the keys up to query i's position first + i that it sees."""
    i = torch.arange(q.shape[0], device="cuda")[:, None] + first
    j = torch.arange(k.shape[0], device="cuda")[None]
    unseen = j > i
    if window:
        unseen = unseen | ((i - j >= window) & (j >= sinks))
    return torch.softmax((q @ k.t() * q.shape[-1] ** -0.5).masked_fill(unseen, -math.inf), -1) @ v


def _sequence64(q, k, v, first, window, sinks):
    """[n, hq, d] for one sequence's q [n, hq, d] and keys and values [m, hkv, d]."""
    g = q.shape[1] // k.shape[1]
    return torch.stack([_rows64(q[:, h], k[:, h // g], v[:, h // g], first, window, sinks)
                        for h in range(q.shape[1])], 1)


def _e4m3_64(x):
    """The nearest e4m3 numbers, the even of two that are as near."""
    size = x.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    return torch.round(x / step) * step


def _append64(codes, exps, x, h):
    """One sequence's codes [m, hkv, d] and exponents [blocks, hkv], with x [n, hkv, d] behind its h tokens."""
    end = h + x.shape[0]
    for b in range(h // BLOCK, -(-end // BLOCK)):
        lo, hi = max(h, b * BLOCK), min(end, (b + 1) * BLOCK)
        new = x[lo - h:hi - h].clamp(-LARGEST, LARGEST)
        most = new.abs().amax((0, 2))
        need = torch.ceil(torch.log2(most.clamp(min=2.0 ** -300) / 448))
        need = torch.where(most > 448 * torch.exp2(need), need + 1, need).clamp(LEAST, MOST)
        if lo > b * BLOCK:
            need = torch.maximum(need, exps[b])
            kept = codes[b * BLOCK:lo]
            codes[b * BLOCK:lo] = _e4m3_64(kept * torch.exp2(exps[b] - need)[:, None])
        exps[b] = need
        codes[lo:hi] = _e4m3_64(new * torch.exp2(-need)[:, None])


def _pools64(s):
    """The cache with the new tokens in place, in 64 bits, and each sequence's keys and values."""
    page, table = s["k_pages"].shape[1], s["table"].tolist()
    pools = [t.double() for t in _cache(s)]
    eight = len(pools) == 4
    k, v = (s[n].double().flatten(0, -3) for n in "kv")
    caches, at = [], 0
    for n, h, row in zip(s["new"], s["held"], table):
        used = torch.tensor(row[:-(-(n + h) // page)], device="cuda")
        seen = []
        for p, x in ((0, k), (1, v)):
            flat = pools[p][used].flatten(0, 1)
            if eight:
                e = pools[2 + p][used].flatten(0, 1)
                _append64(flat, e, x[at:at + n], h)
                pools[2 + p][used] = e.view(-1, *pools[2 + p].shape[1:])
            else:
                flat[h:h + n] = x[at:at + n]
            pools[p][used] = flat.view(-1, *pools[p].shape[1:])
            if eight:
                flat = flat * torch.exp2(e).repeat_interleave(BLOCK, 0)[..., None]
            seen.append(flat[:n + h])
        caches.append(seen)
        at += n
    return pools, caches


def _pages64(s):
    """Pages dealt and returned, one after the other."""
    page, table, free = s["page"], s["table"].tolist(), s["free"].tolist()
    count = int(s["count"][0])
    cu, pos, slots = _offsets(s["new"]), [], []
    given = []
    for row, h, n in zip(table, s["held"], s["new"]):
        for i in range(h // page, -(-(h + n) // page)):
            if row[i] < 0:
                count -= 1
                row[i] = free[count]
                given.append((row, i))
        pos += range(h, h + n)
        slots += [row[p // page] * page + p % page for p in range(h, h + n)]
    while given:
        row, i = given.pop()
        free[count], row[i] = row[i], -1
        count += 1
    return [torch.tensor(x) for x in (cu, pos, slots, [0], table, free, [count])]


def exact(case, seed):
    s = prepare(case, seed)
    kind, new, held = s["kind"], s["new"], s["held"]
    if kind == "pages":
        return _pages64(s)
    cu = _offsets(new)
    spans = list(zip(cu, cu[1:]))
    sight = (s["window"], s["sinks"])
    if kind in ("prompt", "train"):
        shape = s["q"].shape
        flat = [s[n].detach().double().flatten(0, 1) for n in "qkv"]
        if kind == "prompt":
            o = [_sequence64(*(t[a:b] for t in flat), 0, *sight) for a, b in spans]
            return [torch.cat(o).view(shape)]
        do = s["do"].double().flatten(0, 1)
        hkv, g = case["hkv"], case["hq"] // case["hkv"]
        outs = [torch.zeros_like(flat[0]), *(torch.zeros_like(t) for t in flat)]
        for a, b in spans:
            for j in range(hkv):
                heads = slice(j * g, (j + 1) * g)
                q, k, v = (t.clone().requires_grad_(True)
                           for t in (flat[0][a:b, heads], flat[1][a:b, j:j + 1], flat[2][a:b, j:j + 1]))
                o = _sequence64(q, k, v, 0, *sight)
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), do[a:b, heads])
                outs[0][a:b, heads], outs[1][a:b, heads] = o.detach(), dq
                outs[2][a:b, j:j + 1], outs[3][a:b, j:j + 1] = dk, dv
        return [t.view(*shape[:2], *t.shape[1:]) for t in outs]
    pools, caches = _pools64(s)
    if kind == "write":
        return pools
    q = s["q"].double().flatten(0, -3)
    o = [_sequence64(q[a:b], k, v, h, *sight) for (a, b), (k, v), h in zip(spans, caches, held)]
    return [torch.cat(o).view(s["q"].shape), *pools]
