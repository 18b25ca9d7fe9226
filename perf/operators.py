"""Softmax attention beside the gated delta rule: whole prompts, a paged cache, single tokens.

A hybrid decoder mixes tokens by the gated delta rule in most layers and by causal softmax
attention in the others.  The operators are that attention over packed prompts with its
gradient, the append of new keys and values to a paged cache, attention of several new tokens
over such a cache, and the decode step of one token per sequence.  Tokens are bf16 and
token-major; query head h reads key head h / (hq / hkv).

``run`` computes them in plain torch in 32 bits where ``own`` is false, and calls the
framework's operators where it is true.  ``exact`` restates each from its definition in 64
bits, sequence by sequence.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16 = torch.bfloat16


def listed():
    return [
        # one prompt of ordinary length through a layer of few key heads of dim 256
        dict(name="prefill_prompt", kind="prefill", batch=1, tokens=1900, packed=0, hq=16, hkv=2,
             d=256, mix=1),
        # a batch of long prompts
        dict(name="prefill_batch", kind="prefill", batch=4, tokens=4096, packed=0, hq=32, hkv=8,
             d=128, mix=1),
        # eight prompts of uneven lengths in one packed row
        dict(name="prefill_packed", kind="prefill", batch=1, tokens=16384, packed=8, hq=16, hkv=4,
             d=128, mix=2),
        # a training step at the batch of the benchmark
        dict(name="train_batch", kind="train", batch=4, tokens=4096, packed=0, hq=32, hkv=8,
             d=128, mix=1),
        # fine-tuning on one row of packed documents of ragged lengths
        dict(name="train_packed", kind="train", batch=1, tokens=3001, packed=5, hq=16, hkv=2,
             d=256, mix=3),
        # a short turn of one conversation, continued from its cache, with small heads
        dict(name="turn_short", kind="turn", seqs=1, new=77, held=5000, page=16, hq=8, hkv=8,
             d=64, mix=1),
        # the next pieces of several long prompts, each over what its cache holds
        dict(name="turn_batch", kind="turn", seqs=6, new=700, held=7000, page=64, hq=32, hkv=8,
             d=128, mix=4),
        # one user's next token: nothing but latency
        dict(name="decode_one", kind="decode", seqs=1, held=611, page=16, hq=16, hkv=4, d=128,
             mix=1),
        # a serving batch's next tokens over caches of uneven lengths
        dict(name="decode_batch", kind="decode", seqs=64, held=4000, page=64, hq=16, hkv=2, d=256,
             mix=5),
        # the next token behind a very long document
        dict(name="decode_long", kind="decode", seqs=1, held=131000, page=64, hq=32, hkv=4, d=128,
             mix=1),
        # a short turn's keys and values go into the cache
        dict(name="write_turn", kind="write", seqs=1, new=77, held=5000, page=16, hkv=8, d=64,
             mix=1),
        # those of several prompts at once
        dict(name="write_prompts", kind="write", seqs=8, new=4000, held=0, page=64, hkv=8, d=128,
             mix=6),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _fits(case):
    """Whether a case moves and computes no more than the dearest listed ones of its kind."""
    w, listed_work = work(case), [work(c) for c in listed() if c["kind"] == case["kind"]]
    return all(w[n] <= max(x[n] for x in listed_work) for n in ("bytes", "flops"))


def draw(rng):
    """A case of the listed kinds, made smaller until it is no dearer than the listed ones."""
    kind = rng.choice(["prefill", "prefill", "train", "train", "turn", "decode", "decode", "write"])
    c = dict(kind=kind, hkv=rng.choice([1, 2, 4, 8]), d=rng.choice([64, 128, 128, 256]),
             mix=rng.randrange(1, 10000))
    if kind != "write":
        c["hq"] = c["hkv"] * rng.choice([1, 2, 4, 4, 8])
        while c["hq"] > 32:
            c["hq"] //= 2
    if kind in ("prefill", "train"):
        c["packed"] = rng.choice([0, 0, 2, 5, 11])
        c["batch"] = 1 if c["packed"] else rng.choice([1, 1, 2, 3, 5])
        c["tokens"] = _log_int(rng, 16, 16384 // c["batch"])
    else:
        c["page"] = rng.choice([16, 16, 32, 64, 128])
        c["seqs"] = rng.choice([1, 1, 2, 4, 7]) if kind == "turn" else _log_int(rng, 1, 100)
        c["held"] = _log_int(rng, 1, {"turn": 16000, "decode": 130000, "write": 5000}[kind])
        if kind != "decode":
            c["new"] = _log_int(rng, 2, 1500 if kind == "turn" else 8000)
    while not _fits(c):
        for n in ("tokens", "new", "held"):
            if n in c:
                c[n] = max(16, c[n] * 4 // 5)
    return c


# ---------------------------------------------------------------- inputs


def _uneven(total, n, mix):
    """n lengths that sum to the total, at least one token each, the same for one case."""
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
    if kind in ("prefill", "train"):
        if case["packed"]:
            return _uneven(case["tokens"], case["packed"], case["mix"]), [0] * case["packed"]
        return [case["tokens"]] * case["batch"], [0] * case["batch"]
    held = _around(case["held"], case["seqs"], case["mix"])
    if kind == "decode":
        return [1] * case["seqs"], held
    return [max(1, n) for n in _around(case["new"], case["seqs"], case["mix"] + 1)], held


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


class _Draws:
    """Seeded normal draws on the GPU, rounded to bf16."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape, scale=1.0):
        return (torch.randn(shape, generator=self.gen, device="cuda") * scale).to(BF16)


def prepare(case, seed):
    r = _Draws(seed)
    kind, hkv, d = case["kind"], case["hkv"], case["d"]
    new, held = _shape(case)
    s = dict(kind=kind, new=new, held=held)
    if kind in ("prefill", "train"):
        lead = (case["batch"], case["tokens"])
    elif kind == "decode":
        lead = (case["seqs"],)
    else:
        lead = (1, sum(new))
    if kind != "write":
        # normalised queries times a learned weight: scores with a standard deviation of 1.5
        s["q"] = r.normal(*lead, case["hq"], d, scale=1.5)
    s["k"], s["v"] = r.normal(*lead, hkv, d), r.normal(*lead, hkv, d)
    s["cu"] = None
    if case.get("packed") or kind in ("turn", "write"):
        s["cu"] = torch.tensor(_offsets(new), dtype=torch.int32, device="cuda")
    if kind == "train":
        s["do"] = r.normal(*lead, case["hq"], d)
        for n in "qkv":
            s[n].requires_grad_(True)
    if kind in ("turn", "decode", "write"):
        page = case["page"]
        pages = [-(-(n + h) // page) for n, h in zip(new, held)]
        pool = sum(pages) + 3
        s["k_pages"], s["v_pages"] = r.normal(pool, page, hkv, d), r.normal(pool, page, hkv, d)
        order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
        table, at = torch.full((len(new), max(pages)), -1, dtype=torch.int32), 0
        for row, n in enumerate(pages):
            table[row, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        s["table"] = table.cuda()
        s["lengths"] = torch.tensor(held, dtype=torch.int32, device="cuda")
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


def _causal(s, batch, tokens):
    """[1, 1, 1, T, T]: keys at or before the query, within its sequence."""
    at = torch.arange(tokens, device="cuda")
    allowed = at[:, None] >= at[None, :]
    if s["cu"] is not None:
        seq = torch.bucketize(at, s["cu"][1:].long(), right=True)
        allowed = allowed & (seq[:, None] == seq[None, :])
    return allowed[None, None, None]


def _plain_train(s):
    q, k, v = (s[n].detach() for n in "qkv")
    N, T, hq, d = q.shape
    hkv = k.shape[2]
    g = hq // hkv
    p = _weights(q, k, _causal(s, N, T))
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


def _plain_write(s, k, v):
    """New tokens' keys and values into their pages, behind what the sequence holds."""
    page = s["k_pages"].shape[1]
    n = k.shape[0]
    at = torch.arange(n, device="cuda")
    if s["cu"] is None:
        seq, pos = at, s["lengths"].long()
    else:
        seq = torch.bucketize(at, s["cu"][1:].long(), right=True)
        pos = s["lengths"].long()[seq] + at - s["cu"].long()[seq]
    into = s["table"].long()[seq, pos // page]
    s["k_pages"][into, pos % page] = k
    s["v_pages"][into, pos % page] = v
    return seq, pos


def _gathered(s):
    """(k, v) [N, capacity, hkv, d] as the tables lay them out."""
    table = s["table"].long().clamp(min=0)
    flat = lambda t: t[table].flatten(1, 2)
    return flat(s["k_pages"]), flat(s["v_pages"])


def _plain_turn(s):
    q = s["q"][0]
    _, pos = _plain_write(s, s["k"][0], s["v"][0])
    cu = s["cu"].long()
    most = max(s["new"])
    i = torch.arange(most, device="cuda")
    token = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)      # [N, most], rows past the last idle
    k, v = _gathered(s)
    key = torch.arange(k.shape[1], device="cuda")
    allowed = key <= (s["lengths"].long()[:, None] + i)[..., None]
    o = _mixed(_weights(q[token], k, allowed[:, None, None]), v).to(BF16)
    seq = torch.bucketize(torch.arange(q.shape[0], device="cuda"), cu[1:], right=True)
    return [o[seq, torch.arange(q.shape[0], device="cuda") - cu[seq]][None], s["k_pages"], s["v_pages"]]


def _plain_decode(s):
    _plain_write(s, s["k"], s["v"])
    k, v = _gathered(s)
    allowed = torch.arange(k.shape[1], device="cuda") <= s["lengths"].long()[:, None]
    p = _weights(s["q"][:, None], k, allowed[:, None, None, None])
    return [_mixed(p, v)[:, 0].to(BF16), s["k_pages"], s["v_pages"]]


def _own(s):
    import omegalax_amd as om
    kind = s["kind"]
    if kind == "prefill":
        return [om.attention_prefill(s["q"], s["k"], s["v"], cu_seqlens=s["cu"])]
    if kind == "train":
        x = [s[n] for n in "qkv"]
        o = om.attention_prefill(*x, cu_seqlens=s["cu"])
        return [o.detach(), *torch.autograd.grad(o, x, s["do"])]
    cache = (s["k_pages"], s["v_pages"], s["table"], s["lengths"])
    if kind == "decode":
        return [om.attention_decode_step(s["q"], s["k"], s["v"], *cache), s["k_pages"], s["v_pages"]]
    om.kv_pages_write(s["k"], s["v"], *cache, cu_seqlens=s["cu"])
    if kind == "write":
        return [s["k_pages"], s["v_pages"]]
    return [om.attention_prefill_paged(s["q"], *cache, cu_seqlens=s["cu"]), s["k_pages"], s["v_pages"]]


def run(s):
    if own:
        return _own(s)
    kind = s["kind"]
    if kind == "prefill":
        N, T = s["q"].shape[:2]
        return [_mixed(_weights(s["q"], s["k"], _causal(s, N, T)), s["v"]).to(BF16)]
    if kind == "train":
        return _plain_train(s)
    if kind == "turn":
        return _plain_turn(s)
    if kind == "decode":
        return _plain_decode(s)
    _plain_write(s, s["k"][0], s["v"][0])
    return [s["k_pages"], s["v_pages"]]


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    new, held = _shape(case)
    kind, hkv, d = case["kind"], case["hkv"], case["d"]
    tokens, row = sum(new), hkv * d * 2
    if kind == "write":
        return dict(bytes=4 * tokens * row, flops=0)
    hq = case["hq"]
    pairs = sum(n * h + n * (n + 1) // 2 for n, h in zip(new, held))
    if kind in ("prefill", "train"):
        q = tokens * hq * d * 2
        if kind == "prefill":
            return dict(bytes=2 * q + 2 * tokens * row, flops=4 * hq * d * pairs)
        return dict(bytes=4 * q + 4 * tokens * row, flops=14 * hq * d * pairs)
    # new keys and values read and written, held ones read; queries in, outputs out
    return dict(bytes=4 * tokens * row + 2 * sum(held) * row + 4 * tokens * hq * d,
                flops=4 * hq * d * pairs)


# ---------------------------------------------------------------- the definition in 64 bits


def _rows64(q, k, v, first):
    """Attention of one head: query i sees the keys up to first + i."""
    s = q @ k.t() * q.shape[-1] ** -0.5
    unseen = torch.ones_like(s, dtype=torch.bool).triu(first + 1)
    return torch.softmax(s.masked_fill(unseen, -math.inf), -1) @ v


def _sequence64(q, k, v, first):
    """[n, hq, d] for one sequence's q [n, hq, d] and keys and values [m, hkv, d]."""
    g = q.shape[1] // k.shape[1]
    return torch.stack([_rows64(q[:, h], k[:, h // g], v[:, h // g], first)
                        for h in range(q.shape[1])], 1)


def _pages64(s):
    """The pools with the new tokens in place, in 64 bits, and each sequence's keys and values."""
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    page, table = kp.shape[1], s["table"].tolist()
    k, v = (t.double().flatten(0, -3) for t in (s["k"], s["v"]))
    caches, at = [], 0
    for n, h, row in zip(s["new"], s["held"], table):
        used = torch.tensor(row[:-(-(n + h) // page)], device="cuda")
        for pool, x in ((kp, k), (vp, v)):
            flat = pool[used].flatten(0, 1)
            flat[h:h + n] = x[at:at + n]
            pool[used] = flat.view(-1, *pool.shape[1:])
        caches.append([pool[used].flatten(0, 1)[:n + h] for pool in (kp, vp)])
        at += n
    return kp, vp, caches


def exact(case, seed):
    s = prepare(case, seed)
    kind, new, held = s["kind"], s["new"], s["held"]
    cu = _offsets(new)
    spans = list(zip(cu, cu[1:]))
    if kind in ("prefill", "train"):
        shape = s["q"].shape
        outs = []
        flat = [s[n].detach().double().flatten(0, 1) for n in "qkv"]
        if kind == "prefill":
            o = [_sequence64(*(t[a:b] for t in flat), 0) for a, b in spans]
            return [torch.cat(o).view(shape)]
        do = s["do"].double().flatten(0, 1)
        hkv, g = case["hkv"], case["hq"] // case["hkv"]
        outs = [torch.zeros_like(flat[0]), *(torch.zeros_like(t) for t in flat)]
        for a, b in spans:
            for j in range(hkv):
                heads = slice(j * g, (j + 1) * g)
                q, k, v = (t.clone().requires_grad_(True)
                           for t in (flat[0][a:b, heads], flat[1][a:b, j:j + 1], flat[2][a:b, j:j + 1]))
                o = _sequence64(q, k, v, 0)
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), do[a:b, heads])
                outs[0][a:b, heads], outs[1][a:b, heads] = o.detach(), dq
                outs[2][a:b, j:j + 1], outs[3][a:b, j:j + 1] = dk, dv
        return [t.view(*shape[:2], *t.shape[1:]) for t in outs]
    kp, vp, caches = _pages64(s)
    if kind == "write":
        return [kp, vp]
    q = s["q"].double().flatten(0, -3)
    o = [_sequence64(q[a:b], k, v, h) for (a, b), (k, v), h in zip(spans, caches, held)]
    return [torch.cat(o).view(s["q"].shape), kp, vp]
