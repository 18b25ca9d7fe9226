"""Softmax attention of one sequence in 64 bits whose queries see a window of keys and the first
ones, with the bounds that attn_reference derives: the roundings are the same, over fewer keys."""
import torch

from attn_reference import MORE, U


def seen(n, m, first, window=None, sinks=0, allowed=None, device="cuda"):
    """[n, m]: whether query i, at position first + i, sees key j."""
    i = torch.arange(n, device=device)[:, None] + first
    j = torch.arange(m, device=device)[None]
    see = j <= i
    if window is not None:
        see = see & ((i - j < window) | (j < sinks))
    return see if allowed is None else see & allowed[None, :]


def one_sequence(q, k, v, see, do=None, scale=None):
    """q [n,Hq,D], k, v [m,Hkv,D] in 64 bits, see [n,m].  Returns dicts of values and of bounds."""
    n, Hq, D = q.shape
    G = Hq // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    val = dict(o=torch.zeros_like(q), lse=q.new_full((n, Hq), float("-inf")))
    tol = dict(o=torch.zeros_like(q))
    if do is not None:
        for name, t in (("dq", q), ("dk", k), ("dv", v)):
            val[name], tol[name] = torch.zeros_like(t), torch.zeros_like(t)
    used, some = see.any(0)[:, None], see.any(1)
    for h in range(Hq):
        j = h // G
        K, V, Q = torch.where(used, k[:, j], 0.0), torch.where(used, v[:, j], 0.0), q[:, h]  # unseen: anything
        s = (Q @ K.t() * scale).masked_fill(~see, float("-inf"))
        lse = torch.logsumexp(s, -1)
        p = torch.where(some[:, None], torch.exp(s - torch.where(some, lse, 0.0)[:, None]), 0.0)
        o = p @ V
        to = MORE * U * (p @ V.abs() + o.abs())
        val["o"][:, h], val["lse"][:, h], tol["o"][:, h] = o, lse, to
        if do is None:
            continue
        dO = do[:, h]
        ds = p * (dO @ V.t() - (dO * o).sum(-1, keepdim=True))
        spread = U * ds.abs() + p * (dO.abs() * to).sum(-1, keepdim=True)
        val["dq"][:, h] = scale * ds @ K
        val["dk"][:, j] += scale * ds.t() @ Q
        val["dv"][:, j] += p.t() @ dO
        tol["dq"][:, h] = MORE * scale * spread @ K.abs()
        tol["dk"][:, j] += MORE * scale * spread.t() @ Q.abs()
        tol["dv"][:, j] += MORE * U * (p.t() @ dO.abs())
    if do is not None:
        for name in ("dq", "dk", "dv"):
            tol[name] += MORE * U * val[name].abs()
    return val, tol
