"""Causal softmax attention in 64 bits, with bounds of what the kernels' roundings may cost.

A bf16 rounding is off by at most U = 2^-8 of the value.  The forward rounds each weight (relative
to the row's maximum, in fp32 before) for its product with v, and the output once:
  |o - o64| <= U (sum_j p_j |v_j| + |o64|).
The backward rounds p for dv, ds for dq and dk, and each gradient; delta = do . o is formed from the
rounded o, so it is off by E_i <= |do_i| . |o - o64|, which ds carries as p E:
  |dv - dv64| <= U (sum_i p |do| + |dv64|)
  |dq - dq64| <= scale sum_j (U |ds| + p E) |k_j| + U |dq64|,  dk likewise over i with |q_i|.
What fp32 adds (scores, exp2, sums: a few 2^-24 of terms of the same size) is far below 5% of
these; the bounds are taken 1.05 times.
"""
import torch

U = 2.0 ** -8
MORE = 1.05


def one_sequence(q, k, v, first, do=None, allowed=None, scale=None):
    """q [n,Hq,D], k, v [m,Hkv,D] in 64 bits: query i sees keys j <= first + i that `allowed` [m]
    leaves.  Returns dicts of values and of bounds."""
    n, Hq, D = q.shape
    m, Hkv = k.shape[:2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    see = torch.arange(m, device=q.device)[None, :] <= first + torch.arange(n, device=q.device)[:, None]
    if allowed is not None:
        see = see & allowed[None, :]
    val = dict(o=torch.zeros_like(q), lse=q.new_full((n, Hq), float("-inf")))
    tol = dict(o=torch.zeros_like(q))
    if do is not None:
        for name, t in (("dq", q), ("dk", k), ("dv", v)):
            val[name], tol[name] = torch.zeros_like(t), torch.zeros_like(t)
    for h in range(Hq):
        j = h // G
        K, V, Q = k[:, j], v[:, j], q[:, h]
        V = torch.where(see.any(0)[:, None], V, 0.0)  # keys nobody sees may hold anything
        K = torch.where(see.any(0)[:, None], K, 0.0)
        s = (Q @ K.t() * scale).masked_fill(~see, float("-inf"))
        lse = torch.logsumexp(s, -1)
        some = see.any(1)
        p = torch.where(some[:, None], torch.exp(s - torch.where(some, lse, 0.0)[:, None]), 0.0)
        o = p @ V
        val["o"][:, h], val["lse"][:, h] = o, lse
        to = MORE * U * (p @ V.abs() + o.abs())
        tol["o"][:, h] = to
        if do is None:
            continue
        dO = do[:, h]
        ds = p * (dO @ V.t() - (dO * o).sum(-1, keepdim=True))
        E = (dO.abs() * to).sum(-1, keepdim=True)
        spread = U * ds.abs() + p * E
        dq, dk, dv = scale * ds @ K, scale * ds.t() @ Q, p.t() @ dO
        val["dq"][:, h] = dq
        val["dk"][:, j] += dk
        val["dv"][:, j] += dv
        tol["dq"][:, h] = MORE * scale * spread @ K.abs()
        tol["dk"][:, j] += MORE * scale * spread.t() @ Q.abs()
        tol["dv"][:, j] += MORE * U * (p.t() @ dO.abs())
    if do is not None:
        for name in ("dq", "dk", "dv"):
            tol[name] += MORE * U * val[name].abs()
    return val, tol


def check(name, got, want, tol):
    """Every element within its bound, and non-finite ones where they belong."""
    got = got.double()
    far = (got - want).abs() - tol
    bad = ~(far <= 1e-7)
    if bool(bad.any()):
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {i}: "
                             f"{float(got[i])} for {float(want[i])}, bound {float(tol[i])}")
