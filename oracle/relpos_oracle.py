"""64-bit statement of attention with a learned relative position bias, with bounds on what a kernel may be off.

Test infrastructure only. One (sequence, head) at a time, straight from the formulas:

    S = c Q K^T + T[bucket(r), h],  r = j - (i + sk - sq),  P = softmax(S),  O = P V
    dP = dO V^T,  D = rowsum(dO O),  dS = P (dP - D),  dQ = c dS K,  dK = c dS^T Q,  dV = P^T dO,  dT[t, h] = sum of dS over bucket t

Bounds (u = half a step of the inputs' type, e = 2^-24). The kernels hold sums, softmax statistics and dS in float32 and round to
the inputs' type in three places: P and dS where they become operands of a matrix product, and every output once (O is
also what D is computed from).
    a score                 |dS_ij| <= es_ij = (d + 8) e (c |q|.|k| + |T|): d products and sums, the bias, the shift by the row's maximum
    P, relative             ep = 2 max_j es + 16 e: exp of a score that is off, and the row sum likewise; the exponential itself and its argument
    O                       (u + ep + n e) P |V| + u |O|           u: P as an operand; n e: float32 sums over n keys
    D                       dD = u rowsum(|dO| |O|) + (1 + u) (rowsum(|dO| (u + ep + n e) P|V|) + d e |dO| |O|)
    dS                      ds = |dS| ep + P (dD + d e |dO|.|V| )
    dQ                      c (ds + (u + n e) |dS|) |K| + u |dQ|;  dK, dV, dT alike (dT has no operand rounding)
`apart`: the scores are formed as c q.k + (T - top), top the largest entry that the row's keys have, so that |T - top| takes the place of |T|:
    |dS_ij| <= es_ij = (d + 8) e c |q|.|k| + 2^10 e |T - top|     two entries that differ do so by 2^-8 (bf16) of the larger or more, so that their own
                                                                   roundings to log2 units, 2 e |T| each, are within 2^9 e |T - top| each
    P, relative             ep_ij = es_ij + sum_j P_ij es_ij + 16 e
float16 operands (P, dS) below 2^-14 are subnormal: their rounding is off by up to half a step of 2^-24, an absolute w = 2^-25 beside
the relative u. It adds w rowsum(|V|) to O, c w rowsum(|K|) to dQ, and so on; 0 for the other types, whose range is float32's.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch


def bucket(n: int, side: int, far: int) -> int:
    """Bucket of distance n on a side of `side` buckets, in whole numbers: the formula's logarithms compared as powers."""
    e = side // 2
    if n < e:
        return n
    m, t = side - e, 0
    while t + 1 < m and n ** m * e ** (t + 1) >= far ** (t + 1) * e ** m:
        t += 1
    return e + t


def buckets(sq: int, sk: int, num: int, far: int, two: bool) -> torch.Tensor:
    """(sq, sk) bucket of every pair."""
    side = num // 2 if two else num
    memo = {n: bucket(min(n, far), side, far) for n in range(0, max(sq, sk) + abs(sk - sq) + 1)}
    of = lambda r: (memo[-r] if r <= 0 else (side + memo[r] if two else memo[0]))  # noqa: E731
    line = {r: of(r) for r in range(-(max(sq, sk) + abs(sk - sq)), max(sq, sk) + abs(sk - sq) + 1)}
    return torch.tensor([[line[j - (i + sk - sq)] for j in range(sk)] for i in range(sq)], dtype=torch.long).reshape(sq, sk)


class Head(NamedTuple):
    out: torch.Tensor
    dq: Optional[torch.Tensor]
    dk: Optional[torch.Tensor]
    dv: Optional[torch.Tensor]
    dt: Optional[torch.Tensor]
    tol_out: torch.Tensor
    tol_dq: Optional[torch.Tensor]
    tol_dk: Optional[torch.Tensor]
    tol_dv: Optional[torch.Tensor]
    tol_dt: Optional[torch.Tensor]


def head(q, k, v, table, which, scale, causal, u, dout=None, w=0.0, apart=False) -> Head:
    """q (sq, d), k/v (sk, d), table (num,), which (sq, sk) long; everything float64 on one device."""
    e = 2.0 ** -24
    sq, sk, d = q.shape[0], k.shape[0], q.shape[1]
    b = table[which]
    s = scale * (q @ k.T) + b
    hidden = torch.zeros(sq, sk, dtype=torch.bool, device=q.device)
    if causal:
        hidden = torch.arange(sk, device=q.device)[None, :] - torch.arange(sq, device=q.device)[:, None] > sk - sq
    s = s.masked_fill(hidden, -math.inf)
    m = s.amax(-1, keepdim=True) if sk else torch.full((sq, 1), -math.inf, dtype=q.dtype, device=q.device)
    p = torch.exp(s - m.masked_fill(m == -math.inf, 0.0))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    out = p @ v
    mag = (abs(scale) * (q.abs() @ k.abs().T) + b.abs()).masked_fill(hidden | (s == -math.inf), 0.0)
    es = (d + 8) * e * mag
    if apart:
        seen_b = b.masked_fill(hidden | (s == -math.inf), -math.inf)
        top = seen_b.amax(-1, keepdim=True) if sk else torch.zeros(sq, 1, dtype=q.dtype, device=q.device)
        es = (d + 8) * e * abs(scale) * (q.abs() @ k.abs().T) + 2.0 ** 10 * e * (b - top).abs()
        es = es.masked_fill(seen_b == -math.inf, 0.0)
    ep = (2 * es.amax(-1, keepdim=True) + 16 * e) if sk else torch.zeros(sq, 1, dtype=q.dtype, device=q.device)
    if apart:
        ep = es + (p * es).sum(-1, keepdim=True) + 16 * e
    seen = (p > 0).to(q.dtype)
    tol_out = (p * (u + ep + sk * e)) @ v.abs() + w * (seen @ v.abs()) + u * out.abs() * (1 + 2 * u)
    if dout is None:
        return Head(out, None, None, None, None, tol_out, None, None, None, None)
    g = dout
    dp = g @ v.T
    dd = (g * out).sum(-1, keepdim=True)
    ds = p * (dp - dd)
    err_d = ((g.abs() * tol_out).sum(-1, keepdim=True)) + d * e * (g.abs() * out.abs()).sum(-1, keepdim=True) * (1 + u)
    err_s = ds.abs() * ep * (1 + ep) + p * (err_d + d * e * (g.abs() @ v.abs().T) + 2 * e * (dp.abs() + dd.abs())) * (1 + ep)
    op = err_s + (u + 4 * e) * (ds.abs() + err_s) + w * seen  # dS as an operand
    dq, dk, dv = scale * ds @ k, scale * ds.T @ q, p.T @ g
    c = abs(scale)
    tol_dq = c * (op + sk * e * ds.abs()) @ k.abs() * (1 + u) + (u + 2 * e) * dq.abs()
    tol_dk = c * (op + sq * e * ds.abs()).T @ q.abs() * (1 + u) + (u + 2 * e) * dk.abs()
    tol_dv = (p * (ep + u + sq * e) + w * seen).T @ g.abs() * (1 + u) + u * dv.abs()
    num = table.shape[0]
    # the table's gradient: float32 sums over a warp's diagonals, a tile, then in 64 bits over the tiles; at most sk + 256 summands in a row
    dt = torch.zeros(num, dtype=q.dtype, device=q.device).index_add_(0, which.flatten(), ds.flatten())
    tol_dt = torch.zeros_like(dt).index_add_(0, which.flatten(), (err_s + (sk + 256) * e * ds.abs()).flatten())
    return Head(out, dq, dk, dv, dt, tol_out, tol_dq, tol_dk, tol_dv, tol_dt)


class Result(NamedTuple):
    out: torch.Tensor
    dq: Optional[torch.Tensor]
    dk: Optional[torch.Tensor]
    dv: Optional[torch.Tensor]
    dt: Optional[torch.Tensor]
    tol: tuple  # bounds for (out, dq, dk, dv, dt)


def attention(q, k, v, table, far, two, scale, causal, dout=None, lens_q=None, lens_k=None, apart=False) -> Result:
    """Dense (b, s, h, d), or packed (total, h, d) with lens_q, lens_k; inputs of any type, results float64."""
    u = torch.finfo(q.dtype).eps / 2
    packed = q.dim() == 3
    w = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    wide = lambda t: None if t is None else t.detach().double()  # noqa: E731
    q, k, v, table, dout = map(wide, (q, k, v, table, dout))
    shape_q, shape_k = q.shape, k.shape
    if not packed:
        lens_q, lens_k = [q.shape[1]] * q.shape[0], [k.shape[1]] * k.shape[0]
        q, k, v = q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1)
        dout = None if dout is None else dout.flatten(0, 1)
    group = q.shape[1] // k.shape[1]
    z = torch.zeros_like
    out, tol_out, dq, tol_dq = z(q), z(q), z(q), z(q)
    dk, tol_dk, dv, tol_dv = z(k), z(k), z(k), z(k)
    dt, tol_dt = z(table), z(table)
    iq = ik = 0
    for nq, nk in zip(lens_q, lens_k):
        which = buckets(nq, nk, table.shape[0], far, two).to(q.device)
        sl, kl = slice(iq, iq + nq), slice(ik, ik + nk)
        for h in range(q.shape[1]):
            hk = h // group
            r = head(q[sl, h], k[kl, hk], v[kl, hk], table[:, h], which, scale, causal, u, None if dout is None else dout[sl, h], w, apart)
            out[sl, h], tol_out[sl, h] = r.out, r.tol_out
            if dout is not None:
                dq[sl, h], tol_dq[sl, h] = r.dq, r.tol_dq
                dk[kl, hk] += r.dk
                tol_dk[kl, hk] += r.tol_dk
                dv[kl, hk] += r.dv
                tol_dv[kl, hk] += r.tol_dv
                dt[:, h] += r.dt
                tol_dt[:, h] += r.tol_dt
        iq, ik = iq + nq, ik + nk
    tol_dt = tol_dt + u * (dt.abs() + tol_dt)
    if dout is None:
        return Result(out.view(shape_q), None, None, None, None, (tol_out.view(shape_q),))
    return Result(out.view(shape_q), dq.view(shape_q), dk.view(shape_k), dv.view(shape_k), dt,
                  (tol_out.view(shape_q), tol_dq.view(shape_q), tol_dk.view(shape_k), tol_dv.view(shape_k), tol_dt))
