"""Attention in float64 with bounds on how far the kernels' results may be.

The bounds follow one rounding analysis, worst cases added up.  u is half a
step of float32 (2^-24), h half a step of the operands' type (0 where that is
float32).  A sum of n products in any order is off by at most n u times the
sum of their magnitudes; an exponential of an argument that is off by e is off
by a factor of 1 +- (e + 4 u (1 + |argument|)), the second term for the
argument's own rounding in base 2 and for the hardware's exponential.
"""
import numpy as np

U = 2.0 ** -24
H = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
# below the smallest normal number of fp16 a rounding is off by an absolute amount
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}


def visible(nq, nk, causal):
    i, j = np.arange(nq)[:, None], np.arange(nk)[None, :]
    return j <= i + nk - nq if causal else np.ones((nq, nk), bool)


def head(q, k, v, causal, scale, dtype, w=None):
    """One head of one sequence: {name: (value, bound)} for o, lse and, with
    the upstream gradient w, dq, dk, dv (dk and dv of this query head alone)."""
    h, tiny = H[dtype], TINY[dtype]
    nq, size = q.shape
    nk = k.shape[0]
    see = visible(nq, nk, causal)
    s = np.where(see, scale * (q @ k.T), -np.inf)
    s_off = scale * (np.abs(q) @ np.abs(k).T) * (size + 4) * U
    top = s.max(1, initial=-np.inf, keepdims=True)
    ref = np.where(np.isneginf(top), 0.0, top)
    e = np.where(see, np.exp(s - ref), 0.0)
    total = e.sum(1, keepdims=True)
    p = e / np.where(total == 0, 1.0, total)
    # an exponential's error against the row's sum of them
    with np.errstate(invalid="ignore"):
        arg = np.where(see, np.abs(s - ref) + 2 * np.abs(s), 0.0)
    each = np.where(see, s_off + 4 * U * (1 + arg), 0.0)
    most = each.max(1, initial=0.0, keepdims=True) + (nk + 8) * U  # of the sum, relatively
    p_rel = each + most
    o = p @ v
    # 16 bits: each probability is rounded once, relatively to its own size down to the smallest normal
    # number (the largest of a row is at least 2^-8 of its reference), and the result once
    o_off = ((p * (p_rel + h) + 256 * tiny * see) @ np.abs(v)) * (1 + h) + h * np.abs(o) + (nk + 4) * U * (p @ np.abs(v)) + tiny
    out = {"o": (o, o_off)}
    with np.errstate(divide="ignore"):
        lse = np.where(total[:, 0] == 0, -np.inf, ref[:, 0] + np.log(np.where(total[:, 0] == 0, 1, total[:, 0])))
    out["lse"] = (lse, most[:, 0] + 8 * U * (1 + np.abs(np.where(np.isneginf(lse), 0, lse))))
    if w is None:
        return out
    lse_off = out["lse"][1][:, None]
    p_rel = each + lse_off + 4 * U * (1 + np.abs(np.where(see, s, 0)) + np.abs(np.where(np.isneginf(lse), 0, lse))[:, None])
    dp = w @ v.T
    d = (w * o).sum(1, keepdims=True)
    dp_off = (np.abs(w) @ np.abs(v).T) * (size + 4) * U
    d_off = (np.abs(w) * (o_off + np.abs(o) * (size + 4) * U)).sum(1, keepdims=True)
    t = p * (dp - d)
    t_off = np.abs(t) * (p_rel + 2 * U) + p * (dp_off + d_off) * (1 + p_rel)
    t_off = t_off + h * (np.abs(t) + t_off) + tiny * see
    dv, dv_off = p.T @ w, (p * (p_rel + h) + tiny * see).T @ np.abs(w) + (nq + 4) * U * (p.T @ np.abs(w))
    dq, dq_off = scale * t @ k, scale * (t_off @ np.abs(k) + (nk + 4) * U * (np.abs(t) @ np.abs(k)))
    dk, dk_off = scale * t.T @ q, scale * (t_off.T @ np.abs(q) + (nq + 4) * U * (np.abs(t).T @ np.abs(q)))
    for name, x, off in (("dq", dq, dq_off), ("dk", dk, dk_off), ("dv", dv, dv_off)):
        out[name] = (x, off + h * (np.abs(x) + off) + tiny)
    return out


def attention(q, k, v, causal, scale, dtype, spans, w=None):
    """q [rows, heads, size], k, v [rows, kv heads, size] in float64; spans: (first query, queries, first key,
    keys) of each sequence.  {name: (value, bound)} with zeros (bound 0) in rows of no sequence."""
    group = q.shape[1] // k.shape[1]
    names = {"o": q.shape, "lse": q.shape[:2]}
    if w is not None:
        names.update(dq=q.shape, dk=k.shape, dv=k.shape)
    out = {n: (np.zeros(s), np.zeros(s)) for n, s in names.items()}
    for q0, nq, k0, nk in spans:
        for hq in range(q.shape[1]):
            hk = hq // group
            qs, ks = (slice(q0, q0 + nq), hq), (slice(k0, k0 + nk), hk)
            got = head(q[qs], k[ks], v[ks], causal, scale, dtype, None if w is None else w[qs])
            for n, (x, off) in got.items():
                at = ks if n in ("dk", "dv") else qs
                if n in ("dk", "dv"):  # the heads of a group add up, unrounded
                    out[n][0][at] += x
                    out[n][1][at] += off
                else:
                    out[n][0][at], out[n][1][at] = x, off
    return out
