"""Attention whose scores are large: up to 1e12 of both signs, and the range between.  Queries hold powers of two in one
or two elements and zeros elsewhere, and keys small whole numbers there, so that every score is exact in float32 in any
order of sums, and the softmax is known whatever the scores' size."""
import ctypes
import math

import numpy as np
import pytest

import attention_ref as R
from phptensors import CudaArray, _host

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "float16", "bfloat16"]
U = R.U


def head(q, k, v, w, causal, scale, dtype, exact=True):
    """{name: (value, bound)} of one head, in float64, as attention_ref.head, for exact scores: an exponential of
    argument x, taken as one difference, scaled, is off by a factor of 1 +- 4 u (1 + |x|), the sum by u for each term.
    exact False: scores off by their products' roundings, of rows in which one key is so far ahead that its weight is 1
    all the same."""
    h, tiny = R.H[dtype], R.TINY[dtype]
    (nq, size), nk = q.shape, k.shape[0]
    see = R.visible(nq, nk, causal)
    s = np.where(see, scale * (q @ k.T), -np.inf)
    top = s.max(1, keepdims=True)
    assert np.isfinite(top).all()
    e = np.exp(s - top)
    total = e.sum(1, keepdims=True)
    p = e / total
    if not exact:
        off = scale * (np.abs(q) @ np.abs(k).T).max(1) * (size + 4) * U
        gap = np.sort(s, 1)
        assert (gap[:, -1] - gap[:, -2] > 2 * off + 200).all() and (p == e).all()
    arg = np.where(p > 0, top - s, 0.0)
    p_rel = 4 * U * (1 + arg) + (4 * U * (1 + arg)).max(1, keepdims=True) + (nk + 8) * U
    # (exponentials below the smallest float32 vanish)
    o = p @ v
    o_off = (p * (p_rel + h) + 256 * tiny * see) @ np.abs(v) * (1 + h) + h * np.abs(o) + (nk + 4) * U * (p @ np.abs(v)) + tiny
    lse = (top + np.log(total))[:, 0]
    # Rows whose lse is 512 or less keep it as one rounded number, as attention_ref counts it: lse's own bound, and the
    # roundings of its product with log2(e) and of the exponent.  (513: its value here may be a rounding larger.)
    size_of = np.where(np.abs(lse) <= 513, np.abs(lse), 0.0)[:, None]
    p_rel = p_rel + np.where(size_of > 0, 8 * U * (1 + size_of) + 4 * U * (1 + size_of + np.where(see, np.abs(s), 0.0)), 0.0)
    dp, d = w @ v.T, (w * o).sum(1, keepdims=True)
    dp_off = (np.abs(w) @ np.abs(v).T) * (size + 4) * U
    d_off = (np.abs(w) * (o_off + np.abs(o) * (size + 4) * U)).sum(1, keepdims=True)
    t = p * (dp - d)
    t_off = np.abs(t) * (p_rel + 2 * U) + p * (dp_off + d_off) * (1 + p_rel)
    t_off = t_off + h * (np.abs(t) + t_off) + tiny * see
    dv, dv_off = p.T @ w, (p * (p_rel + h) + tiny * see).T @ np.abs(w) + (nq + 4) * U * (p.T @ np.abs(w))
    dq, dq_off = scale * t @ k, scale * (t_off @ np.abs(k) + (nk + 4) * U * (np.abs(t) @ np.abs(k)))
    dk, dk_off = scale * t.T @ q, scale * (t_off.T @ np.abs(q) + (nq + 4) * U * (np.abs(t).T @ np.abs(q)))
    out = {"o": (o, o_off), "lse": (lse, 8 * U * (1 + np.abs(lse)))}
    for name, x, off in (("dq", dq, dq_off), ("dk", dk, dk_off), ("dv", dv, dv_off)):
        out[name] = (x, off + h * (np.abs(x) + off) + tiny)
    return out


def check(q, k, v, w, causal, scale, dtype, exact=True):
    """q, w [tokens, heads, size], k, v [tokens, key heads, size] as CudaArrays: everything against float64."""
    qv, kv, vv, wv = (t.toNumpy().astype(np.float64) for t in (q, k, v, w))
    (nq, heads, _), (nk, kv_heads, _) = qv.shape, kv.shape
    want = {n: (np.zeros(s), np.zeros(s)) for n, s in (("o", qv.shape), ("lse", (heads, nq)), ("dq", qv.shape), ("dk", kv.shape),
                                                       ("dv", kv.shape))}
    for i in range(heads):
        j = i // (heads // kv_heads)
        for n, x in head(qv[:, i], kv[:, j], vv[:, j], wv[:, i], causal, scale, dtype, exact).items():
            at = (i,) if n == "lse" else (slice(None), j if n in ("dk", "dv") else i)
            for a, b in zip(want[n], x):
                a[at] += b   # the heads of a group add up, unrounded
    lib, kept, got = _host.load(), (ctypes.c_void_p * 2)(), (ctypes.c_void_p * 3)()
    o = CudaArray._wrap(lib.phpt_attention(q._h, k._h, v._h, int(causal), scale, None, None, kept))
    lse, rest = (CudaArray._wrap(h) if h else None for h in kept)
    assert not lib.phpt_attention_backward(q._h, k._h, v._h, o._h, lse._h, rest._h if rest is not None else None, w._h,
                                           int(causal), scale, None, None, got)
    for n, t in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *(CudaArray._wrap(h) for h in got))):
        x, off = want[n]
        t = t.toNumpy().astype(np.float64).reshape(x.shape)
        if dtype == "float16" and n != "lse":   # (elements whose bounds leave the type show nothing: few)
            fits = np.abs(x) + off < 65504
            assert fits.mean() > 0.9, n
            t, x, off = (np.where(fits, y, 0.0) for y in (t, x, off))
        far = np.abs(t - x) - off
        assert not np.isnan(t).any() and far.max() <= 0, (n, np.unravel_index(far.argmax(), far.shape), t.flat[far.argmax()],
                                                           x.flat[far.argmax()], off.flat[far.argmax()])


def operands(nq, nk, heads, kv, size, dtype, q, k, w):
    """Random arrays with the first elements of the queries' and keys' heads given, all other elements of queries 0."""
    rng = np.random.default_rng(nq + nk)
    a = np.zeros((nq, heads, size), np.float32)
    b, c = rng.standard_normal((2, nk, kv, size)).astype(np.float32)
    for i, x in enumerate(q):
        a[:, :, i] = x(rng, (nq, heads))
    for i, x in enumerate(k):
        b[:, :, i] = x(rng, (nk, kv))
    return [CudaArray.fromNumpy(x.astype(np.float32), dtype) for x in (a, b, c, w * rng.standard_normal(a.shape))]


# queries, keys, heads, key heads, size: one block, tiles and a ragged end, elements staged one by one, split prompts,
# single tokens alone and split, wide heads
SHAPES = [(5, 9, 2, 1, 64), (70, 190, 4, 2, 64), (140, 70, 2, 2, 128), (20, 45, 3, 1, 24), (40, 900, 2, 1, 64), (1, 33, 4, 2, 64),
          (1, 1500, 8, 2, 128), (2, 515, 2, 1, 256), (50, 600, 1, 1, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("power", [30, 34, 40])
def test_scores_of_any_size(shape, power, dtype):
    """Scores of 3 to 7 times +- 2^(power - 2), so that the largest of a row, several times there, share the weight;
    rows of all zeros and of ordinary scores beside them."""
    nq, nk, heads, kv, size = shape

    def queries(rng, n):
        x = 256 * rng.choice([-1.0, 1.0], n)
        x[rng.random(n) < 0.2] = 0.0
        # 4096 of a key times this times the scale: of order 1
        x[rng.random(n) < 0.2] = 2.0 ** -(12 + power - 22)
        return x
    ops = operands(*shape, dtype, [queries], [lambda rng, n: 4096.0 * rng.integers(3, 8, n)],
                   2.0 ** (-10 if power == 30 else -16))
    if dtype == "float16":   # (what is below its numbers is another score, and a known one)
        assert np.abs(ops[0].toNumpy()).max() == 256
    for causal in (False, True) if nk >= nq else (False,):
        check(*ops, causal, 2.0 ** (power - 22), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES[1:7], ids=str)
@pytest.mark.parametrize("base", [10, 14, 18, 22])
def test_neighbouring_scores_of_any_size(shape, base, dtype):
    """Scores of +- 2^base and some ones more or less: the weights are those of the differences."""
    nq, nk, heads, kv, size = shape
    half = base // 2
    ops = operands(*shape, dtype, [lambda rng, n: rng.choice([-1.0, 1.0], n) * 2.0 ** half, lambda rng, n: np.ones(n)],
                   [lambda rng, n: np.full(n, 2.0 ** (base - half)), lambda rng, n: rng.integers(-40, 41, n)], 2.0 ** -6)
    for scale in (0.25, 1.0) if base < 22 else (0.25, 8.0):   # 8: beyond 2^24 in base 2
        check(*ops, False, scale, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(60, 90, 4, 2, 64), (33, 600, 2, 2, 128), (1, 800, 8, 2, 64), (30, 20, 2, 1, 40)], ids=str)
def test_random_products(shape, dtype):
    """Scores of order 1e9 that are sums of roundings: both gradient kernels see the same ones, and the key that is
    ahead has all the weight."""
    nq, nk, heads, kv, size = shape
    rng = np.random.default_rng(sum(shape))
    ops = [CudaArray.fromNumpy((s * rng.standard_normal((n, h, size))).astype(np.float32), dtype)
           for n, h, s in ((nq, heads, 1.0), (nk, kv, 1.0), (nk, kv, 1.0), (nq, heads, 2.0 ** -24))]
    if dtype == "float16":
        ops[3] = CudaArray.fromNumpy(np.zeros((nq, heads, size), np.float32) + 2.0 ** -24, dtype)
    q, k = (t.toNumpy().astype(np.float64) for t in ops[:2])
    # rows whose two largest scores are too close to tell in float32 are made zeros but for one element
    for i in range(heads):
        s = 2.0 ** 27 * np.sort(q[:, i] @ k[:, i // (heads // kv)].T, 1)
        near = s[:, -1] - s[:, -2] < 2.0 ** 27 * 140 * U * np.abs(q[:, i]) @ np.abs(k[:, i // (heads // kv)]).T.max(1) + 300
        q[near, i] = 0.0
        q[near, i, 0] = 4.0
    ops[0] = CudaArray.fromNumpy(q.astype(np.float32), dtype)
    check(*ops, False, 2.0 ** 27, dtype, exact=False)
