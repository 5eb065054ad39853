"""CudaArray.attention and its gradients against float64, within bounds that
count the roundings (attention_ref)."""
import ctypes
import math

import numpy as np
import pytest

import attention_ref as R
import oracle_lib as O
from phptensors import CudaArray, Fusion, Sequences, _abi, _host

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "float16", "bfloat16"]
CODE = {"float32": O.F32, "float16": O.F16, "bfloat16": O.BF16}


def values(shape, dtype, seed, scale=1.0):
    """(CudaArray, its values in float64), rounded to the dtype first."""
    x = np.random.default_rng(seed).standard_normal(shape).astype(np.float32) * np.float32(scale)
    a = CudaArray.fromNumpy(x, dtype)
    return a, a.toNumpy().astype(np.float64).reshape(shape)


def close(got, want, what):
    x, off = want
    got = got.toNumpy().astype(np.float64).reshape(x.shape)
    assert np.array_equal(np.isneginf(got), np.isneginf(x)), what
    with np.errstate(invalid="ignore"):
        far = np.abs(got - x) - off
    far = np.where(np.isneginf(x) & np.isneginf(got), -1.0, far)
    worst = np.unravel_index(np.argmax(np.where(np.isnan(far), np.inf, far)), far.shape) if far.size else None
    assert not np.isnan(got).any() and (not far.size or far.max() <= 0), (what, worst, got[worst], x[worst], off[worst])


def check(q, k, v, causal, dtype, spans, got, w=None, scale=None, grads=None):
    """`got` and `grads` against float64; q, k, v, w are float64 [rows, heads, size]."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    ref = R.attention(q, k, v, causal, scale, dtype, spans, w)
    close(got, ref["o"], "o")
    if grads is not None:
        for n, g in zip(("dq", "dk", "dv"), grads):
            close(g, ref[n], n)
            assert g.getDtype() == dtype


# tokens of queries and keys, heads, key heads, size
SHAPES = [
    (1, 1, 1, 1, 64), (1, 1, 2, 1, 1), (3, 2, 2, 2, 8), (37, 37, 4, 2, 64), (64, 64, 2, 2, 64), (65, 129, 2, 1, 128),
    (130, 257, 3, 3, 128), (128, 128, 1, 1, 256), (33, 70, 2, 1, 200), (40, 50, 4, 4, 80), (50, 40, 4, 2, 96),
    (31, 33, 8, 1, 32), (20, 45, 3, 1, 33), (9, 140, 2, 2, 7), (1, 1000, 8, 2, 64), (1, 700, 4, 4, 128), (2, 515, 6, 2, 256),
    (5, 300, 16, 2, 72), (100, 1, 2, 2, 16), (200, 520, 2, 2, 48),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_one_sequence(shape, causal, dtype):
    nq, nk, heads, kv, size = shape
    q, qv = values((nq, heads, size), dtype, 1)
    k, kvv = values((nk, kv, size), dtype, 2)
    v, vv = values((nk, kv, size), dtype, 3)
    w, wv = values((nq, heads, size), dtype, 4)
    for t in (q, k, v):
        t.requiresGrad()
    o = q.attention(k, v, causal=causal)
    assert o.getDtype() == dtype and o.getShape() == [nq, heads, size]
    o.backward(w)
    check(qv, kvv, vv, causal, dtype, [(0, nq, 0, nk)], o, wv, grads=[q.grad(), k.grad(), v.grad()])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [64, 24, 128])
def test_batch_of_one_length(dtype, size):
    """[sequences, tokens, heads, size], also as views of [sequences, heads, tokens, size]."""
    b, nq, nk, heads, kv = 3, 70, 90, 4, 2
    q, qv = values((b, nq, heads, size), dtype, 1)
    k, kvv = values((b, nk, kv, size), dtype, 2)
    v, vv = values((b, nk, kv, size), dtype, 3)
    w, wv = values((b, nq, heads, size), dtype, 4)

    def rows(x):
        return x.reshape((-1,) + x.shape[2:])
    spans = [(i * nq, nq, i * nk, nk) for i in range(b)]
    for t in (q, k, v):
        t.requiresGrad()
    o = q.attention(k, v, causal=True)
    o.backward(w)
    check(rows(qv), rows(kvv), rows(vv), True, dtype, spans, o, rows(wv), grads=[t.grad() for t in (q, k, v)])
    # the same values with the heads before the tokens in memory
    views = []
    for x in (q, k, v):
        bits = np.ascontiguousarray(x.toBits().swapaxes(1, 2))
        views.append(CudaArray.fromBuffer(bits.tobytes(), list(bits.shape), dtype).swapaxes(1, 2))
    o2 = views[0].attention(views[1], views[2], causal=True)
    assert np.array_equal(o2.toBits(), o.toBits())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_packed_sequences(dtype, causal):
    """Prompts behind each other, an empty one among them, and rows of no sequence at the end."""
    lengths = [5, 0, 130, 1, 64]
    heads, kv, size, spare = 4, 2, 64, 7
    rows = sum(lengths) + spare
    q, qv = values((rows, heads, size), dtype, 1)
    k, kvv = values((rows, kv, size), dtype, 2)
    v, vv = values((rows, kv, size), dtype, 3)
    w, wv = values((rows, heads, size), dtype, 4)
    at = np.cumsum([0] + lengths)
    spans = [(int(a), n, int(a), n) for a, n in zip(at, lengths)]
    for t in (q, k, v):
        t.requiresGrad()
    o = q.attention(k, v, causal=causal, queries=Sequences(lengths))
    o.backward(w)
    check(qv, kvv, vv, causal, dtype, spans, o, wv, grads=[t.grad() for t in (q, k, v)])
    for t in (o, q.grad(), k.grad(), v.grad()):
        assert not t.toNumpy()[-spare:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 3])
def test_cache_slots(dtype, new):
    """New tokens of several requests against slots of a cache; what lies behind a slot's tokens is NaN."""
    slots, size, heads, kv = 700, 64, 8, 2
    kept = [1, 700, 0, 333, 64, 513]
    starts = [i * slots for i in (2, 0, 5, 1, 4, 3)]
    queries, keys = Sequences([new] * 6), Sequences(kept, starts)
    q, qv = values((6 * new, heads, size), dtype, 1)
    fill = np.full((6 * slots, kv, size), np.nan, np.float32)
    for n, s in zip(kept, starts):
        fill[s:s + n] = np.random.default_rng(s).standard_normal((n, kv, size))
    k, v = CudaArray.fromNumpy(fill, dtype), CudaArray.fromNumpy(fill[:, :, ::-1].copy(), dtype)
    o = q.attention(k, v, causal=True, queries=queries, keys=keys)
    kvv, vv = (t.toNumpy().astype(np.float64) for t in (k, v))
    check(qv, kvv, vv, True, dtype, [(i * new, new, s, n) for i, (n, s) in enumerate(zip(kept, starts))], o)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_cache_is_split(dtype):
    """One token against a long cache: the keys are split between workgroups."""
    n, heads, kv, size = 20000, 4, 2, 64
    q, qv = values((1, heads, size), dtype, 1, 2.0)
    k, kvv = values((n, kv, size), dtype, 2)
    v, vv = values((n, kv, size), dtype, 3)
    check(qv, kvv, vv, True, dtype, [(0, 1, 0, n)], q.attention(k, v, causal=True))


def test_shared_prefix():
    """Sequences of keys may share rows in the forward pass; their gradient is refused."""
    q, qv = values((4, 2, 32), "float32", 1)
    k, kvv = values((50, 2, 32), "float32", 2)
    v, vv = values((50, 2, 32), "float32", 3)
    queries, keys = Sequences([2, 2]), Sequences([40, 50], [0, 0])
    o = q.requiresGrad().attention(k, v, queries=queries, keys=keys)
    check(qv, kvv, vv, False, "float32", [(0, 2, 0, 40), (2, 2, 0, 50)], o)
    with pytest.raises(_abi.InvalidArgumentException):
        o.backward(o.detach())


def test_large_scores_and_scale():
    """Rows whose scores differ by hundreds: one key takes all the weight, and nothing overflows."""
    q, qv = values((70, 2, 64), "float32", 1, 30.0)
    k, kvv = values((90, 2, 64), "float32", 2, 5.0)
    v, vv = values((90, 2, 64), "float32", 3)
    check(qv, kvv, vv, False, "float32", [(0, 70, 0, 90)], q.attention(k, v, scale=0.7), scale=float(np.float32(0.7)))


def test_infinite_scores_of_hidden_keys():
    """Keys that a query does not see may hold anything finite or not in the scores' product."""
    q, _ = values((40, 1, 64), "float32", 1)
    kept = np.random.default_rng(2).standard_normal((40, 1, 64)).astype(np.float32)
    v, _ = values((40, 1, 64), "float32", 3)
    clean = q.attention(CudaArray.fromNumpy(kept), v, causal=True).toNumpy()
    for bad in (np.inf, np.nan, -np.inf):
        k = kept.copy()
        k[39] = bad
        got = q.attention(CudaArray.fromNumpy(k), v, causal=True).toNumpy()
        assert np.array_equal(got[:39], clean[:39])


def test_gradient_against_differences():
    q, qv = values((6, 2, 5), "float32", 1)
    k, kvv = values((8, 1, 5), "float32", 2)
    v, vv = values((8, 1, 5), "float32", 3)
    w, wv = values((6, 2, 5), "float32", 4)
    for t in (q, k, v):
        t.requiresGrad()
    q.attention(k, v, causal=True).backward(w)

    def loss(a, b, c):
        return float((R.attention(a, b, c, True, 1 / math.sqrt(5), "float32", [(0, 6, 0, 8)])["o"][0] * wv).sum())
    base = [qv, kvv, vv]
    for n, t in enumerate((q, k, v)):
        g = t.grad().toNumpy()
        for at in [(0, 0, 0), (3, 0, 2), (5, 0, 4)]:
            step = 1e-5
            up, down = [x.copy() for x in base], [x.copy() for x in base]
            up[n][at] += step
            down[n][at] -= step
            # the difference quotient is off by step^2 times a third derivative of order 1
            assert abs((loss(*up) - loss(*down)) / (2 * step) - g[at]) < 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_compiled_plan(dtype):
    """Forward and backward inside Fusion.compile, replayed on other inputs, give the eager results."""
    heads, kv, size = 4, 2, 64
    seqs = Sequences([30, 66])

    def step(q, k, v, w):
        q, k, v = q.detach(), k.detach(), v.detach()
        for t in (q, k, v):
            t.requiresGrad()
        o = q.attention(k, v, causal=True, queries=seqs)
        o.backward(w)
        return [o, q.grad(), k.grad(), v.grad()]

    def inputs(seed):
        return [values((96, n, size), dtype, seed + i)[0] for i, n in enumerate((heads, kv, kv, heads))]
    plans = [Fusion.compile(step, inputs(1), cudaGraph=graph) for graph in (True, False)]
    for seed in (10, 20, 30, 10):
        ins = inputs(seed)
        want = [t.toBits() for t in step(*ins)]
        for plan in plans:
            got = plan.run(*ins)
            assert all(np.array_equal(a, b.toBits()) for a, b in zip(want, got))


def test_strided_views_of_one_projection():
    """q, k and v as slices of one product's result, read in place."""
    t, heads, size = 50, 3, 32
    x, xv = values((t, 3 * heads, size), "bfloat16", 1)
    q, k, v = (x.slice(None, [i * heads, (i + 1) * heads]) for i in range(3))
    o = q.attention(k, v)
    xs = [xv[:, i * heads:(i + 1) * heads] for i in range(3)]
    check(*xs, False, "bfloat16", [(0, t, 0, t)], o)
    # a view that starts inside a 16-byte pack, and one whose elements are not side by side
    y, yv = values((t, heads, size + 3), "bfloat16", 2)
    o = y.slice(None, None, [3, size + 3]).attention(k, v)
    check(yv[:, :, 3:], xs[1], xs[2], False, "bfloat16", [(0, t, 0, t)], o)
    z, zv = values((t, size, heads), "bfloat16", 3)
    o = z.swapaxes(1, 2).attention(k, v)
    check(zv.swapaxes(1, 2), xs[1], xs[2], False, "bfloat16", [(0, t, 0, t)], o)


def test_no_tokens():
    q, k = CudaArray.zeros([0, 2, 16]), CudaArray.zeros([5, 2, 16])
    assert q.attention(k, k).getShape() == [0, 2, 16]
    q = values((4, 2, 16), "float32", 1)[0].requiresGrad()
    none = CudaArray.zeros([0, 2, 16])
    o = q.attention(none, none)
    o.backward(CudaArray.ones([4, 2, 16]))
    assert not o.toNumpy().any() and not q.grad().toNumpy().any()


def test_refusals():
    a, b = CudaArray.zeros([4, 4, 16]), CudaArray.zeros([6, 2, 16])
    bad = _abi.InvalidArgumentException
    two = Sequences([2, 2])
    for call in [
            lambda: a.attention(b, CudaArray.zeros([5, 2, 16])),                    # values of another shape
            lambda: a.attention(CudaArray.zeros([6, 3, 16]), CudaArray.zeros([6, 3, 16])),  # 3 does not divide 4
            lambda: a.attention(CudaArray.zeros([6, 2, 8]), CudaArray.zeros([6, 2, 8])),
            lambda: a.attention(b.astype("float64"), b.astype("float64")),
            lambda: CudaArray.zeros([4, 16]).attention(CudaArray.zeros([4, 16]), CudaArray.zeros([4, 16])),
            lambda: CudaArray.zeros([2, 2, 257]).attention(*[CudaArray.zeros([2, 2, 257])] * 2),
            lambda: a.attention(b, b, scale=0.0), lambda: a.attention(b, b, scale=-1.0),
            lambda: a.attention(b, b, scale=float("nan")), lambda: a.attention(b, b, scale=float("inf")),
            lambda: a.attention(b, b, queries=two, keys=Sequences([6])),            # another count
            lambda: a.attention(b, b, queries=Sequences([2, 3])),                   # past the tokens
            lambda: a.attention(b, b, queries=Sequences([3, 2], [0, 2]), keys=two),  # shared query rows
            lambda: a.attention(b, b, keys=two), lambda: a.attention(b, 3),
            lambda: a.attention(b, b, queries=[2, 2]),
            lambda: Sequences([]), lambda: Sequences([-1]), lambda: Sequences([1], [-1]),
            lambda: Sequences([1, 2], [0]), lambda: Sequences([2 ** 31 - 1, 5]),
    ]:
        with pytest.raises(bad):
            call()
    four = CudaArray.zeros([1, 4, 4, 16])
    with pytest.raises(bad):
        four.attention(four, four, queries=Sequences([4]))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("size", [64, 20])
def test_float32_upstream_gradient(dtype, size):
    """16-bit operands, the upstream gradient in float32: rounded once to the operands' type.  Also without what the
    forward pass kept of the output's rounding, which the bounds allow for."""
    lengths, starts, rows, heads, kv = [40, 0, 33], [2, 45, 50], 90, 4, 2
    q, qv = values((rows, heads, size), dtype, 1)
    k, kvv = values((rows, kv, size), dtype, 2)
    v, vv = values((rows, kv, size), dtype, 3)
    w, w32 = values((rows, heads, size), "float32", 4)
    wv = CudaArray.fromNumpy(w32.astype(np.float32), dtype).toNumpy().astype(np.float64).reshape(w32.shape)
    seqs = Sequences(lengths, starts)
    spans = [(a, n, a, n) for a, n in zip(starts, lengths)]
    lib = _host.load()
    kept = (ctypes.c_void_p * 2)()
    out = CudaArray._wrap(lib.phpt_attention(q._h, k._h, v._h, 1, 0.0, seqs._h, seqs._h, kept))
    lse, rest = (CudaArray._wrap(h) for h in kept)
    assert rest.getDtype() == dtype
    for given in (rest._h, None):
        got = (ctypes.c_void_p * 3)()
        assert not lib.phpt_attention_backward(q._h, k._h, v._h, out._h, lse._h, given, w._h, 1, 0.0, seqs._h, seqs._h, got)
        check(qv, kvv, vv, True, dtype, spans, out, wv, grads=[CudaArray._wrap(h) for h in got])


def test_bounds_past_the_tensors():
    """pt_attention's `queries` and `keys` are bounds: larger ones than the tensors hold give the same results."""
    lib = _abi.load()
    heads, kv, size, rows = 4, 2, 64, 300
    arrays = [np.random.default_rng(i).standard_normal((rows, n, size)).astype(np.float32) for i, n in enumerate((heads, kv, kv, heads))]
    dev = [_abi.to_device(a) for a in arrays]
    seq = [_abi.to_device(np.array(a, np.int32)) for a in ([0, 130], [130, 170])]
    names = [("out", arrays[0]), ("lse", np.zeros((heads, rows), np.float32)), ("dq", arrays[0]), ("dk", arrays[1]), ("dv", arrays[1])]
    bits = []
    for most in (170, 300, 100000):
        d = _abi.PtAttentionDesc()
        for n, h in (("q", heads), ("k", kv), ("v", kv)):
            setattr(d, n + "_strides", (ctypes.c_size_t * 3)(0, h * size, size))
        for n, x in dict(dtype=_abi.FLOAT32, sequences=2, heads=heads, kv_heads=kv, head_size=size, queries=most, keys=most,
                         q_starts=seq[0].ptr, q_lengths=seq[1].ptr, k_starts=seq[0].ptr, k_lengths=seq[1].ptr, q_rows=rows,
                         k_rows=rows, causal=1, scale=0.125).items():
            setattr(d, n, x)
        to = {n: _abi.to_device(np.zeros_like(a)) for n, a in names}
        p = {n: t.ptr for n, t in to.items()}
        _abi.check(lib.pt_attention(ctypes.byref(d), *(a.ptr for a in dev[:3]), p["out"], p["lse"], None, None))
        _abi.check(lib.pt_attention_backward(ctypes.byref(d), *(a.ptr for a in dev[:3]), p["out"], p["lse"], None, dev[3].ptr,
                                             _abi.FLOAT32, p["dq"], p["dk"], p["dv"], None))
        _abi.synchronize()
        bits.append([to[n].download(np.uint32, a.shape) for n, a in names])
    spans = [(0, 130, 0, 130), (130, 170, 130, 170)]
    x = [a.astype(np.float64) for a in arrays]
    ref = R.attention(*x[:3], True, 0.125, "float32", spans, x[3])
    for got in bits:   # (another bound may split the work otherwise: the same within the bounds, not always bit for bit)
        for (n, a), b in zip(names, got):
            want, off = (x.reshape(a.shape) if n != "lse" else x.T for x in ref["o" if n == "out" else n])
            assert (np.abs(b.view(np.float32).astype(np.float64) - want) <= off).all(), n
    assert all(np.array_equal(a, b) for a, b in zip(bits[1], bits[2]))
