"""Gradients of CudaArray.layerNorm against float64, within bounds that count
the roundings (u: half a step of float32, h: of the result's type)."""
import numpy as np
import pytest

from phptensors import CudaArray, Fusion, _abi

pytestmark = pytest.mark.gpu
HALF = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
# the smallest step of fp16 rounds absolutely
TINY = {"float64": 0.0, "float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}


def values(shape, dtype, seed, scale=1.0, shift=0.0):
    x = (np.random.default_rng(seed).standard_normal(shape) * scale + shift).astype(
        np.float64 if dtype == "float64" else np.float32)
    a = CudaArray.fromNumpy(x, dtype)
    return a, a.toNumpy().astype(np.float64).reshape(shape)


def reference(x, g, gamma, eps, u):
    """{name: (value, bound before its rounding to the result's type)} of rows x."""
    n, rows = x.shape[1], x.shape[0]
    m = x.mean(1, keepdims=True)
    d = x - m
    d_off = u * np.abs(x) + (n + 3) * u * np.abs(x).mean(1, keepdims=True) + u * np.abs(d)
    q = (d * d).mean(1, keepdims=True) + eps
    r = 1 / np.sqrt(q)
    r_rel = (np.abs(d) * d_off + d_off * d_off).mean(1, keepdims=True) / q + (n + 8) * u
    xn, xn_off = d * r, (np.abs(d) * r_rel + d_off) * r * (1 + r_rel)
    h = g * gamma
    h1, h1_off = h.mean(1, keepdims=True), (n + 4) * u * np.abs(h).mean(1, keepdims=True)
    h2 = (h * xn).mean(1, keepdims=True)
    h2_off = (np.abs(h) * xn_off).mean(1, keepdims=True) + (n + 8) * u * np.abs(h * xn).mean(1, keepdims=True)
    inner = h - h1 - xn * h2
    off = (h1_off + np.abs(xn) * h2_off + xn_off * (np.abs(h2) + h2_off)
           + 4 * u * (np.abs(h) + np.abs(h1) + np.abs(xn * h2)))
    return {"dx": (r * inner, r * (1 + r_rel) * (off + r_rel * np.abs(inner))),
            "dgamma": ((g * xn).sum(0), (np.abs(g) * xn_off).sum(0) + (rows + 8) * u * np.abs(g * xn).sum(0)),
            "dbeta": (g.sum(0), (rows + 8) * u * np.abs(g).sum(0))}


def close(got, want, what):
    h, tiny = HALF[got.getDtype()], TINY[got.getDtype()]
    x, off = want
    v = got.toNumpy().astype(np.float64).reshape(x.shape)
    far = np.abs(v - x) - (off + h * (np.abs(x) + off) + tiny)
    assert far.size == 0 or (not np.isnan(v).any() and far.max() <= 0), (what, float(far.max()))


# widths on both sides of each kernel's range, one element, odd ones, the general kernel's
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (1, 8), (5, 9), (37, 64), (700, 100), (4, 511), (9, 512), (130, 513),
                                    (64, 1024), (33, 1025), (20, 2048), (11, 2049), (600, 4096), (7, 4097), (5, 8192),
                                    (3, 8193), (2, 16384), (2, 16385), (1, 40001), (5000, 16), (600, 5003), (300, 16000)])
def test_gradients(rows, n, dtype):
    x, xv = values((rows, n), dtype, 1, 2.0, 0.5)
    scale, sv = values((n,), dtype, 2, 0.2, 1.0)
    bias, _ = values((n,), dtype, 3)
    g, gv = values((rows, n), "float32", 4)
    for t in (x, scale, bias):
        t.requiresGrad()
    y = x.layerNorm([1], 1e-5, scale, bias)
    y.backward(g)
    ref = reference(xv, gv, sv, 1e-5, HALF["float32"])
    for t, name in ((x, "dx"), (scale, "dgamma"), (bias, "dbeta")):
        assert t.grad().getDtype() == t.getDtype() and t.grad().getShape() == t.getShape()
        close(t.grad(), ref[name], name)


@pytest.mark.parametrize("n", [5, 300, 20000])
@pytest.mark.parametrize("scale_dtype,dtype", [("float64", "float64"), ("float64", "float32"), ("float64", "bfloat16")])
def test_float64(dtype, scale_dtype, n):
    x, xv = values((13, n), dtype, 1)
    scale, sv = values((n,), scale_dtype, 2, 0.2, 1.0)
    bias, _ = values((n,), scale_dtype, 3)
    g, gv = values((13, n), "float64", 4)
    for t in (x, scale, bias):
        t.requiresGrad()
    x.layerNorm([1], 1e-5, scale, bias).backward(g)
    ref = reference(xv, gv, sv, 1e-5, HALF["float64"])
    for t, name in ((x, "dx"), (scale, "dgamma"), (bias, "dbeta")):
        assert t.grad().getDtype() == t.getDtype()
        close(t.grad(), ref[name], name)


def test_mixed_parameter_dtypes_and_missing_ones():
    x, xv = values((40, 96), "bfloat16", 1)
    scale, sv = values((96,), "bfloat16", 2, 0.2, 1.0)
    bias, _ = values((96,), "float32", 3)
    g, gv = values((40, 96), "float32", 4)
    ref, plain = reference(xv, gv, sv, 1e-5, 2.0 ** -24), reference(xv, gv, np.ones(96), 1e-5, 2.0 ** -24)
    for t in (x, scale, bias):
        t.requiresGrad()
    x.layerNorm([1], 1e-5, scale, bias).backward(g)
    for t, name in ((x, "dx"), (scale, "dgamma"), (bias, "dbeta")):
        assert t.grad().getDtype() == t.getDtype()
        close(t.grad(), ref[name], name)
        t.zeroGrad()
    x.layerNorm([1]).backward(g)
    close(x.grad(), plain["dx"], "dx")
    x.zeroGrad()
    x.layerNorm([1], 1e-5, None, bias).backward(g)
    close(x.grad(), plain["dx"], "dx")
    close(bias.grad(), plain["dbeta"], "dbeta")
    # whole numbers have no gradient, their parameters do
    whole = CudaArray.fromNumpy(np.arange(12, dtype=np.int32).reshape(3, 4))
    s = CudaArray.ones([4], "float64").requiresGrad()
    whole.layerNorm([1], 1e-5, s).backward(CudaArray.ones([3, 4], "float64"))
    want = reference(np.arange(12.0).reshape(3, 4), np.ones((3, 4)), np.ones(4), 1e-5, 2.0 ** -53)
    close(s.grad(), want["dgamma"], "dgamma")


@pytest.mark.parametrize("axes", [[0], [0, 2], [2, 0], [1, 2], [-1, 1, 0]])
def test_other_axes(axes):
    """Normalized axes anywhere and in any order: the parameters' dimensions follow the list."""
    shape = (4, 5, 6)
    x, xv = values(shape, "float32", 1)
    pshape = tuple(shape[a] for a in axes)
    scale, sv = values(pshape, "float32", 2, 0.2, 1.0)
    bias, _ = values(pshape, "float32", 3)
    g, gv = values(shape, "float32", 4)
    for t in (x, scale, bias):
        t.requiresGrad()
    x.layerNorm(axes, 1e-5, scale, bias).backward(g)
    ax = [a % 3 for a in axes]
    last = sorted(ax)
    perm = [d for d in range(3) if d not in ax] + last
    n = int(np.prod([shape[a] for a in ax]))
    order = [ax.index(a) for a in last]  # parameter dimensions in ascending order of the axes
    ref = reference(xv.transpose(perm).reshape(-1, n), gv.transpose(perm).reshape(-1, n),
                    sv.transpose(order).reshape(-1), 1e-5, 2.0 ** -24)

    def back(v, dims, p):
        return v.reshape([dims[i] for i in p]).transpose(np.argsort(p))
    close(x.grad(), [back(v, shape, perm) for v in ref["dx"]], "dx")
    close(scale.grad(), [back(v, pshape, order) for v in ref["dgamma"]], "dgamma")
    close(bias.grad(), [back(v, pshape, order) for v in ref["dbeta"]], "dbeta")


def test_strided_input_and_row_values():
    x, xv = values((60, 50), "float32", 1, 1.0, 1000.0)  # a mean far from zero
    g, gv = values((50, 60), "float32", 4)
    x.requiresGrad()
    x.T.layerNorm([1]).backward(g)
    ref = reference(xv.T, gv, np.ones(60), 1e-5, 2.0 ** -24)["dx"]
    close(x.grad(), [v.T for v in ref], "dx")
    # equal elements: the variance is 0 and eps alone holds the division
    c = CudaArray.full([3, 40], 2.5).requiresGrad()
    c.layerNorm([1]).backward(CudaArray.fromNumpy(gv[:3, :40].astype(np.float32)))
    close(c.grad(), reference(np.full((3, 40), 2.5), gv[:3, :40], np.ones(40), 1e-5, 2.0 ** -24)["dx"], "dx")


def test_no_rows_and_determinism():
    scale = CudaArray.ones([32]).requiresGrad()
    x = CudaArray.zeros([0, 32]).requiresGrad()
    x.layerNorm([1], 1e-5, scale).backward(CudaArray.zeros([0, 32]))
    assert x.grad().getShape() == [0, 32] and not scale.grad().toNumpy().any()
    x, _ = values((3000, 700), "float32", 1)
    g, _ = values((3000, 700), "float32", 2)
    seen = []
    for _ in range(3):
        s = CudaArray.ones([700]).requiresGrad()
        x.layerNorm([1], 1e-5, s).backward(g)
        seen.append(s.grad().toBits())
    assert np.array_equal(seen[0], seen[1]) and np.array_equal(seen[0], seen[2])


def test_compiled_plan():
    def step(x, scale, bias, g):
        x, scale, bias = x.detach(), scale.detach(), bias.detach()
        for t in (x, scale, bias):
            t.requiresGrad()
        y = x.layerNorm([1], 1e-5, scale, bias)
        (y * g).sum().backward()
        return [y.detach(), x.grad(), scale.grad(), bias.grad()]

    def inputs(seed):
        return [values(s, "float32", seed + i)[0] for i, s in enumerate(((48, 300), (300,), (300,), (48, 300)))]
    for graph in (True, False):
        plan = Fusion.compile(step, inputs(1), cudaGraph=graph)
        for seed in (10, 20, 30, 10):
            ins = inputs(seed)
            assert all(np.array_equal(a.toBits(), b.toBits()) for a, b in zip(step(*ins), plan.run(*ins)))


def test_refusals():
    lib = _abi.load()
    x = _abi.to_device(np.zeros(64, np.float32))

    def call(dt=0, ct=0, rows=4, n=16, eps=1e-5, pdt=0, inp=x.ptr):
        return lib.pt_layernorm_backward(inp, x.ptr, dt, ct, rows, n, eps, None, pdt, x.ptr, None, None, None)
    for bad in (dict(eps=0.0), dict(eps=float("nan")), dict(ct=11), dict(dt=4), dict(dt=1), dict(pdt=12), dict(n=0),
                dict(ct=1, dt=12, pdt=1), dict(n=2 ** 31), dict(inp=None)):
        assert call(**bad) == _abi.PT_ERR_INVALID, bad
    assert call() == _abi.PT_OK
