"""CudaArray.gatedProjection and its gradients where values are small or large: the activations and their slopes relative
to themselves, element by element, and float16 gradients whose inner values leave float16's range.  U: half a step of
float32, HALF: of the operands' type."""
import math

import numpy as np
import pytest

import test_gpu_gated
from phptensors import CudaArray

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "float16", "bfloat16"]
U = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}


def within(got, want, off, dtype, what):
    """off: the bound before the result's own rounding."""
    y = got.toNumpy().astype(np.float64).reshape(want.shape)
    far = np.abs(y - want) - (off * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want) + TINY[dtype])
    far = np.where(np.isnan(far), np.inf, far)
    at = np.unravel_index(far.argmax(), far.shape)
    assert far.max() <= 0, (what, at, y[at], want[at])


def below(g):
    """The standard normal's distribution, by the tail that keeps its digits."""
    return np.vectorize(lambda v: 0.5 * math.erfc(-v / math.sqrt(2)), otypes=[float])(g)


def activation(name, g):
    """{value, slope: (exact, bound)}.  exp takes its argument with one rounding more (U |g| of the result) and is off by
    2 U at most, as the reciprocal or the division is; with the sum before it and the product behind it a sigmoid is within
    (8 + 2 |g|) U of itself.  erfc's argument and the bell's exponent are off by 2 U of themselves, which their slopes make
    2 g^2 U and g^2 U of the results, and both are within 16 U besides (a fit of 3.2 U and its ten operations, or the
    library's).  Sums of terms of both signs are within their terms' magnitudes.  Sigmoids and bells below the least normal
    float32 may be zeros."""
    a = np.abs(g)
    none = a * 2.0 ** -126
    if name == "relu":
        return {"value": (np.maximum(g, 0.0), 0 * g), "slope": ((g > 0).astype(float), 0 * g)}
    if name == "gelu":
        part, bell = below(g), np.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        rel = (24 + 4 * g * g) * U
        return {"value": (g * part, rel * np.abs(g * part) + none),
                "slope": (part + g * bell, rel * (part + a * bell) + none + 2.0 ** -126)}
    with np.errstate(over="ignore"):
        s, t = 1 / (1 + np.exp(-g)), 1 / (1 + np.exp(g))
    rel = (12 + 3 * a) * U
    if name == "sigmoid":
        return {"value": (s, rel * s + 2.0 ** -126), "slope": (s * t, 2 * rel * s * t + 2.0 ** -126)}
    # (1 - s by subtraction: off by U of 1)
    return {"value": (g * s, rel * np.abs(g * s) + none),
            "slope": (s * (1 + g * t), 2 * rel * s * (1 + a * t) + 4 * U * a * s + none + 2.0 ** -126)}


def unit(m, f, dtype, sizes):
    """Products of one term each: x is the unit matrix, so both products are the weights and the weights' gradients are
    the gradients of both products, each element by itself.  Returns arrays and float64 values."""
    rng = np.random.default_rng(7)
    g = sizes(rng, (m, f))
    u = 0.5 + rng.random((m, f))
    made = [CudaArray.fromNumpy(np.asarray(v, np.float32), dtype).requiresGrad() for v in (np.eye(m), g, u)]
    return made, [t.toNumpy().astype(np.float64).reshape(s) for t, s in zip(made, [(m, m), (m, f), (m, f)])]


# few rows, and more, which take other kernels
@pytest.mark.parametrize("rows", [24, 200])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["silu", "gelu", "relu", "sigmoid"])
def test_activations_keep_their_digits(name, dtype, rows):
    def sizes(rng, shape):
        return rng.uniform(-14, 14, shape)
    (x, gate, up), (_, g, u) = unit(rows, 40, dtype, sizes)
    h = x.gatedProjection(gate, up, name)
    h.backward(CudaArray.ones([rows, 40], dtype))
    (v, v_off), (s, s_off) = activation(name, g).values()
    # (the products are values of the operands' type, which the 24 bits that the gradient keeps of them hold)
    within(h, v * u, (v_off + U * np.abs(v)) * u, dtype, "h")
    for got, (want, off) in ((gate, (s * u, (s_off + 2 * U * np.abs(s)) * u)), (up, (v, v_off + U * np.abs(v)))):
        # dg and du are rounded to the type once, and the sum of that one term again, which leaves it
        within(got.grad(), want, off, dtype, "gradient")


# ------------------------------------------- float16: gradients of both products past float16's range
# The gradients are linear in the upstream one, so rows (and columns) of that which are scaled by powers of two scale the
# exact rows of dx (columns of dgate and dup) and all of their bounds, those of test_gpu_gated.reference for upstream
# gradients of order 1.  Its 2^-25 for each of dg and du stays far above what they are held with: 2^-39 of their row's or
# column's largest, which is below 2^7 here.
# rows, inner, outer: few and more, odd widths, several chunks of columns, split contractions of both, tall and narrow
RANGED = [(24, 64, 40), (300, 40, 77), (5, 48, 1203), (24, 64, 8000), (2100, 40, 24), (70001, 8, 9), (1, 9, 3)]


def ranged(shape, x_scale=1.0, w_scale=1.0, up_scale=1.0):
    """(arrays, float64 values) of x, gate and up in float16, and upstream values of order 1."""
    m, k, f = shape
    rng = np.random.default_rng(11)
    made = [CudaArray.fromNumpy((rng.standard_normal(s) * c).astype(np.float32), "float16").requiresGrad()
            for s, c in (((m, k), x_scale), ((k, f), w_scale * k ** -0.5), ((k, f), w_scale * up_scale * k ** -0.5))]
    return made, [t.toNumpy().astype(np.float64).reshape(t.getShape()) for t in made], \
        rng.standard_normal((m, f)).astype(np.float32).astype(np.float64)


def gradients(made, dh, dtype="float32"):
    for t in made:
        t.zeroGrad()
    h = made[0].gatedProjection(made[1], made[2], "silu")
    g = CudaArray.fromNumpy(np.asarray(dh, np.float32), dtype)
    if dtype == "float16":
        h.backward(g)
    else:
        (h * g).sum().backward()
    return [t.grad() for t in made]


def ranged_close(got, want, scales, what):
    for t, n, c in zip(got, ("dx", "dgate", "dup"), scales):
        if c is not None:
            assert t.getDtype() == "float16"
            within(t, want[n][0] * c, want[n][1] * c, "float16", (what, n))


# (past 65504 only the results that float16 holds)
@pytest.mark.parametrize("power,x_scale,wanted", [(-27, 2.0 ** 9, (1, 1, 1)), (-27, 2.0 ** -12, (1, 1, 1)), (-40, 2.0 ** 12, (1, 1, 1)),
                                                  (15, 2.0 ** -9, (0, 1, 1)), (15, 2.0 ** 9, (1, 0, 0))])
@pytest.mark.parametrize("shape", RANGED, ids=str)
def test_float16_upstream_gradients_of_any_size(shape, power, x_scale, wanted):
    made, values, dh = ranged(shape, x_scale, 1 / x_scale)
    got = gradients(made, dh * 2.0 ** power)
    want = test_gpu_gated.reference(*values, "silu", "float16", dh)
    ranged_close(got, want, [2.0 ** power if w else None for w in wanted], "scaled")


@pytest.mark.parametrize("shape", RANGED, ids=str)
def test_float16_rows_and_columns_of_their_own_size(shape):
    """Small rows keep dx, and small columns dgate and dup, beside large ones; some have no gradient at all."""
    m, _, f = shape
    rng = np.random.default_rng(12)
    for axis, n, x_scale in ((0, m, 2.0 ** -8), (1, f, 2.0 ** 3)):
        made, values, dh = ranged(shape, x_scale, 1 / x_scale)
        c = 2.0 ** rng.integers(-24, 2, n).astype(np.float64)
        c[rng.random(n) < 0.1] = 0.0
        c = c[:, None] if axis == 0 else c[None, :]
        got = gradients(made, dh * c)
        want = test_gpu_gated.reference(*values, "silu", "float16", dh)
        ranged_close(got, want, (c, None, None) if axis == 0 else (None, c, c), axis)
        # each gradient alone is what it is among all
        for i, t in enumerate(made):
            for o in made:
                o.requiresGrad(o is t)
            alone = gradients(made, dh * c)[i]
            assert np.array_equal(alone.toBits(), got[i].toBits())
        for o in made:
            o.requiresGrad()


@pytest.mark.parametrize("shape", RANGED[:5], ids=str)
@pytest.mark.parametrize("value", [np.inf, np.nan, 1e30, -3e38])
def test_one_float16_outlier_stays_in_its_row_and_column(shape, value):
    m, _, f = shape
    made, values, dh = ranged(shape)
    want = test_gpu_gated.reference(*values, "silu", "float16", dh)
    row, column = m // 2, f - 2
    dh[row, column] = value
    dx, *dw = gradients(made, dh)
    rows, columns = np.arange(m) != row, np.arange(f) != column
    for t, n, keep in ((dx, "dx", np.s_[rows]), (dw[0], "dgate", np.s_[:, columns]), (dw[1], "dup", np.s_[:, columns])):
        v = t.toNumpy().reshape(t.getShape()).astype(np.float32)
        if v[keep].size:
            within(CudaArray.fromNumpy(np.ascontiguousarray(v[keep]), "float16"), want[n][0][keep], want[n][1][keep], "float16", n)
        # (a float32 product with 3e38 may end before infinity, its share of a float16 result does not)
        assert not np.isfinite(v[~rows] if n == "dx" else v[:, ~columns]).any()


def test_float16_products_of_large_values():
    """dg past 65504 from float16 operands and upstream gradients, dx and dgate within it."""
    for shape in ((24, 64, 16), (300, 64, 16)):
        made, values, dh = ranged(shape, 2.0 ** -6, 2.0 ** -3, 2.0 ** 14)
        dh = (dh * 2.0 ** 11).astype(np.float16).astype(np.float64)
        want = test_gpu_gated.reference(*values, "silu", "float16", dh)
        x, gate, up = values
        g, u = x @ gate, x @ up
        assert (np.abs(dh * u) * 0.5).max() > 70000 and max(np.abs(want[n][0]).max() for n in ("dx", "dgate", "dup")) < 60000
        ranged_close(gradients(made, dh, "float16"), want, (1, 1, 1), shape)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_upstream_gradient(dtype):
    for m in (3, 100):
        x, a, b = (CudaArray.ones(s, dtype).requiresGrad() for s in ((m, 24), (24, 33), (24, 33)))
        x.gatedProjection(a, b).backward(CudaArray.zeros([m, 33], dtype))
        assert not any(t.grad().toNumpy().any() for t in (x, a, b))
