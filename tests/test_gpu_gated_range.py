"""CudaArray.gatedProjection and its gradients where values are small: the activations and their slopes relative to
themselves, element by element.  U: half a step of float32, HALF: of the operands' type."""
import math

import numpy as np
import pytest

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
