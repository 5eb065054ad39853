"""16-bit gradients of one tensor add up in float32, over its uses and over backward calls, and are rounded once."""
import numpy as np
import pytest

import attention_ref as R
from phptensors import CudaArray, Fusion

pytestmark = pytest.mark.gpu


def made(shape, seed, dtype, scale=1.0):
    x = np.random.default_rng(seed).standard_normal(shape).astype(np.float32) * np.float32(scale)
    return CudaArray.fromNumpy(x, dtype)


def once_rounded(got, total, size, additions, dtype):
    """`additions` roundings to float32 of sums no larger than `size`, and one to the type."""
    assert got.getDtype() == dtype
    off = additions * R.U * size
    assert (np.abs(got.toNumpy().astype(np.float64) - total) <= off + R.H[dtype] * (np.abs(total) + off) + R.TINY[dtype]).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_several_uses(dtype):
    x, w = made((40, 3, 16), 1, dtype), made((40, 3, 16), 2, dtype)

    def apart(x, w):
        a, b, c = (x.detach().requiresGrad() for _ in range(3))
        a.attention(b, c, causal=True).backward(w)
        return [t.grad().toNumpy().astype(np.float64) for t in (a, b, c)]

    def together(x, w):
        one = x.detach().requiresGrad()
        one.attention(one, one, causal=True).backward(w)
        return one.grad()
    each = apart(x, w)
    total, size = sum(each), sum(np.abs(t) for t in each)
    once_rounded(together(x, w), total, size, 2, dtype)
    once_rounded(Fusion.compile(together, [x, w]).run(x, w), total, size, 2, dtype)
    kept = []
    Fusion.run(lambda: kept.append(together(x, w)) or kept[0])
    once_rounded(kept[0], total, size, 2, dtype)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_many_backward_calls(dtype):
    """Sums of bfloat16 would stay where they are once they are 256 times what is added."""
    n = 700
    q, k = made((20, 2, 16), 1, dtype).requiresGrad(), made((20, 2, 16), 2, dtype)
    w = made((20, 2, 16), 3, dtype, 2.0 ** -4)
    q.attention(k, k).backward(w)
    first = q.grad().toNumpy().astype(np.float64)
    for i in range(1, n):
        q.attention(k, k).backward(w)
        if i % 97 == 0:   # reading the sum on the way leaves it as it is
            once_rounded(q.grad(), (i + 1) * first, (i + 1) * np.abs(first), i, dtype)
    once_rounded(q.grad(), n * first, n * np.abs(first), n - 1, dtype)
    q.zeroGrad()
    q.attention(k, k).backward(w)
    assert np.array_equal(q.grad().toNumpy().astype(np.float64), first)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_a_sum_of_both_types(dtype):
    """A float32 gradient beside 16-bit ones: all of them in float32, as a single float32 one is."""
    x, w = made((30, 2, 16), 1, dtype).requiresGrad(), made((30, 2, 16), 2, dtype)
    o = x.attention(x, x)
    o.backward(w)
    low = x.grad().toNumpy().astype(np.float64)
    (x * 3.0).sum().backward()
    got = x.grad()
    assert got.getDtype() == "float32"
    # (the three uses' sum was rounded above, and is not here)
    assert (np.abs(got.toNumpy().astype(np.float64) - (low + 3.0)) <= R.H[dtype] * np.abs(low) * 1.01 + 4 * R.U * (np.abs(low) + 3.0) + R.TINY[dtype]).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_results_that_meet_float64(dtype):
    """An upstream gradient in float64, of a factor that float32 holds: the bits of the same factor in float32."""
    factor = np.random.default_rng(5).standard_normal((20, 2, 16)).astype(np.float32)
    tokens = CudaArray.fromNumpy(np.arange(20, dtype=np.int32))
    bits = []
    for up in ("float32", "float64"):
        q, x = made((20, 2, 16), 1, dtype).requiresGrad(), made((20, 40), 2, dtype).requiresGrad()
        (q.attention(q, q) * CudaArray.fromNumpy(factor.astype(up), up)).sum().backward()
        (x.logProbs(tokens)["entropy"] * CudaArray.fromNumpy(factor[:, 0, 0].astype(up), up)).sum().backward()
        assert q.grad().getDtype() == x.grad().getDtype() == dtype
        bits.append((q.grad().toBits(), x.grad().toBits()))
    assert all(np.array_equal(a, b) for a, b in zip(*bits))
