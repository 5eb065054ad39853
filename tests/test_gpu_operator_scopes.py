"""Results of attention, layerNorm's gradients and logProbs read inside and after a Fusion.run scope are the eager ones."""
import itertools

import numpy as np
import pytest

from phptensors import CudaArray, Fusion, Sequences

pytestmark = pytest.mark.gpu


def made(shape, seed, dtype="float32"):
    return CudaArray.fromNumpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float32), dtype)


def logprobs():
    x = made((7, 300), 1).requiresGrad()
    got = x.logProbs(CudaArray.fromNumpy(np.array([0, 5, -1, 299, 7, 8, 9], np.int32)), top=3)
    (got["logProbs"].sum() + got["entropy"].sum()).backward()
    return [*(t.detach() for t in got.values()), x.grad()]


def norm():
    x, s, b = (made(n, i).requiresGrad() for i, n in enumerate(((9, 40), (40,), (40,))))
    y = x.layerNorm([1], 1e-5, s, b)
    y.backward(made((9, 40), 5))
    return [y.detach(), x.grad(), s.grad(), b.grad()]


def attention(dtype):
    q, k, v = (made((50, n, 16), n + i, dtype).requiresGrad() for i, n in enumerate((4, 2, 2)))
    o = q.attention(k, v, causal=True, queries=Sequences([20, 30]))
    o.backward(made((50, 4, 16), 9, dtype))
    return [o.detach(), q.grad(), k.grad(), v.grad()]


@pytest.mark.parametrize("op", [logprobs, norm, lambda: attention("float32"), lambda: attention("float16")],
                         ids=["logprobs", "norm", "attention", "attention16"])
def test_scopes(op):
    want = [t.toBits() for t in op()]
    n = len(want)
    for order in itertools.permutations(range(n), 2):
        kept = []

        def inside():
            kept[:] = op()
            for i in order:
                assert np.array_equal(kept[i].toBits(), want[i]), order
            return kept[order[0]]
        Fusion.run(inside)
        for i in range(n):
            assert np.array_equal(kept[i].toBits(), want[i]), (order, i)
