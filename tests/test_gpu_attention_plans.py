"""Plans of attention without gradients, which are captured into a graph: replays on other inputs give the eager bits."""
import numpy as np
import pytest

from phptensors import CudaArray, Fusion, Sequences

pytestmark = pytest.mark.gpu


def made(shape, seed, dtype):
    return CudaArray.fromNumpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float32), dtype)


def same_bits(step, inputs, launches):
    plan = Fusion.compile(step, inputs(0), cudaGraph=True)
    for seed in (1, 2, 3, 1):
        ins = inputs(seed)
        want = [t.toBits() for t in step(*ins)]
        for _ in range(2):
            assert all(np.array_equal(a, b.toBits()) for a, b in zip(want, plan.run(*ins)))
    assert plan.getStats()["graphLaunches"] >= launches, plan.getStats()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_attention_alone(dtype):
    at = Sequences([30, 66])
    same_bits(lambda q, k, v: [q.attention(k, v, causal=True, queries=at)],
              lambda seed: [made((96, n, 64), seed + i, dtype) for i, n in enumerate((4, 2, 2))], 6)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_a_layer(dtype):
    """Three projections, which may run beside each other, attention behind them, and a projection of its result; and a
    split cache, whose parts lie in the plan's workspace."""
    at, one, kept = Sequences([30, 66]), Sequences([1, 1]), Sequences([700, 513], [0, 700])

    def step(x, wq, wk, wv, wo, q, cache):
        a, b, c = (x.matmul(w).reshape([96, -1, 32]) for w in (wq, wk, wv))
        y = a.attention(b, c, causal=True, queries=at).reshape([96, 128]).matmul(wo)
        return [y, q.attention(cache, cache, causal=True, queries=one, keys=kept)]
    shapes = [(96, 128), (128, 128), (128, 64), (128, 64), (128, 128), (2, 4, 32), (1400, 2, 32)]
    same_bits(step, lambda seed: [made(s, 10 * seed + i, dtype) for i, s in enumerate(shapes)], 6)
