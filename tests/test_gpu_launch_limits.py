"""Calls of more than one launch holds, which counts its threads in 32 bits: AdamW over many tensors and 8-bit moments
(through the C entries), elementwise operations, reductions, rows, products, plans.  Up to 155 GB of the card's 288."""
import ctypes

import numpy as np
import pytest

from phptensors import CudaArray, Fusion, _abi
from test_gpu_block_sizes import big, end

pytestmark = pytest.mark.gpu


def download(pointer, like):
    out = np.empty_like(like)
    _abi.check(_abi.load().pt_memcpy_d2h(out.ctypes.data, pointer, out.nbytes, None))
    return out


def test_adamw():
    """Sixteen tensors of 2^31 elements and one of 700 in 8 bits, moments in place.  All read the same old values and
    gradients, zeros but for 700 at the end, so each one's last elements step as those alone do."""
    lib, rng, last, each, many = _abi.load(), np.random.default_rng(3), 700, 2 ** 31, 16
    p, g = (rng.standard_normal(last).astype(np.float16) for _ in range(2))
    old, grad = big(each * 2, p), big(each * 2, g)

    def run(sizes):
        total = sum(-(-n // 256) * 256 for n in sizes)
        new, m, v = big(sum(sizes) * 2), big(total), big(total)
        e = [big(total // 256) for _ in range(2)]
        numbers, draws = _abi.to_device(np.ones(4, np.float32)), _abi.to_device(np.array([7, 0], np.int32))
        d, t, at, ends = _abi.PtAdamwDesc(), (_abi.PtAdamwTensor * len(sizes))(), 0, []
        for i, n in enumerate(sizes):
            skip = (each - n) * 2
            t[i] = _abi.PtAdamwTensor(old.ptr + skip, grad.ptr + skip, new.ptr + sum(sizes[:i]) * 2, n, at, _abi.FLOAT16,
                                      _abi.FLOAT16, 1)
            at += -(-n // 256) * 256
            ends.append(new.ptr + sum(sizes[:i + 1]) * 2 - p.nbytes)
        for name, x in dict(bits=8, beta1=0.9, beta2=0.99, epsilon=1e-8, weight_decay=0.1, rate_value=0.1, first=m.ptr,
                            second=v.ptr, new_first=m.ptr, new_second=v.ptr, power1=numbers.ptr, power2=numbers.ptr + 4,
                            new_power1=numbers.ptr + 8, new_power2=numbers.ptr + 12, first_exponent=e[0].ptr,
                            second_exponent=e[1].ptr, new_first_exponent=e[0].ptr, new_second_exponent=e[1].ptr, draws=draws.ptr,
                            new_draws=draws.ptr + 4).items():
            setattr(d, name, x)
        _abi.check(lib.pt_adamw(ctypes.byref(d), t, len(sizes), None))
        moments = end(m, np.empty(768, np.uint8))
        return [download(x, p) for x in ends], moments, download(numbers.ptr, np.empty(4, np.float32)), download(
            draws.ptr, np.empty(2, np.int32))
    (want,), _, numbers, _ = run([last])
    got, moments, powers, draws = run([each] * many + [last])
    assert not np.array_equal(want, p) and all(np.array_equal(x, want) for x in got)
    assert np.array_equal(powers, numbers) and draws[1] == 8
    assert (moments[:last] != 0).mean() > 0.9 and not moments[last:].any()


def test_moments():
    lib, n = _abi.load(), 2 ** 34 + 512
    tail = np.random.default_rng(4).integers(0, 256, 512).astype(np.uint8)
    code, exponent = big(n, tail), big(n // 256, np.array([3, -5], np.int8))
    out = [_abi.DeviceBuffer(n * 4) for _ in range(2)]
    for b in out:
        _abi.check(lib.pt_memset(b.ptr, 0xFF, n * 4, None))

    def run(code, exponent, values, n):
        _abi.check(lib.pt_adamw_moments(code, exponent, code, exponent, *values, n, None))
    run(code.ptr, exponent.ptr, [b.ptr for b in out], n)
    few = [_abi.DeviceBuffer(512 * 4) for _ in range(2)]
    run(code.ptr + n - 512, exponent.ptr + n // 256 - 2, [b.ptr for b in few], 512)
    for a, b in zip(out, few):
        assert np.array_equal(end(a, np.empty(512, np.float32)), download(b.ptr, np.empty(512, np.float32)))
        for at in (0, n // 2, n - 1536):
            assert not download(a.ptr + at * 4, np.empty(1024, np.float32)).any()


# Tensors of one value: a tensor's first, middle and last rows.  No two results that follow each other are alike, so
# memory that is used again holds nothing that passes.
def same(t, want):
    n = t.getShape()[0]
    for at in (0, n // 2, n - 3):
        x = t.slice([at, at + 3]).toNumpy()
        assert np.array_equal(x, np.broadcast_to(np.asarray(want, x.dtype), x.shape)), (at, want)


@pytest.mark.parametrize("rows", [2 ** 16, 2 ** 16 + 1])
def test_elements(rows):
    """A thread for each of 2^32 elements, and of more."""
    x = CudaArray.full([rows, 2 ** 16], 3, "uint8")
    same(x, 3)
    same(x + x, 6)
    same(x.astype("int16"), 3)
    same(CudaArray.where(x, CudaArray.full([1], 9, "uint8"), CudaArray.full([1], 1, "uint8")), 9)


@pytest.mark.parametrize("dtype,rows", [("float32", 2 ** 17 + 1), ("bfloat16", 2 ** 18 + 1)])
def test_packs(dtype, rows):
    """A thread for each 16 bytes."""
    x = CudaArray.full([rows, 2 ** 17], 1.5, dtype)
    same(x, 1.5)
    same(x * 2.0, 3.0)
    same(x.neg(), -1.5)


# Tensors that repeat 1021 rows: every row's result is that of the row alone.
def repeated(shape, dtype, seed=1):
    base = np.random.default_rng(seed).integers(-8, 9, (1021, *shape[1:])).astype(np.int32 if dtype == "int32" else np.float32)
    return CudaArray.fromNumpy(np.resize(base, shape), dtype), CudaArray.fromNumpy(base, dtype)


def repeats(many, few, what):
    a, b = many.toBits(), few.toBits()
    assert np.array_equal(a, np.resize(b, a.shape)), what


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows(dtype):
    """A wave for each of more than 2^26 rows."""
    x, y = repeated((2 ** 26 + 64, 4), dtype)
    for name in ("sum", "mean", "max", "min", "prod", "argMax", "argMin", "var", "softmax"):
        repeats(getattr(x, name)(-1), getattr(y, name)(-1), name)
    repeats(x.layerNorm([1], 1e-3), y.layerNorm([1], 1e-3), "layerNorm")


def test_long_rows():
    """512 threads for each of more than 2^23 rows."""
    x = CudaArray.full([2 ** 23 + 64, 1028], 0.5)
    same(x.sum(-1), 514.0)
    same(x.max(-1), 0.5)
    few = CudaArray.full([1, 1028], 0.5).softmax(-1).toNumpy()[0, 0]
    same(x.softmax(-1), few)


@pytest.mark.parametrize("dtype", ["float32", "int32"])
def test_strided_reductions(dtype):
    """128 threads for each of more than 2^25 results."""
    x, y = repeated((2 ** 25 + 64, 3, 2), dtype)
    for name in ("sum", "max"):
        repeats(getattr(x, name)(1), getattr(y, name)(1), name)
    repeats(x.swapaxes(1, 2).sum(-1), y.swapaxes(1, 2).sum(-1), "swapped")
    repeats(x.sum(-1), y.sum(-1), "last")


def test_empty_axes():
    same(CudaArray.zeros([2 ** 16 + 1, 0, 2 ** 16]).prod(1), 1.0)


def test_columns():
    """64 columns of bytes to a workgroup, 512 of bfloat16."""
    x = CudaArray.full([2, 2 ** 30 + 1], 3, "uint8")
    got = x.sum(0)
    same(got, 6)
    del x, got
    x = CudaArray.full([2, 2 ** 16 + 1, 2 ** 16], 1.0, "bfloat16")
    same(x.sum(0), 2.0)


def test_softmax_of_another_axis():
    """An element to a thread, moved there and back."""
    x = CudaArray.full([2 ** 11 + 1, 2, 2 ** 20], 1.0, "bfloat16")
    same(x.softmax(1), 0.5)


@pytest.mark.parametrize("lead", [(2 ** 24 + 8,), (4099, 1, 4097)], ids=str)
@pytest.mark.parametrize("shared", ["left", "right"])
def test_small_products(lead, shared):
    """A tile for each of more than 2^24 products, one factor common to all."""
    n = int(np.prod(lead))
    x, y = repeated((n, 2, 2), "float32")
    w = CudaArray.fromNumpy(np.array([[1, 2], [-3, 4]], np.float32))
    a, b = (w.matmul(x.reshape([*lead, 2, 2])), w.matmul(y)) if shared == "left" else (x.reshape([*lead, 2, 2]).matmul(w), y.matmul(w))
    assert a.getShape() == [*lead, 2, 2]
    repeats(a.reshape([n, 2, 2]), b, shared)


def test_small_products_of_pairs():
    x, y = repeated((2 ** 24 + 8, 2, 3), "bfloat16")
    u, v = repeated((2 ** 24 + 8, 3, 2), "bfloat16", 2)
    repeats(x.matmul(u), y.matmul(v), "pairs")


def test_empty_products():
    same(CudaArray.zeros([2 ** 16 + 1, 0], "float16").matmul(CudaArray.zeros([0, 2 ** 16], "float16")), 0.0)


def test_plan_of_elements():
    x = CudaArray.full([2 ** 16, 2 ** 16], 3, "int32")
    plan = Fusion.compile(lambda t: [t * t + t], [x])
    same(plan.run(x)[0], 12)


def test_plan_of_rows():
    """Reductions and what follows them, a workgroup for each of more than 2^26 rows."""
    x, y = repeated((2 ** 26 + 64, 4), "float32")

    def body(t):
        return [(t - t.max(-1).reshape([-1, 1])).exp().sum(-1) * 0.5]
    repeats(Fusion.compile(body, [x]).run(x)[0], body(y)[0], "plan")
