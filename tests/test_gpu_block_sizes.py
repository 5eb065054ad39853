"""Rotary positions, the gated projection and AdamW over many tensors past 2^31 elements (AdamW in 8 bits past 2^32): the
last rows of operands that are zeros before them, through the C entries, against the same rows alone or float64."""
import ctypes

import numpy as np
import pytest

import test_gpu_gated
from phptensors import _abi

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -11


def big(size, tail=None):
    """A buffer of `size` bytes, zeros but for the array at its end."""
    b = _abi.DeviceBuffer(size)
    _abi.check(_abi.load().pt_memset(b.ptr, 0, size, None))
    if tail is not None:
        _abi.check(_abi.load().pt_memcpy_h2d(b.ptr + size - tail.nbytes, np.ascontiguousarray(tail).ctypes.data, tail.nbytes, None))
    _abi.synchronize()
    return b


def end(b, like):
    out = np.empty_like(like)
    _abi.check(_abi.load().pt_memcpy_d2h(out.ctypes.data, b.ptr + b.nbytes - out.nbytes, out.nbytes, None))
    return out


def pair(*pointers):
    return (ctypes.c_void_p * 2)(*pointers)


def test_rotary():
    lib, rng, heads, size, last = _abi.load(), np.random.default_rng(1), (80, 48), 256, 3
    tokens = 2 ** 31 // (heads[0] * size) + 7
    x, g = ([rng.standard_normal((last, h, size)).astype(np.float16) for h in heads] for _ in range(2))
    scale, turns = rng.standard_normal(size).astype(np.float16), _abi.to_device(rng.random(size // 2))
    w = _abi.to_device(scale)

    def run(n, positions):
        bx, bg = ([big(n * h * size * 2, t) for h, t in zip(heads, ts)] for ts in (x, g))
        by = [big(n * h * size * 2) for h in heads]
        ds = [big(size * 2) for _ in heads]
        d = _abi.PtRotaryDesc()
        for name, v in dict(dtype=_abi.FLOAT16, sequences=1, tokens=n, size=size, part=size, magnitude=1.0, epsilon=1e-6,
                            turns=turns.ptr, positions=positions).items():
            setattr(d, name, v)
        d.position_strides = (ctypes.c_size_t * 2)(0, 1)
        for i, h in enumerate(heads):
            d.heads[i], d.strides[i] = h, (ctypes.c_size_t * 3)(0, h * size, size)
        p = [pair(*(b.ptr for b in bs)) for bs in (bx, bg, by, ds)]
        _abi.check(lib.pt_rotary(ctypes.byref(d), p[0], pair(w.ptr, w.ptr), p[2], None))
        out = [end(b, t) for b, t in zip(by, x)]
        _abi.check(lib.pt_rotary_backward(ctypes.byref(d), p[0], pair(w.ptr, w.ptr), p[1], _abi.FLOAT16, p[2], p[3], None))
        return out + [end(b, t) for b, t in zip(by, x)], [end(b, scale).astype(np.float64) for b in ds]
    at = _abi.to_device(np.arange(tokens - last, tokens, dtype=np.int32))
    (many, ds), (few, ds_few) = run(tokens, None), run(last, at.ptr)
    assert all(np.array_equal(a, b) for a, b in zip(many, few)) and all(np.abs(a).max() > 0.1 for a in many)
    for a, b, t in zip(ds, ds_few, g):
        # sums of the same last * heads products in another order, then each its rounding
        off = t.size // size * 2.0 ** -24 * np.abs(t.astype(np.float64)).sum((0, 1)) * 16
        assert (np.abs(a - b) <= off + 2 * HALF * np.abs(b)).all()


def test_gated():
    lib, rng, m, k, f, last = _abi.load(), np.random.default_rng(2), 2 ** 21, 8, 1032, 100
    x, dh = rng.standard_normal((last, k)).astype(np.float16), rng.standard_normal((last, f)).astype(np.float16)
    gate, up = ((rng.standard_normal((k, f)) / 3).astype(np.float16) for _ in range(2))
    bx, bdh, bh, kept, dx = (big(m * n * 2, t) for n, t in ((k, x), (f, dh), (f, None), (3 * f, None), (k, None)))
    weights, grads = [_abi.to_device(t) for t in (gate, up)], [big(t.nbytes) for t in (gate, up)]
    d = _abi.PtGatedDesc(_abi.FLOAT16, 0, m, k, f)
    _abi.check(lib.pt_gated(ctypes.byref(d), bx.ptr, *(b.ptr for b in weights), bh.ptr, kept.ptr, None))
    _abi.check(lib.pt_gated_backward(ctypes.byref(d), bx.ptr, *(b.ptr for b in weights), kept.ptr, bdh.ptr, _abi.FLOAT16, dx.ptr,
                                     *(b.ptr for b in grads), None))
    want = test_gpu_gated.reference(*(t.astype(np.float64) for t in (x, gate, up)), "silu", "float16", dh.astype(np.float64))
    for name, got in (("h", end(bh, dh)), ("dx", end(dx, x)), ("dgate", end(grads[0], gate)), ("dup", end(grads[1], up))):
        v, off = want[name]
        assert (np.abs(got.astype(np.float64) - v) <= off * (1 + HALF) + HALF * np.abs(v) + 2.0 ** -25).all(), name
        assert np.abs(v).max() > 0.1


@pytest.mark.parametrize("bits,n", [(32, 2 ** 31 + 700), (8, 2 ** 32 + 700)])
def test_adamw(bits, n):
    """In the old ones' place.  The last elements' step is that of a tensor of them alone; of the 8-bit moments, whose drawn
    numbers go by the index, the values are within a step of their codes of it: 2^-3 and, squared, 2 * 2^-4 + 2^-8."""
    lib, rng, last = _abi.load(), np.random.default_rng(3), 700
    p, g = (rng.standard_normal(last).astype(np.float16) for _ in range(2))
    wide = 4 if bits == 32 else 1

    def run(n):
        blocks = (n + 255) // 256
        bp, bg, m, v = big(n * 2, p), big(n * 2, g), big(blocks * 256 * wide), big(blocks * 256 * wide)
        e = [big(blocks) for _ in range(2)]
        numbers = _abi.to_device(np.ones(4, np.float32))
        draws = _abi.to_device(np.array([7, 0], np.int32))
        d, t = _abi.PtAdamwDesc(), _abi.PtAdamwTensor(bp.ptr, bg.ptr, bp.ptr, n, 0, _abi.FLOAT16, _abi.FLOAT16, 1)
        for name, x in dict(bits=bits, beta1=0.9, beta2=0.99, epsilon=1e-8, weight_decay=0.1, rate_value=0.1, first=m.ptr,
                            second=v.ptr, new_first=m.ptr, new_second=v.ptr, power1=numbers.ptr, power2=numbers.ptr + 4,
                            new_power1=numbers.ptr + 8, new_power2=numbers.ptr + 12, first_exponent=e[0].ptr,
                            second_exponent=e[1].ptr, new_first_exponent=e[0].ptr, new_second_exponent=e[1].ptr, draws=draws.ptr,
                            new_draws=draws.ptr + 4).items():
            setattr(d, name, x)
        _abi.check(lib.pt_adamw(ctypes.byref(d), ctypes.byref(t), 1, None))
        out = [end(bp, p)]
        tail = np.zeros((last + 255) // 256 * 256, np.float32)
        if bits == 32:
            return out + [end(b, tail) for b in (m, v)]
        size = blocks * 256 * 4
        f = [big(size) for _ in range(2)]
        _abi.check(lib.pt_adamw_moments(m.ptr, e[0].ptr, v.ptr, e[1].ptr, f[0].ptr, f[1].ptr, blocks * 256, None))
        return out + [end(b, tail) for b in f]
    assert n % 256 == last % 256
    many, few = run(n), run(last)
    assert np.array_equal(many[0], few[0]) and not np.array_equal(many[0], p)
    if bits == 32:
        assert all(np.array_equal(a, b) for a, b in zip(many, few))
    for a, b, off in zip(many[1:], few[1:], (2.0 ** -3, 2 * 2.0 ** -4 + 2.0 ** -8)):
        a, b = a.astype(np.float64), b.astype(np.float64)
        # a code's neighbours are at most `off` of the smaller one apart, and below 2^-6 of 2^e a step is the same all the way
        assert (np.abs(a - b) <= off * np.maximum(np.abs(a), np.abs(b)) + 2.0 ** -9 * np.abs(b).max() / 128).all()
        assert np.abs(b).max() > 0 and not a[last:].any()
