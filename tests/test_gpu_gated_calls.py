"""The gated projection's few-row kernel with a split contraction in each of its forms, and the C entries' operands and
results at addresses between packs."""
import ctypes

import numpy as np
import pytest

import test_gpu_gated
from phptensors import _abi

pytestmark = pytest.mark.gpu


# rows of one, two and four groups of 16 (the last in strips of half the width); columns that end inside a strip, a
# contraction that ends inside a step
@pytest.mark.parametrize("dtype", test_gpu_gated.DTYPES)
@pytest.mark.parametrize("shape", [(9, 2050, 137), (24, 2048, 300), (32, 1030, 260), (48, 2048, 300), (64, 4100, 301), (33, 1001, 71)],
                         ids=str)
def test_split_contractions_of_few_rows(shape, dtype):
    test_gpu_gated.test_both_directions(shape, dtype)


@pytest.mark.parametrize("shape", [(96, 1000, 27000), (511, 1200, 5600), (512, 1200, 5600)], ids=str)
def test_large_float32_weights(shape):
    """Past 2.5e9 multiplications for a matrix with few rows, and on both sides of the rows where the gradients go another
    way."""
    test_gpu_gated.test_both_directions(shape, "float32")


@pytest.mark.parametrize("dtype", test_gpu_gated.DTYPES)
@pytest.mark.parametrize("shape", [(1, 64, 40), (20, 72, 136), (40, 64, 128), (80, 64, 128), (150, 65, 77), (2048, 640, 2048)], ids=str)
def test_any_address(shape, dtype):
    """Everything an element behind a pack's boundary: the bits of calls at boundaries, but for large float32 gradients, whose
    plain products add in another order there; those are within the bounds against float64."""
    lib, (m, k, f), rng = _abi.load(), shape, np.random.default_rng(1)
    code = {"float32": _abi.FLOAT32, "float16": _abi.FLOAT16, "bfloat16": _abi.BFLOAT16}[dtype]
    store = {"float32": lambda v: v, "float16": lambda v: v.astype(np.float16),
             "bfloat16": lambda v: (v.view(np.uint32) >> 16).astype(np.uint16)}[dtype]
    made = {n: store((rng.standard_normal(s) * c).astype(np.float32)) for n, s, c in
            (("x", (m, k), 1), ("gate", (k, f), k ** -0.5), ("up", (k, f), k ** -0.5), ("g", (m, f), 1))}
    sizes = {"h": m * f, "dx": m * k, "dgate": k * f, "dup": k * f}
    d, wide = _abi.PtGatedDesc(code, 0, m, k, f), 4 if dtype == "float32" else 2

    def run(skip):
        held = {n: _abi.DeviceBuffer(t.nbytes + skip) for n, t in made.items()}
        held.update({n: _abi.DeviceBuffer(s * wide + skip + 64) for n, s in sizes.items()})
        kept = _abi.DeviceBuffer((8 if wide == 4 else 6) * m * f)
        for n, b in held.items():
            _abi.check(lib.pt_memset(b.ptr, 0x5A, b.nbytes, None))
            if n in made:
                _abi.check(lib.pt_memcpy_h2d(b.ptr + skip, np.ascontiguousarray(made[n]).ctypes.data, made[n].nbytes, None))
        p = {n: b.ptr + skip for n, b in held.items()}
        _abi.check(lib.pt_gated(ctypes.byref(d), p["x"], p["gate"], p["up"], p["h"], kept.ptr, None))
        _abi.check(lib.pt_gated_backward(ctypes.byref(d), p["x"], p["gate"], p["up"], kept.ptr, p["g"], code, p["dx"], p["dgate"],
                                         p["dup"], None))
        out = {n: held[n].download(np.uint8, (held[n].nbytes,)) for n in sizes}
        for n, s in sizes.items():  # nothing in front or behind
            assert (out[n][:skip] == 0x5A).all() and (out[n][skip + s * wide:] == 0x5A).all(), n
        return {n: out[n][skip:skip + s * wide] for n, s in sizes.items()}
    want, got = run(0), run(wide)
    if dtype == "float32" and m * k * f > 2e9:
        exact = test_gpu_gated.reference(*(made[n].astype(np.float64) for n in ("x", "gate", "up")), "silu", dtype,
                                         made["g"].astype(np.float64))
        for out in (want, got):
            for n, (v, off) in exact.items():
                y = out[n].view(np.float32).reshape(v.shape).astype(np.float64)
                assert (np.abs(y - v) <= off * (1 + test_gpu_gated.U) + test_gpu_gated.U * np.abs(v) + 2.0 ** -126).all(), n
        sizes = {"h": sizes["h"]}
    for n in sizes:
        assert np.array_equal(want[n], got[n]), n
        assert (want[n] != 0x5A).any()
