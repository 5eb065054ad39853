"""Packed prompts of very different lengths whose keys or queries are split between workgroups: results, and the
scratch they take, which goes by the rows there are and not by the longest prompt's."""
import ctypes

import numpy as np
import pytest

import attention_ref as R
from phptensors import CudaArray, Sequences, _abi, _host

pytestmark = pytest.mark.gpu


def peak_of(call):
    """Bytes of scratch that the call asks for."""
    lib, peak = _abi.load(), ctypes.c_size_t()
    _abi.check(lib.pt_workspace_begin(None, 0))
    try:
        out = call()
    finally:
        _abi.check(lib.pt_workspace_end(ctypes.byref(peak)))
    return out, peak.value


# sequences of one query beside a chunk, keys of each, heads, key heads, size
MIXED = [(126, 386, 520, 32, 1, 128), (40, 150, 700, 8, 2, 64), (9, 300, 300, 4, 4, 40), (60, 200, 300, 6, 3, 32)]


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("case", MIXED, ids=str)
def test_a_chunk_among_single_tokens(case, dtype):
    ones, chunk, keys, heads, kv, size = case
    lengths = [1] * (ones // 2) + [chunk] + [1] * (ones - ones // 2)
    count, rows = len(lengths), sum(lengths) + 3
    rng = np.random.default_rng(ones)
    kept = [int(n) for n in rng.integers(1, keys + 1, count)]
    kept[ones // 2] = keys
    starts = [int(n) + 1 for n in np.cumsum([0] + lengths)[:-1]]
    q, k, v, w = (CudaArray.fromNumpy(rng.standard_normal(s).astype(np.float32), dtype)
                  for s in ((rows, heads, size), (count * keys, kv, size), (count * keys, kv, size), (rows, heads, size)))
    queries, at = Sequences(lengths, starts), Sequences(kept, [i * keys for i in range(count)])
    lib, held, got = _host.load(), (ctypes.c_void_p * 2)(), (ctypes.c_void_p * 3)()
    q.attention(k, v, causal=True, queries=queries, keys=at)   # (what a first call allocates for itself)
    o, forward = peak_of(lambda: CudaArray._wrap(lib.phpt_attention(q._h, k._h, v._h, 1, 0.0, queries._h, at._h, held)))
    lse, rest = (CudaArray._wrap(h) if h else None for h in held)
    status, backward = peak_of(lambda: lib.phpt_attention_backward(
        q._h, k._h, v._h, o._h, lse._h, rest._h if rest is not None else None, w._h, 1, 0.0, queries._h, at._h, got))
    assert not status
    spans = [(a, n, i * keys, m) for i, (a, n, m) in enumerate(zip(starts, lengths, kept))]
    ref = R.attention(*(t.toNumpy().astype(np.float64) for t in (q, k, v)), True, size ** -0.5, dtype, spans,
                      w.toNumpy().astype(np.float64))
    for n, t in zip(("o", "dq", "dk", "dv"), (o, *(CudaArray._wrap(h) for h in got))):
        want, off = ref[n]
        assert (np.abs(t.toNumpy().astype(np.float64).reshape(want.shape) - want) <= off).all(), n
    # at most 64 ranges of keys, fewer the more tiles there are: a row's sums for each, 512 workgroups of 128 rows in all
    tiles = -(-rows * (heads // kv) // 128) * kv
    assert forward <= min(64, 512 // tiles + 1) * rows * heads * (size + 2) * 4 + 4096
    # shares of the queries' gradient, or of the keys' and values', in float32, beside three numbers a row
    assert backward <= 16 * max(rows * heads, 2 * count * keys * kv) * size * 4 + 3 * rows * heads * 4 + 8192
