"""What the C entries of attention, layerNorm's gradients and the log probabilities refuse, before they touch a
device: no call here reaches one."""
import ctypes

import pytest

from phptensors import _abi

LIB = _abi.load()
P = ctypes.c_void_p(4096)   # never read: every call below is refused first


def refused(status, code=_abi.PT_ERR_INVALID):
    assert status == code and _abi.last_error()


def desc(**change):
    d = _abi.PtAttentionDesc()
    base = dict(dtype=_abi.BFLOAT16, sequences=2, heads=4, kv_heads=2, head_size=64, queries=8, keys=16, causal=1,
                scale=0.125, q_rows=0, k_rows=0)
    strides = dict(q_strides=(2048, 256, 64), k_strides=(2048, 128, 64), v_strides=(2048, 128, 64))
    for n, v in {**base, **strides, **change}.items():
        setattr(d, n, (ctypes.c_size_t * 3)(*v) if n.endswith("strides") else v)
    return d


BAD = [dict(dtype=_abi.FLOAT64), dict(dtype=_abi.INT32), dict(sequences=-1), dict(queries=-1), dict(keys=-2),
       dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(head_size=0), dict(scale=0.0), dict(scale=-1.0),
       dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-40), dict(q_starts=4096), dict(k_lengths=4096),
       dict(q_starts=4096, q_lengths=4096, q_rows=-1), dict(k_starts=4096, k_lengths=4096, k_rows=-1),
       dict(queries=1 << 30), dict(sequences=1 << 30), dict(sequences=1 << 20, keys=1 << 24)]


@pytest.mark.parametrize("change", BAD, ids=str)
def test_attention_descriptions(change):
    d = ctypes.byref(desc(**change))
    refused(LIB.pt_attention(d, P, P, P, P, P, P, None))
    refused(LIB.pt_attention_backward(d, P, P, P, P, P, P, P, _abi.BFLOAT16, P, P, P, None))


def test_attention_operands():
    d = ctypes.byref(desc())
    refused(LIB.pt_attention(None, P, P, P, P, P, P, None))
    refused(LIB.pt_attention(ctypes.byref(desc(head_size=257)), P, P, P, P, P, None, None), _abi.PT_ERR_UNSUPPORTED)
    for missing in range(4):
        args = [None if i == missing else P for i in range(4)]
        refused(LIB.pt_attention(d, *args, None, None, None))
    for missing in range(9):  # q, k, v, out, lse, grad, dq, dk, dv
        a = [None if i == missing else P for i in range(9)]
        refused(LIB.pt_attention_backward(d, *a[:5], None, a[5], _abi.BFLOAT16, *a[6:], None))
    refused(LIB.pt_attention_backward(d, P, P, P, P, P, None, P, _abi.FLOAT16, P, P, P, None))
    refused(LIB.pt_attention_backward(d, P, P, P, P, P, None, P, _abi.FLOAT64, P, P, P, None))


def test_layernorm_gradients():
    def call(input=P, grad=P, dt=_abi.FLOAT32, cdt=_abi.FLOAT32, rows=4, n=8, eps=1e-5, pdt=_abi.FLOAT32):
        refused(LIB.pt_layernorm_backward(input, grad, dt, cdt, rows, n, eps, None, pdt, P, P, P, None))
    for change in [dict(input=None), dict(grad=None), dict(dt=_abi.INT32), dict(dt=_abi.FLOAT64), dict(cdt=_abi.FLOAT16),
                   dict(dt=_abi.FLOAT16, cdt=_abi.FLOAT64, pdt=_abi.FLOAT64), dict(pdt=_abi.FLOAT64),
                   dict(dt=_abi.FLOAT16, pdt=_abi.BFLOAT16), dict(n=0), dict(n=1 << 32), dict(rows=1 << 32), dict(eps=0.0),
                   dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(eps=1e-60)]:
        call(**change)


def test_log_probabilities():
    def call(x=P, dt=_abi.FLOAT32, rows=4, classes=10, pitch=10, tokens=P, top=2):
        refused(LIB.pt_logprobs(x, dt, rows, classes, pitch, tokens, top, P, P, P, P, P, None))
        refused(LIB.pt_logprobs_backward(x, dt, rows, classes, pitch, tokens, top, P, P, P, P, P, P, P, None))
    for change in [dict(x=None), dict(dt=_abi.FLOAT64), dict(dt=_abi.INT64), dict(rows=1 << 32), dict(classes=0),
                   dict(classes=1 << 31), dict(pitch=9), dict(tokens=None), dict(top=-1), dict(top=11),
                   dict(top=65, classes=100, pitch=100)]:
        call(**change)
    for missing in range(4):  # the indices, the statistics, the entropy, the result
        index, stats, entropy, out = [None if i == missing else P for i in range(4)]
        refused(LIB.pt_logprobs_backward(P, _abi.FLOAT32, 4, 10, 10, P, 2, index, stats, entropy, P, P, P, out, None))
