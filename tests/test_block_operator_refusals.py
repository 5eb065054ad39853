"""What the C entries of rotary, the gated projection and AdamW over many tensors refuse, before they touch a device: no
call here reaches one."""
import ctypes

import pytest

from phptensors import _abi

LIB = _abi.load()
A = 4096
P = ctypes.c_void_p(A)   # never read: every call below is refused first


def refused(status, code=_abi.PT_ERR_INVALID):
    assert status == code and _abi.last_error()


def pair(a=A, b=A):
    return (ctypes.c_void_p * 2)(a, b)


def rotary(**change):
    d = _abi.PtRotaryDesc()
    base = dict(dtype=_abi.BFLOAT16, sequences=2, tokens=8, size=64, part=32, interleaved=0, magnitude=1.0, epsilon=1e-6, turns=A)
    for n, v in {**base, **change}.items():
        if n != "heads":
            setattr(d, n, v)
    d.heads[0], d.heads[1] = change.get("heads", (4, 2))
    for side in range(2):
        for i, v in enumerate((2048, 256, 64)):
            d.strides[side][i] = v
    return ctypes.byref(d)


@pytest.mark.parametrize("change", [
    dict(dtype=_abi.FLOAT64), dict(dtype=_abi.INT32), dict(sequences=-1), dict(tokens=-1), dict(heads=(-1, 2)), dict(heads=(4, -1)),
    dict(heads=(1 << 20, 1)), dict(sequences=1 << 20, tokens=1 << 20), dict(size=0), dict(part=0), dict(part=33), dict(part=66),
    dict(turns=0), dict(magnitude=float("nan")), dict(magnitude=1e300), dict(epsilon=0.0), dict(epsilon=-1.0),
    dict(epsilon=float("nan")), dict(epsilon=1e-60)], ids=str)
def test_rotary_descriptions(change):
    refused(LIB.pt_rotary(rotary(**change), pair(), pair(), pair(), None))
    refused(LIB.pt_rotary_backward(rotary(**change), pair(), pair(), pair(), _abi.BFLOAT16, pair(), pair(), None))


def test_rotary_operands():
    refused(LIB.pt_rotary(None, pair(), pair(), pair(), None))
    refused(LIB.pt_rotary(rotary(size=300, part=32), pair(), None, pair(), None), _abi.PT_ERR_UNSUPPORTED)
    refused(LIB.pt_rotary(rotary(), None, None, pair(), None))
    refused(LIB.pt_rotary(rotary(), pair(), None, None, None))
    for a, b in ((None, A), (A, None)):
        refused(LIB.pt_rotary(rotary(), pair(a, b), None, pair(), None))
        refused(LIB.pt_rotary(rotary(), pair(), None, pair(a, b), None))
        refused(LIB.pt_rotary_backward(rotary(), pair(a, b), pair(), pair(), _abi.BFLOAT16, pair(), pair(), None))
        refused(LIB.pt_rotary_backward(rotary(), pair(), pair(), pair(a, b), _abi.BFLOAT16, pair(), pair(), None))
        refused(LIB.pt_rotary_backward(rotary(), pair(), pair(), pair(), _abi.BFLOAT16, pair(a, b), None, None))
    for dtype in (_abi.FLOAT16, _abi.FLOAT64):
        refused(LIB.pt_rotary_backward(rotary(), pair(), pair(), pair(), dtype, pair(), pair(), None))
    refused(LIB.pt_rotary_backward(rotary(), pair(), pair(), None, _abi.BFLOAT16, pair(), pair(), None))
    refused(LIB.pt_rotary_backward(rotary(), pair(), pair(), pair(), _abi.BFLOAT16, None, pair(), None))


def gated(**change):
    d = _abi.PtGatedDesc()
    for n, v in {**dict(dtype=_abi.FLOAT16, activation=0, rows=4, inner=8, outer=16), **change}.items():
        setattr(d, n, v)
    return ctypes.byref(d)


def test_gated_projection():
    def both(d, code=_abi.PT_ERR_INVALID):
        refused(LIB.pt_gated(d, P, P, P, P, P, None), code)
        refused(LIB.pt_gated_backward(d, P, P, P, P, P, _abi.FLOAT32, P, P, P, None), code)
    both(None)
    for change in [dict(dtype=_abi.FLOAT64), dict(dtype=_abi.INT8), dict(activation=-1), dict(activation=4), dict(rows=-1),
                   dict(inner=-1), dict(outer=-1)]:
        both(gated(**change))
    for change in [dict(rows=(1 << 21) + 1), dict(inner=(1 << 21) + 1), dict(outer=(1 << 21) + 1)]:
        both(gated(**change), _abi.PT_ERR_UNSUPPORTED)
    for missing in range(4):  # x, gate, up, h
        refused(LIB.pt_gated(gated(), *(None if i == missing else P for i in range(4)), None, None))
    for missing in range(5):  # x, gate, up, kept, grad
        refused(LIB.pt_gated_backward(gated(), *(None if i == missing else P for i in range(5)), _abi.FLOAT32, P, P, P, None))
    refused(LIB.pt_gated_backward(gated(), P, P, P, P, P, _abi.BFLOAT16, P, P, P, None))
    for results in ((None, None, None), (P, P, None), (P, None, P)):
        refused(LIB.pt_gated_backward(gated(), P, P, P, P, P, _abi.FLOAT16, *results, None))


def adamw(**change):
    d = _abi.PtAdamwDesc()
    for name, kind in d._fields_:
        setattr(d, name, A if kind is ctypes.c_void_p else 0)
    for n, v in {**dict(bits=8, beta1=0.9, beta2=0.99, epsilon=1e-8, weight_decay=0.1, rate_value=0.1, rate=0,
                      new_power1=A + 4, new_power2=A + 8, new_draws=A + 12), **change}.items():
        setattr(d, n, v)
    return ctypes.byref(d)


def tensors(*changes):
    t = (_abi.PtAdamwTensor * max(1, len(changes)))()
    for i, change in enumerate(changes):
        base = dict(param=A, grad=A, new_param=A, n=300, at=512 * i, param_dtype=_abi.BFLOAT16, grad_dtype=_abi.FLOAT32, decay=1)
        for n, v in {**base, **change}.items():
            setattr(t[i], n, v)
    return t


@pytest.mark.parametrize("change", [
    dict(bits=16), dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=float("nan")), dict(epsilon=-1.0), dict(epsilon=float("inf")),
    dict(weight_decay=-1.0), dict(rate_value=-1.0), dict(rate_value=float("nan")), dict(first=0), dict(second=0), dict(new_first=0),
    dict(new_second=0), dict(power1=0), dict(power2=0), dict(new_power1=0), dict(new_power2=0), dict(master=0), dict(new_master=0),
    dict(first_exponent=0), dict(second_exponent=0), dict(new_first_exponent=0), dict(new_second_exponent=0), dict(draws=0),
    dict(new_draws=0), dict(new_power1=A), dict(new_power2=A), dict(new_draws=A)], ids=str)
def test_adamw_descriptions(change):
    refused(LIB.pt_adamw(adamw(**change), tensors({}), 1, None))


@pytest.mark.parametrize("changes", [
    [dict(grad=0)], [dict(new_param=0)], [dict(param_dtype=_abi.FLOAT64)], [dict(grad_dtype=_abi.INT32)], [dict(at=100)],
    [dict(n=1 << 41)], [{}, dict(at=256)], [{}, dict(at=0)]], ids=str)
def test_adamw_tensors(changes):
    refused(LIB.pt_adamw(adamw(), tensors(*changes), len(changes), None))


def test_adamw_operands():
    refused(LIB.pt_adamw(None, tensors({}), 1, None))
    refused(LIB.pt_adamw(adamw(), None, 1, None))
    refused(LIB.pt_adamw(adamw(), tensors({}), -1, None))
    refused(LIB.pt_adamw(adamw(master=0, new_master=0), tensors(dict(param=0)), 1, None))
    refused(LIB.pt_adamw_moments(P, P, P, P, P, P, 100, None))
    for missing in range(6):
        refused(LIB.pt_adamw_moments(*(None if i == missing else P for i in range(6)), 256, None))
