"""Optimizer.fusedStep: float32 bit for bit as Optimizer.step, 16-bit parameters against float64, 8-bit moments code for
code against their definition in numpy."""
import ctypes
import math

import numpy as np
import pytest

from phptensors import CudaArray, Fusion, InvalidArgumentException, _abi, _host
from phptensors.optimizer import Optimizer

pytestmark = pytest.mark.gpu
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
U = 2.0 ** -24
# one element, odd sizes, whole and broken blocks, nothing, a long one
SHAPES = [(1,), (3, 5), (256,), (257,), (0, 4), (16, 16), (1, 1024), (129, 65), (2048,), (2049,), (5001, 3)]


def made(shape, dtype, seed, scale=1.0):
    return CudaArray.fromNumpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float32) * np.float32(scale), dtype)


def flat(shapes, arrays):
    """Arrays in one, each from a multiple of 256 on, zeros between."""
    out = []
    for s, a in zip(shapes, arrays):
        a = np.asarray(a, np.float32).reshape(-1)
        out.append(np.pad(a, (0, -a.size % 256)))
    return np.concatenate(out)


def same(a, b):
    return np.array_equal(np.asarray(a).view(np.uint8), np.asarray(b).view(np.uint8))


@pytest.mark.parametrize("rate", [None, 0.01, "device"])
@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_float32_is_step_bit_for_bit(decay, rate):
    opt = Optimizer.adamW(0.002, 0.9, 0.99, 1e-6, decay)
    params = [made(s, "float32", i) for i, s in enumerate(SHAPES)]
    mask = [i % 3 != 1 for i in range(len(SHAPES))]
    lr = CudaArray.full([1], 0.003) if rate == "device" else rate
    want, plain = params, opt.initState(params)
    got, state = params, opt.initFusedState(params)
    for t in range(3):
        grads = [made(s, "float32", 100 * t + 50 + i, 0.1) for i, s in enumerate(SHAPES)]
        r = opt.step(want, grads, plain, lr, mask)
        want, plain = r["parameters"], r["state"]
        r = opt.fusedStep(got, grads, state, lr, mask)
        got, state = r["parameters"], r["state"]
        assert all(same(a.toBits(), b.toBits()) and a.getShape() == b.getShape() for a, b in zip(want, got))
        for name in ("firstMoment", "secondMoment"):
            assert same(flat(SHAPES, [m.toNumpy() for m in plain[name]]).reshape(-1, 256), state[name].toNumpy())
        for name in ("beta1Power", "beta2Power"):
            assert same(plain[name].toNumpy(), state[name].toNumpy())


def test_gradients_that_are_not_finite():
    opt = Optimizer.adamW(0.01)
    p = made((300,), "float32", 1)
    g = made((300,), "float32", 2).toNumpy()
    g[[0, 7, 299]], g[11] = np.nan, np.inf
    g = CudaArray.fromNumpy(g)
    want = opt.step([p], [g], opt.initState([p]))
    got = opt.fusedStep([p], [g], opt.initFusedState([p]))
    # (which NaN infinity over infinity gives is not promised)
    assert np.array_equal(want["parameters"][0].toNumpy(), got["parameters"][0].toNumpy(), equal_nan=True)
    # with 8 bits an infinite one is left out too, as a block has one scale
    got = opt.fusedStep([p], [g], opt.initFusedState([p], bits=8))
    x, m = got["parameters"][0].toNumpy(), opt.moments(got["state"])
    bad = np.isin(np.arange(300), [0, 7, 11, 299])
    assert np.array_equal(x[bad], p.toNumpy()[bad]) and (x[~bad] != p.toNumpy()[~bad]).all()
    for n in m:
        v = m[n].toNumpy().reshape(-1)
        assert np.isfinite(v).all() and not v[:300][bad].any() and not v[300:].any()


@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("dtype,grad", [("bfloat16", "bfloat16"), ("float16", "float32"), ("bfloat16", "float16")])
def test_16_bit_parameters(dtype, grad, master):
    """The update of float32 arithmetic: at most 12 roundings of the step (moments 3 and 4, divisions, root, sum, rate),
    two of the decayed parameter, one of the difference; then one to the parameter's type."""
    opt = Optimizer.adamW(0.05, 0.9, 0.99, 1e-6, 0.1)
    params = [made(s, dtype, i) for i, s in enumerate(SHAPES)]
    state = opt.initFusedState(params, master=master)
    if master:
        assert same(flat(SHAPES, [p.toNumpy() for p in params]).reshape(-1, 256), state["master"].toNumpy())
    for t in range(2):
        grads = [made(s, grad, 100 * t + 50 + i, 0.1) for i, s in enumerate(SHAPES)]
        m0, v0 = (state[n].toNumpy().astype(np.float64).reshape(-1) for n in ("firstMoment", "secondMoment"))
        old = flat(SHAPES, [p.toNumpy() for p in params]) if not master else state["master"].toNumpy().reshape(-1)
        powers = [float(state[n].toNumpy()[0]) for n in ("beta1Power", "beta2Power")]
        r = opt.fusedStep(params, grads, state)
        params, state = r["parameters"], r["state"]
        g = flat(SHAPES, [x.toNumpy().astype(np.float32) for x in grads]).astype(np.float64)
        m, v = 0.9 * m0 + 0.1 * g, 0.99 * v0 + 0.01 * g * g
        c1, c2 = 1 - powers[0] * 0.9, 1 - powers[1] * 0.99
        step = m / c1 / (np.sqrt(v / c2) + 1e-6) * 0.05
        want = old * (1 - 0.05 * 0.1) - step
        # (the moments add terms of both signs; c1 and c2 are differences of numbers near 1)
        off = 0.05 * (0.9 * np.abs(m0) + 0.1 * np.abs(g)) / c1 / (np.sqrt(v / c2) + 1e-6) * (12 + 2 / c1 + 2 / c2) * U + 4 * U * np.abs(old)
        if master:
            held = state["master"].toNumpy().reshape(-1)
            assert (np.abs(held - want) <= off + U * np.abs(want)).all()
            for p, x in zip(params, np.split(held, np.cumsum([-(-math.prod(s) // 256) * 256 for s in SHAPES])[:-1])):
                rounded = CudaArray.fromNumpy(x[:p.getSize()].reshape(p.getShape()), dtype)
                assert same(rounded.toBits(), p.toBits())
        else:
            got = flat(SHAPES, [p.toNumpy().astype(np.float32) for p in params])
            assert (np.abs(got - want) <= off + HALF[dtype] * (np.abs(want) + off) + 2.0 ** -25).all()
        assert {p.getDtype() for p in params} == {dtype}


# ---------------------------------------------------------------- 8 bits
def mix(h):
    h = h.astype(np.uint32)
    for shift, factor in ((16, 0x85EBCA6B), (13, 0xC2B2AE35)):
        h = (h ^ (h >> np.uint32(shift))) * np.uint32(factor)
    return h ^ (h >> np.uint32(16))


def decode(code, exponent, root):
    """By the definition: sign, exponent with bias 7, mantissa, times the block's power of two."""
    c = code.reshape(-1, 256).astype(np.int64)
    bits = 4 if root else 3
    e, f = (c >> bits) & 15, c & ((1 << bits) - 1)
    x = np.where(e == 0, f * 2.0 ** (-6 - bits), (1 + f * 2.0 ** -bits) * 2.0 ** (e - 7.0))
    x = x * 2.0 ** exponent.reshape(-1, 1).astype(np.float64)
    return x if root else np.where(c >= 128, -x, x)


def encode(x, root, drawn):
    x = np.asarray(x, np.float32).reshape(-1, 256)
    top = np.abs(x).max(1)
    exponent = np.maximum(np.where(top > 0, np.frexp(top)[1] - 1, -127) - 7, -126).astype(np.int8)
    y = np.abs(x).astype(np.float64) * 2.0 ** -exponent.astype(np.float64)[:, None]
    bits = 4 if root else 3
    e = np.maximum(np.floor(np.log2(np.maximum(y, 2.0 ** -6))), -6.0)
    steps = y / 2.0 ** (e - bits)                       # from the power of two below: whole and a fraction
    # the fraction, cut or rounded to what float32's subnormals hold of it, against 16 drawn bits and a half
    ulp = 2.0 ** (19 if root else 20)
    whole = np.floor(steps)
    part = np.round((steps - whole) * ulp)
    up = part + drawn.reshape(-1, 256).astype(np.float64) * (ulp / 65536) + ulp / 131072 >= ulp
    code = (whole + up + (e + 6) * (1 << bits)).astype(np.int64)
    return np.where(x < 0, code | 128, code).astype(np.uint8) if not root else code.astype(np.uint8), exponent


def drawn(state, n):
    with np.errstate(over="ignore"):
        key = mix(np.array([int(state["draws"].toNumpy()[0])], np.int64).astype(np.uint32))
        h = mix(np.arange(n, dtype=np.uint32) + key)
    return h & np.uint32(0xFFFF), h >> np.uint32(16)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [1.0, 1e-12, 1e9])
def test_8_bit_moments(scale, dtype):
    opt = Optimizer.adamW(0.01, 0.9, 0.999, 1e-12, 0.1)
    params = [made(s, dtype, i) for i, s in enumerate(SHAPES)]
    state = opt.initFusedState(params, bits=8, seed=-7)
    f = np.float32
    for t in range(3):
        # gradients over many binades, so that subnormal codes are met
        grads = [CudaArray.fromNumpy((made(s, "float32", 9 * t + i).toNumpy() * scale
                                      * np.exp2(-np.random.default_rng(i).integers(0, 30, s))).astype(f)) for i, s in enumerate(SHAPES)]
        m0 = decode(state["firstMoment"].toNumpy(), state["firstExponent"].toNumpy(), False).astype(f)
        v0 = decode(state["secondMoment"].toNumpy(), state["secondExponent"].toNumpy(), True).astype(f)
        held = opt.moments(state)
        assert same(held["firstMoment"].toNumpy() + f(0), m0 + f(0)) and same(held["secondMoment"].toNumpy(), v0 * v0)
        g = flat(SHAPES, [x.toNumpy() for x in grads]).reshape(-1, 256)
        m, v = m0 * f(0.9) + g * f(1 - 0.9), (v0 * v0) * f(0.999) + (g * g) * f(1 - 0.999)
        r = drawn(state, g.size)
        new = opt.fusedStep(params, grads, state)
        codes, exponents = encode(m, False, r[0])
        assert np.array_equal(new["state"]["firstExponent"].toNumpy(), exponents)
        assert np.array_equal(new["state"]["firstMoment"].toNumpy(), codes)
        held_m = codes & 127
        codes, exponents = encode(np.sqrt(v), True, r[1])
        codes = np.maximum(codes, np.minimum(held_m, 1))  # (no root of zero under a first moment that is not)
        assert np.array_equal(new["state"]["secondExponent"].toNumpy(), exponents)
        assert np.array_equal(new["state"]["secondMoment"].toNumpy(), codes)
        assert int(new["state"]["draws"].toNumpy()[0]) == -6 + t
        # the parameters step from the moments before their rounding: those of 32 bits
        wide = opt.initFusedState(params)
        wide.update(firstMoment=held["firstMoment"], secondMoment=held["secondMoment"], beta1Power=state["beta1Power"],
                    beta2Power=state["beta2Power"])
        for a, b, old in zip(opt.fusedStep(params, grads, wide)["parameters"], new["parameters"], params):
            a, b, old = (x.toNumpy().astype(np.float64) for x in (a, b, old))
            # (at most 24 roundings of the step either way, and the parameter's own)
            assert (np.abs(a - b) <= 24 * U * (np.abs(a - old) + np.abs(old)) + 2 * HALF[dtype] * np.abs(a)).all()
        params, state = new["parameters"], new["state"]


def test_8_bit_rounding_favours_neither_side():
    """The mean of many roundings of one value is the value: off by at most 5 deviations of a half step a draw, and the
    drawn bits' own 2^-17 of a step.  A second moment that is only kept decays though it moves by 1 / 1000 a step."""
    n, opt = 256 * 4096, Optimizer.adamW(0.0, 0.0, 0.999, 1e-8, 0.0)
    x = np.full(n, 1.3, np.float32)
    x[::256] = 1.9  # the block's largest
    p = CudaArray.zeros([n])
    state = opt.fusedStep([p], [CudaArray.fromNumpy(x)], opt.initFusedState([p], bits=8, seed=3))["state"]
    m = opt.moments(state)["firstMoment"].toNumpy().astype(np.float64).reshape(-1)[x < 1.5]
    assert abs(m.mean() - np.float32(1.3)) <= 0.125 * (5 * 0.5 / math.sqrt(m.size) + 2.0 ** -17)
    assert set(np.unique(m)) == {1.25, 1.375}
    start = opt.moments(state)["secondMoment"].toNumpy().astype(np.float64).mean()
    zero = CudaArray.zeros([n])
    for _ in range(100):
        state = opt.fusedStep([p], [zero], state)["state"]
    end = opt.moments(state)["secondMoment"].toNumpy().astype(np.float64).mean()
    # the root is kept in the mean, so the square grows by the rounding's variance: below (1 / 16)^2 / 4 of it a step
    # that rounds, which few do; 0.999^100 = 0.905
    assert 0.85 < end / start < 0.96


def test_8_bit_steps_of_small_gradients():
    """A gradient of 1e-7 of its block's largest rounds to zero or to the smallest code, its first moment and its root each
    for themselves.  A first moment that is held steps by at most 0.92 of its smallest code, 2^-9 / 128 of the block's
    largest, over a root of at least sqrt(0.999) of its own, 2^-10 / 256 of the largest: 3.7 times the largest element's
    quotient.  That is 1 but for the codes' roundings, by 1 / 8 and 1 / 16 a step: after 20 steps m is at most 2.6 times
    what it should be (0.1 sum 1.0125^k / (1 - 0.9^20)), the root 0.3 times (16 / 17)^20.  3.7 * 2.6 / 0.3 = 32 rates; with
    roots of zero it would be 1e-6 / (0.03 * 1e-7) and more."""
    n, opt = 256 * 512, Optimizer.adamW(1.0, 0.9, 0.999, 1e-12, 0.0)
    g = np.full(n, 1e-7, np.float32)
    g[::256] = 1.0
    grad, p = CudaArray.fromNumpy(g), CudaArray.zeros([n])
    state, seen = opt.initFusedState([p], bits=8, seed=11), 0
    for _ in range(20):
        new = opt.fusedStep([p], [grad], state)
        step = (new["parameters"][0] - p).toNumpy()[g < 1]
        assert np.abs(step).max() < 32
        p, state = new["parameters"][0], new["state"]
        m, v = (opt.moments(state)[x].toNumpy().reshape(-1)[g < 1] for x in ("firstMoment", "secondMoment"))
        assert not ((m != 0) & (v == 0)).any()
        seen += int((m != 0).sum())
    assert seen > 0


def test_8_bit_without_epsilon():
    """An element that never had a gradient stays, whatever epsilon is."""
    p = CudaArray.fromNumpy(np.arange(600, dtype=np.float32))
    for epsilon in (0.0, 1e-40, 1e-300):
        opt = Optimizer.adamW(0.01, 0.9, 0.999, epsilon, 0.0)
        got = opt.fusedStep([p], [CudaArray.zeros([600])], opt.initFusedState([p], bits=8))["parameters"][0]
        assert same(got.toNumpy(), p.toNumpy())


# ------------------------------------------------------------- the calls
def test_more_tensors_than_a_launch_takes_and_views():
    opt = Optimizer.adamW(0.01)
    base = made((400, 40), "float32", 1)
    params = [base.slice([i, 400, 7], ":").swapaxes(0, 1) if i % 2 else base.slice([i, i + 3]) for i in range(150)]
    grads = [made(p.getShape(), "float32", 7 + i) for i, p in enumerate(params)]
    want = opt.step(params, grads, opt.initState(params))
    got = opt.fusedStep(params, grads, opt.initFusedState(params))
    assert all(same(a.toBits(), b.toBits()) for a, b in zip(want["parameters"], got["parameters"]))
    master = opt.initFusedState(params, master=True)["master"].toNumpy()
    assert same(flat([p.getShape() for p in params], [p.toNumpy() for p in params]).reshape(-1, 256), master)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_plan_steps_as_the_calls_do(bits):
    opt = Optimizer.adamW(0.01)
    shapes = [(33, 20), (20,), (300,)]
    names = ["firstMoment", "secondMoment", "beta1Power", "beta2Power"] + (["firstExponent", "secondExponent", "draws"] if bits == 8 else [])

    def body(rate, *tensors):
        p, g, s = tensors[:3], tensors[3:6], dict(zip(names, tensors[6:]), bits=bits)
        r = opt.fusedStep([x * 1.5 for x in p], list(g), s, rate)
        m = opt.moments(r["state"])
        return [*r["parameters"], *(r["state"][n] for n in names), m["firstMoment"], m["secondMoment"]]
    p = [made(s, "float32", i) for i, s in enumerate(shapes)]
    state = opt.initFusedState(p, bits=bits)
    ins = [CudaArray.full([1], 0.02), *p, *[made(s, "float32", 9 + i) for i, s in enumerate(shapes)], *(state[n] for n in names)]
    plan = Fusion.compile(body, ins)
    for _ in range(3):
        want = [t.toBits() for t in body(*ins)]
        out = plan.run(*ins)
        assert all(same(a, b.toBits()) for a, b in zip(want, out))
        ins = [ins[0], *[t.copy() for t in out[:3]], *ins[4:7], *[t.copy() for t in out[3:3 + len(names)]]]


@pytest.mark.parametrize("bits", [32, 8])
def test_new_values_in_the_old_ones_place(bits):
    """The C entry takes results that are its operands."""
    opt = Optimizer.adamW(0.01)
    p, g = made((700,), "bfloat16", 1), made((700,), "bfloat16", 2)
    state = opt.initFusedState([p], bits=bits, master=True)
    want = opt.fusedStep([p], [g], state)
    at = lambda t: _host.load().phpt_device_pointer(t._h)  # noqa: E731
    d, t, fresh = _abi.PtAdamwDesc(), _abi.PtAdamwTensor(), [CudaArray.zeros([1]) for _ in range(2)] + [CudaArray.zeros([1], "int32")]
    values = dict(bits=bits, beta1=0.9, beta2=0.999, epsilon=1e-8, weight_decay=0.01, rate_value=0.01,
                  power1=at(state["beta1Power"]), power2=at(state["beta2Power"]), new_power1=at(fresh[0]), new_power2=at(fresh[1]))
    for name, field in (("firstMoment", "first"), ("secondMoment", "second"), ("master", "master"),
                        ("firstExponent", "first_exponent"), ("secondExponent", "second_exponent")):
        if name in state:
            values[field] = values["new_" + field] = at(state[name])
    if bits == 8:
        values.update(draws=at(state["draws"]), new_draws=at(fresh[2]))
    for n, v in values.items():
        setattr(d, n, v)
    t.param, t.grad, t.new_param, t.n, t.param_dtype, t.grad_dtype, t.decay = at(p), at(g), at(p), 700, _abi.BFLOAT16, _abi.BFLOAT16, 1
    _abi.check(_abi.load().pt_adamw(ctypes.byref(d), ctypes.byref(t), 1, None))
    assert same(p.toBits(), want["parameters"][0].toBits())
    assert all(same(state[n].toBits(), want["state"][n].toBits()) for n in state if n not in ("bits", "beta1Power", "beta2Power", "draws"))


def test_refusals():
    opt, p = Optimizer.adamW(), [CudaArray.zeros([5]), CudaArray.zeros([2, 3], "bfloat16")]
    s, s8 = opt.initFusedState(p), opt.initFusedState(p, bits=8)
    bad = [lambda: Optimizer.sgd().initFusedState(p), lambda: opt.initFusedState(p, bits=16), lambda: opt.initFusedState([]),
           lambda: opt.initFusedState([1]), lambda: opt.initFusedState(p, bits=8, seed=2 ** 40), lambda: opt.fusedStep([], [], s),
           lambda: Optimizer.sgd().fusedStep(p, p, s),
           lambda: opt.fusedStep(p, p[:1], s), lambda: opt.fusedStep(p[:1], p[:1], dict(s, firstMoment=None)), lambda: opt.fusedStep(p, p[::-1], s),
           lambda: opt.fusedStep([CudaArray.zeros([5], "float64")] * 2, p, s), lambda: opt.fusedStep(p, [CudaArray.zeros([5], "int32"), p[1]], s),
           lambda: opt.fusedStep(p[:1], p[:1], s), lambda: opt.fusedStep(p, p, dict(s, bits=8)), lambda: opt.fusedStep(p, p, dict(s8, bits=32)),
           lambda: opt.fusedStep(p, p, dict(s8, draws=CudaArray.zeros([2], "int32"))), lambda: opt.fusedStep(p, p, s, -1.0),
           lambda: opt.fusedStep(p, p, s, float("nan")), lambda: opt.fusedStep(p, p, s, "x"), lambda: opt.fusedStep(p, p, s, CudaArray.zeros([2])),
           lambda: opt.fusedStep(p, p, s, CudaArray.zeros([1], "float64")), lambda: opt.fusedStep(p, p, s, None, [True]),
           lambda: opt.moments({}), lambda: opt.moments(dict(s8, firstExponent=None)), lambda: opt.moments(dict(s, bits=8)),
           lambda: opt.moments(dict(s8, bits=4)), lambda: opt.moments(dict(s8, secondExponent=CudaArray.zeros([9], "int8"))),
           lambda: opt.fusedStep(p, p, s, None, [1, 0]), lambda: opt.fusedStep(p, p, dict(s, master=CudaArray.zeros([1, 256])))]
    for i, call in enumerate(bad):
        with pytest.raises(InvalidArgumentException):
            call()
            pytest.fail(f"call {i} was taken")
