"""CudaArray.rotary and its gradients against float64, within bounds that count the roundings (u: half a step of
float32, h: of the result's type)."""
import math

import numpy as np
import pytest

from phptensors import CudaArray, Fusion, InvalidArgumentException, Rotary

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "float16", "bfloat16"]
U = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}  # smallest steps round absolutely
EPS = 1e-6


def values(shape, dtype, seed, scale=1.0, shift=0.0):
    x = np.random.default_rng(seed).standard_normal(shape).astype(np.float32) * np.float32(scale) + np.float32(shift)
    a = CudaArray.fromNumpy(x, dtype)
    return a, a.toNumpy().astype(np.float64).reshape(shape)


def frequencies(part, base=10000.0, factor=1.0, context=None, low=1.0, high=32.0):
    f = base ** (-np.arange(0, part, 2) / part)
    if context is None:
        return f / factor
    keep = np.clip((context * f / (2 * math.pi) - low) / (high - low), 0.0, 1.0)
    return f * keep + f / factor * (1.0 - keep) if factor != 1.0 else f


def turned(x, angle, magnitude, interleaved, back=False):
    """x [.., heads, size] turned by angle [.., part / 2], and by the same with every product's magnitude."""
    part = 2 * angle.shape[-1]
    c, s = magnitude * np.cos(angle)[..., None, :], magnitude * np.sin(angle)[..., None, :] * (-1.0 if back else 1.0)
    p, q = (np.s_[..., 0:part:2], np.s_[..., 1:part:2]) if interleaved else (np.s_[..., :part // 2], np.s_[..., part // 2:part])
    y, most = x.copy(), np.abs(x)
    y[p], y[q] = x[p] * c - x[q] * s, x[p] * s + x[q] * c
    both = abs(magnitude) * (np.abs(x[p]) + np.abs(x[q]))
    most[p], most[q] = both, both
    return y, most


def reference(x, w, angle, magnitude, interleaved, g=None):
    """{name: (value, bound before its rounding)}.  A head's sum of squares takes at most 16 products in a lane and 6
    exchanges; with the mean, the root and the division r is off by 28 u, a product of two cosines and sines (u each,
    rounded from double) by 6 u more."""
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) if w is not None else 1.0
    n = x * r * (1.0 if w is None else w)
    y, most = turned(n, angle, magnitude, interleaved)
    out = {"y": (y, (6 + (32 if w is not None else 0)) * U * most)}
    if g is None:
        return out
    dn, dmost = turned(g, angle, magnitude, interleaved, back=True)
    if w is None:
        out["dx"] = (dn, 6 * U * dmost)
        return out
    u, h, hmost = x * r, dn * w, dmost * np.abs(w)
    mean, mmost = (h * u).mean(-1, keepdims=True), (hmost * np.abs(u)).mean(-1, keepdims=True)
    out["dx"] = (r * (h - u * mean), 128 * U * r * (hmost + np.abs(u) * mmost))
    rows = int(np.prod(x.shape[:-1]))
    axes = tuple(range(x.ndim - 1))
    out["dw"] = ((dn * u).sum(axes), (64 + rows) * U * (dmost * np.abs(u)).sum(axes))
    return out


def close(got, want, what):
    dt = got.getDtype()
    x, off = want
    y = got.toNumpy().astype(np.float64).reshape(x.shape)
    far = np.abs(y - x) - (off * (1 + HALF[dt]) + HALF[dt] * np.abs(x) + TINY[dt])
    worst = float(np.where(np.isnan(far), np.inf, far).max()) if far.size else 0.0
    assert worst <= 0, (what, worst, np.unravel_index(far.argmax(), far.shape))


# tokens (or sequences and tokens), heads, key heads, size, part
SHAPES = [((1,), 1, 1, 2, 2), ((1,), 4, 2, 128, 128), ((7,), 3, 1, 64, 32), ((33,), 8, 2, 80, 20), ((5, 13), 2, 2, 96, 96),
          ((3, 1), 5, 5, 7, 6), ((2, 9), 1, 3, 256, 256), ((40,), 2, 1, 255, 254), ((17,), 2, 2, 129, 2), ((300,), 6, 3, 48, 16),
          ((2, 2300), 2, 1, 32, 32), ((4, 1), 70, 7, 40, 24)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_both_directions(shape, norm, interleaved, dtype):
    lead, heads, kv, size, part = shape
    plan = Rotary(part, interleaved=interleaved, magnitude=1.25)
    at = np.random.default_rng(5).integers(-50, 100000, lead).astype(np.int32)
    angle = at[..., None].astype(np.float64) * frequencies(part)
    q, k = values((*lead, heads, size), dtype, 1, 2.0, 0.5), values((*lead, kv, size), dtype, 2, 2.0, -0.5)
    scales = [values((size,), dtype, 3 + i, 0.2, 1.0) if norm else (None, None) for i in range(2)]
    grads = [values((*lead, n, size), dtype, 6 + i, 0.5) for i, n in enumerate((heads, kv))]
    leaves = [t for t in (q[0], k[0], scales[0][0], scales[1][0]) if t is not None]
    for t in leaves:
        t.requiresGrad()
    got = q[0].rotary(plan, CudaArray.fromNumpy(at), k[0], scales[0][0], scales[1][0], EPS)
    for y, g in zip(got, grads):
        y.backward(g[0])
    for y, x, w, g in zip(got, (q, k), scales, grads):
        want = reference(x[1], w[1], angle, 1.25, interleaved, g[1])
        close(y, want["y"], "y")
        close(x[0].grad(), want["dx"], "dx")
        assert y.getDtype() == x[0].grad().getDtype() == dtype
        if norm:
            close(w[0].grad(), want["dw"], "dw")


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_pass_of_both_gradients_and_float32_upstream(dtype):
    """A loss of queries and keys together: float32 upstream gradients, one gradient call."""
    plan, size = Rotary(24), 40
    (q, qx), (k, kx), (w, wx) = values((11, 4, size), dtype, 1), values((11, 2, size), dtype, 2), values((size,), dtype, 3, 0.1, 1)
    (a, ax), (b, bx) = values((11, 4, size), "float32", 4), values((11, 2, size), "float32", 5)
    for t in (q, k, w):
        t.requiresGrad()
    x, y = q.rotary(plan, None, k, w, w, EPS)
    ((x * a).sum() + (y * b).sum()).backward()
    angle = np.arange(11)[:, None] * frequencies(24)
    wants = [reference(t, wx, angle, 1.0, False, g) for t, g in ((qx, ax), (kx, bx))]
    close(q.grad(), wants[0]["dx"], "dq")
    close(k.grad(), wants[1]["dx"], "dk")
    # the shared scale takes both, each rounded to its type before the sum
    total = wants[0]["dw"][0] + wants[1]["dw"][0]
    off = sum(t["dw"][1] + HALF[dtype] * np.abs(t["dw"][0]) for t in wants) + U * np.abs(total)
    close(w.grad(), (total, off), "dw")


def test_gradient_against_differences():
    """Along random directions, in float64 of the values that the calls return for float32 inputs a step apart."""
    plan, size, h = Rotary(8, interleaved=True), 12, 2.0 ** -8
    x, w, g = values((5, 3, size), "float32", 1)[1], values((size,), "float32", 2, 0.2, 1)[1], values((5, 3, size), "float32", 3)[1]
    a, s = CudaArray.fromNumpy(x.astype(np.float32)).requiresGrad(), CudaArray.fromNumpy(w.astype(np.float32)).requiresGrad()
    a.rotary(plan, scale=s, epsilon=EPS).backward(CudaArray.fromNumpy(g.astype(np.float32)))

    def loss(x, w):
        y = CudaArray.fromNumpy(x.astype(np.float32)).rotary(plan, scale=CudaArray.fromNumpy(w.astype(np.float32)), epsilon=EPS)
        return float((y.toNumpy().astype(np.float64) * g).sum())
    for seed in range(4):
        # directions of whole steps, so that x + h d is a float32 number
        r = np.random.default_rng(seed)
        dx, dw = r.integers(-1, 2, x.shape), r.integers(-1, 2, w.shape)
        xr, wr = np.round(x * 2 ** 14) / 2 ** 14, np.round(w * 2 ** 14) / 2 ** 14
        slope = (loss(xr + h * dx, wr + h * dw) - loss(xr - h * dx, wr - h * dw)) / (2 * h)
        want = float((a.grad().toNumpy() * dx).sum() + (s.grad().toNumpy() * dw).sum())
        # the third derivative's part of a central difference, h^2 / 6 of sums whose terms are below about 60, and
        # rounding of the losses: 180 terms off by 40 u each, over 2 h
        assert abs(slope - want) <= h * h * 60 * 6 + 180 * 3 * 40 * U / h + 180 * 2.0 ** -13, (slope, want)


@pytest.mark.parametrize("scaling", [dict(factor=4.0), dict(factor=8.0, context=2048), dict(base=500000.0),
                                     dict(factor=2.0, context=100, low=0.5, high=3.0)], ids=str)
def test_scaled_frequencies_and_far_positions(scaling):
    """Angles are exact to 2^-22 turns at positions up to 2^30: the bound of a float64 product, not of a float32 one."""
    at = np.array([0, 1, 2047, 10 ** 6, 2 ** 24 + 1, 2 ** 30, -(2 ** 30)], np.int32)
    x, xv = values((len(at), 2, 64), "float32", 1)
    got = x.rotary(Rotary(64, **scaling), CudaArray.fromNumpy(at))
    angle = at[:, None].astype(np.float64) * frequencies(64, **scaling)
    y, most = turned(xv, angle, 1.0, False)
    # both sides round position * frequency to 53 bits, by two and three roundings of at most 2^-53 of it
    close(got, (y, most * (6 * U + 5 * 2.0 ** -53 * np.abs(angle).max(1)[:, None, None])), "y")


def test_given_frequencies_and_shared_positions():
    f = [1.0, 0.25, -0.125]
    at = np.array([3, 1, 4, 1, 5], np.int32)
    x, xv = values((2, 5, 3, 6), "float32", 1)
    want, most = turned(xv, np.broadcast_to(at[:, None] * np.array(f), (2, 5, 3)), 1.0, True)
    got = x.rotary(Rotary(6, interleaved=True, frequencies=f), CudaArray.fromNumpy(at))
    close(got, (want, 6 * U * most), "y")
    # the same positions through strides, and a sequence's own
    many = CudaArray.fromNumpy(np.stack([at, at * 0]).T.copy()).transpose().slice([0, 1]).broadcastTo([2, 5])
    assert np.array_equal(got.toBits(), x.rotary(Rotary(6, interleaved=True, frequencies=f), many).toBits())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_heads(dtype):
    """Queries and keys as slices of one projection, and heads in front of tokens; a head's elements apart are packed."""
    plan, size = Rotary(32), 32
    whole, wv = values((2, 21, 6, size), dtype, 1)
    (s, _), gq, gk = values((size,), dtype, 2, 0.1, 1.0), values((2, 21, 4, size), dtype, 3)[0], values((2, 21, 1, size), dtype, 4)[0]

    def both(q, k):
        for t in (q, k, s):
            t.requiresGrad().zeroGrad()
        out = q.rotary(plan, None, k, s, s)
        out[0].backward(gq)
        out[1].backward(gk)
        return [t.toBits() for t in (*out, q.grad(), k.grad(), s.grad())]
    parts = [whole.slice(":", ":", [0, 4]), whole.slice(":", ":", [4, 5])]
    want = both(*(p.copy() for p in parts))
    assert all(np.array_equal(a, b) for a, b in zip(want, both(*parts)))
    swapped = [p.swapaxes(1, 2).copy().swapaxes(1, 2) for p in parts]
    assert all(np.array_equal(a, b) for a, b in zip(want, both(*swapped)))
    apart = [p.swapaxes(2, 3).copy().swapaxes(2, 3) for p in parts]
    assert all(np.array_equal(a, b) for a, b in zip(want, both(*apart)))


@pytest.mark.parametrize("shape", [(0, 2, 8), (3, 0, 8), (0, 4, 2, 8), (2, 0, 2, 8)], ids=str)
def test_nothing_to_turn(shape):
    x, s = CudaArray.zeros(shape).requiresGrad(), CudaArray.ones([8]).requiresGrad()
    y = x.rotary(Rotary(8), scale=s)
    y.backward(CudaArray.zeros(shape))
    assert y.getShape() == x.grad().getShape() == list(shape) and not s.grad().toNumpy().any()


def test_rows_past_one_turn_of_the_blocks():
    """More tokens than the gradient's blocks take in one turn, and a token group that ends inside."""
    x, xv = values((70001, 1, 2), "float32", 1)
    s, sv = values((2,), "float32", 2, 0.1, 1.0)
    g, gv = values((70001, 1, 2), "float32", 3)
    x.requiresGrad(), s.requiresGrad()
    y = x.rotary(Rotary(2), scale=s, epsilon=EPS)
    y.backward(g)
    want = reference(xv, sv, np.arange(70001)[:, None] * np.ones(1), 1.0, False, gv)
    close(y, want["y"], "y"), close(x.grad(), want["dx"], "dx"), close(s.grad(), want["dw"], "dw")


# few heads of many tokens, several of which share a wave: groups of heads that fill it or not, last groups that end inside
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("shape", [((4097,), 1, 1, 2, 2), ((3, 1401), 2, 1, 20, 8), ((2, 2200), 1, 1, 64, 64), ((4500,), 3, 1, 7, 6),
                                   ((4099,), 2, 2, 32, 30), ((4200,), 5, 1, 16, 16), ((4100,), 1, 3, 128, 96)], ids=str)
def test_tokens_that_share_a_wave(shape, norm, interleaved, dtype):
    test_both_directions(shape, norm, interleaved, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_together_and_in_parts(dtype):
    """Many tokens' values and gradients, both sides' in one call, are those of parts of them, which go another way."""
    plan, n = Rotary(12), 4500
    q, k, s = values((n, 3, 18), dtype, 1)[0], values((n, 1, 18), dtype, 2)[0], values((18,), dtype, 3, 0.1, 1.0)[0]
    a, b = values((n, 3, 18), dtype, 4)[0], values((n, 1, 18), dtype, 5)[0]

    def run(lo, hi, at):
        x, y = (t.slice([lo, hi]).copy().requiresGrad() for t in (q, k))
        u, v = x.rotary(plan, at, y, s, s, EPS)
        ((u * a.slice([lo, hi])).sum() + (v * b.slice([lo, hi])).sum()).backward()
        return [t.toBits() for t in (u, v, x.grad(), y.grad())]
    whole = run(0, n, None)
    for lo, hi in ((0, 1500), (1500, 3000), (3000, n)):
        part = run(lo, hi, CudaArray.fromNumpy(np.arange(lo, hi, dtype=np.int32)))
        assert all(np.array_equal(w[lo:hi], p) for w, p in zip(whole, part))


def test_no_norm_leaves_what_is_not_finite_in_its_pair():
    x = np.zeros((2, 1, 8), np.float32)
    x[0, 0, 1], x[1, 0, 7] = np.nan, np.inf
    y = CudaArray.fromNumpy(x).rotary(Rotary(4), CudaArray.fromNumpy(np.array([1, 2], np.int32))).toNumpy()
    assert np.array_equal(np.isfinite(y), np.array([[[1, 0, 1, 0, 1, 1, 1, 1]], [[1] * 7 + [0]]], bool))


def test_plans_follow_positions():
    """A captured graph of the forward pass alone, and a plan with gradients, give the eager bits on other inputs."""
    plan = Rotary(16)

    def forward(x, s, at):
        return [x.rotary(plan, at, scale=s)]

    def step(x, s, at, k):
        for t in (x, s, k):
            t.requiresGrad()
        a, b = x.rotary(plan, at, k, s, s)
        y = a.rotary(plan, at)
        (y.sum() + (b * b).sum()).backward()
        out = [t.detach() for t in (a, b, y)] + [t.grad() for t in (x, s, k)]
        for t in (x, s, k):
            t.requiresGrad(False).zeroGrad()
        return out
    for body, graph in ((forward, True), (step, False)):
        def inputs(seed):
            return [values((9, 3, 20), "float32", seed)[0], values((20,), "float32", seed + 50)[0],
                    CudaArray.fromNumpy(np.random.default_rng(seed).integers(0, 9999, 9).astype(np.int32)),
                    *([] if graph else [values((9, 1, 20), "float32", seed + 70)[0]])]
        compiled = Fusion.compile(body, inputs(0), cudaGraph=graph)
        for seed in (1, 2, 3, 1):
            ins = inputs(seed)
            want = [t.toBits() for t in body(*ins)]
            for _ in range(2):
                assert all(np.array_equal(a, b.toBits()) for a, b in zip(want, compiled.run(*ins)))
        if graph:
            assert compiled.getStats()["graphLaunches"] >= 6


def test_refusals():
    x, k = CudaArray.zeros([4, 2, 8]), CudaArray.zeros([4, 1, 8])
    plan, at = Rotary(8), CudaArray.zeros([4], "int32")
    bad = [lambda: Rotary(3), lambda: Rotary(0), lambda: Rotary(258), lambda: Rotary(8, base=0.0), lambda: Rotary(8, factor=0.0),
           lambda: Rotary(8, factor=float("nan")), lambda: Rotary(8, context=-1.0), lambda: Rotary(8, low=2.0, high=2.0),
           lambda: Rotary(8, frequencies=[1.0]), lambda: Rotary(4, frequencies=[1.0, float("inf")]),
           lambda: Rotary(8, magnitude=float("inf")),
           lambda: x.rotary(None), lambda: x.rotary(plan, 3), lambda: x.rotary(Rotary(10)), lambda: x.rotary(plan, CudaArray.zeros([3], "int32")),
           lambda: x.rotary(plan, CudaArray.zeros([4])), lambda: x.rotary(plan, at, CudaArray.zeros([3, 1, 8])),
           lambda: x.rotary(plan, at, CudaArray.zeros([4, 1, 10])), lambda: x.rotary(plan, at, CudaArray.zeros([4, 1, 8], "float16")),
           lambda: x.rotary(plan, at, scale=CudaArray.ones([4])), lambda: x.rotary(plan, at, scale=CudaArray.ones([8], "bfloat16")),
           lambda: x.rotary(plan, at, keyScale=CudaArray.ones([8])), lambda: x.rotary(plan, at, k, epsilon=0.0),
           lambda: x.rotary(plan, at, k, epsilon=1e-60), lambda: CudaArray.zeros([4, 8]).rotary(plan),
           lambda: CudaArray.zeros([4, 2, 8], "float64").rotary(plan), lambda: CudaArray.zeros([4, 2, 300]).rotary(plan)]
    for i, call in enumerate(bad):
        with pytest.raises(InvalidArgumentException):
            call()
            pytest.fail(f"call {i} was taken")
