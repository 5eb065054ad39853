"""CudaArray.gatedProjection and its gradients against float64, within bounds that count the roundings (U: half a step of
float32, h: of the operands' type)."""
import math

import numpy as np
import pytest

from phptensors import CudaArray, Fusion, InvalidArgumentException

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "float16", "bfloat16"]
ACTS = ["silu", "gelu", "relu", "sigmoid"]
U = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}
erf = np.vectorize(math.erf, otypes=[float])


def values(shape, dtype, seed, scale=1.0):
    x = np.random.default_rng(seed).standard_normal(shape).astype(np.float32) * np.float32(scale)
    a = CudaArray.fromNumpy(x, dtype)
    return a, a.toNumpy().astype(np.float64).reshape(shape)


def act(name, g):
    """(value, slope, the most that the slope and the slope's slope reach)."""
    if name == "relu":
        return np.maximum(g, 0.0), (g > 0).astype(float), 1.0, 0.0
    if name == "gelu":
        below, bell = 0.5 * (1 + erf(g / math.sqrt(2))), np.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        return g * below, below + g * bell, 1.13, 0.8
    s = 1 / (1 + np.exp(-g))
    if name == "sigmoid":
        return s, s * (1 - s), 0.25, 0.1
    return g * s, s * (1 + g * (1 - s)), 1.1, 0.5


def reference(x, gate, up, name, dtype, dh=None):
    """{name: (value, bound before the result's own rounding)}.  A product of K terms is off by at most K + 2 of U in the
    terms' magnitudes; an activation is computed within 16 U of its value and its argument's magnitude."""
    h, tiny = HALF[dtype], TINY[dtype]
    k = x.shape[1]
    g, u = x @ gate, x @ up
    g_off, u_off = (k + 2) * U * (np.abs(x) @ np.abs(gate)), (k + 2) * U * (np.abs(x) @ np.abs(up))
    a, slope, steep, curve = act(name, g)
    a_off = steep * g_off + 16 * U * (np.abs(a) + np.abs(a) * np.abs(g) + steep * np.abs(g))
    out = {"h": (a * u, np.abs(a) * u_off + a_off * (np.abs(u) + u_off) + U * np.abs(a * u))}
    if dh is None:
        return out
    # the gradient takes the products as they are kept, cut to 15 bits behind the first, and rounds dg and du to the type
    low, cut = (0.0, 0.0) if dtype == "float32" else (h, 2.0 ** -15)
    gk, uk = g_off * (1 + cut) + cut * np.abs(g), u_off * (1 + cut) + cut * np.abs(u)
    s_off = curve * gk + 32 * U * (1 + np.abs(g)) * (1 + np.abs(slope))
    ak = steep * gk + 16 * U * (np.abs(a) + np.abs(a) * np.abs(g) + steep * np.abs(g))
    if name == "relu":  # a product whose sign is not certain may fall on either side
        s_off = s_off + (np.abs(g) <= gk)
    dg, du = dh * u * slope, dh * a
    dg_off = np.abs(dh) * (uk * (np.abs(slope) + s_off) + np.abs(u) * s_off) + 2 * U * np.abs(dg)
    du_off = np.abs(dh) * ak + U * np.abs(du)
    dg_off, du_off = (off * (1 + low) + low * np.abs(d) + tiny for off, d in ((dg_off, dg), (du_off, du)))

    def product(a, a_off, b):
        n = a.shape[1]
        return a @ b, a_off @ np.abs(b) * (1 + (n + 2) * U) + (n + 2) * U * (np.abs(a) @ np.abs(b))
    p, q = product(dg, dg_off, gate.T), product(du, du_off, up.T)
    out["dx"] = p[0] + q[0], p[1] + q[1] + U * (np.abs(p[0]) + np.abs(q[0]))
    for n, d, off in (("dgate", dg, dg_off), ("dup", du, du_off)):
        v, o = product(d.T, off.T, x)
        out[n] = v.T, o.T
    return out


def close(got, want, what):
    dt = got.getDtype()
    x, off = want
    y = got.toNumpy().astype(np.float64).reshape(x.shape)
    far = np.abs(y - x) - (off * (1 + HALF[dt]) + HALF[dt] * np.abs(x) + TINY[dt])
    worst = float(np.where(np.isnan(far), np.inf, far).max()) if far.size else 0.0
    assert worst <= 0, (what, worst, np.unravel_index(far.argmax(), far.shape))


# rows, inner, outer: single tokens, few rows, tiles that end anywhere, contractions shorter than a stage and split ones
SHAPES = [(1, 1, 1), (1, 7, 5), (2, 64, 128), (1, 2048, 300), (5, 33, 129), (16, 100, 256), (17, 31, 24), (32, 500, 1000), (33, 64, 128),
          (40, 1, 8), (64, 72, 136), (50, 300, 77), (100, 37, 3), (129, 8, 7), (130, 200, 260), (257, 65, 129), (300, 129, 64), (128, 4096, 128),
          (513, 96, 640), (70, 2000, 40), (2100, 40, 24), (300, 48, 40), (390, 61, 130)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_both_directions(shape, dtype):
    m, k, f = shape
    name = ACTS[(m + k + f) % 4]
    (x, xv), (a, av), (b, bv) = values((m, k), dtype, 1), values((k, f), dtype, 2, k ** -0.5), values((k, f), dtype, 3, k ** -0.5)
    plain = x.gatedProjection(a, b, name)
    for t in (x, a, b):
        t.requiresGrad()
    h = x.gatedProjection(a, b, name)
    assert np.array_equal(plain.toBits(), h.toBits()) and h.getDtype() == dtype and h.getShape() == [m, f]
    for up in ("same", "float32"):
        g, gv = values((m, f), dtype if up == "same" else "float32", 4)
        if up == "float32" and dtype == "float32":
            continue
        for t in (x, a, b):
            t.zeroGrad()
        if up == "same":
            h.backward(g, retainGraph=True)
        else:
            (h * g).sum().backward()
        want = reference(xv, av, bv, name, dtype, gv)
        close(h, want["h"], "h")
        for t, n in ((x, "dx"), (a, "dgate"), (b, "dup")):
            close(t.grad(), want[n], n)
            assert t.grad().getDtype() == dtype


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("shape", [(1024, 512, 1024), (600, 1024, 2056), (2048, 264, 520)], ids=str)
def test_many_tiles(shape, dtype):
    test_both_directions(shape, dtype)


@pytest.mark.parametrize("shape", [(2048, 640, 2048), (2500, 1004, 1000)], ids=str)
def test_large_float32(shape):
    """Past 2.5e9 multiplications for a matrix, where the gradients go another way."""
    test_both_directions(shape, "float32")


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_activations_over_their_range(name, dtype):
    """A gate of one element: products from -200 to 200 and their neighbourhood of zero."""
    xs = np.concatenate([np.linspace(-200, 200, 501), np.linspace(-4, 4, 301), [0.0, -0.0, 1e-6, -1e-6]]).astype(np.float32)
    for rows in (xs[:, None], xs[:24, None]):
        x = CudaArray.fromNumpy(rows, dtype).requiresGrad()
        xv = x.toNumpy().astype(np.float64)
        one, two = CudaArray.fromNumpy(np.full((1, 8), 1.0, np.float32), dtype), CudaArray.fromNumpy(np.full((1, 8), 0.5, np.float32), dtype)
        h = x.gatedProjection(one, two, name)
        h.backward(CudaArray.ones([len(rows), 8], dtype))
        want = reference(xv, np.ones((1, 8)), np.full((1, 8), 0.5), name, dtype, np.ones((len(rows), 8)))
        close(h, want["h"], "h")
        close(x.grad(), want["dx"], "dx")


def test_gradient_against_differences():
    x, a, b, g = (values(s, "float32", i, 0.5)[1] for i, s in enumerate([(6, 9), (9, 7), (9, 7), (6, 7)]))
    x, a, b, g = (np.round(v * 2 ** 12) / 2 ** 12 for v in (x, a, b, g))
    step = 2.0 ** -7
    for name in ("silu", "gelu", "sigmoid"):
        leaves = [CudaArray.fromNumpy(v.astype(np.float32)).requiresGrad() for v in (x, a, b)]
        leaves[0].gatedProjection(leaves[1], leaves[2], name).backward(CudaArray.fromNumpy(g.astype(np.float32)))
        for i, v in enumerate((x, a, b)):
            d = np.random.default_rng(i).integers(-1, 2, v.shape)

            def loss(sign):
                moved = [w + sign * step * d if j == i else w for j, w in enumerate((x, a, b))]
                h = CudaArray.fromNumpy(moved[0].astype(np.float32)).gatedProjection(
                    *(CudaArray.fromNumpy(w.astype(np.float32)) for w in moved[1:]), name)
                return float((h.toNumpy().astype(np.float64) * g).sum())
            slope = (loss(1) - loss(-1)) / (2 * step)
            want = float((leaves[i].grad().toNumpy().astype(np.float64) * d).sum())
            # 42 results of at most 20, each off by 60 U, over 2 steps; and a third derivative of at most 9^3 times 6 a result
            assert abs(slope - want) <= 42 * 20 * 60 * U / step + step ** 2 / 6 * 42 * 6 * 9 ** 3 * 0.5, (name, i, slope, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_leading_axes_views_and_wanted_gradients(dtype):
    (x, xv), (w, wv) = values((3, 4, 24), dtype, 1), values((40, 24), dtype, 2, 0.2)
    gate, up = w.slice([0, 20]).transpose(), w.slice([20, 40]).transpose()
    want = x.reshape([12, 24]).gatedProjection(gate.copy(), up.copy()).toBits()
    got = x.gatedProjection(gate, up)
    assert got.getShape() == [3, 4, 20] and np.array_equal(got.toBits().reshape(12, 20), want)
    assert np.array_equal(x.swapaxes(0, 1).gatedProjection(gate, up).toBits(), want.reshape(3, 4, 20).swapaxes(0, 1))
    assert x.slice(0, 0).gatedProjection(gate, up).getShape() == [20]
    # each operand's gradient alone is what it is among all
    g = values((3, 4, 20), dtype, 3)[0]
    leaves = [x, gate.copy(), up.copy()]
    for t in leaves:
        t.requiresGrad()
    leaves[0].gatedProjection(*leaves[1:]).backward(g)
    every = [t.grad().toBits() for t in leaves]
    for i, t in enumerate(leaves):
        for o in leaves:
            o.requiresGrad(o is t).zeroGrad()
        leaves[0].gatedProjection(*leaves[1:]).backward(g)
        assert np.array_equal(t.grad().toBits(), every[i]) and all(o.grad() is None for o in leaves if o is not t)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(0, 8, 8), (3, 0, 8), (3, 8, 0), (40, 0, 16)], ids=str)
def test_empty(shape, dtype):
    m, k, f = shape
    x, a, b = (CudaArray.ones(s, dtype).requiresGrad() for s in ((m, k), (k, f), (k, f)))
    h = x.gatedProjection(a, b, "sigmoid")
    h.backward(CudaArray.ones([m, f], dtype))
    assert h.getShape() == [m, f] and not h.toNumpy().any()
    for t in (x, a, b):
        assert t.grad().getShape() == t.getShape() and not t.grad().toNumpy().any()


@pytest.mark.parametrize("shape", [(3, 90, 40), (70, 90, 40), (70, 91, 41)], ids=str)
def test_what_is_not_finite_stays_in_its_row_and_column(shape):
    """Edges re-read rows and columns, and the end of a contraction meets other rows' values: none may leak."""
    m, k, f = shape
    for dtype in DTYPES:
        x, a = np.ones((m, k), np.float32), np.ones((k, f), np.float32) * 0.1
        x[m - 1, 0], x[0, k - 1], a[0, f - 1] = np.nan, np.inf, np.inf
        h = CudaArray.fromNumpy(x, dtype).gatedProjection(CudaArray.fromNumpy(a, dtype), CudaArray.fromNumpy(a, dtype), "relu")
        finite = np.ones((m, f), bool)
        finite[[0, m - 1]] = finite[:, f - 1] = False
        assert np.array_equal(np.isfinite(h.toNumpy().astype(np.float32)), finite), dtype


def test_runs_give_the_same_bits_and_plans_the_eager_ones():
    for dtype, shape in (("bfloat16", (200, 1024, 96)), ("float16", (9, 520, 72)), ("float32", (50, 64, 48))):
        m, k, f = shape

        def forward(x, a, b):
            return [x.gatedProjection(a, b, "gelu")]

        def step(x, a, b):
            for t in (x, a, b):
                t.requiresGrad()
            h = x.gatedProjection(a, b)
            (h * h).sum().backward()
            out = [h.detach(), x.grad(), a.grad(), b.grad()]
            for t in (x, a, b):
                t.requiresGrad(False).zeroGrad()
            return out

        def inputs(seed):
            return [values(s, dtype, seed * 10 + i, k ** -0.25)[0] for i, s in enumerate([(m, k), (k, f), (k, f)])]
        for body, graph in ((forward, True), (step, False)):
            plan = Fusion.compile(body, inputs(0), cudaGraph=graph)
            for seed in (1, 2, 3, 1):
                ins = inputs(seed)
                want = [t.toBits() for t in body(*ins)]
                for _ in range(2):
                    assert all(np.array_equal(p, q.toBits()) for p, q in zip(want, plan.run(*ins)))
            if graph:
                assert plan.getStats()["graphLaunches"] >= 6


def test_refusals():
    x, w = CudaArray.zeros([4, 8]), CudaArray.zeros([8, 6])
    bad = [lambda: x.gatedProjection(w, 3), lambda: x.gatedProjection(w, CudaArray.zeros([8, 5])),
           lambda: x.gatedProjection(CudaArray.zeros([7, 6]), CudaArray.zeros([7, 6])), lambda: x.gatedProjection(w, w, "tanh"),
           lambda: x.gatedProjection(w, w, None), lambda: x.gatedProjection(w, CudaArray.zeros([8, 6], "float16")),
           lambda: CudaArray.zeros([4, 8], "float64").gatedProjection(CudaArray.zeros([8, 6], "float64"), CudaArray.zeros([8, 6], "float64")),
           lambda: x.gatedProjection(w.reshape([8, 6, 1]), w.reshape([8, 6, 1])), lambda: CudaArray.zeros([]).gatedProjection(w, w)]
    for i, call in enumerate(bad):
        with pytest.raises(InvalidArgumentException):
            call()
            pytest.fail(f"call {i} was taken")
