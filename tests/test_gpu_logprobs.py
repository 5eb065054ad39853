"""CudaArray.logProbs and its gradients against float64, within bounds that
count the roundings (u: half a step of float32, h: of the gradient's type)."""
import numpy as np
import pytest

from phptensors import CudaArray, Fusion, _abi

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {"float32": U, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}


def scores(shape, dtype, seed, scale=2.5):
    a = CudaArray.fromNumpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float32) * np.float32(scale), dtype)
    return a, a.toNumpy().astype(np.float64).reshape(shape)


def reference(x, tokens):
    """{name: (value, bound)} of rows of finite scores or -inf, one finite at least.

    An exponential's argument (base 2) is off by one rounding of the maximum's product, which all of a row
    share, and one of its own: a factor of 1 +- e.  The sum of n of them adds n u."""
    rows, n = x.shape
    m = x.max(1, keepdims=True)
    gap = np.where(np.isneginf(x), 0.0, m - x)
    ex = np.where(np.isneginf(x), 0.0, np.exp(-gap))
    s = ex.sum(1, keepdims=True)
    p, lse = ex / s, m + np.log(s)
    e = 4 * U * (1 + np.minimum(gap, 200) + np.abs(m))
    s_rel = (p * e).sum(1, keepdims=True) + (n + 8) * U
    lse_off = s_rel + 6 * U * (np.abs(m) + np.abs(lse) + 1)
    t = (p * gap).sum(1, keepdims=True)
    ent = np.log(s) + t
    ent_off = (p * (gap + 1) * e).sum(1, keepdims=True) + (s_rel + (n + 8) * U) * (1 + t) + 8 * U * (np.abs(ent) + np.abs(m) + 1)
    lp = x - lse
    lp_off = lse_off + 6 * U * (np.where(np.isneginf(x), 0, np.abs(x)) + np.abs(m) + np.where(np.isneginf(lp), 0, np.abs(lp)))
    at = np.clip(tokens, 0, n - 1)
    one = np.arange(rows)
    named = tokens >= 0
    return {"p": p, "lp": (lp, lp_off), "entropy": (ent[:, 0], ent_off[:, 0]),
            "logProbs": (np.where(named, lp[one, at], 0.0), np.where(named, lp_off[one, at], 0.0))}


def near(got, want, what):
    x, off = want
    v = got.toNumpy().astype(np.float64).reshape(x.shape)
    same = np.isneginf(v) & np.isneginf(x)
    with np.errstate(invalid="ignore"):
        far = np.where(same, -1.0, np.abs(v - x) - off)
    assert not np.isnan(far).any() and (far.size == 0 or far.max() <= 0), (what, float(np.nanmax(far)))


def listed(x, top):
    """Indices of the largest, the lower index first among equals."""
    return np.argsort(-x, axis=1, kind="stable")[:, :top]


def check(a, x, tokens, top, dtype):
    got = a.logProbs(CudaArray.fromNumpy(tokens.astype(np.int32)), top=top)
    ref = reference(x, tokens)
    near(got["logProbs"], ref["logProbs"], "logProbs")
    near(got["entropy"], ref["entropy"], "entropy")
    if top:
        best = listed(x, top)
        assert np.array_equal(got["topTokens"].toNumpy(), best)
        at = np.arange(len(x))[:, None]
        near(got["topLogProbs"], (ref["lp"][0][at, best], ref["lp"][1][at, best]), "topLogProbs")


# widths around the packs, the turns of the blocks and the split; few rows and many
SIZES = [(1, 1), (3, 2), (5, 63), (2, 64), (70, 65), (9, 1000), (4, 2047), (3, 2048), (6, 2049), (600, 300), (520, 4099),
         (2, 8192), (7, 8191), (1, 20001), (2, 131072), (515, 2500)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,n", SIZES)
def test_values(rows, n, dtype):
    a, x = scores((rows, n), dtype, rows + n)
    tokens = np.random.default_rng(3).integers(-1, n, rows)
    for top in sorted({0, 1, min(5, n), min(20, n), min(64, n)}):
        check(a, x, tokens, top, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [40, 3000, 50000])
def test_equal_and_ordered_scores(dtype, n):
    """Many equal scores, rising and falling rows: the order of the alternatives is by index."""
    rng = np.random.default_rng(1)
    rows = [np.zeros(n), rng.integers(0, 3, n), np.arange(n) % 256, -(np.arange(n) % 256.0), np.arange(n)[::-1] % 7]
    a = CudaArray.fromNumpy(np.stack(rows).astype(np.float32), dtype)
    check(a, a.toNumpy().astype(np.float64), np.array([0, n - 1, -1, 5, 3]), min(n, 33), dtype)


def test_masked_scores():
    """-inf scores: no probability, last among the alternatives; a row of nothing else; NaN; an infinite score."""
    x = np.random.default_rng(2).standard_normal((7, 4500)).astype(np.float32)
    x[0, 1::2] = -np.inf
    x[1, :] = -np.inf
    x[1, 4100] = 0.25
    x[2, :4400] = -np.inf
    a = CudaArray.fromNumpy(x[:3])
    check(a, x[:3].astype(np.float64), np.array([1, 4100, 4450]), 8, "float32")
    lowest = np.where(np.isneginf(x), np.finfo(np.float32).min, x)  # the type's lowest value as the mask
    check(CudaArray.fromNumpy(lowest[:3]), lowest[:3].astype(np.float64), np.array([0, 4100, 4450]), 8, "float32")
    # a row of the lowest value alone is a row of equal scores
    flat = CudaArray.fromNumpy(np.full((1, 3000), np.finfo(np.float32).min, np.float32)).requiresGrad()
    got = flat.logProbs(CudaArray.fromNumpy(np.array([7], np.int32)), top=2)
    got["logProbs"].backward(CudaArray.ones([1]))
    want = np.full((1, 3000), -1 / 3000)
    want[0, 7] += 1
    near(flat.grad(), (want, np.abs(want) * 4000 * U), "dx of equal scores")  # a sum of 3000 terms
    assert abs(got["entropy"].item() - np.log(3000)) < 4000 * U * 9 and got["topTokens"].toNumpy().tolist() == [[0, 1]]
    x[3, :] = -np.inf
    x[4, 17] = np.nan
    x[5, 18] = np.inf
    x[6, 2:] = np.nan
    for width in (4500, 30):
        b = CudaArray.fromNumpy(np.ascontiguousarray(x[:, :width])).requiresGrad()
        got = b.logProbs(CudaArray.fromNumpy(np.zeros(7, np.int32)), top=4)
        lp, ent, tv, ti = (got[k].toNumpy() for k in ("logProbs", "entropy", "topLogProbs", "topTokens"))
        assert np.isneginf(lp[3]) and ent[3] == 0 and np.isneginf(tv[3]).all() and ti[3].tolist() == [0, 1, 2, 3]
        assert np.isnan(lp[4]) and np.isnan(ent[4]) and np.isnan(tv[4]).all() and 17 not in ti[4]
        assert np.isnan(lp[5]) and np.isnan(ent[5]) and ti[5, 0] == 18
        assert np.isnan(lp[6]) and ti[6].tolist() == sorted([0, 1], key=lambda i: -x[6, i]) + [-1, -1]
        (got["logProbs"] + got["entropy"] + got["topLogProbs"].sum(1)).backward(CudaArray.ones([7]))
        g = b.grad().toNumpy()
        assert not g[3].any() and np.isnan(g[4]).any() and np.isnan(g[6]).any()
    # a token past the classes is not looked up
    c = scores((2, 10), "float32", 1)[0]
    lp = c.logProbs(CudaArray.fromNumpy(np.array([10, 2 ** 31 - 1], np.int32)))["logProbs"].toNumpy()
    assert np.isnan(lp).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (70, 65), (9, 1000), (4, 2049), (600, 300), (520, 4099), (7, 20001),
                                    (1, 131072)])
def test_gradients(rows, n, dtype):
    a, x = scores((rows, n), dtype, 5)
    rng = np.random.default_rng(6)
    tokens = rng.integers(-1, n, rows)
    top = min(n, 6)
    ga, gh = (rng.standard_normal(rows).astype(np.float32) for _ in range(2))
    gu = rng.standard_normal((rows, top)).astype(np.float32)
    best = listed(x, top)
    tokens[::3] = best[::3, 0]  # some tokens are alternatives too
    ref = reference(x, tokens)
    p, (lp, lp_off), (ent, ent_off) = ref["p"], ref["lp"], ref["entropy"]
    at = np.arange(rows)
    t32 = CudaArray.fromNumpy(tokens.astype(np.int32))
    for use in ("a", "h", "u", "ahu"):
        g = np.where(tokens >= 0, ga, 0.0).astype(np.float64) if "a" in use else np.zeros(rows)
        h = gh.astype(np.float64) if "h" in use else np.zeros(rows)
        u = gu.astype(np.float64) if "u" in use else np.zeros((rows, top))
        own = np.zeros((rows, n))
        own[at[tokens >= 0], tokens[tokens >= 0]] = g[tokens >= 0]
        np.add.at(own, (at[:, None], best), u)
        all_ = (g + u.sum(1))[:, None]
        weight = all_ + h[:, None] * (lp + ent[:, None])
        want = own - p * weight
        size = np.abs(all_) + np.abs(u).sum(1)[:, None] + np.abs(h[:, None]) * (np.abs(lp) + np.abs(ent[:, None]))
        off = p * (2 * lp_off + 8 * U * (1 + np.abs(lp))) * size + p * np.abs(h[:, None]) * (lp_off + ent_off[:, None])
        off = off + p * size * (top + 8) * U + 4 * U * (np.abs(own) + np.abs(u).sum(1)[:, None] * (own != 0))
        off = off + HALF[dtype] * (np.abs(want) + off) + TINY[dtype]
        a.requiresGrad().zeroGrad()
        got = a.logProbs(t32, top=top)
        loss = None
        for k, name, w in (("a", "logProbs", ga), ("h", "entropy", gh), ("u", "topLogProbs", gu)):
            if k in use:
                part = (got[name] * CudaArray.fromNumpy(w)).sum()
                loss = part if loss is None else loss + part
        loss.backward()
        assert a.grad().getDtype() == dtype
        near(a.grad(), (want, off), use)


def test_gradient_against_differences():
    a, x = scores((2, 9), "float32", 1)
    a.requiresGrad()
    tokens = np.array([3, 8])
    got = a.logProbs(CudaArray.fromNumpy(tokens.astype(np.int32)), top=2)
    (got["logProbs"] * 2.0 + got["entropy"] * 3.0 + got["topLogProbs"].sum(1)).backward(CudaArray.ones([2]))
    g = a.grad().toNumpy()

    def loss(v):
        r = reference(v, tokens)
        best = listed(v, 2)
        return (2 * r["logProbs"][0] + 3 * r["entropy"][0]).sum() + r["lp"][0][np.arange(2)[:, None], best].sum()
    for at in np.ndindex(2, 9):
        up, down = x.copy(), x.copy()
        up[at] += 1e-5
        down[at] -= 1e-5
        assert abs((loss(up) - loss(down)) / 2e-5 - g[at]) < 1e-4


def test_shapes_and_views():
    a, x = scores((3, 4, 50), "float32", 1)
    tokens = np.random.default_rng(1).integers(0, 50, (3, 4))
    t = CudaArray.fromNumpy(tokens.astype(np.int32))
    got = a.logProbs(t, top=3)
    assert got["entropy"].getShape() == [3, 4] and got["topTokens"].getShape() == [3, 4, 3]
    ref = reference(x.reshape(12, 50), tokens.reshape(-1))
    near(got["logProbs"], ref["logProbs"], "logProbs")
    # rows further apart than they are long, rows in another order, classes not side by side
    for view, values in ((a.slice(None, None, [5, 45]), x[:, :, 5:45]), (a.slice(None, [1, 3]), x[:, 1:3]),
                         (a.swapaxes(0, 1), x.swapaxes(0, 1)), (a.swapaxes(1, 2), x.swapaxes(1, 2)),
                         (a.slice(1), x[1]), (a.slice(2, 3), x[2, 3])):
        rows = view.getShape()[:-1] or [1]
        n = values.shape[-1]
        tok = np.random.default_rng(2).integers(0, n, rows)
        got = view.detach().requiresGrad().logProbs(CudaArray.fromNumpy(tok.astype(np.int32)), top=2)
        ref = reference(values.reshape(-1, n), tok.reshape(-1))
        near(got["logProbs"], ref["logProbs"], "view")
        assert got["entropy"].getShape() == list(rows)
    leaf = a.slice(None, None, [5, 45]).requiresGrad()
    leaf.logProbs(CudaArray.fromNumpy(np.minimum(tokens, 39).astype(np.int32)))["logProbs"].sum().backward()
    r = reference(x[:, :, 5:45].reshape(12, 40), np.minimum(tokens, 39).reshape(-1))
    want = -r["p"]
    want[np.arange(12), np.minimum(tokens, 39).reshape(-1)] += 1
    # p is off by its exponent's bound, twice u for the sum and the rounding
    near(leaf.grad(), (want, r["p"] * (2 * r["lp"][1] + 16 * U) + 4 * U * np.abs(want)), "dx of a view")
    assert a.slice(None, [0, 0]).logProbs(CudaArray.zeros([3, 0], "int32"))["entropy"].getShape() == [3, 0]


@pytest.mark.parametrize("top", [0, 4])
def test_compiled_plan(top):
    tokens = CudaArray.fromNumpy(np.random.default_rng(4).integers(-1, 900, 30).astype(np.int32))

    def step(x):
        x = x.detach().requiresGrad()
        got = x.logProbs(tokens, top=top)
        loss = (got["logProbs"] * 0.5 - got["entropy"] * 0.1).sum()
        if top:
            loss = loss + got["topLogProbs"].sum()
        loss.backward()
        return [*(t.detach() for t in got.values()), x.grad()]
    for graph in (True, False):
        plan = Fusion.compile(step, [scores((30, 900), "float32", 1)[0]], cudaGraph=graph)
        for seed in (10, 20, 30, 10):
            x = scores((30, 900), "float32", seed)[0]
            assert all(np.array_equal(a.toBits(), b.toBits()) for a, b in zip(step(x), plan.run(x)))


def test_refusals():
    a = CudaArray.zeros([4, 10])
    t = CudaArray.zeros([4], "int32")
    for call in [lambda: a.logProbs(CudaArray.zeros([4], "int64")), lambda: a.logProbs(CudaArray.zeros([5], "int32")),
                 lambda: a.logProbs(CudaArray.zeros([4, 1], "int32")), lambda: a.logProbs(t, top=11),
                 lambda: a.logProbs(t, top=-1), lambda: CudaArray.zeros([4, 100]).logProbs(t, top=65),
                 lambda: a.astype("float64").logProbs(t), lambda: CudaArray.zeros([4, 0]).logProbs(t),
                 lambda: a.logProbs(3), lambda: a.logProbs(t, top=2 ** 40)]:
        with pytest.raises(_abi.InvalidArgumentException):
            call()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_alternatives_of_unsplit_rows(dtype):
    """Many rows of four waves each: rising, falling, equal and nearly all masked scores, the best in one wave's share
    or at either end, in rows that start at any element of a pack."""
    rows, n, top = 512, 5005, 30
    rng = np.random.default_rng(11)
    x = rng.standard_normal((rows, n)).astype(np.float32)
    x[0], x[1], x[2] = np.arange(n) % 256, -(np.arange(n) % 256.0), 1.0
    x[3, 40:] = -np.inf
    x[4, :-40] = -np.inf
    x[5, 256:320] += 9
    x[6, :7], x[6, -7:] = 9, 9
    x[7] = np.arange(n)[::-1] // 64
    x[8, 1:] = np.float32(-60000)
    x[9, 2048:4096] = -np.inf
    a = CudaArray.fromNumpy(x, dtype)
    check(a, a.toNumpy().astype(np.float64), rng.integers(-1, n, rows), top, dtype)


def test_more_rows_than_one_launch_counts():
    rows, n = (1 << 22) + 3, 3
    x = np.random.default_rng(1).integers(-3, 4, (rows, n)).astype(np.float32)
    tokens = (np.arange(rows) % n).astype(np.int32)
    a = CudaArray.fromNumpy(x).requiresGrad()
    got = a.logProbs(CudaArray.fromNumpy(tokens), top=1)
    (got["logProbs"] + got["topLogProbs"].reshape([rows])).sum().backward()
    r = reference(x.astype(np.float64), tokens)
    near(got["logProbs"], r["logProbs"], "logProbs")
    best = listed(x, 1)
    assert np.array_equal(got["topTokens"].toNumpy(), best)
    want = -2 * r["p"]
    want[np.arange(rows), tokens] += 1
    want[np.arange(rows), best[:, 0]] += 1
    # as for the view above, for two upstream gradients
    near(a.grad(), (want, r["p"] * (4 * r["lp"][1] + 32 * U) + 8 * U * (np.abs(want) + 1)), "dx")
