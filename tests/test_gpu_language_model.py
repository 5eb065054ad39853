"""layerNorm, attention and logProbs as a small language model uses them together: a training step against float64,
the same step from a compiled plan, a prompt and single tokens from a cache; and their C entries on another stream and
in captured graphs."""
import ctypes
import math

import numpy as np
import pytest

import attention_ref as R
from phptensors import CudaArray, Fusion, Sequences, _abi

pytestmark = pytest.mark.gpu

WIDTH, HEADS, KV, SIZE, CLASSES, LENGTHS = 48, 6, 2, 8, 101, [17, 1, 30]
ROWS = sum(LENGTHS)


def weights(seed):
    rng = np.random.default_rng(seed)
    shapes = {"s1": (WIDTH,), "b1": (WIDTH,), "wq": (WIDTH, HEADS * SIZE), "wk": (WIDTH, KV * SIZE), "wv": (WIDTH, KV * SIZE),
              "wo": (HEADS * SIZE, WIDTH), "s2": (WIDTH,), "b2": (WIDTH,), "head": (WIDTH, CLASSES)}
    out = {n: (rng.standard_normal(s) / math.sqrt(s[0])).astype(np.float32) for n, s in shapes.items()}
    for n in ("s1", "s2"):
        out[n] = np.float32(1) + out[n]
    return out


def inputs(seed):
    rng = np.random.default_rng(seed)
    return rng.standard_normal((ROWS, WIDTH)).astype(np.float32), rng.integers(-1, CLASSES, ROWS).astype(np.int32)


def loss_of(x, w, tokens, seqs):
    """The framework's step: the sum of a row's log probability, its entropy and its two likeliest classes'."""
    h = x.layerNorm([1], 1e-5, w["s1"], w["b1"])
    q, k, v = (h.matmul(w[n]).reshape([ROWS, heads, SIZE]) for n, heads in (("wq", HEADS), ("wk", KV), ("wv", KV)))
    y = x + q.attention(k, v, causal=True, queries=seqs).reshape([ROWS, HEADS * SIZE]).matmul(w["wo"])
    got = y.layerNorm([1], 1e-5, w["s2"], w["b2"]).matmul(w["head"]).logProbs(tokens, top=2)
    return got["logProbs"].sum() * -0.1 + got["entropy"].sum() * 0.01 + got["topLogProbs"].sum() * 0.02


def norm(t, scale, bias):
    c = t - t.mean(1, keepdims=True)
    r = 1 / np.sqrt((c * c).mean(1, keepdims=True) + 1e-5)
    return c * r * scale + bias, c * r, r


def norm_back(g, unit, r, scale):
    h = g * scale
    return r * (h - h.mean(1, keepdims=True) - unit * (h * unit).mean(1, keepdims=True)), (g * unit).sum(0), g.sum(0)


def reference(x, w, tokens, gradients=True):
    """The loss and, by hand, its gradients in float64."""
    x, w = x.astype(np.float64), {n: t.astype(np.float64) for n, t in w.items()}
    h, unit1, r1 = norm(x, w["s1"], w["b1"])
    q, k, v = ((h @ w[n]).reshape(ROWS, heads, SIZE) for n, heads in (("wq", HEADS), ("wk", KV), ("wv", KV)))
    c, o, probs, at = 1 / math.sqrt(SIZE), np.zeros((ROWS, HEADS, SIZE)), {}, 0
    for n in LENGTHS:
        rows = slice(at, at + n)
        for i in range(HEADS):
            j = i // (HEADS // KV)
            e = np.where(np.tri(n) > 0, np.exp(c * q[rows, i] @ k[rows, j].T), 0.0)
            probs[at, i] = p = e / e.sum(1, keepdims=True)
            o[rows, i] = p @ v[rows, j]
        at += n
    y = x + o.reshape(ROWS, -1) @ w["wo"]
    z, unit2, r2 = norm(y, w["s2"], w["b2"])
    logits = z @ w["head"]
    lp = logits - np.log(np.exp(logits).sum(1, keepdims=True))
    p, one, named = np.exp(lp), np.arange(ROWS), tokens >= 0
    entropy, best = -(p * lp).sum(1, keepdims=True), np.argsort(-lp, 1, kind="stable")[:, :2]
    loss = -0.1 * lp[one, tokens][named].sum() + 0.01 * entropy.sum() + 0.02 * np.take_along_axis(lp, best, 1).sum()
    if not gradients:
        return loss
    d = p * (0.1 * named[:, None] - 0.04) - 0.01 * p * (lp + entropy)
    d[one[named], tokens[named]] -= 0.1
    for i in range(2):
        d[one, best[:, i]] += 0.02
    out = {"loss": loss, "head": z.T @ d}
    dy, out["s2"], out["b2"] = norm_back(d @ w["head"].T, unit2, r2, w["s2"])
    out["wo"] = o.reshape(ROWS, -1).T @ dy
    do = (dy @ w["wo"].T).reshape(o.shape)
    dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    for at, n in zip(np.cumsum([0] + LENGTHS), LENGTHS):
        rows = slice(at, at + n)
        for i in range(HEADS):
            j, p = i // (HEADS // KV), probs[at, i]
            dp = do[rows, i] @ v[rows, j].T
            ds = c * p * (dp - (dp * p).sum(1, keepdims=True))
            dv[rows, j] += p.T @ do[rows, i]
            dq[rows, i] = ds @ k[rows, j]
            dk[rows, j] += ds.T @ q[rows, i]
    dh = 0
    for n, g in (("wq", dq), ("wk", dk), ("wv", dv)):
        g = g.reshape(ROWS, -1)
        out[n] = h.T @ g
        dh = dh + g @ w[n].T
    dx, out["s1"], out["b1"] = norm_back(dh, unit1, r1, w["s1"])
    out["x"] = dy + dx
    return out


def leaves(x, w):
    x = CudaArray.fromNumpy(x).requiresGrad()
    return x, {n: CudaArray.fromNumpy(t).requiresGrad() for n, t in w.items()}


def test_training_step():
    """Tolerance: some twenty operations forwards and back, each off by at most 128 terms' roundings (the longest sums
    are of 101) relatively to the largest magnitude, which conditions of order 8 (the norms' scales, the softmax) carry
    on: 20 * 128 * 8 * 2^-24 = 1.2e-3 of a gradient's largest element."""
    (x, tokens), w = inputs(1), weights(2)
    want = reference(x, w, tokens)
    # the reference itself, against differences along a direction of every operand (step 1e-5: off by 1e-10 times
    # third derivatives and 1e-16 / 1e-5 of the loss)
    rng = np.random.default_rng(3)
    for n in ("x", *w):
        step = 1e-5 * rng.standard_normal(want[n].shape)
        sides = [reference(x + s if n == "x" else x, {m: t + s if m == n else t for m, t in w.items()}, tokens, False)
                 for s in (step, -step)]
        slope = (want[n] * step).sum()
        assert abs((sides[0] - sides[1]) / 2 - slope) < 1e-10, n   # slopes are of order 1e-5
    a, p = leaves(x, w)
    loss = loss_of(a, p, CudaArray.fromNumpy(tokens), Sequences(LENGTHS))
    loss.backward()
    assert abs(loss.item() - want["loss"]) < 1.2e-3 * abs(want["loss"])
    for n, t in [("x", a), *p.items()]:
        got = t.grad().toNumpy().astype(np.float64).reshape(want[n].shape)
        assert np.abs(got - want[n]).max() < 1.2e-3 * np.abs(want[n]).max(), n


@pytest.mark.parametrize("graph", [True, False])
def test_compiled_training_step(graph):
    """A plan of the whole step gives the eager bits on every replay, recorded and run while an eager history of the
    same leaves is alive, which then still gives its own gradients."""
    w0, seqs = weights(2), Sequences(LENGTHS)
    names = list(w0)
    tokens = CudaArray.fromNumpy(inputs(1)[1])

    def step(x, *params):
        x = x.detach().requiresGrad()
        p = {n: t.detach().requiresGrad() for n, t in zip(names, params)}
        loss = loss_of(x, p, tokens, seqs)
        loss.backward()
        return [loss.detach(), x.grad(), *(p[n].grad() for n in names)]

    def arrays(seed):
        return [CudaArray.fromNumpy(inputs(seed)[0]), *(CudaArray.fromNumpy(t) for t in weights(seed + 1).values())]
    held, p = leaves(inputs(1)[0], w0)
    alive = loss_of(held, p, tokens, seqs)
    plan = Fusion.compile(step, [held.detach(), *(t.detach() for t in p.values())], cudaGraph=graph)
    for seed in (1, 5, 9, 1):
        ins = arrays(seed)
        want = [t.toBits() for t in step(*ins)]
        assert all(np.array_equal(a, b.toBits()) for a, b in zip(want, plan.run(*ins)))
    # operators with several results are not captured, also where a graph is asked for
    assert plan.getStats()["backend"] == "stream" and plan.getStats()["graphLaunches"] == 0
    assert not graph or plan.getStats()["cudaGraphIncompatibility"] == "several-results"
    alive.backward()
    want = step(held.detach(), *(t.detach() for t in p.values()))
    assert all(np.array_equal(a.toBits(), b.toBits()) for a, b in zip([held.grad(), *(t.grad() for t in p.values())], want[1:]))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_prompt_then_tokens(dtype):
    """The rows of a cache written up to a length and one query at a time give the rows of the whole prompt."""
    heads, kv, size, slot, lengths = 8, 2, 64, 160, [150, 3, 77]
    rng = np.random.default_rng(3)
    q, k, v = (CudaArray.fromNumpy(rng.standard_normal((3 * slot, n, size)).astype(np.float32), dtype) for n in (heads, kv, kv))
    qv, kval, vv = (t.toNumpy().astype(np.float64) for t in (q, k, v))
    starts = [i * slot for i in range(3)]
    spans = [(a, n, a, n) for a, n in zip(starts, lengths)]
    want, off = R.attention(qv, kval, vv, True, size ** -0.5, dtype, spans)["o"]
    whole = Sequences(lengths, starts)
    got = q.attention(k, v, causal=True, queries=whole).toNumpy()
    assert (np.abs(got - want) <= off).all()
    for back in (1, 2, 40):  # the last tokens, the third of a sequence of two queries or none among them
        n = [max(0, m - back + 1) for m in lengths]
        at = [a + m - 1 if m else a for a, m in zip(starts, n)]
        one = Sequences([min(1, m) for m in n], at)
        got = q.attention(k, v, causal=True, queries=one, keys=Sequences(n, starts)).toNumpy()
        for a, m in zip(at, n):
            if m:
                assert (np.abs(got[a] - want[a]) <= off[a]).all()
        left = np.ones(3 * slot, bool)
        left[[a for a, m in zip(at, n) if m]] = False
        assert not got[left].any()


def test_gradients_do_not_depend_on_timing():
    """Runs of split keys and queries, with shared heads, give the same bits."""
    rng = np.random.default_rng(1)
    for dtype, rows, heads, kv, size in (("bfloat16", 700, 4, 1, 128), ("float32", 530, 6, 3, 40), ("float16", 900, 2, 2, 256)):
        q, k, v, w = (CudaArray.fromNumpy(rng.standard_normal((rows, n, size)).astype(np.float32), dtype)
                      for n in (heads, kv, kv, heads))
        bits = []
        for _ in range(4):
            a, b, c = (t.detach().requiresGrad() for t in (q, k, v))
            a.attention(b, c, causal=True).backward(w)
            bits.append([t.grad().toBits() for t in (a, b, c)])
        assert all(np.array_equal(x, y) for other in bits[1:] for x, y in zip(bits[0], other))


class Buffers:
    """Device copies of host arrays by name, and results of given sizes."""

    def __init__(self, **arrays):
        self.kept = {n: _abi.to_device(a) for n, a in arrays.items()}

    def __getattr__(self, name):
        return self.kept[name].ptr

    def bytes(self, name):
        return self.kept[name].download(np.uint8, (self.kept[name].nbytes,))

    def blank(self, *names):
        for n in names:
            _abi.check(_abi.load().pt_memset(self.kept[n].ptr, 0xFF, self.kept[n].nbytes, None))
        _abi.synchronize()


def test_captured_graphs_share_a_workspace():
    """A cache's attention (keys split, the parts in scratch) and its training gradients, and the log probabilities of
    few long rows, captured on a stream of their own into two graphs with one workspace: replayed in turn they give
    the eager results, and follow lengths that change on the device."""
    lib, rng = _abi.load(), np.random.default_rng(7)
    heads, kv, size, slot, count = 4, 2, 64, 3000, 2
    f = lambda *s: rng.standard_normal(s).astype(np.float16)
    b = Buffers(q=f(count, heads, size), k=f(count * slot, kv, size), v=f(count * slot, kv, size), w=f(count, heads, size),
                out=f(count, heads, size), lse=np.zeros((heads, count), np.float32), dq=f(count, heads, size), rest=f(count, heads, size),
                dk=f(count * slot, kv, size), dv=f(count * slot, kv, size),
                qs=np.arange(count, dtype=np.int32), qn=np.ones(count, np.int32),
                ks=(np.arange(count) * slot).astype(np.int32), kn=np.array([slot, 1700], np.int32),
                x=rng.standard_normal((3, 40000)).astype(np.float32), tokens=np.array([5, -1, 39999], np.int32),
                lp=np.zeros(3, np.float32), ent=np.zeros(3, np.float32), stats=np.zeros(6, np.float32),
                tv=np.zeros(24, np.float32), ti=np.zeros(24, np.int32), dx=np.zeros((3, 40000), np.float32),
                g=rng.standard_normal(3).astype(np.float32), gt=rng.standard_normal(24).astype(np.float32))
    d = _abi.PtAttentionDesc()
    strides = dict(q=heads, k=kv, v=kv)
    for n, h in strides.items():
        setattr(d, n + "_strides", (ctypes.c_size_t * 3)(0, h * size, size))
    for n, x in dict(dtype=_abi.FLOAT16, sequences=count, heads=heads, kv_heads=kv, head_size=size, queries=1, keys=slot,
                     q_starts=b.qs, q_lengths=b.qn, k_starts=b.ks, k_lengths=b.kn, q_rows=count, k_rows=count * slot,
                     causal=1, scale=0.125).items():
        setattr(d, n, x)

    def attend(stream):
        _abi.check(lib.pt_attention(ctypes.byref(d), b.q, b.k, b.v, b.out, b.lse, b.rest, stream))
        _abi.check(lib.pt_attention_backward(ctypes.byref(d), b.q, b.k, b.v, b.out, b.lse, b.rest, b.w, _abi.FLOAT16, b.dq, b.dk,
                                             b.dv, stream))

    def score(stream):
        _abi.check(lib.pt_logprobs(b.x, _abi.FLOAT32, 3, 40000, 40000, b.tokens, 8, b.lp, b.ent, b.stats, b.tv, b.ti, stream))
        _abi.check(lib.pt_logprobs_backward(b.x, _abi.FLOAT32, 3, 40000, 40000, b.tokens, 8, b.ti, b.stats, b.ent, b.g, b.g,
                                            b.gt, b.dx, stream))
    results = {attend: ("out", "lse", "rest", "dq", "dk", "dv"), score: ("lp", "ent", "stats", "tv", "ti", "dx")}

    def eager(call):
        b.blank(*results[call])
        call(None)
        _abi.synchronize()
        return [b.bytes(n) for n in results[call]]
    want = {call: eager(call) for call in results}
    peak = ctypes.c_size_t()
    need = 0
    for call in results:
        _abi.check(lib.pt_workspace_begin(None, 0))
        call(None)
        _abi.check(lib.pt_workspace_end(ctypes.byref(peak)))
        need = max(need, peak.value)
    assert need > 0
    _abi.synchronize()
    space = _abi.DeviceBuffer(need)
    stream = ctypes.c_void_p()
    _abi.check(lib.pt_stream_create(ctypes.byref(stream)))
    graphs = {}
    for call in results:
        _abi.check(lib.pt_workspace_begin(space.ptr, need))
        _abi.check(lib.pt_graph_begin_capture(stream))
        call(stream)
        g = ctypes.c_void_p()
        _abi.check(lib.pt_graph_end_capture(stream, ctypes.byref(g)))
        _abi.check(lib.pt_workspace_end(None))
        graphs[call] = g

    def replay():
        b.blank(*results[attend], *results[score])
        for _ in range(2):
            for call in results:
                _abi.check(lib.pt_graph_launch(graphs[call], stream))
        _abi.check(lib.pt_stream_synchronize(stream))
        for call, names in results.items():
            assert all(np.array_equal(x, b.bytes(n)) for x, n in zip(want[call], names))
    for _ in range(3):
        replay()
    # a result on the stream alone, without graph or workspace
    b.blank(*results[attend])
    attend(stream)
    _abi.check(lib.pt_stream_synchronize(stream))
    assert all(np.array_equal(x, b.bytes(n)) for x, n in zip(want[attend], results[attend]))
    b.kept["kn"].upload(np.array([64, 2999], np.int32))
    want[attend] = eager(attend)
    for _ in range(2):
        replay()
    # a workspace too small is refused, nothing written past it
    _abi.check(lib.pt_workspace_begin(space.ptr, 256))
    assert lib.pt_attention(ctypes.byref(d), b.q, b.k, b.v, b.out, b.lse, b.rest, None) != _abi.PT_OK
    _abi.check(lib.pt_workspace_end(None))
    for g in graphs.values():
        _abi.check(lib.pt_graph_destroy(g))
    _abi.check(lib.pt_stream_destroy(stream))


RAGGED = [(150, 6, 3, 64, "bfloat16"), (70, 5, 5, 40, "float32"), (40, 32, 16, 16, "float16"), (9, 12, 12, 128, "bfloat16"),
          (300, 2, 1, 256, "float16")]


@pytest.mark.parametrize("count,heads,kv,size,dtype", RAGGED, ids=str)
def test_many_ragged_sequences(count, heads, kv, size, dtype):
    """Sequences of none to some hundred tokens, out of order and with rows of no sequence between them."""
    rng = np.random.default_rng(count)
    lengths = rng.integers(0, 40, count)
    lengths[rng.integers(0, count, 3)] = [200, 129, 128]
    order = rng.permutation(count)
    starts, at = np.zeros(count, int), 2
    for i in order:
        starts[i] = at
        at += int(lengths[i]) + int(rng.integers(0, 3))
    seqs = Sequences([int(n) for n in lengths], [int(a) for a in starts])
    arrays = [CudaArray.fromNumpy(rng.standard_normal((at + 5, n, size)).astype(np.float32), dtype)
              for n in (heads, kv, kv, heads)]
    qv, kval, vv, wv = (t.toNumpy().astype(np.float64) for t in arrays)
    q, k, v = (t.requiresGrad() for t in arrays[:3])
    o = q.attention(k, v, causal=True, queries=seqs)
    o.backward(arrays[3])
    spans = [(int(a), int(n), int(a), int(n)) for a, n in zip(starts, lengths)]
    ref = R.attention(qv, kval, vv, True, size ** -0.5, dtype, spans, wv)
    for name, t in (("o", o), ("dq", q.grad()), ("dk", k.grad()), ("dv", v.grad())):
        want, off = ref[name]
        got = t.toNumpy().astype(np.float64).reshape(want.shape)
        assert (np.abs(got - want) <= off).all(), name


def test_operand_in_several_places_and_sequences_of_a_plan():
    """One tensor as queries, keys and values gets the sum of the three gradients; Sequences made while a plan is
    recorded belong to it."""
    x = CudaArray.fromNumpy(np.random.default_rng(1).standard_normal((40, 3, 16)).astype(np.float32))
    w = CudaArray.fromNumpy(np.random.default_rng(2).standard_normal((40, 3, 16)).astype(np.float32))

    def step(x, w):
        a, b, c = (x.detach().requiresGrad() for _ in range(3))
        a.attention(b, c, causal=True, queries=Sequences([30, 10])).backward(w)
        return [a.grad(), b.grad(), c.grad()]
    each = step(x, w)
    one = x.detach().requiresGrad()
    one.attention(one, one, causal=True, queries=Sequences([30, 10])).backward(w)
    total, size = sum(t.toNumpy().astype(np.float64) for t in each), sum(np.abs(t.toNumpy()) for t in each)
    assert (np.abs(one.grad().toNumpy() - total) <= 2 * R.U * size).all()   # two additions
    for graph in (True, False):
        plan = Fusion.compile(step, [x, w], cudaGraph=graph)
        for _ in range(3):
            assert all(np.array_equal(a.toBits(), b.toBits()) for a, b in zip(each, plan.run(x, w)))


def test_gradient_calls_of_the_host_refuse_what_the_forward_calls_refuse():
    from phptensors import _host
    lib = _host.load()
    x, g, s = CudaArray.zeros([4, 6]), CudaArray.zeros([4, 6]), CudaArray.zeros([6])
    got = (ctypes.c_void_p * 3)()

    def call(axes, eps=1e-5, x=x, g=g, scale=s):
        a = (ctypes.c_int * len(axes))(*axes)
        return lib.phpt_layernorm_backward(x._h, g._h, a, len(axes), eps, scale._h if scale is not None else None, None, got)
    for args in [dict(axes=[2]), dict(axes=[-3]), dict(axes=[1, 1], scale=None), dict(axes=[0]), dict(axes=[1], eps=0.0),
                 dict(axes=[1], g=CudaArray.zeros([4, 5])), dict(axes=[1], g=CudaArray.zeros([4, 6], "int32")),
                 dict(axes=[1], scale=CudaArray.zeros([6], "int32")), dict(axes=[0, 1, 2], scale=None)]:
        assert call(**args) != 0, args
    q = CudaArray.zeros([4, 2, 8])
    kept = (ctypes.c_void_p * 2)()
    o = CudaArray._wrap(lib.phpt_attention(q._h, q._h, q._h, 0, 0.0, None, None, kept))
    lse = CudaArray._wrap(kept[0])
    assert not kept[1]   # float32 keeps no rest
    for bad in [dict(o=CudaArray.zeros([4, 2, 4])), dict(lse=CudaArray.zeros([4, 2])), dict(g=CudaArray.zeros([3, 2, 8])),
                dict(g=CudaArray.zeros([4, 2, 8], "bfloat16")), dict(rest=q)]:
        a = {"o": o, "lse": lse, "rest": None, "g": q, **bad}
        assert lib.phpt_attention_backward(q._h, q._h, q._h, a["o"]._h, a["lse"]._h, a["rest"]._h if a["rest"] is not None else None,
                                           a["g"]._h, 0, 0.0, None, None, got) != 0, bad
