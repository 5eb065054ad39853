"""Rotary positions, the gated projection and AdamW over many tensors as a language model's block uses them together: a
training step against float64, the same from a compiled plan, tokens one by one against the prompt; and their C entries on
another stream, in captured graphs that share a workspace, and from two threads at once."""
import ctypes
import math
import threading

import numpy as np
import pytest

import test_gpu_gated
from phptensors import CudaArray, Fusion, Rotary, Sequences, _abi
from phptensors.optimizer import Optimizer

pytestmark = pytest.mark.gpu

WIDTH, HEADS, KV, SIZE, HIDDEN, CLASSES, LENGTHS = 40, 4, 2, 12, 56, 67, [13, 1, 22]
ROWS = sum(LENGTHS)
AT = np.concatenate([np.arange(n) for n in LENGTHS]).astype(np.int32)


def weights(seed):
    rng = np.random.default_rng(seed)
    shapes = {"n1": (WIDTH,), "wq": (WIDTH, HEADS * SIZE), "wk": (WIDTH, KV * SIZE), "wv": (WIDTH, KV * SIZE), "sq": (SIZE,),
              "sk": (SIZE,), "wo": (HEADS * SIZE, WIDTH), "n2": (WIDTH,), "gate": (WIDTH, HIDDEN), "up": (WIDTH, HIDDEN),
              "down": (HIDDEN, WIDTH), "head": (WIDTH, CLASSES)}
    out = {n: (rng.standard_normal(s) / math.sqrt(s[0])).astype(np.float32) for n, s in shapes.items()}
    for n in ("n1", "n2", "sq", "sk"):
        out[n] = np.float32(1) + out[n] * np.float32(0.3)
    return out


def inputs(seed):
    rng = np.random.default_rng(seed)
    return rng.standard_normal((ROWS, WIDTH)).astype(np.float32), rng.integers(0, CLASSES, ROWS).astype(np.int32)


def loss_of(x, w, tokens, seqs, plan, at):
    h = x.layerNorm([1], 1e-5, w["n1"])
    q, k, v = (h.matmul(w[n]).reshape([ROWS, heads, SIZE]) for n, heads in (("wq", HEADS), ("wk", KV), ("wv", KV)))
    q, k = q.rotary(plan, at, k, w["sq"], w["sk"])
    y = x + q.attention(k, v, causal=True, queries=seqs).reshape([ROWS, HEADS * SIZE]).matmul(w["wo"])
    z = y + y.layerNorm([1], 1e-5, w["n2"]).gatedProjection(w["gate"], w["up"]).matmul(w["down"])
    return z.matmul(w["head"]).logProbs(tokens)["logProbs"].sum() * (-1.0 / ROWS)


def reference(x, w, tokens):
    """The loss in float64."""
    x, w = x.astype(np.float64), {n: t.astype(np.float64) for n, t in w.items()}

    def norm(t, scale):
        c = t - t.mean(-1, keepdims=True)
        return c / np.sqrt((c * c).mean(-1, keepdims=True) + 1e-5) * scale

    def turn(t, scale):
        t = t / np.sqrt((t * t).mean(-1, keepdims=True) + 1e-6) * scale
        z = (t[..., :SIZE // 2] + 1j * t[..., SIZE // 2:]) * np.exp(1j * AT[:, None] * 10000.0 ** (-np.arange(0, SIZE, 2) / SIZE))[:, None]
        return np.concatenate([z.real, z.imag], -1)
    h = norm(x, w["n1"])
    q, k, v = ((h @ w[n]).reshape(ROWS, heads, SIZE) for n, heads in (("wq", HEADS), ("wk", KV), ("wv", KV)))
    q, k, o, at = turn(q, w["sq"]), turn(k, w["sk"]), np.zeros((ROWS, HEADS, SIZE)), 0
    for n in LENGTHS:
        rows = slice(at, at + n)
        for i in range(HEADS):
            j = i // (HEADS // KV)
            e = np.where(np.tri(n) > 0, np.exp(q[rows, i] @ k[rows, j].T / math.sqrt(SIZE)), 0.0)
            o[rows, i] = e / e.sum(1, keepdims=True) @ v[rows, j]
        at += n
    y = x + o.reshape(ROWS, -1) @ w["wo"]
    h = norm(y, w["n2"])
    g = h @ w["gate"]
    logits = (y + (g / (1 + np.exp(-g)) * (h @ w["up"])) @ w["down"]) @ w["head"]
    return -(logits[np.arange(ROWS), tokens] - np.log(np.exp(logits).sum(1))).sum() / ROWS


def test_training_step():
    """Gradients against differences of the float64 loss along two directions of each operand.  Some thirty operations
    forwards and back, each off by at most 128 roundings relatively to the largest magnitude, which conditions of order 8
    carry on: 30 * 128 * 8 * 2^-24 = 1.9e-3 of a gradient's largest element; along a direction at most that times the
    direction's sum of magnitudes.  The differences themselves (step 1e-5) are off by 1e-10 times third derivatives."""
    (x, tokens), w = inputs(1), weights(2)
    a, p = CudaArray.fromNumpy(x).requiresGrad(), {n: CudaArray.fromNumpy(t).requiresGrad() for n, t in w.items()}
    plan = Rotary(SIZE)
    loss = loss_of(a, p, CudaArray.fromNumpy(tokens), Sequences(LENGTHS), plan, CudaArray.fromNumpy(AT))
    loss.backward()
    want = reference(x, w, tokens)
    assert abs(loss.item() - want) < 1.9e-3 * abs(want)
    rng = np.random.default_rng(3)
    for n, t in [("x", a), *p.items()]:
        g = t.grad().toNumpy().astype(np.float64)
        assert t.grad().getShape() == t.getShape()
        for _ in range(2):
            step = 1e-5 * rng.standard_normal(g.shape)
            sides = [reference(x + s if n == "x" else x, {m: v + s if m == n else v for m, v in w.items()}, tokens)
                     for s in (step, -step)]
            off = 1.9e-3 * np.abs(g).max() * np.abs(step).sum() + 1e-12
            assert abs((sides[0] - sides[1]) / 2 - (g * step).sum()) < off, n
    # and the step that follows, over all of them at once
    opt = Optimizer.adamW(0.01)
    params, grads = list(p.values()), [t.grad() for t in p.values()]
    mask = [len(t.getShape()) > 1 for t in params]
    one = opt.step(params, grads, opt.initState(params), None, mask)["parameters"]
    many = opt.fusedStep(params, grads, opt.initFusedState(params), None, mask)["parameters"]
    assert all(np.array_equal(s.toBits(), t.toBits()) for s, t in zip(one, many))


@pytest.mark.parametrize("bits", [32, 8])
def test_compiled_training_step(bits):
    """A plan of the whole step, update included, gives the eager bits on every replay, recorded and run while an eager
    history of the same leaves is alive."""
    opt, plan, seqs = Optimizer.adamW(0.01), Rotary(SIZE), Sequences(LENGTHS)
    names = list(weights(0))
    tokens, at = CudaArray.fromNumpy(inputs(1)[1]), CudaArray.fromNumpy(AT)
    held = ["firstMoment", "secondMoment", "beta1Power", "beta2Power"] + (["firstExponent", "secondExponent", "draws"] if bits == 8 else [])

    def step(x, *tensors):
        p = {n: t.detach().requiresGrad() for n, t in zip(names, tensors)}
        loss = loss_of(x, p, tokens, seqs, plan, at)
        loss.backward()
        r = opt.fusedStep(list(p.values()), [t.grad() for t in p.values()], dict(zip(held, tensors[len(names):]), bits=bits))
        return [loss.detach(), *r["parameters"], *(r["state"][n] for n in held)]
    x, p = CudaArray.fromNumpy(inputs(1)[0]), [CudaArray.fromNumpy(t).requiresGrad() for t in weights(2).values()]
    alive = loss_of(x, dict(zip(names, p)), tokens, seqs, plan, at)
    state = opt.initFusedState(p, bits=bits)
    ins = [x, *(t.detach() for t in p), *(state[n] for n in held)]
    compiled = Fusion.compile(step, ins)
    for _ in range(4):
        want = [t.toBits() for t in step(*ins)]
        out = compiled.run(*ins)
        assert all(np.array_equal(a, b.toBits()) for a, b in zip(want, out))
        ins = [x, *(t.copy() for t in out[1:])]
    alive.backward()
    assert all(np.isfinite(t.grad().toNumpy()).all() for t in p)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_prompt_then_tokens(dtype):
    """A token alone, at its position, is turned to the bits of the prompt's row; through the gated projection, whose
    kernels for a row and for a prompt add in different orders, both are within the bounds against float64."""
    rng, plan, rows, k, f = np.random.default_rng(1), Rotary(32, factor=4.0, context=256), 80, 96, 136
    x, s = (CudaArray.fromNumpy(rng.standard_normal(n).astype(np.float32), dtype) for n in ((rows, 6, 32), (32,)))
    whole = x.rotary(plan, None, scale=s).toBits()
    y, a, b = (CudaArray.fromNumpy(rng.standard_normal(n).astype(np.float32) * 0.2, dtype) for n in ((rows, k), (k, f), (k, f)))
    yv, av, bv = (t.toNumpy().astype(np.float64) for t in (y, a, b))
    want, off = test_gpu_gated.reference(yv, av, bv, "silu", dtype)["h"]
    test_gpu_gated.close(y.gatedProjection(a, b), (want, off), "prompt")
    for t in (0, 1, 41, 79):
        one = x.slice([t, t + 1]).rotary(plan, CudaArray.fromNumpy(np.array([t], np.int32)), scale=s)
        assert np.array_equal(one.toBits()[0], whole[t])
        test_gpu_gated.close(y.slice([t, t + 1]).gatedProjection(a, b), (want[t:t + 1], off[t:t + 1]), t)


class Buffers:
    """Device copies of host arrays by name."""

    def __init__(self, **arrays):
        self.kept = {n: _abi.to_device(a) for n, a in arrays.items()}

    def __getattr__(self, name):
        return self.kept[name].ptr

    def bytes(self, name):
        return self.kept[name].download(np.uint8, (self.kept[name].nbytes,))

    def blank(self, names):
        for n in names:
            _abi.check(_abi.load().pt_memset(self.kept[n].ptr, 0xFF, self.kept[n].nbytes, None))
        _abi.synchronize()


def test_captured_graphs_share_a_workspace():
    """Both directions of rotary (partial sums in scratch) and of the gated projection (split contractions, packed
    weights, float32 products), and a step of AdamW, captured on a stream of their own into graphs with one workspace: replayed in
    turn they give the eager results, and follow positions that change on the device."""
    lib, rng = _abi.load(), np.random.default_rng(7)
    h = lambda *s: rng.standard_normal(s).astype(np.float16)  # noqa: E731
    e = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    m, k, f = 70, 500, 203
    b = Buffers(x=h(90, 3, 24), g=h(90, 3, 24), y=h(90, 3, 24), dx=h(90, 3, 24), s=h(24), ds=h(24), turns=rng.random(12),
                at=np.arange(90, dtype=np.int32), gx=h(m, k), ga=h(k, f), gu=h(k, f), gh=h(m, f), gk=np.zeros(6 * m * f, np.uint8),
                gg=h(m, f), gdx=h(m, k), gda=h(k, f), gdu=h(k, f), fx=e(m, k), fa=e(k, f), fu=e(k, f), fh=e(m, f),
                fk=np.zeros(8 * m * (f + 1), np.uint8), fg=e(m, f), fdx=e(m, k), fda=e(k, f), fdu=e(k, f),
                p=e(700), pg=e(700), pn=e(700), m0=e(768), v0=np.abs(e(768)), m1=e(768), v1=e(768), b1=np.ones(1, np.float32),
                b2=np.ones(1, np.float32), n1=e(1), n2=e(1))
    r = _abi.PtRotaryDesc()
    for n, v in dict(dtype=_abi.FLOAT16, sequences=1, tokens=90, size=24, part=24, interleaved=1, magnitude=1.0, epsilon=1e-6,
                     turns=b.turns, positions=b.at).items():
        setattr(r, n, v)
    r.heads[0], r.strides[0], r.position_strides = 3, (ctypes.c_size_t * 3)(0, 72, 24), (ctypes.c_size_t * 2)(0, 1)
    one = lambda p: (ctypes.c_void_p * 2)(p, None)  # noqa: E731
    gd = {t: _abi.PtGatedDesc(t, 1, m, k, f) for t in (_abi.FLOAT16, _abi.FLOAT32)}
    d, t = _abi.PtAdamwDesc(), _abi.PtAdamwTensor(b.p, b.pg, b.pn, 700, 0, _abi.FLOAT32, _abi.FLOAT32, 1)
    for n, v in dict(bits=32, beta1=0.9, beta2=0.99, epsilon=1e-8, weight_decay=0.1, rate_value=0.01, first=b.m0, second=b.v0,
                     new_first=b.m1, new_second=b.v1, power1=b.b1, power2=b.b2, new_power1=b.n1, new_power2=b.n2).items():
        setattr(d, n, v)

    def turn(stream):
        _abi.check(lib.pt_rotary(ctypes.byref(r), one(b.x), one(b.s), one(b.y), stream))
        _abi.check(lib.pt_rotary_backward(ctypes.byref(r), one(b.x), one(b.s), one(b.g), _abi.FLOAT16, one(b.dx), one(b.ds), stream))

    def gate(stream, c="g", dt=_abi.FLOAT16):
        q = {n: getattr(b, c + n) for n in ("x", "a", "u", "h", "k", "g", "dx", "da", "du")}
        _abi.check(lib.pt_gated(ctypes.byref(gd[dt]), q["x"], q["a"], q["u"], q["h"], q["k"], stream))
        _abi.check(lib.pt_gated_backward(ctypes.byref(gd[dt]), q["x"], q["a"], q["u"], q["k"], q["g"], dt, q["dx"], q["da"], q["du"], stream))

    def wide(stream):
        gate(stream, "f", _abi.FLOAT32)

    def update(stream):
        _abi.check(lib.pt_adamw(ctypes.byref(d), ctypes.byref(t), 1, stream))
    results = {turn: ("y", "dx", "ds"), gate: ("gh", "gk", "gdx", "gda", "gdu"), wide: ("fh", "fdx", "fda", "fdu"),
               update: ("pn", "m1", "v1", "n1", "n2")}

    def eager(call):
        b.blank(results[call])
        call(None)
        _abi.synchronize()
        return [b.bytes(n) for n in results[call]]
    want = {call: eager(call) for call in results}
    peak, need = ctypes.c_size_t(), 0
    for call in results:
        _abi.check(lib.pt_workspace_begin(None, 0))
        call(None)
        _abi.check(lib.pt_workspace_end(ctypes.byref(peak)))
        need = max(need, peak.value)
    _abi.synchronize()
    assert need > 0
    space, stream, graphs = _abi.DeviceBuffer(need), ctypes.c_void_p(), {}
    _abi.check(lib.pt_stream_create(ctypes.byref(stream)))
    for call in results:
        _abi.check(lib.pt_workspace_begin(space.ptr, need))
        _abi.check(lib.pt_graph_begin_capture(stream))
        call(stream)
        g = ctypes.c_void_p()
        _abi.check(lib.pt_graph_end_capture(stream, ctypes.byref(g)))
        _abi.check(lib.pt_workspace_end(None))
        graphs[call] = g

    def replay():
        for names in results.values():
            b.blank(names)
        for _ in range(2):
            for call in results:
                _abi.check(lib.pt_graph_launch(graphs[call], stream))
        _abi.check(lib.pt_stream_synchronize(stream))
        for call, names in results.items():
            assert all(np.array_equal(x, b.bytes(n)) for x, n in zip(want[call], names)), call
    for _ in range(3):
        replay()
    # on the stream alone, without graph or workspace
    for call, names in results.items():
        b.blank(names)
        call(stream)
        _abi.check(lib.pt_stream_synchronize(stream))
        assert all(np.array_equal(x, b.bytes(n)) for x, n in zip(want[call], names)), call
    b.kept["at"].upload(np.arange(90, dtype=np.int32)[::-1].copy() * 1000)
    before, want[turn] = want[turn], eager(turn)
    assert not np.array_equal(before[0], want[turn][0])
    for _ in range(2):
        replay()
    # a workspace too small is refused, nothing written past it
    _abi.check(lib.pt_workspace_begin(space.ptr, 256))
    q = ctypes.byref(gd[_abi.FLOAT16])
    assert lib.pt_gated(q, b.gx, b.ga, b.gu, b.gh, b.gk, None) != _abi.PT_OK
    assert lib.pt_rotary_backward(ctypes.byref(r), one(b.x), one(b.s), one(b.g), _abi.FLOAT16, one(b.dx), one(b.ds), None) != _abi.PT_OK
    _abi.check(lib.pt_workspace_end(None))
    for g in graphs.values():
        _abi.check(lib.pt_graph_destroy(g))
    _abi.check(lib.pt_stream_destroy(stream))


def test_two_threads_at_once():
    """Calls of two threads; only one of them records a history at a time, as the recording belongs to the process."""
    opt, plan, lock = Optimizer.adamW(0.01), Rotary(16), threading.Lock()

    def work(seed):
        rng = np.random.default_rng(seed)
        x, a, u, h = (CudaArray.fromNumpy(rng.standard_normal(s).astype(np.float32), "bfloat16") for s in
                      ((90, 257), (257, 80), (257, 80), (90, 5, 16)))
        out = []
        for _ in range(10):
            with lock:
                leaves = [t.detach().requiresGrad() for t in (x, a, u)]
                y = leaves[0].gatedProjection(*leaves[1:])
                y.backward(y.detach())
                g = [t.grad() for t in leaves]
            r = opt.fusedStep([x, a, u], g, opt.initFusedState([x, a, u], bits=8))
            z = x.gatedProjection(a, u)
            out.append([t.toBits() for t in (y, z, *g, *r["parameters"], r["state"]["firstMoment"], h.rotary(plan))])
        return out
    want, got = {s: work(s) for s in (1, 2)}, {}
    threads = [threading.Thread(target=lambda s=s: got.update({s: work(s)})) for s in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for s in (1, 2):
        assert all(np.array_equal(p, q) for one, other in zip(want[s], got[s]) for p, q in zip(one, other))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_one_tensor_in_several_places(dtype):
    """The same queries as keys, the same scale twice, one matrix as gate and up, a parameter listed twice."""
    rng = np.random.default_rng(8)

    def made(*shape):
        return CudaArray.fromNumpy(rng.standard_normal(shape).astype(np.float32), dtype)
    plan, q, s, gq, gk = Rotary(16), made(40, 3, 16), made(16), made(40, 3, 16), made(40, 3, 16)

    def turn(q, k, s, t):
        for x in (q, k, s, t):
            x.requiresGrad().zeroGrad()
        a, b = q.rotary(plan, None, k, s, t)
        (a * gq + b * gk).sum().backward()
        return a, b
    a, b = turn(q, q, s, s)
    one = [x.grad().toNumpy().astype(np.float64) for x in (q, s)]
    k, t = q.copy(), s.copy()
    c, d = turn(q, k, s, t)
    assert all(np.array_equal(x.toBits(), y.toBits()) for x, y in ((a, c), (b, d)))
    h = test_gpu_gated.HALF[dtype]
    for got, x, y in ((one[0], q, k), (one[1], s, t)):
        x, y = (v.grad().toNumpy().astype(np.float64) for v in (x, y))
        # the parts are each rounded to the type, and their sum once more
        assert (np.abs(got - (x + y)) <= 2 * h * (np.abs(x) + np.abs(y)) + 2.0 ** -120).all()
    x, w, g = made(70, 24), made(24, 40), made(70, 40)

    def project(gate, up):
        for v in (x, gate, up):
            v.requiresGrad().zeroGrad()
        y = x.gatedProjection(gate, up, "gelu")
        y.backward(g)
        return y
    y = project(w, w)
    both, dx = w.grad().toNumpy().astype(np.float64), x.grad().toBits()
    u = w.copy()
    z = project(w, u)
    p, r = (v.grad().toNumpy().astype(np.float64) for v in (w, u))
    assert np.array_equal(y.toBits(), z.toBits()) and np.array_equal(dx, x.grad().toBits())
    assert (np.abs(both - (p + r)) <= 2 * h * (np.abs(p) + np.abs(r)) + 2.0 ** -120).all()
    opt, grads = Optimizer.adamW(0.1), [made(24, 40), made(24, 40)]
    w.requiresGrad(False)
    new = opt.fusedStep([w, w], grads, opt.initFusedState([w, w]))["parameters"]
    for n, gr in zip(new, grads):
        assert np.array_equal(n.toBits(), opt.fusedStep([w], [gr], opt.initFusedState([w]))["parameters"][0].toBits())


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_broadcast_and_strided_operands(dtype):
    """Views with steps of zero and others give what their copies do, gradients of broadcast leaves summed."""
    rng = np.random.default_rng(9)

    def made(*shape):
        return CudaArray.fromNumpy(rng.standard_normal(shape).astype(np.float32), dtype)
    plan, at = Rotary(8, interleaved=True), CudaArray.fromNumpy(np.arange(66, dtype=np.int32))
    for x in (made(33, 1, 12).broadcastTo([33, 5, 12]), made(1, 5, 12).broadcastTo([33, 5, 12]), made(5, 33, 12).swapaxes(0, 1)):
        for p in (at.slice([0, 66, 2]), at.slice([7, 8]).broadcastTo([33])):
            assert np.array_equal(x.rotary(plan, p).toBits(), x.copy().rotary(plan, p.copy()).toBits())
    row, g = made(1, 5, 12), made(33, 5, 12)
    row.requiresGrad()
    row.broadcastTo([33, 5, 12]).rotary(plan, at.slice([0, 33])).backward(g)
    back = row.grad().toNumpy().astype(np.float64)
    full = row.detach().broadcastTo([33, 5, 12]).copy().requiresGrad()
    full.rotary(plan, at.slice([0, 33])).backward(g)
    each = full.grad().toNumpy().astype(np.float64)
    h = test_gpu_gated.HALF[dtype]
    # 33 rounded terms, added in float32 and rounded, or added with a rounding each
    assert (np.abs(back - each.sum(0, keepdims=True)) <= 34 * h * np.abs(each).sum(0, keepdims=True)).all()
    w, v = made(1, 40).broadcastTo([24, 40]), made(48, 40).slice([0, 48, 2])
    for rows in (1, 30, 90):
        for x in (made(1, 24).broadcastTo([rows, 24]), made(24, rows).T, made(rows, 48).slice(":", [0, 48, 2])):
            assert np.array_equal(x.gatedProjection(w, v).toBits(), x.copy().gatedProjection(w.copy(), v.copy()).toBits())
    opt = Optimizer.adamW(0.1)
    state = opt.initFusedState([v], bits=8, master=True)
    got, want = (opt.fusedStep([p], [g], state)["parameters"][0].toBits() for p, g in ((v, w), (v.copy(), w.copy())))
    assert np.array_equal(got, want)
