"""What the host runtime does with the rotation of heads, the gated projection and AdamW over many tensors in Fusion scopes
and plans, shown on a double of the device library: no GPU."""
from unittest import mock

import pytest

import device_double

# what the calls write: a value of their own into each result, what the forward pass left read back for the gradients
BODY = {
    "pt_rotary": "for (int i = 0; i < 2; i++) if (desc->heads[i])"
                 " values(y[i], desc->sequences * desc->tokens * desc->heads[i] * desc->size, 1.5f + i, desc->dtype);",
    "pt_rotary_backward": "for (int i = 0; i < 2; i++) if (desc->heads[i]) {"
                          " values(dx[i], desc->sequences * desc->tokens * desc->heads[i] * desc->size, 3.0f + i, desc->dtype);"
                          " if (dscale) values(dscale[i], desc->size, 5.0f + i, desc->dtype); }",
    "pt_gated": "const size_t n = (size_t)desc->rows * desc->outer; values(h, n, 1.5f, desc->dtype);"
                " if (kept) memset(kept, 7, (desc->dtype == PT_FLOAT32 ? 8 : 6) * n);",
    "pt_gated_backward": "const float at = *(const unsigned char *)kept;"
                         " values(dx, (size_t)desc->rows * desc->inner, at + 1.0f, desc->dtype);"
                         " values(dgate, (size_t)desc->inner * desc->outer, at + 2.0f, desc->dtype);"
                         " values(dup, (size_t)desc->inner * desc->outer, at + 3.0f, desc->dtype);",
    "pt_adamw": "size_t end = 0;"
                " for (int i = 0; i < count; i++) {"
                "  values(tensors[i].new_param, tensors[i].n, 2.0f + i, tensors[i].param_dtype);"
                "  end = tensors[i].at + (tensors[i].n + 255) / 256 * 256; }"
                " if (desc->bits == 8) {"
                "  memset(desc->new_first, 21, end); memset(desc->new_second, 22, end);"
                "  memset(desc->new_first_exponent, 23, end / 256); memset(desc->new_second_exponent, 24, end / 256);"
                "  *desc->new_draws = 25;"
                " } else { floats(desc->new_first, end, 21.0f); floats(desc->new_second, end, 22.0f); }"
                " floats(desc->new_master, end, 26.0f); floats(desc->new_power1, 1, 27.0f); floats(desc->new_power2, 1, 28.0f);",
    "pt_adamw_moments": "floats(first_values, n, 31.0f); floats(second_values, n, 32.0f);",
}


@pytest.fixture(scope="module")
def double(tmp_path_factory):
    folder = str(tmp_path_factory.mktemp("double"))
    with mock.patch.dict(device_double.BODY, BODY):
        device_double.build(folder)
    return lambda code: device_double.run(folder, OPERATORS + code)


OPERATORS = """
import itertools
from phptensors import Rotary
from phptensors.optimizer import Optimizer
plan = Rotary(8)
opt = Optimizer.adamW(0.1)

def leaves(*shapes, dtype="float32"):
    return [CudaArray.zeros(list(s), dtype).requiresGrad() for s in shapes]

def rotary(read, dtype="float32"):
    q, k, s, t = leaves((6, 4, 10), (6, 2, 10), (10,), (10,), dtype=dtype)
    a, b = q.rotary(plan, CudaArray.zeros([6], "int32"), k, s, t)
    (a * 2.0).sum().backward(), (b * 3.0).sum().backward()
    return read([(a, 1.5), (b, 2.5), (q.grad(), 3.0), (k.grad(), 4.0), (s.grad(), 5.0), (t.grad(), 6.0)])

def gated(read, dtype="float32"):
    x, a, b = leaves((5, 9), (9, 7), (9, 7), dtype=dtype)
    h = x.gatedProjection(a, b)
    h.backward(CudaArray.zeros([5, 7], dtype))
    return read([(h, 1.5), (x.grad(), 8.0), (a.grad(), 9.0), (b.grad(), 10.0)])

def adamw(read, bits=8, dtype="float32"):
    ps = [CudaArray.zeros([300], dtype), CudaArray.zeros([], dtype), CudaArray.zeros([3, 0], dtype), CudaArray.zeros([2, 3], dtype)]
    r = opt.fusedStep(ps, [CudaArray.zeros(p.getShape(), dtype) for p in ps], states[bits], CudaArray.zeros([1]))
    s, p = r["state"], r["parameters"]
    small = [(s["firstExponent"], 23), (s["secondExponent"], 24), (s["draws"], 25)] if bits == 8 else []
    return read([(p[0], 2.0), (p[1], 3.0), (p[3], 5.0), (s["firstMoment"], 21), (s["secondMoment"], 22), (s["master"], 26.0),
                 (s["beta1Power"], 27.0), (s["beta2Power"], 28.0), *small])

def moments(read):
    m = opt.moments(states[8])
    return read([(m["firstMoment"], 31.0), (m["secondMoment"], 32.0)])

states = {bits: opt.initFusedState([CudaArray.zeros(s) for s in ([300], [], [3, 0], [2, 3])], bits, master=True) for bits in (8, 32)}
KERNELS = {rotary: {"pt_rotary": 1, "pt_rotary_backward": 2}, gated: {"pt_gated": 1, "pt_gated_backward": 1},
           adamw: {"pt_adamw": 1}, moments: {"pt_adamw_moments": 1}}
SIZES = {rotary: 6, gated: 4, adamw: 11, moments: 2}

def orders(op):
    # all of few results, else each first, forwards and backwards
    n = SIZES[op]
    if n <= 4:
        return list(itertools.permutations(range(n)))
    return [[(s * i + f) % n for i in range(n)] for f in range(n) for s in (1, -1)]

def holds(t, x):
    got = t.toNumpy()
    assert (got == x).all(), (got.ravel()[:3], x)

class Calls:
    def __init__(self, op):
        self.op = op
    def __enter__(self):
        self.before = {k: count(k) for k in KERNELS[self.op]}
    def __exit__(self, *_):
        for k, n in KERNELS[self.op].items():
            assert count(k) - self.before[k] == n, (self.op.__name__, k, count(k) - self.before[k])
"""


def test_eager_results(double):
    double("""
for op in KERNELS:
    with Calls(op):
        op(lambda results: [holds(*r) for r in results])
for dtype in ("float16", "bfloat16"):
    for op in (rotary, gated, adamw):
        with Calls(op):
            op(lambda results: [holds(*r) for r in results], dtype=dtype)
adamw(lambda results: [holds(*r) for r in results], 32)
""")


def test_results_read_one_by_one_inside_a_scope(double):
    """In many orders; each operator runs once."""
    double("""
for op in KERNELS:
    for order in orders(op):
        def read(results):
            for i in order:
                holds(*results[i])
            return [t for t, _ in results]
        with Calls(op):
            Fusion.run(lambda: op(read))
Fusion.run(lambda: adamw(lambda results: [holds(*r) for r in results] and [t for t, _ in results], 32))
""")


def test_results_read_after_their_scope(double):
    """One result is returned, the others are kept by the program and read later."""
    double("""
for op, n in SIZES.items():
    for first in range(n):
        kept = []
        def read(results):
            kept[:] = results
            return results[first][0]
        with Calls(op):
            Fusion.run(lambda: op(read))
            for i in range(n):
                holds(*kept[(first + 1 + i) % n])
""")


def test_results_of_operators_whose_first_was_dropped(double):
    double("""
for op, n in SIZES.items():
    for first in range(1, n):
        kept = []
        def read(results):
            kept[:] = results[first:]
            return CudaArray.zeros([3]) + 1.0
        Fusion.run(lambda: op(read))
        for t, x in kept:
            holds(t, x)
""")


def test_gradients_after_the_scope_of_their_forward_pass(double):
    double("""
x, a, b = leaves((5, 9), (9, 7), (9, 7), dtype="bfloat16")
h = Fusion.run(lambda: x.gatedProjection(a, b))
h.backward(CudaArray.zeros([5, 7], "bfloat16"))
holds(x.grad(), 8.0), holds(a.grad(), 9.0), holds(b.grad(), 10.0)
q, s = leaves((2, 3, 1, 9), (9,))
y = Fusion.run(lambda: q.rotary(plan, None, scale=s))
y.backward(CudaArray.zeros([2, 3, 1, 9]))
holds(q.grad(), 3.0), holds(s.grad(), 5.0)
assert [count(k) for k in ("pt_gated", "pt_gated_backward", "pt_rotary", "pt_rotary_backward")] == [1] * 4
""")


def test_only_the_gradients_that_are_wanted(double):
    double("""
for wanted in itertools.product((0, 1), repeat=3):
    if not any(wanted):
        continue
    x, a, b = (CudaArray.zeros(s) for s in ([5, 9], [9, 7], [9, 7]))
    for t, w in zip((x, a, b), wanted):
        if w:
            t.requiresGrad()
    for run in (lambda f: f(), Fusion.run):
        h = run(lambda: x.gatedProjection(a, b))
        h.backward(CudaArray.zeros([5, 7]))
        for t, w, v in zip((x, a, b), wanted, (8.0, 9.0, 10.0)):
            if w:
                holds(t.grad(), v)
                t.zeroGrad()
# queries alone, keys alone, and one of a pair whose other has no part in the loss
q, k, s, t = leaves((6, 4, 10), (6, 2, 10), (10,), (10,))
a, b = q.rotary(plan, None, k, s, t)
b.sum().backward()
assert q.grad() is None or not q.grad().toNumpy().any()
holds(k.grad(), 4.0), holds(t.grad(), 6.0)
# constants beside what learns
q, k, s = CudaArray.zeros([6, 4, 10]), CudaArray.zeros([6, 2, 10]), leaves((10,))[0]
a, b = q.rotary(plan, None, k, s)
a.sum().backward()
holds(s.grad(), 5.0)
""")


def test_results_read_while_a_plan_is_recorded(double):
    """Of an operator that depends on no input of the plan, which may be read then."""
    double("""
def read(results):
    for r in results[::turn]:
        holds(*r)
    return [t for t, _ in results]
for op, turn in itertools.product(KERNELS, (1, -1)):
    values = []
    def step(y):
        def keep(results):
            values[:] = [x for _, x in results]
            return read(results)
        return [y + 1.0] + [t.detach() for t in op(keep)]
    compiled = Fusion.compile(step, [CudaArray.zeros([3])])
    for t, x in zip(compiled.run(CudaArray.zeros([3]))[1:], values):
        holds(t, x)
""")


def test_captured_forms_of_one_result(double):
    """One result a call, and what a capture may hold: a rotation of queries alone, a projection without gradients."""
    double("""
q, x, a = CudaArray.zeros([6, 4, 10]), CudaArray.zeros([5, 9]), CudaArray.zeros([9, 7])
for step, ins in ((lambda q: q.rotary(plan), [q]), (lambda x, a: x.gatedProjection(a, a), [x, a])):
    compiled = Fusion.compile(step, ins, cudaGraph=True)
    for _ in range(3):
        compiled.run(*ins)
    assert compiled.getStats()["graphLaunches"] > 0, compiled.getStats()
for step, ins in ((lambda q: list(q.rotary(plan, None, q)), [q]),):
    compiled = Fusion.compile(step, ins, cudaGraph=True)
    for _ in range(3):
        holds(compiled.run(*ins)[1], 2.5)
    assert compiled.getStats()["graphLaunches"] == 0 and compiled.getStats()["cudaGraphIncompatibility"] == "several-results"
""")


def test_empty_values(double):
    double("""
for run in (lambda f: f(), Fusion.run):
    assert run(lambda: CudaArray.zeros([0, 4, 8]).rotary(plan)).getShape() == [0, 4, 8]
    assert run(lambda: CudaArray.zeros([3, 0, 8]).rotary(plan)).getShape() == [3, 0, 8]
    assert run(lambda: CudaArray.zeros([0, 9]).gatedProjection(*leaves((9, 7), (9, 7)))).getShape() == [0, 7]
    assert run(lambda: CudaArray.zeros([2, 0, 9]).gatedProjection(*leaves((9, 7), (9, 7)))).getShape() == [2, 0, 7]
    assert run(lambda: CudaArray.zeros([5, 9]).gatedProjection(*leaves((9, 0), (9, 0)))).getShape() == [5, 0]
    for bits, master in itertools.product((32, 8), (False, True)):
        p = [CudaArray.zeros([0]), CudaArray.zeros([2, 0])]
        state = opt.initFusedState(p, bits, master)
        def step():
            r = opt.fusedStep(p, p, state)
            return [*r["parameters"], r["state"]["firstMoment"], r["state"]["beta1Power"]]
        r = run(step)
        assert [t.getShape() for t in r] == [[0], [2, 0], [0, 256], [1]], [t.getShape() for t in r]
        holds(r[3], 27.0)
""")
