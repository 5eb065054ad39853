"""What the host runtime does with operators of several results in Fusion scopes and plans, shown on a double of the
device library: no GPU."""
import pytest

import device_double


@pytest.fixture(scope="module")
def double(tmp_path_factory):
    folder = str(tmp_path_factory.mktemp("double"))
    device_double.build(folder)
    return lambda code: device_double.run(folder, code)


OPERATORS = """
import itertools

def logprobs(read):
    x, t = CudaArray.zeros([5, 30]), CudaArray.zeros([5], "int32")
    got = x.logProbs(t, top=2)
    return read([(got["logProbs"], 1.5), (got["entropy"], 2.5), (got["topLogProbs"], 4.5), (got["topTokens"], 7)])

def norm(read):
    x, s, b = (CudaArray.zeros(n).requiresGrad() for n in ([4, 6], [6], [6]))
    x.layerNorm([1], 1e-5, s, b).backward(CudaArray.zeros([4, 6]))
    return read([(x.grad(), 5.0), (s.grad(), 6.0), (b.grad(), 7.0)])

def attention(read):
    q, k, v = (CudaArray.zeros([6, n, 8]).requiresGrad() for n in (4, 2, 2))
    o = q.attention(k, v, causal=True)
    o.backward(CudaArray.zeros([6, 4, 8]))
    return read([(o, 1.5), (q.grad(), 5.0), (k.grad(), 6.0), (v.grad(), 7.0)])

KERNELS = {logprobs: ["pt_logprobs"], norm: ["pt_layernorm_backward"], attention: ["pt_attention", "pt_attention_backward"]}

def holds(t, x):
    got = t.toNumpy()
    assert (got == x).all(), (got.ravel()[:3], x)
"""


def test_results_read_one_by_one_inside_a_scope(double):
    """In every order; each operator runs once."""
    double(OPERATORS + """
for op, kernels in KERNELS.items():
    for order in itertools.permutations(range({logprobs: 4, norm: 3, attention: 4}[op])):
        before = [count(k) for k in kernels]
        def read(results):
            for i in order:
                holds(*results[i])
            return [t for t, _ in results]
        Fusion.run(lambda: op(read))
        assert [count(k) - n for k, n in zip(kernels, before)] == [1] * len(kernels), (op.__name__, order)
""")


def test_results_read_after_their_scope(double):
    """One result is returned, the others are kept by the program and read later."""
    double(OPERATORS + """
for op, kernels in KERNELS.items():
    n = {logprobs: 4, norm: 3, attention: 4}[op]
    for first in range(n):
        before, kept = [count(k) for k in kernels], []
        def read(results):
            kept[:] = results
            return results[first][0]
        Fusion.run(lambda: op(read))
        for i in range(n):
            holds(*kept[(first + 1 + i) % n])
        assert [count(k) - m for k, m in zip(kernels, before)] == [1] * len(kernels), (op.__name__, first)
""")


def test_results_of_an_operator_whose_first_was_dropped(double):
    double(OPERATORS + """
for n in (1, 2, 3):
    kept, before = [], count("pt_logprobs")
    def read(results):
        kept[:] = results[1:1 + n]
        return CudaArray.zeros([3]) + 1.0
    Fusion.run(lambda: logprobs(read))
    for t, x in kept:
        holds(t, x)
    assert count("pt_logprobs") == before + 1
""")


def test_gradients_after_the_scope_of_their_forward_pass(double):
    """What the forward pass leaves for the gradients is there when the gradients are asked for outside the scope."""
    double(OPERATORS + """
q, k, v = (CudaArray.zeros([6, n, 8]).requiresGrad() for n in (4, 2, 2))
o = Fusion.run(lambda: q.attention(k, v))
o.backward(CudaArray.zeros([6, 4, 8]))
holds(o, 1.5), holds(q.grad(), 5.0), holds(k.grad(), 6.0), holds(v.grad(), 7.0)
assert count("pt_attention") == count("pt_attention_backward") == 1
x, t, kept = CudaArray.zeros([5, 30]).requiresGrad(), CudaArray.zeros([5], "int32"), []
def read():
    kept.append(x.logProbs(t))
    return kept[0]["entropy"]
Fusion.run(read)
kept[0]["logProbs"].backward(CudaArray.zeros([5]))
holds(x.grad(), 6.0)   # stats and entropy
""")


def test_results_read_while_a_plan_is_recorded(double):
    """Of an operator that depends on no input of the plan, which may be read then."""
    double(OPERATORS + """
def read(results):
    for r in results[::turn]:
        holds(*r)
    return [t for t, _ in results]
for op, turn in itertools.product(KERNELS, (1, -1)):
    plan = Fusion.compile(lambda y: [y + 1.0] + [t.detach() for t in op(read)], [CudaArray.zeros([3])])
    for t, x in zip(plan.run(CudaArray.zeros([3]))[1:], {logprobs: (1.5, 2.5, 4.5, 7), norm: (5, 6, 7), attention: (1.5, 5, 6, 7)}[op]):
        holds(t, x)
""")


def test_types_of_gradients_that_add_up(double):
    """16-bit gradients of several uses, and of several backward calls, add up in float32 and are handed out in the
    operand's type; an operation in front gets its operand's type too."""
    double("""
from phptensors import autograd
for dtype in ("float16", "bfloat16"):
    q = CudaArray.zeros([6, 2, 8], dtype).requiresGrad()
    for n in range(3):
        before = count("pt_cast")
        o = q.attention(q, q)
        o.backward(o.detach())
        assert isinstance(q._grad, autograd.Sum) and q._grad.total.getDtype() == "float32"
        assert q.grad().getDtype() == dtype and q.grad() is q.grad()
        # the first of the walk's gradients is widened, and what is handed out rounded once
        assert count("pt_cast") - before == 2, count("pt_cast") - before
    w = CudaArray.zeros([16, 16], dtype).requiresGrad()
    y = CudaArray.zeros([6, 16], dtype).matmul(w).reshape([6, 2, 8])
    o = y.attention(y, y)
    o.backward(o.detach())
    assert w.grad().getDtype() == dtype
    plan = Fusion.compile(lambda a, g: (lambda b: (b.attention(b, b).backward(g), b.grad())[1])(a.detach().requiresGrad()),
                          [q.detach(), o.detach()])
    assert plan.run(q.detach(), o.detach()).getDtype() == dtype
""")


def test_upstream_gradients_of_every_floating_type(double):
    """Results that meet a float64 or a 16-bit tensor on the way to the loss."""
    double("""
def attention(dtype, up):
    q = CudaArray.zeros([6, 2, 8], dtype).requiresGrad()
    (q.attention(q, q) * CudaArray.ones([6, 2, 8], up)).sum().backward()
    return q
def logprobs(dtype, up):
    x = CudaArray.zeros([6, 9], dtype).requiresGrad()
    got = x.logProbs(CudaArray.zeros([6], "int32"), top=2)
    (got["entropy"] * CudaArray.ones([6], up) + got["topLogProbs"].sum(1) * CudaArray.ones([6], up)).sum().backward()
    return x
def norm(dtype, up):
    x = CudaArray.zeros([6, 9], dtype).requiresGrad()
    (x.layerNorm([1]) * CudaArray.ones([6, 9], up)).sum().backward()
    return x
for op in (attention, logprobs, norm):
    for dtype in ("float32", "float16", "bfloat16"):
        for up in ("float32", "float64", "float16", "bfloat16"):
            assert op(dtype, up).grad().getDtype() == dtype, (op.__name__, dtype, up)
""")


CAPTURES = """
def captured(step, inputs):
    plan = Fusion.compile(step, inputs, cudaGraph=True)
    for _ in range(2):   # the first run sizes the workspace, the second captures
        plan.run(*inputs)
    assert plan.getStats()["graphLaunches"] == 1, plan.getStats()
    return record()

def rules(calls, kernels):
    # every event stands for work on its stream (the first for the capture itself), waits are for recorded events, and
    # the plan's first kernel is on the capture's own stream
    assert sum(w == "launch" for w, _, _ in calls) == kernels, calls
    worked, events = set(), {}
    for n, (what, a, b) in enumerate(calls):
        if what == "launch":
            assert worked or a == 0, calls
            worked.add(a)
        elif what == "record":
            assert a not in events and (n == 0 or b in worked), (n, calls)
            events[a] = b
        else:
            assert b in events, calls
    # the capture's own stream ends behind all others
    waited = {events[b] for w, a, b in calls if w == "wait" and a == 0}
    assert worked - {0} <= waited, calls
"""


def test_branches_of_a_capture(double):
    """Steps that launch nothing (empty values) take no branch, wherever they stand."""
    double(CAPTURES + """
a, b, none = CudaArray.zeros([40, 40]), CudaArray.zeros([40, 40]), CudaArray.zeros([0, 40])
rules(captured(lambda x, y, e: [e * 2.0, x.matmul(y), y.matmul(x), x.sum(0)], [a, b, none]), 3)
rules(captured(lambda x, y, e: [e * 2.0, e.matmul(x), x.matmul(y), e.matmul(y), y.matmul(x).matmul(x)], [a, b, none]), 3)
rules(captured(lambda x, y, e: [x.matmul(y).matmul(x.matmul(x)), e + 1.0, y.matmul(x)], [a, b, none]), 4)
""")


def test_captured_attention_without_gradients(double):
    """Projections on several branches, attention behind them, and attention alone."""
    double(CAPTURES + """
for dtype in ("float32", "float16", "bfloat16"):
    x, w = CudaArray.zeros([24, 32], dtype), [CudaArray.zeros([32, n], dtype) for n in (32, 16, 16, 32)]
    at = Sequences([10, 14])
    def layer(x, wq, wk, wv, wo):
        q, k, v = (x.matmul(p).reshape([24, -1, 8]) for p in (wq, wk, wv))
        return q.attention(k, v, causal=True, queries=at).reshape([24, 32]).matmul(wo)
    rules(captured(layer, [x, *w]), 5)
    q, k = CudaArray.zeros([24, 4, 8], dtype), CudaArray.zeros([24, 2, 8], dtype)
    rules(captured(lambda q, k: [q.attention(k, k), k.attention(k, k)], [q, k]), 2)
""")


def test_plans_of_several_results_are_not_captured(double):
    double("""
x, t = CudaArray.zeros([5, 30]), CudaArray.zeros([5], "int32")
plan = Fusion.compile(lambda x: list(x.logProbs(t).values()), [x], cudaGraph=True)
for _ in range(3):
    plan.run(x)
stats = plan.getStats()
assert stats["graphLaunches"] == 0 and stats["cudaGraphIncompatibility"] == "several-results" and count("pt_graph_begin_capture") == 0
""")
