"""More operators of language models that are timed: their plain forms in torch and the framework's calls.

Three operators that stand beside the matrix products and the attention of a block: the rotation of queries and keys by
their positions, with the norm of each head in the same pass; the gated projection act(x gate) * (x up); and the AdamW
step over all of a model's tensors, with moments in 32 or in 8 bits.  A case names its `kind`, sizes and types.  `run`
computes it from elementary torch operations in 32 bits, or, with `own`, through the framework as a program calls it.
"""
import math
import os
import sys

import torch

own = False

TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
EPSILON = 1e-6
# AdamW's numbers, those of a usual training program
RATE, BETA1, BETA2, ADAM_EPSILON, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
STEPS = 20      # steps that the moments stand for
BLOCK = 256     # elements that share a power of two in 8-bit moments


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one new token for each of 32 requests, far into a stretched context: launches and host time
        {"name": "rotary_token_bf16", "kind": "rotary", "dtype": "bfloat16", "sequences": 0, "tokens": 32, "heads": 32,
         "kv_heads": 8, "size": 128, "part": 128, "interleaved": False, "norm": True, "factor": 8.0, "context": 8192,
         "far": 1000000, "train": False},
        # a training step's queries and keys, normalised, both directions from memory
        {"name": "rotary_train_bf16", "kind": "rotary", "dtype": "bfloat16", "sequences": 0, "tokens": 8192, "heads": 32,
         "kv_heads": 8, "size": 128, "part": 128, "interleaved": False, "norm": True, "factor": 1.0, "context": 0,
         "far": 8192, "train": True},
        # a quarter of each head rotated in neighbouring pairs, in 32 bits, sequences of an odd length
        {"name": "rotary_f32_odd", "kind": "rotary", "dtype": "float32", "sequences": 3, "tokens": 1001, "heads": 12,
         "kv_heads": 12, "size": 80, "part": 20, "interleaved": True, "norm": False, "factor": 1.0, "context": 0,
         "far": 1001, "train": True},
        # one token through a wide layer: both weights stream from memory
        {"name": "gated_token_bf16", "kind": "gated", "dtype": "bfloat16", "rows": 1, "inner": 4096, "outer": 16384,
         "activation": "silu", "train": False},
        # a step of several requests together
        {"name": "gated_few_bf16", "kind": "gated", "dtype": "bfloat16", "rows": 24, "inner": 2048, "outer": 8192,
         "activation": "silu", "train": False},
        # a prompt through a layer whose widths fill no whole packs or tiles
        {"name": "gated_prompt_f16_odd", "kind": "gated", "dtype": "float16", "rows": 1733, "inner": 1000, "outer": 2731,
         "activation": "gelu", "train": False},
        # a training step's layer, forward and backward
        {"name": "gated_train_bf16", "kind": "gated", "dtype": "bfloat16", "rows": 8192, "inner": 2048, "outer": 8192,
         "activation": "silu", "train": True},
        # the first layer of the benchmark's classifier, gated, in 32 bits, forward and backward
        {"name": "gated_train_f32", "kind": "gated", "dtype": "float32", "rows": 4096, "inner": 784, "outer": 1024,
         "activation": "silu", "train": True},
        # the tensors of the benchmark's classifier: the latency of a step
        {"name": "adamw_classifier_f32", "kind": "adamw", "dtype": "float32", "grad": "float32", "bits": 32,
         "master": False, "layers": 0, "width": 0, "hidden": 0, "rows": 0},
        # a small language model in 16 bits with float32 masters
        {"name": "adamw_model_bf16", "kind": "adamw", "dtype": "bfloat16", "grad": "bfloat16", "bits": 32,
         "master": True, "layers": 6, "width": 1024, "hidden": 4096, "rows": 32768},
        # the same with moments in 8 bits, as a program holds them that has little memory left
        {"name": "adamw_model_8bit", "kind": "adamw", "dtype": "bfloat16", "grad": "bfloat16", "bits": 8,
         "master": False, "layers": 6, "width": 1024, "hidden": 4096, "rows": 32768},
    ]


def _size(rng, low, high):
    """A size between low and high, even over the logarithm; half of them multiples of 16 where that fits."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 16:
        v -= v % 16
    return max(low, min(high, v))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "gated", "gated", "few", "adamw"])
    wide = ["float32", "float16", "bfloat16"]
    while True:
        if kind == "rotary":
            size = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
            kv = rng.choice([1, 2, 4, 8])
            case = {"kind": "rotary", "dtype": rng.choice(wide), "sequences": rng.choice([0, 0, 1, 4]),
                    "tokens": _size(rng, 1, 8192), "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "size": size,
                    "part": rng.choice([size, size, size // 2, size // 4]), "interleaved": rng.random() < 0.4,
                    "norm": rng.random() < 0.6, "factor": rng.choice([1.0, 1.0, 4.0, 8.0]),
                    "context": rng.choice([0, 4096]), "far": _size(rng, 8192, 1000000), "train": rng.random() < 0.5}
        elif kind in ("gated", "few"):
            case = {"kind": "gated", "dtype": rng.choice(wide), "rows": _size(rng, 1, 32 if kind == "few" else 8192),
                    "inner": _size(rng, 64, 4096), "outer": _size(rng, 64, 16384),
                    "activation": rng.choice(["silu", "silu", "gelu", "relu", "sigmoid"]),
                    "train": kind == "gated" and rng.random() < 0.6}
        else:
            dt = rng.choice(wide)
            case = {"kind": "adamw", "dtype": dt, "grad": rng.choice([dt, "float32"]), "bits": rng.choice([32, 32, 8]),
                    "master": dt != "float32" and rng.random() < 0.5, "layers": _size(rng, 1, 6),
                    "width": _size(rng, 64, 1024), "hidden": _size(rng, 64, 4096), "rows": _size(rng, 100, 32768)}
        w = work(case)
        # no more than the largest listed calls: 1.6 TFLOP in 16 bits, 40 GFLOP in 32 bits, 3.8 GB moved
        most = 4e10 if case["dtype"] == "float32" else 1.6e12
        if (case["kind"] == "adamw" or w["flops"] <= most) and w["bytes"] <= (3.8e9 if case["kind"] == "adamw" else 5e8):
            return case


# ------------------------------------------------------------------ inputs
class _Inputs:
    """Random tensors on the GPU from one seed, in one order."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, shape, dtype="float32", std=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * std).to(TORCH[dtype])

    def integers(self, shape, low, high, dtype=torch.int32):
        return torch.randint(low, high, shape, generator=self.g, device="cuda", dtype=dtype)


def _shapes(c):
    """The model's tensors: the benchmark's classifier, or embeddings and, a layer, two norms, four square weights and
    the three of a gated block."""
    if not c["layers"]:
        return [(784, 1024), (1, 1024), (1024, 1024), (1, 1024), (1024, 10), (1, 10)]
    w, h = c["width"], c["hidden"]
    return [(c["rows"], w)] + [s for _ in range(c["layers"])
                               for s in ((w,), (w, w), (w, w), (w, w), (w, w), (w,), (w, h), (w, h), (h, w))]


def _places(shapes):
    """Where each tensor's moments begin in the one array of blocks that holds them all, and the array's size."""
    at = [0]
    for s in shapes:
        at.append(at[-1] + -(-math.prod(s) // BLOCK) * BLOCK)
    return at[:-1], at[-1]


def _joined(shapes, tensors):
    """Tensors in one array, zeros between them."""
    at, size = _places(shapes)
    out = torch.zeros(size, device="cuda")
    for a, t in zip(at, tensors):
        out[a:a + t.numel()] = t.reshape(-1)
    return out


def _decays(shapes):
    return [len(s) > 1 and s[0] > 1 for s in shapes]  # weights decay, norms and biases do not


def _frequencies(c):
    part, factor, context = c["part"], c["factor"], c["context"]
    f = 10000.0 ** (-torch.arange(0, part, 2, dtype=torch.float64, device="cuda") / part)
    if factor == 1.0:
        return f
    if not context:
        return f / factor
    keep = ((context * f / (2.0 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return f * keep + f / factor * (1.0 - keep)


def _magnitude(c):
    """Scores grow a little as the context is stretched."""
    return 0.1 * math.log(c["factor"]) + 1.0 if c["context"] else 1.0


def _make(c, seed):
    """The inputs as torch tensors by name (lists of tensors for AdamW)."""
    r, dt = _Inputs(seed), c["dtype"]
    if c["kind"] == "rotary":
        lead = (c["sequences"], c["tokens"]) if c["sequences"] else (c["tokens"],)
        made = {}
        for name, heads in (("q", c["heads"]), ("k", c["kv_heads"])):
            made[name] = r.normal((*lead, heads, c["size"]), dt, 2.0)
            if c["norm"]:
                made[name + "s"] = r.normal((c["size"],), dt, 0.1) + 1.0
            if c["train"]:
                made[name + "g"] = r.normal((*lead, heads, c["size"]), dt, 0.1)
        made["positions"] = r.integers(lead, 0, c["far"])
        return made
    if c["kind"] == "gated":
        made = {"x": r.normal((c["rows"], c["inner"]), dt)}
        for name in ("gate", "up"):
            made[name] = r.normal((c["inner"], c["outer"]), dt, 1.0 / math.sqrt(c["inner"]))
        if c["train"]:
            made["g"] = r.normal((c["rows"], c["outer"]), dt, 0.1)
        return made
    shapes = _shapes(c)
    made = {"p": [r.normal(s, std=0.02) for s in shapes], "g": [r.normal(s, c["grad"], 1e-3) for s in shapes]}
    if c["master"]:
        made["master"] = _joined(shapes, made["p"]).reshape(-1, BLOCK)
    made["p"] = [p.to(TORCH[dt]) for p in made["p"]]
    made["m"] = _joined(shapes, [r.normal(t, std=3e-4) for t in shapes]).reshape(-1, BLOCK)
    made["v"] = _joined(shapes, [r.normal(t, std=1e-3) ** 2 * 0.02 for t in shapes]).reshape(-1, BLOCK)
    if c["bits"] == 8:
        made["m"], made["me"] = _encode(made["m"], False, None)
        made["v"], made["ve"] = _encode(made["v"], True, None)
        made["draws"] = r.integers((1,), 0, 1 << 30)
    return made


def _powers():
    return [torch.full((1,), b ** STEPS, device="cuda", dtype=torch.float32) for b in (BETA1, BETA2)]


def _framework():
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "php-gpu-tensors_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import phptensors
    return phptensors


def _array(framework, t):
    """A CudaArray with the tensor's values, copied on the GPU."""
    from phptensors import _abi, _host
    a = framework.CudaArray.zeros(list(t.shape), str(t.dtype).replace("torch.", ""))
    torch.cuda.synchronize()
    _abi.check(_abi.load().pt_memcpy_d2d(_host.load().phpt_device_pointer(a._h), t.data_ptr(),
                                         t.numel() * t.element_size(), None))
    # the framework's stream does not wait for torch's, nor torch's for it: the copy ends before t's memory is used again
    torch.cuda.synchronize()
    return a


class _Memory:
    """A CudaArray's memory as __cuda_array_interface__ describes it (bfloat16, which has no spelling there, as
    16-bit integers); the tensor made of it keeps the array alive."""
    SPELLED = {"float32": "<f4", "float16": "<f2", "bfloat16": "<i2"}

    def __init__(self, array, pointer, dtype):
        self.array = array
        self.__cuda_array_interface__ = {"data": (pointer, False), "shape": array.shape, "version": 2,
                                         "typestr": self.SPELLED[dtype]}


def _tensors(arrays):
    from phptensors import _host
    pointer, out = _host.load().phpt_device_pointer, []
    for a in arrays:
        dt = a.getDtype()
        t = torch.as_tensor(_Memory(a, pointer(a._h), dt), device="cuda")
        out.append(t.view(torch.bfloat16) if dt == "bfloat16" else t)
    return out


def prepare(case, seed):
    c = dict(case)
    s = _make(c, seed)
    if own:
        # the same inputs in the arrays that a program of the framework holds
        framework = _framework()
        s = {n: [_array(framework, t) for t in v] if isinstance(v, list) else _array(framework, v) for n, v in s.items()}
    s["case"] = c
    if c["kind"] == "rotary" and own:
        s["angles"] = framework.Rotary(c["part"], interleaved=c["interleaved"], factor=c["factor"],
                                       context=c["context"] or None, magnitude=_magnitude(c))
    if c["kind"] == "rotary" and not own:
        s["angles"] = _frequencies(c)
    if c["kind"] == "adamw":
        s["decays"] = _decays(_shapes(c))
        s["powers"] = _powers()
        if own:
            from phptensors.optimizer import Optimizer
            s["powers"] = [_array(framework, t) for t in s["powers"]]
            s["optimizer"] = Optimizer.adamW(RATE, BETA1, BETA2, ADAM_EPSILON, DECAY)
            state = s["optimizer"].initFusedState(s["p"], bits=c["bits"], master=c["master"])
            state.update(firstMoment=s["m"], secondMoment=s["v"], beta1Power=s["powers"][0], beta2Power=s["powers"][1])
            if c["master"]:
                state.update(master=s["master"])
            if c["bits"] == 8:
                state.update(firstExponent=s["me"], secondExponent=s["ve"], draws=s["draws"])
            s["state"] = state
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _tensors({"rotary": _own_rotary, "gated": _own_gated, "adamw": _own_adamw}[kind](s))
    return {"rotary": _plain_rotary, "gated": _plain_gated, "adamw": _plain_adamw}[kind](s)


def _own_rotary(s):
    c = s["case"]
    leaves = [s["q"], s["k"]] + ([s["qs"], s["ks"]] if c["norm"] else [])
    if c["train"]:
        for t in leaves:
            t.requiresGrad().zeroGrad()
    q, k = s["q"].rotary(s["angles"], s["positions"], key=s["k"], scale=s.get("qs"), keyScale=s.get("ks"),
                         epsilon=EPSILON)
    if not c["train"]:
        return [q, k]
    q.backward(s["qg"])
    k.backward(s["kg"])
    return [q, k] + [t.grad() for t in leaves]


def _own_gated(s):
    leaves = [s["x"], s["gate"], s["up"]]
    if not s["case"]["train"]:
        return [s["x"].gatedProjection(s["gate"], s["up"], s["case"]["activation"])]
    for t in leaves:
        t.requiresGrad().zeroGrad()
    h = s["x"].gatedProjection(s["gate"], s["up"], s["case"]["activation"])
    h.backward(s["g"])
    return [h] + [t.grad() for t in leaves]


def _own_adamw(s):
    got = s["optimizer"].fusedStep(s["p"], s["g"], s["state"], weightDecayMask=s["decays"])
    moments = s["optimizer"].moments(got["state"]) if s["case"]["bits"] == 8 else got["state"]
    return (got["parameters"] + ([got["state"]["master"]] if s["case"]["master"] else [])
            + [moments["firstMoment"], moments["secondMoment"]])


def _turn(c, x, cos, sin):
    """The rotated part of x [.., size] by angles [.., 1, part / 2]."""
    part, half = c["part"], c["part"] // 2
    head = x[..., :part]
    a, b = (head[..., 0::2], head[..., 1::2]) if c["interleaved"] else (head[..., :half], head[..., half:])
    turned = [a * cos - b * sin, a * sin + b * cos]
    turned = torch.stack(turned, -1).flatten(-2) if c["interleaved"] else torch.cat(turned, -1)
    return torch.cat([turned, x[..., part:]], -1)


def _plain_rotary(s):
    c, m = s["case"], _magnitude(s["case"])
    angle = (s["positions"].double()[..., None] * s["angles"])[..., None, :]  # (32 bits lose far positions)
    cos, sin = (angle.cos() * m).float(), (angle.sin() * m).float()
    out, grads, scales = [], [], []
    for name in "qk":
        given = s[name]
        x = given.float()
        if c["norm"]:
            inverse = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPSILON)
            unit, scale = x * inverse, s[name + "s"].float()
            out.append(_turn(c, unit * scale, cos, sin).to(given.dtype))
        else:
            out.append(_turn(c, x, cos, sin).to(given.dtype))
        if not c["train"]:
            continue
        d = _turn(c, s[name + "g"].float(), cos, -sin)
        if c["norm"]:
            scales.append((d * unit).flatten(0, -2).sum(0).to(given.dtype))
            d = d * scale
            d = inverse * (d - unit * (d * unit).mean(-1, keepdim=True))
        grads.append(d.to(given.dtype))
    return out + grads + scales


def _act(name, g):
    """The activation and its derivative."""
    if name == "relu":
        return torch.where(g > 0.0, g, 0.0), torch.where(g > 0.0, 1.0, 0.0)
    if name == "gelu":
        below = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * below, below + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    part = 1.0 / (1.0 + torch.exp(-g))
    if name == "sigmoid":
        return part, part * (1.0 - part)
    return g * part, part * (1.0 + g * (1.0 - part))


def _plain_gated(s):
    c, dt = s["case"], s["x"].dtype
    x, gate, up = s["x"].float(), s["gate"].float(), s["up"].float()
    g, u = x @ gate, x @ up
    act, slope = _act(c["activation"], g)
    h = (act * u).to(dt)
    if not c["train"]:
        return [h]
    dh = s["g"].float()
    dg, du = dh * u * slope, dh * act
    dx = dg @ gate.t() + du @ up.t()
    return [h, dx.to(dt), (x.t() @ dg).to(dt), (x.t() @ du).to(dt)]


# 8-bit moments: 256 elements in a row share the power of two 2^e that takes the largest of them into [128, 256).  A first
# moment is held as a sign, 4 bits of exponent and 3 of mantissa, the root of a second one as 4 and 4 bits.
def _decode(code, exponent, root):
    bits = code.int()
    size = ((bits << 19) if root else ((bits & 127) << 20)).view(torch.float32) * 2.0 ** 120
    scale = ((exponent.int() + 127) << 23).view(torch.float32)[:, None]
    x = size * scale
    return x * x if root else torch.where(bits >= 128, -x, x)


def _encode(x, root, rounding):
    """(codes, exponents); rounding: a number of 16 bits an element, None to round to the nearest."""
    blocks = torch.sqrt(x) if root else x
    top = blocks.abs().amax(1).view(torch.int32) >> 23
    exponent = (top - 127 - 7).clamp_min(-126)
    scale = ((127 - exponent) << 23).view(torch.float32)[:, None]
    size = ((blocks.abs() * scale) * 2.0 ** -120).view(torch.int32)
    low = 19 if root else 20
    if rounding is None:
        code = (size + (1 << (low - 1))) >> low
    else:
        code = (size + (rounding << (low - 16)) + (1 << (low - 17))) >> low
    if not root:
        code = code | torch.where(blocks < 0.0, 128, 0)
    return code.to(torch.uint8), exponent.to(torch.int8)


def _mix(h):
    """32 bits spread over 32 bits: xor-shifts and multiplications (the finalizer of MurmurHash3)."""
    h = h ^ (h >> 16)
    h = h * 0x85EBCA6B & 0xFFFFFFFF
    h = h ^ (h >> 13)
    h = h * 0xC2B2AE35 & 0xFFFFFFFF
    return h ^ (h >> 16)


def _rounding(draws, like):
    """Numbers of 16 bits for the first and for the second moment of each element."""
    h = _mix((torch.arange(like.numel(), device="cuda") + _mix(draws.long())) & 0xFFFFFFFF).reshape(like.shape)
    return (h & 0xFFFF).int(), (h >> 16).int()


def _plain_adamw(s):
    c, small = s["case"], s["case"]["bits"] == 8
    c1, c2 = ((p * b - 1.0) * -1.0 for p, b in zip(s["powers"], (BETA1, BETA2)))
    m0, v0 = (_decode(s["m"], s["me"], False), _decode(s["v"], s["ve"], True)) if small else (s["m"], s["v"])
    first, second, params = torch.zeros_like(m0), torch.zeros_like(v0), []
    masters = torch.zeros_like(m0) if c["master"] else None
    m0, v0, m1, v1 = (t.reshape(-1) for t in (m0, v0, first, second))
    for i, (at, given) in enumerate(zip(_places(_shapes(c))[0], s["p"])):
        here = slice(at, at + given.numel())
        g = s["g"][i].float().reshape(-1)
        p = s["master"].reshape(-1)[here] if c["master"] else given.float().reshape(-1)
        m1[here] = m = m0[here] * BETA1 + g * (1.0 - BETA1)
        v1[here] = v = v0[here] * BETA2 + (g * g) * (1.0 - BETA2)
        step = (m / c1) / (torch.sqrt(v / c2) + ADAM_EPSILON) * RATE
        new = p * (1.0 - RATE * DECAY) - step if s["decays"][i] else p - step
        params.append(new.to(given.dtype).reshape(given.shape))
        if c["master"]:
            masters.reshape(-1)[here] = new
    if small:
        r = _rounding(s["draws"], first)
        first, second = _decode(*_encode(first, False, r[0]), False), _decode(*_encode(second, True, r[1]), True)
    return params + ([masters] if c["master"] else []) + [first, second]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "rotary":
        b = SIZE[c["dtype"]]
        n = max(1, c["sequences"]) * c["tokens"]
        x = n * (c["heads"] + c["kv_heads"]) * c["size"]
        # each head in and out; with gradients the upstream one in and the head's out
        return {"bytes": x * b * (4 if c["train"] else 2) + 4 * n, "flops": (20.0 if c["train"] else 8.0) * x}
    if c["kind"] == "gated":
        b, m, k, f = SIZE[c["dtype"]], c["rows"], c["inner"], c["outer"]
        if not c["train"]:
            return {"bytes": b * (m * k + 2 * k * f + m * f), "flops": 4.0 * m * k * f}
        return {"bytes": b * (2 * m * k + 4 * k * f + 2 * m * f), "flops": 12.0 * m * k * f}
    n = sum(math.prod(s) for s in _shapes(c))
    p, g = SIZE[c["dtype"]], SIZE[c["grad"]]
    # parameters, masters and moments in and out, gradients in; of 8-bit moments also the values they stand for
    moments = 16 if c["bits"] == 32 else 4 + 8
    return {"bytes": n * (g + moments + (p + 8 if c["master"] else 2 * p)), "flops": 16.0 * n}


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    made = _make(case, seed)
    return {"rotary": _exact_rotary, "gated": _exact_gated, "adamw": _exact_adamw}[case["kind"]](case, made)


def _exact_rotary(c, d):
    """The pairs as complex numbers, the gradients by torch's own differentiation."""
    turn = torch.polar(torch.full((), _magnitude(c), dtype=torch.float64, device="cuda"),
                       d["positions"].double()[..., None, None] * _frequencies(c))
    out, grads, scales = [], [], []
    for name in "qk":
        x = d[name].double().requires_grad_(c["train"])
        y = x
        if c["norm"]:
            scale = d[name + "s"].double().requires_grad_(c["train"])
            y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPSILON) * scale
        head = y[..., :c["part"]]
        if c["interleaved"]:
            pairs = torch.view_as_complex(head.reshape(*head.shape[:-1], -1, 2)) * turn
            head = torch.view_as_real(pairs).flatten(-2)
        else:
            pairs = torch.complex(*head.chunk(2, -1)) * turn
            head = torch.cat([pairs.real, pairs.imag], -1)
        y = torch.cat([head, y[..., c["part"]:]], -1)
        out.append(y.detach())
        if c["train"]:
            got = torch.autograd.grad(y, [x, scale] if c["norm"] else [x], d[name + "g"].double())
            grads.append(got[0])
            scales.extend(got[1:])
    return out + grads + scales


def _exact_gated(c, d):
    x, gate, up = (d[n].double().requires_grad_(c["train"]) for n in ("x", "gate", "up"))
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
         "sigmoid": torch.sigmoid}[c["activation"]]
    h = f(x @ gate) * (x @ up)
    if not c["train"]:
        return [h]
    return [h.detach(), *torch.autograd.grad(h, [x, gate, up], d["g"].double())]


def _exact_adamw(c, d):
    """The moments of 8 bits have no value in 64 bits: they are rounded by drawn numbers."""
    p1, p2 = (p.double() for p in _powers())
    shapes, small = _shapes(c), c["bits"] == 8
    m0, v0 = (_decode(d["m"], d["me"], False), _decode(d["v"], d["ve"], True)) if small else (d["m"], d["v"])
    grads = _joined(shapes, d["g"]).double().reshape(-1, BLOCK)
    m, v = torch.lerp(grads, m0.double(), BETA1), torch.lerp(grads.square(), v0.double(), BETA2)
    rate = v.div(1.0 - p2 * BETA2).sqrt().add(ADAM_EPSILON).reciprocal().mul(RATE / (1.0 - p1 * BETA1))
    old = (d["master"] if c["master"] else _joined(shapes, d["p"]).reshape(-1, BLOCK)).double()
    keep = _joined(shapes, [torch.full(t, float(y), device="cuda") for t, y in zip(shapes, _decays(shapes))])
    new = old - m * rate - RATE * DECAY * keep.double().reshape(-1, BLOCK) * old
    params = [new.reshape(-1)[a:a + math.prod(t)].reshape(t) for a, t in zip(_places(shapes)[0], shapes)]
    return params + ([new] if c["master"] else []) + [None if small else m, None if small else v]
