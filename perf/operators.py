"""The operators of language models that are timed: their plain forms in torch and the framework's calls.

Three operators that a program needs around its matrix products to train and to serve such a model: layer
normalisation with its gradients, attention over whole prompts and over caches with its gradients, and the log
probabilities of given tokens with their gradients.  A case names its `kind`, sizes, types and lengths.  `run`
computes it from elementary torch operations in 32 bits, or, with `own`, through CudaArray as a program calls it.
"""
import math
import os
import sys

import torch

own = False

TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
EPSILON = 1e-5


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one layer's normalisation in a small model's training step: launches and host time
        {"name": "norm_small_f32", "kind": "norm", "dtype": "float32", "rows": 64, "cols": 1024},
        # a large activation, both directions from memory
        {"name": "norm_f32", "kind": "norm", "dtype": "float32", "rows": 8192, "cols": 4096},
        # the same in 16 bits over an odd width, rows that start anywhere in a 16-byte pack
        {"name": "norm_bf16_odd", "kind": "norm", "dtype": "bfloat16", "rows": 6000, "cols": 1001},
        # prompts of several requests packed one behind the other, four query heads to a key head
        {"name": "prompt_bf16", "kind": "attention", "dtype": "bfloat16", "heads": 16, "kv_heads": 4, "size": 128,
         "queries": "4096,1733,2048,517,3001,1", "keys": "", "slots": 0, "causal": True, "train": False},
        # an encoder over texts that were not padded: no causal limit, odd lengths, small heads
        {"name": "prompt_f16_odd", "kind": "attention", "dtype": "float16", "heads": 12, "kv_heads": 12, "size": 64,
         "queries": "1021,333,777,129,64,999,1500,31", "keys": "", "slots": 0, "causal": False, "train": False},
        # one new token for each of many requests, each with its own slot of a cache
        {"name": "token_bf16", "kind": "attention", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "size": 128,
         "queries": ",".join(["1"] * 32), "keys": ",".join(str(977 + 229 * i) for i in range(32)), "slots": 8192,
         "causal": True, "train": False},
        # one request alone: the latency of a token
        {"name": "token_alone_f16", "kind": "attention", "dtype": "float16", "heads": 16, "kv_heads": 4, "size": 64,
         "queries": "1", "keys": "700", "slots": 1024, "causal": True, "train": False},
        # a training step's attention, forward and backward
        {"name": "train_bf16", "kind": "attention", "dtype": "bfloat16", "heads": 16, "kv_heads": 8, "size": 128,
         "queries": "2048,2048,2048,2048", "keys": "", "slots": 0, "causal": True, "train": True},
        # the same in 32 bits over lengths that fill no whole tiles
        {"name": "train_f32_odd", "kind": "attention", "dtype": "float32", "heads": 8, "kv_heads": 8, "size": 64,
         "queries": "777,1001,50", "keys": "", "slots": 0, "causal": True, "train": True},
        # scoring texts: each token's log probability, the entropy and the likeliest alternatives, an odd vocabulary
        {"name": "score_bf16", "kind": "logprobs", "dtype": "bfloat16", "rows": 2000, "cols": 50021, "top": 8,
         "train": False},
        # a training step's loss and its gradient by the scores; some positions carry no token
        {"name": "loss_f32", "kind": "logprobs", "dtype": "float32", "rows": 4096, "cols": 32768, "top": 0,
         "train": True},
        # a few requests' next tokens, reported with their alternatives: the latency of a step
        {"name": "step_f32", "kind": "logprobs", "dtype": "float32", "rows": 4, "cols": 131072, "top": 20,
         "train": False},
    ]


def _size(rng, low, high):
    """A size between low and high, even over the logarithm; half of them multiples of 16 where that fits."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 16:
        v -= v % 16
    return max(low, min(high, v))


def draw(rng):
    kind = rng.choice(["norm", "prompt", "token", "train", "score", "loss"])
    wide = ["float32", "float16", "bfloat16"]
    while True:
        if kind == "norm":
            case = {"kind": "norm", "dtype": rng.choice(wide), "rows": _size(rng, 1, 16384),
                    "cols": _size(rng, 16, 16384)}
        elif kind in ("score", "loss"):
            case = {"kind": "logprobs", "dtype": rng.choice(wide), "rows": _size(rng, 1, 8192),
                    "cols": _size(rng, 256, 140000), "top": rng.choice([0, 1, 5, 8, 20]) if kind == "score" else 0,
                    "train": kind == "loss"}
        else:
            kv = rng.choice([1, 2, 4, 8])
            case = {"kind": "attention", "dtype": rng.choice(wide), "heads": kv * rng.choice([1, 2, 4]),
                    "kv_heads": kv, "size": rng.choice([32, 64, 80, 96, 128, 128]), "keys": "", "slots": 0,
                    "causal": rng.random() < 0.75, "train": kind == "train"}
            if kind == "token":
                slots = _size(rng, 64, 8192)
                keys = [_size(rng, 1, slots) for _ in range(_size(rng, 1, 32))]
                case.update(queries=",".join(["1"] * len(keys)), keys=",".join(map(str, keys)), slots=slots,
                            causal=True)
            else:
                case["queries"] = ",".join(str(_size(rng, 1, 2048)) for _ in range(_size(rng, 1, 8)))
        w = work(case)
        # no more than the largest listed calls: 0.3 TFLOP in 16 bits, 15 GFLOP in fp32, 1.1 GB moved
        most = 1.5e10 if case["dtype"] == "float32" else 3e11
        if w["flops"] <= most and w["bytes"] <= 1.1e9:
            return case


# ------------------------------------------------------------------ inputs
class _Inputs:
    """Random tensors on the GPU from one seed, in one order."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, shape, dtype="float32", std=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * std).to(TORCH[dtype])

    def integers(self, shape, high):
        return torch.randint(high, shape, generator=self.g, device="cuda", dtype=torch.int32)


def _lengths(text):
    return [int(v) for v in text.split(",")] if text else []


def _sequences(c):
    """(lengths, starts) of the queries and of the keys; the keys lie packed as the queries do, or in slots."""
    q = _lengths(c["queries"])
    qs = [sum(q[:i]) for i in range(len(q))]
    if not c["keys"]:
        return (q, qs), (q, qs)
    return (q, qs), (_lengths(c["keys"]), [i * c["slots"] for i in range(len(q))])


def _make(c, seed):
    """The inputs as torch tensors by name."""
    r, dt = _Inputs(seed), c["dtype"]
    if c["kind"] == "norm":
        return {"x": r.normal((c["rows"], c["cols"]), dt, 2.0) + 0.5, "scale": r.normal((c["cols"],), dt, 0.1) + 1.0,
                "bias": r.normal((c["cols"],), dt, 0.1), "g": r.normal((c["rows"], c["cols"]), "float32", 0.1)}
    if c["kind"] == "logprobs":
        x = r.normal((c["rows"], c["cols"]), dt, 2.5)
        tokens = r.integers((c["rows"],), c["cols"])
        made = {"x": x, "tokens": tokens}
        if c["train"]:
            made["tokens"] = torch.where(r.integers((c["rows"],), 16) == 0, -1, tokens)
            made["g"] = r.normal((c["rows"],), "float32", 0.1) - 1.0
            made["h"] = r.normal((c["rows"],), "float32", 0.01)
        return made
    rows = sum(_lengths(c["queries"]))
    kept = len(_lengths(c["queries"])) * c["slots"] or rows
    made = {"q": r.normal((rows, c["heads"], c["size"]), dt), "k": r.normal((kept, c["kv_heads"], c["size"]), dt),
            "v": r.normal((kept, c["kv_heads"], c["size"]), dt)}
    if c["train"]:
        made["g"] = r.normal((rows, c["heads"], c["size"]), dt)
    return made


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
    SPELLED = {"float32": "<f4", "float16": "<f2", "bfloat16": "<i2", "int32": "<i4"}

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
        s = {n: _array(framework, t) for n, t in s.items()}
    s["case"] = c
    if c["kind"] == "attention":
        queries, keys = _sequences(c)
        if own:
            s["queries"] = framework.Sequences(*queries)
            s["keys"] = framework.Sequences(*keys) if c["keys"] else s["queries"]
        else:
            s["queries"], s["keys"] = ([torch.tensor(v, device="cuda") for v in side] for side in (queries, keys))
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _tensors({"norm": _own_norm, "attention": _own_attention, "logprobs": _own_logprobs}[kind](s))
    return {"norm": _plain_norm, "attention": _plain_attention, "logprobs": _plain_logprobs}[kind](s)


def _own_norm(s):
    leaves = [s["x"], s["scale"], s["bias"]]
    for t in leaves:
        t.requiresGrad().zeroGrad()
    y = s["x"].layerNorm([1], EPSILON, s["scale"], s["bias"])
    y.backward(s["g"])
    return [y] + [t.grad() for t in leaves]


def _own_attention(s):
    c, leaves = s["case"], [s["q"], s["k"], s["v"]]
    if not c["train"]:
        return [s["q"].attention(s["k"], s["v"], causal=c["causal"], queries=s["queries"], keys=s["keys"])]
    for t in leaves:
        t.requiresGrad().zeroGrad()
    o = s["q"].attention(s["k"], s["v"], causal=c["causal"], queries=s["queries"], keys=s["keys"])
    o.backward(s["g"])
    return [o] + [t.grad() for t in leaves]


def _own_logprobs(s):
    if not s["case"]["train"]:
        got = s["x"].logProbs(s["tokens"], top=s["case"]["top"])
        out = [got["logProbs"], got["entropy"]]
        return out + [got["topLogProbs"], got["topTokens"]] if s["case"]["top"] else out
    s["x"].requiresGrad().zeroGrad()
    got = s["x"].logProbs(s["tokens"])
    # the mean log probability with a small reward for entropy: one weight a row and output
    loss = (got["logProbs"] * s["g"] + got["entropy"] * s["h"]).sum()
    loss.backward()
    return [got["logProbs"], got["entropy"], s["x"].grad()]


def _plain_norm(s):
    dt = s["x"].dtype
    x, scale, bias, g = s["x"].float(), s["scale"].float(), s["bias"].float(), s["g"]
    centred = x - x.mean(1, keepdim=True)
    inverse = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPSILON)
    unit = centred * inverse
    gs = g * scale
    dx = (gs - gs.mean(1, keepdim=True) - unit * (gs * unit).mean(1, keepdim=True)) * inverse
    return [unit * scale + bias, dx.to(dt), (g * unit).sum(0).to(dt), g.sum(0).to(dt)]


def _plain_attention(s):
    c, dt = s["case"], s["q"].dtype
    heads, kv, size = c["heads"], c["kv_heads"], c["size"]
    group, scale = heads // kv, 1.0 / math.sqrt(size)
    (lq, q0), (lk, k0) = s["queries"], s["keys"]
    b, tq, tk = len(lq), max(_lengths(c["queries"])), max(_lengths(c["keys"] or c["queries"]))
    i, j = torch.arange(tq, device="cuda"), torch.arange(tk, device="cuda")
    rows_q = (q0[:, None] + torch.minimum(i, lq[:, None] - 1)).reshape(-1)
    rows_k = (k0[:, None] + torch.minimum(j, lk[:, None] - 1)).reshape(-1)

    def by_query(t):  # [rows, heads, size] -> [b * kv, group * tq, size]
        t = t[rows_q].float().reshape(b, tq, kv, group, size).permute(0, 2, 3, 1, 4)
        return t.reshape(b * kv, group * tq, size)

    def by_key(t):
        return t[rows_k].float().reshape(b, tk, kv, size).permute(0, 2, 1, 3).reshape(b * kv, tk, size)

    q, k, v = by_query(s["q"]), by_key(s["k"]), by_key(s["v"])
    live = (i < lq[:, None])[:, :, None] & (j < lk[:, None])[:, None, :]
    if c["causal"]:
        live = live & (j[None, None, :] <= (i + (lk - lq)[:, None])[:, :, None])
    live = live[:, None, None].expand(b, kv, group, tq, tk).reshape(b * kv, group * tq, tk)
    scores = (torch.bmm(q, k.transpose(1, 2).contiguous()) * scale).masked_fill_(~live, -math.inf)
    top = scores.amax(2, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(2, keepdim=True)
    p = e / torch.where(total == 0.0, 1.0, total)
    kept_q = (torch.arange(tq, device="cuda") < lq[:, None]).reshape(-1)
    kept_k = (torch.arange(tk, device="cuda") < lk[:, None]).reshape(-1)

    def from_query(t):
        t = t.reshape(b, kv, group, tq, size).permute(0, 3, 1, 2, 4).reshape(b * tq, heads, size)
        return torch.zeros_like(s["q"]).index_copy_(0, rows_q[kept_q], t[kept_q].to(dt))

    def from_key(t):
        t = t.reshape(b, kv, tk, size).permute(0, 2, 1, 3).reshape(b * tk, kv, size)
        return torch.zeros_like(s["k"]).index_copy_(0, rows_k[kept_k], t[kept_k].to(dt))

    out = from_query(torch.bmm(p, v))
    if not c["train"]:
        return [out]
    g = by_query(s["g"])
    dp = torch.bmm(g, v.transpose(1, 2).contiguous())
    ds = p * (dp - (p * dp).sum(2, keepdim=True)) * scale
    dv = torch.bmm(p.transpose(1, 2).contiguous(), g * (kept_q.reshape(b, 1, 1, tq, 1).expand(
        b, kv, group, tq, 1).reshape(b * kv, group * tq, 1)))
    return [out, from_query(torch.bmm(ds, k)), from_key(torch.bmm(ds.transpose(1, 2).contiguous(), q)), from_key(dv)]


def _plain_logprobs(s):
    c, dt = s["case"], s["x"].dtype
    x, tokens = s["x"].float(), s["tokens"].long()
    shifted = x - x.amax(1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    named = tokens >= 0
    at = tokens.clamp_min(0)[:, None]
    log_p = torch.where(named, (shifted.gather(1, at) - log_total)[:, 0], 0.0)
    entropy = (log_total - (e * shifted).sum(1, keepdim=True) / total)[:, 0]
    if not c["train"]:
        if not c["top"]:
            return [log_p, entropy]
        order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :c["top"]].contiguous()
        return [log_p, entropy, shifted.gather(1, order) - log_total, order.int()]
    g, h = torch.where(named, s["g"], 0.0)[:, None], s["h"][:, None]
    dx = -(e / total) * (g + h * (shifted - log_total + entropy[:, None]))
    dx.scatter_add_(1, at, g)
    return [log_p, entropy, dx.to(dt)]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, b = case, SIZE[case["dtype"]]
    if c["kind"] == "norm":
        x = c["rows"] * c["cols"]
        # x and the upstream gradient in, the result and the input's gradient out, four vectors of parameters
        return {"bytes": x * (b + 4 + 4 + b) + 4 * b * c["cols"], "flops": 18.0 * x}
    if c["kind"] == "logprobs":
        x = c["rows"] * c["cols"]
        return {"bytes": x * b * (2 if c["train"] else 1) + c["rows"] * (12 + 8 * c["top"] + (8 if c["train"] else 0)),
                "flops": (10.0 if c["train"] else 5.0) * x}
    (lq, _), (lk, _) = _sequences(c)
    pairs = 0
    for n, m in zip(lq, lk):
        if not c["causal"]:
            pairs += n * m
        else:  # query i sees i + m - n + 1 keys, none where that is negative
            first, last = max(0, n - m), n
            pairs += sum((first + m - n + 1, last + m - n)) * (last - first) // 2
    q, k = sum(lq) * c["heads"] * c["size"], sum(lk) * c["kv_heads"] * c["size"]
    if not c["train"]:
        return {"bytes": b * (2 * q + 2 * k), "flops": 4.0 * c["size"] * c["heads"] * pairs}
    # q, k, v and the upstream gradient in, the result and three gradients out; two products and five
    return {"bytes": b * (4 * q + 4 * k), "flops": 14.0 * c["size"] * c["heads"] * pairs}


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    d = {n: t.double() if t.is_floating_point() else t for n, t in _make(case, seed).items()}
    return {"norm": _exact_norm, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["kind"]](case, d)


def _exact_norm(c, d):
    x, scale, bias = (d[n].requires_grad_() for n in ("x", "scale", "bias"))
    y = torch.nn.functional.layer_norm(x, (c["cols"],), scale, bias, EPSILON)
    return [y.detach(), *torch.autograd.grad(y, [x, scale, bias], d["g"])]


def _exact_attention(c, d):
    """One sequence and one key head at a time, the gradients by torch's own differentiation."""
    (lq, q0), (lk, k0) = _sequences(c)
    group = c["heads"] // c["kv_heads"]
    out = [torch.zeros_like(d["q"])] + ([torch.zeros_like(d[n]) for n in "qkv"] if c["train"] else [])
    for n, a, m, b in zip(lq, q0, lk, k0):
        hidden = torch.zeros(n, m, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        for h in range(c["kv_heads"]):
            at_q, at_k = (slice(a, a + n), slice(h * group, (h + 1) * group)), (slice(b, b + m), h)
            q = d["q"][at_q].transpose(0, 1).contiguous().requires_grad_(c["train"])
            k, v = (d[name][at_k].clone().requires_grad_(c["train"]) for name in "kv")
            weight = (q @ k.t().contiguous() / math.sqrt(c["size"])).masked_fill(hidden, -math.inf)
            weight = torch.where(hidden, 0.0, torch.softmax(weight, 2))
            o = weight @ v
            out[0][at_q] = o.detach().transpose(0, 1)
            if c["train"]:
                g = torch.autograd.grad(o, [q, k, v], d["g"][at_q].transpose(0, 1).contiguous())
                out[1][at_q], out[2][at_k], out[3][at_k] = g[0].transpose(0, 1), g[1], g[2]
    return out


def _exact_logprobs(c, d):
    x, tokens = d["x"], d["tokens"].long()
    log_p = torch.log_softmax(x, 1)
    p = log_p.exp()
    entropy = -(p * log_p).sum(1)
    of_token = torch.where(tokens >= 0, log_p.gather(1, tokens.clamp_min(0)[:, None])[:, 0], 0.0)
    if not c["train"]:
        if not c["top"]:
            return [of_token, entropy]
        return [of_token, entropy, torch.sort(log_p, dim=1, descending=True)[0][:, :c["top"]], None]
    one = torch.zeros_like(x)
    one[torch.arange(c["rows"], device="cuda")[tokens >= 0], tokens[tokens >= 0]] = 1.0
    g = torch.where(tokens >= 0, d["g"], 0.0)[:, None]
    return [of_token, entropy, g * (one - p) - d["h"][:, None] * p * (log_p + entropy[:, None])]
