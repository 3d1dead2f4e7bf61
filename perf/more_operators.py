"""The operators of a decoder with 4-bit microscaled weights and activations, as timed cases.

In a microscaled (MXFP4) tensor 32 neighbouring features of a row share a scale, a
power of two in one byte (2^(byte - 127)), and each is one of the sixteen e2m1
numbers 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, two to a byte with the even
feature in the low half.  Four operators that a model held so runs:

* ``quant_mxfp4``: rows to 4 bits; a block's scale is the smallest power of two at
  which its largest magnitude rounds to 6 at most, its numbers the nearest ones;
* ``dequant_mxfp4``: such rows as 16- or 32-bit values;
* ``linear_mxfp4``: the product of such rows with such weights, optionally with the
  SwiGLU gate and with the result in 4 bits for the next product;
* ``expert_mlp_mxfp4``: the chosen experts' SwiGLU layers, weighted and summed.

Sizes are this repository's decoder's (hidden 2048, FFN 6144, 16/8 heads of 128,
8192 tokens of vocabulary, requests of 128 beams, prompts of 2048 tokens) and generic
ones around them: 64 experts of 768 features, eight to a token, have the active size
of its FFN.

``run`` without ``own`` computes the operators from elementary torch operations in
32 bits, and in 64 for the roundings to 4; ``exact`` computes them in 64 bits
another way.
"""

import math
import os
import sys

import torch

own = False

_DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- cases -------------------------------------------------------------------

def _quant(T, K, dtype):
    """T rows of K features to 4 bits and back."""
    return {"kind": "quant", "T": T, "K": K, "dtype": dtype}


def _dequant(T, K, dtype):
    """T rows of K 4-bit features as values of dtype."""
    return {"kind": "dequant", "T": T, "K": K, "dtype": dtype}


def _linear(M, K, N, out, *, swiglu=False):
    """M rows of K 4-bit features by N columns (SwiGLU: 2 N weight rows)."""
    return {"kind": "linear", "M": M, "K": K, "N": N, "out": out, "swiglu": swiglu}


def _mlp(T, H, Fe, dtype):
    """T rows of H features to 4 bits, through gate and up to Fe 4-bit features and down again."""
    return {"kind": "mlp", "T": T, "H": H, "F": Fe, "dtype": dtype}


def _experts(T, E, k, H, Fe, dtype, *, local=1.0):
    """T tokens through k of E experts, hidden H, expert size Fe.  local: the share
    of the chosen experts that live here (the others are another rank's, id -1)."""
    return {"kind": "experts", "T": T, "E": E, "k": k, "H": H, "F": Fe, "dtype": dtype, "local": local}


def listed():
    named = {
        # one small request's step, the layer's input: latency
        "quant_few": _quant(4, 2048, "float16"),
        # the FFN's activations of four whole prompts: bandwidth
        "quant_prompt": _quant(8192, 6144, "bfloat16"),
        # a layer's gate and up weights read back for work in 16 bits
        "dequant_weights": _dequant(12288, 2048, "bfloat16"),
        # qkv of a small request's step: latency and the weights
        "linear_few": _linear(8, 2048, 4096, "bfloat16"),
        # scores of the vocabulary for a step of four requests x 128 beams
        "linear_scores": _linear(512, 2048, 8192, "float32"),
        # down projection of an odd number of rows
        "linear_down": _linear(1001, 6144, 2048, "float16"),
        # gate and up of four whole prompts, without the gate
        "linear_prompt": _linear(8192, 2048, 12288, "bfloat16"),
        # the feed-forward layer of a step of four requests x 128 beams
        "mlp_step": _mlp(512, 2048, 6144, "float16"),
        # and of four whole prompts
        "mlp_prompt": _mlp(8192, 2048, 6144, "bfloat16"),
        # experts of a small request's step: a few rows each, the weights' way from memory
        "experts_few": _experts(8, 64, 8, 2048, 768, "bfloat16"),
        # experts of a step of four requests x 128 beams
        "experts_step": _experts(512, 64, 8, 2048, 768, "bfloat16"),
        # experts of three odd prompts
        "experts_prompt": _experts(5001, 64, 8, 2048, 768, "float16"),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "dequant", "linear", "linear", "linear", "mlp", "mlp", "experts", "experts", "experts"])
    if kind in ("quant", "dequant"):
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        return (_quant if kind == "quant" else _dequant)(_log(rng, 1, 8192), 32 * rng.randint(1, 192), dtype)
    if kind == "linear":
        M, K, N = _log(rng, 1, 8192), 32 * _log(rng, 4, 192), _log(rng, 16, 12288)
        swiglu = rng.random() < 0.4
        if swiglu:
            N = max(16, N // 32 * 16)
        while M * K * N * (1 + swiglu) > 8192 * 2048 * 12288:
            M = (M + 1) // 2
        return _linear(M, K, N, rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), swiglu=swiglu)
    if kind == "mlp":
        return _mlp(_log(rng, 1, 8192), 32 * _log(rng, 4, 64), 32 * _log(rng, 4, 192), rng.choice(["bfloat16", "float16"]))
    H, Fe = 32 * _log(rng, 8, 64), 32 * _log(rng, 2, 32)
    E = _log(rng, 4, 128)
    while E * H * Fe > 64 * 2048 * 768:
        E = (E + 1) // 2
    k = rng.randint(1, min(8, E))
    T = _log(rng, 1, 8192)
    while T * k * H * Fe > 8192 * 8 * 2048 * 768:
        T = (T + 1) // 2
    return _experts(T, E, k, H, Fe, rng.choice(["bfloat16", "bfloat16", "float16"]), local=rng.choice([1.0, 1.0, 0.5]))


# ---- what a program has in hand ------------------------------------------------

def _acts(g, T, H, dtype):
    """Rows as a norm leaves them: channels of unequal size."""
    size = torch.exp(0.5 * torch.randn(H, generator=g, device="cuda"))
    return (torch.randn(T, H, generator=g, device="cuda") * size).to(dtype)


def _weights4(g, *shape):
    """Weights ~ N(0, 0.02) in 4 bits, with their scales."""
    K = shape[-1]
    rows = math.prod(shape[:-1])
    w4 = torch.empty(rows, K // 2, dtype=torch.uint8, device="cuda")
    ws = torch.empty(rows, K // 32, dtype=torch.uint8, device="cuda")
    at = max(1, (1 << 25) // K)  # rows at a time
    for r in range(0, rows, at):
        n = min(at, rows - r)
        w4[r:r + n], ws[r:r + n] = _quantise(0.02 * torch.randn(n, K, generator=g, device="cuda"))
    return w4.view(*shape[:-1], K // 2), ws.view(*shape[:-1], K // 32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    kind = case["kind"]
    s = {"case": case}
    if kind == "quant":
        s["x"] = _acts(g, case["T"], case["K"], _DT[case["dtype"]])
    elif kind == "dequant":
        s["x4"], s["xs"] = _weights4(g, case["T"], case["K"])
    elif kind == "linear":
        s["x4"], s["xs"] = _quantise(_acts(g, case["M"], case["K"], torch.bfloat16))
        s["w4"], s["ws"] = _weights4(g, case["N"] * (2 if case["swiglu"] else 1), case["K"])
    elif kind == "mlp":
        s["x"] = _acts(g, case["T"], case["H"], _DT[case["dtype"]])
        s["gate_up"], s["gate_up_scale"] = _weights4(g, 2 * case["F"], case["H"])
        s["down"], s["down_scale"] = _weights4(g, case["H"], case["F"])
    else:
        T, E, k, H, Fe = case["T"], case["E"], case["k"], case["H"], case["F"]
        # tokens lean towards some experts
        logits = torch.randn(T, E, generator=g, device="cuda") + 0.3 * torch.randn(E, generator=g, device="cuda")
        weights, ids = torch.softmax(logits, 1).topk(k, 1)
        weights = weights / weights.sum(1, keepdim=True)
        away = torch.rand(T, k, generator=g, device="cuda") >= case["local"]
        s["x"] = _acts(g, T, H, _DT[case["dtype"]])
        s["weights"], s["ids"] = weights.contiguous(), torch.where(away, -1, ids).to(torch.int32).contiguous()
        s["gate_up"], s["gate_up_scale"] = _weights4(g, E, 2 * Fe, H)
        s["down"], s["down_scale"] = _weights4(g, E, H, Fe)
    return s


# ---- the plain forms -----------------------------------------------------------

def _power(e):
    """2^e in float64, by its bits."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _quantise(x):
    """[..., K] to (two numbers a byte [..., K / 2], scales' bytes [..., K / 32])."""
    v = x.double().unflatten(-1, (x.shape[-1] // 32, 32))
    top = v.abs().amax(-1)
    half, power = torch.frexp(top)  # half in [0.5, 1) times 2^power
    e = torch.where(top > 0, power - 3 + (half >= 0.875).int(), -127).clamp(-127, 127)
    v = v * _power(-e[..., None])
    a = v.abs()
    # steps of 0.5, 1 and 2: the numbers' codes count them from 0, 2 and 4 on
    code = torch.where(a < 2, (2 * a).round(), torch.where(a < 4, a.round() + 2, (a / 2).round() + 4)).clamp_max(7)
    code = (code + 8 * torch.signbit(v)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, (e + 127).to(torch.uint8)


def _values(x4, scale):
    """The float32 values of a 4-bit tensor."""
    code = torch.stack([x4 & 15, x4 >> 4], -1).flatten(-2).long()
    number = torch.tensor(_E2M1 + tuple(-n for n in _E2M1), device=x4.device)
    unit = _power(scale.int() - 127).float()
    return number[code] * unit.repeat_interleave(32, -1)


def _gated(y):
    gate, up = y.chunk(2, -1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _plain_experts(s):
    c = s["case"]
    T, E, k, H = c["T"], c["E"], c["k"], c["H"]
    gate_up, down = _values(s["gate_up"], s["gate_up_scale"]), _values(s["down"], s["down_scale"])
    x = _values(*_quantise(s["x"]))
    # every expert's rows side by side, padded to the longest; another rank's rows get expert 0 and weight 0
    flat = s["ids"].long().reshape(-1)
    weights = torch.where(s["ids"] < 0, 0.0, s["weights"])
    flat = flat.clamp_min(0)
    order = torch.argsort(flat, stable=True)
    expert = flat[order]
    count = torch.bincount(flat, minlength=E)
    slot = torch.arange(T * k, device=x.device) - (count.cumsum(0) - count)[expert]
    rows = torch.zeros(E, int(count.max()), H, device=x.device)
    rows[expert, slot] = x[order // k]
    act = _values(*_quantise(_gated(torch.bmm(rows, gate_up.transpose(1, 2)))))
    y = torch.empty(T * k, H, device=x.device)
    y[order] = torch.bmm(act, down.transpose(1, 2))[expert, slot]
    return (y.view(T, k, H) * weights[..., None]).sum(1).to(s["x"].dtype)


def _own(s):
    if "vllm_gr_amd" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "vllm-gr-ehaleva_amd"))
    from vllm_gr_amd import ops
    c = s["case"]
    kind = c["kind"]
    if kind == "quant":
        x4, scale = ops.quant_mxfp4(s["x"])
        return ops.dequant_mxfp4(x4, scale, dtype=s["x"].dtype), scale.view(torch.float8_e8m0fnu)
    if kind == "dequant":
        return ops.dequant_mxfp4(s["x4"], s["xs"], dtype=_DT[c["dtype"]])
    if kind == "linear":
        return ops.linear_mxfp4(s["x4"], s["xs"], s["w4"], s["ws"], swiglu=c["swiglu"], out_dtype=_DT[c["out"]])
    if kind == "mlp":
        act = ops.linear_mxfp4(*ops.quant_mxfp4(s["x"]), s["gate_up"], s["gate_up_scale"], swiglu=True, quantized=True)
        return ops.linear_mxfp4(*act, s["down"], s["down_scale"], out_dtype=s["x"].dtype)
    return ops.expert_mlp_mxfp4(s["x"], s["gate_up"], s["gate_up_scale"], s["down"], s["down_scale"], s["weights"],
                                s["ids"])


def run(s):
    if own:
        return _own(s)
    c = s["case"]
    kind = c["kind"]
    if kind == "quant":
        x4, scale = _quantise(s["x"])
        return _values(x4, scale).to(s["x"].dtype), scale.view(torch.float8_e8m0fnu)
    if kind == "dequant":
        return _values(s["x4"], s["xs"]).to(_DT[c["dtype"]])
    if kind == "linear":
        y = _values(s["x4"], s["xs"]) @ _values(s["w4"], s["ws"]).t()
        return (_gated(y) if c["swiglu"] else y).to(_DT[c["out"]])
    if kind == "mlp":
        y = _gated(_values(*_quantise(s["x"])) @ _values(s["gate_up"], s["gate_up_scale"]).t())
        return (_values(*_quantise(y)) @ _values(s["down"], s["down_scale"]).t()).to(s["x"].dtype)
    return _plain_experts(s)


# ---- what each has to move and compute -------------------------------------------

def work(case):
    size = {"float32": 4, "float16": 2, "bfloat16": 2}
    packed = 0.5 + 1 / 32  # bytes of a 4-bit feature and its share of a scale
    kind = case["kind"]
    if kind == "quant":
        n = case["T"] * case["K"]
        return {"bytes": n * (2 * size[case["dtype"]] + packed), "flops": 4 * n}
    if kind == "dequant":
        n = case["T"] * case["K"]
        return {"bytes": n * (size[case["dtype"]] + packed), "flops": n}
    if kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        rows = N * (1 + case["swiglu"])
        return {"bytes": (M + rows) * K * packed + M * N * size[case["out"]], "flops": 2 * M * rows * K}
    T, H, Fe = case["T"], case["H"], case["F"]
    if kind == "mlp":
        return {"bytes": 3 * H * Fe * packed + 2 * T * H * 2, "flops": 6 * T * H * Fe}
    E, k = case["E"], case["k"]
    rows = T * k * case["local"]
    touched = E * (1.0 - (1.0 - case["local"] * k / E) ** T)  # experts that any token chose
    return {"bytes": touched * 3 * H * Fe * packed + 2 * T * H * 2 + 8 * T * k, "flops": 6 * rows * H * Fe}


# ---- the definitions in 64 bits ---------------------------------------------------

def _exact_quant(x):
    """Values [T, K] and scales of the 4-bit form, in float64: the scale by a search
    among the powers of two, the numbers by one among the borders between them."""
    T, K = x.shape
    x = x.double()
    table = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    border = (table[1:] + table[:-1]) / 2
    power = torch.pow(2.0, torch.arange(-127, 128, dtype=torch.float64, device=x.device))
    top = x.abs().view(T, K // 32, 32).max(2)[0]
    scale = power[torch.searchsorted(7.0 * power, top, right=True)]  # the least with top < 7 scale
    unit = scale.repeat_interleave(32, 1)
    a = x.abs() / unit
    i = torch.bucketize(a, border)  # the lower of two at a border
    i = i + ((a == border[i.clamp_max(6)]) & (i < 7) & (i % 2 == 1)).long()
    return table[i] * torch.sign(x) * unit, scale


def _exact_values(x4, scale):
    K = 2 * x4.shape[-1]
    out = torch.empty(*x4.shape[:-1], K, dtype=torch.float64, device=x4.device)
    for odd, code in ((0, x4 % 16), (1, x4 // 16)):
        c = code.int()
        m, p = c % 2, c // 2 % 4
        a = torch.where(p == 0, 0.5 * m.double(), (1.0 + 0.5 * m.double()) * torch.pow(2.0, (p - 1).double()))
        out[..., odd::2] = torch.where(c >= 8, -a, a)
    for b in range(K // 32):
        out[..., 32 * b:32 * b + 32] *= torch.pow(2.0, scale[..., b:b + 1].double() - 127.0)
    return out


def _exact_layer(v, gate_up, gate_up_scale, down, down_scale):
    w = _exact_values(gate_up, gate_up_scale)
    half = len(w) // 2
    gate, up = v @ w[:half].t(), v @ w[half:].t()
    act = _exact_quant(gate * torch.sigmoid(gate) * up)[0]
    return act @ _exact_values(down, down_scale).t()


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return _exact_quant(s["x"])
    if kind == "dequant":
        return _exact_values(s["x4"], s["xs"])
    if kind == "linear":
        x, w = _exact_values(s["x4"], s["xs"]), _exact_values(s["w4"], s["ws"])
        if not case["swiglu"]:
            return x @ w.t()
        gate, up = x @ w[:case["N"]].t(), x @ w[case["N"]:].t()
        return gate * torch.sigmoid(gate) * up
    v = _exact_quant(s["x"])[0]
    if kind == "mlp":
        return _exact_layer(v, s["gate_up"], s["gate_up_scale"], s["down"], s["down_scale"])
    out = torch.zeros_like(v)
    for e in range(case["E"]):
        tok, j = torch.nonzero(s["ids"] == e, as_tuple=True)
        if len(tok):
            y = _exact_layer(v[tok], s["gate_up"][e], s["gate_up_scale"][e], s["down"][e], s["down_scale"][e])
            out.index_add_(0, tok, y * s["weights"][tok, j].double()[:, None])
    return out
