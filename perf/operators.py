"""The calls a serving stack makes around the experts of a block-quantised FP8 model, as cases for timing.

Three kinds of operator, in the order in which a token row meets them:

    norm     "before": the last block's output joins the residual stream (gate, residual scale) and is normalised for the
             next block, in 16 bits or quantised to e4m3 per 1 x 128 group;  "after": a block's output is normalised first,
             gated, scaled and added;  "between": both, for layers that normalise on either side of a block
    linear   e4m3 weights [N, K] with one scale per 128 x 128 block; activations quantised per 1 x 128 group, by the call
             ("bf16", "fp16") or before it ("fp8")
    act      a gated activation of [M, 2I] rows, its result in 16 bits or quantised per 1 x 128 group

A case holds plain values; the layers' sizes are those of the repository's configurations (7168 x 2048, 4096, 5120) and odd ones.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_ROOT = Path(__file__).resolve().parent.parent
_FP8 = torch.float8_e4m3fn
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.bfloat16}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}


def _package():
    for p in (Path.cwd() / "flaggems-sglang_b200", _ROOT / "flaggems-sglang_b200"):
        if p.is_dir():
            if str(p) not in sys.path:
                sys.path.insert(0, str(p))
            break
    import flaggems_sglang_b200
    return flaggems_sglang_b200


def _linear(m, n, k, x="bf16", bias=False):
    return {"op": "linear", "m": m, "n": n, "k": k, "x": x, "bias": bias}


def _norm(form, m, h, x="bf16", residual="bf16", kind="rms", offset=0.0, gate="none", scale=1.0, quantize=False):
    return {"op": "norm", "form": form, "m": m, "h": h, "x": x, "residual": residual, "kind": kind, "offset": offset,
            "gate": gate, "scale": scale, "quantize": quantize}


def _act(m, i, x="bf16", kind="silu", quantize=True):
    return {"op": "act", "m": m, "i": i, "x": x, "kind": kind, "quantize": quantize}


def _named(name, case):
    return {"name": name, **case}


def listed():
    return [
        # one user's decode step: gate and up rows of a shared expert, bound by its weights and the launch
        _named("linear one token", _linear(1, 4096, 7168)),
        # a decode batch through the shared expert's down projection, activations in 16 bits
        _named("linear decode batch", _linear(48, 7168, 2048, bias=True)),
        # a chunk of a prompt through a projection whose rows are no multiple of a block, already quantised by the norm
        _named("linear ragged chunk", _linear(333, 2112, 7168, "fp8")),
        # prefill of the shared expert, activations in 16 bits
        _named("linear prefill", _linear(4096, 4096, 7168, "fp16")),
        # prefill of a dense layer, already quantised
        _named("linear large prefill", _linear(8192, 18432, 7168, "fp8")),
        # one user's decode step: residual add, norm and quantisation in one launch
        _named("norm before one token", _norm("before", 1, 7168, quantize=True)),
        # prefill: the same for a batch of prompts
        _named("norm before prefill", _norm("before", 4096, 7168, quantize=True)),
        # a layer norm in fp16 with unit offset on weights, an odd number of rows of a size that is no multiple of a group
        _named("norm before ragged", _norm("before", 1001, 2600, "fp16", "fp16", "layer", 1.0, "channel", 0.5)),
        # decode batch with norms on either side of the block and the residual stream in fp32
        _named("norm between decode", _norm("between", 33, 4096, residual="fp32", offset=1.0, quantize=True)),
        # prefill with a norm after the block, one gate per token
        _named("norm after prefill", _norm("after", 8192, 5120, gate="token", scale=0.25)),
        # decode batch between the two products of a shared expert
        _named("activation decode", _act(48, 2048)),
        # prefill between the two products of a dense layer
        _named("activation prefill", _act(4096, 18432)),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "norm", "act"])
    m = _log(rng, 1, 8192)
    if op == "linear":
        return _linear(m, _log(rng, 64, 18432), 16 * _log(rng, 8, 448), rng.choice(["bf16", "fp16", "fp8"]), rng.random() < 0.3)
    if op == "act":
        return _act(m, 8 * _log(rng, 16, 2304), rng.choice(["bf16", "fp16"]), rng.choice(["silu", "gelu", "swiglu_oai"]),
                    rng.random() < 0.6)
    x = rng.choice(["bf16", "bf16", "fp16"])
    return _norm(rng.choice(["before", "after", "between"]), m, 8 * _log(rng, 32, 1024), x, rng.choice([x, x, "fp32"]),
                 rng.choice(["rms", "rms", "layer"]), rng.choice([0.0, 1.0]), rng.choice(["none", "channel", "token", "full"]),
                 rng.choice([1.0, 0.25]), rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------- inputs
def _quantised(x):
    """(e4m3, scales) of rows per group of 128, the last group as long as it is: scale = max(amax, 1e-10) / 448."""
    m, k = x.shape
    g = -(-k // 128)
    v = torch.nn.functional.pad(x.float(), (0, g * 128 - k)).view(m, g, 128)
    s = v.abs().amax(-1).clamp_min(1e-10) / 448.0
    q = (v / s[..., None]).clamp(-448.0, 448.0).to(_FP8)
    return q.view(m, g * 128)[:, :k].contiguous(), s


def _spread(s, k):
    return s.repeat_interleave(128, dim=1)[:, :k]


def _rows(shape, dtype, gen, scale=1.0, outliers=True):
    """Unit normal rows with a few channels that are larger throughout, as residual streams have."""
    x = torch.randn(shape, device="cuda", generator=gen) * scale
    if outliers:
        big = torch.rand(shape[-1], device="cuda", generator=gen) < 0.01
        x *= torch.where(big, 8.0, 1.0)
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    t = _TYPES[case["x"]]
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        gn, gk = -(-n // 128), -(-k // 128)
        w = torch.zeros(gn * 128, gk * 128, device="cuda")
        w[:n, :k] = torch.randn(n, k, device="cuda", generator=gen) * 0.02
        w = w.view(gn, 128, gk, 128)
        ws = w.abs().amax((1, 3)).clamp_min(1e-10) / 448.0
        state["w"] = (w / ws[:, None, :, None]).clamp(-448.0, 448.0).to(_FP8).view(gn * 128, gk * 128)[:n, :k].contiguous()
        state["ws"] = ws
        x = _rows((m, k), t, gen)
        state["x"], state["xs"] = _quantised(x) if case["x"] == "fp8" else (x, None)
        state["bias"] = torch.randn(n, device="cuda", generator=gen) if case["bias"] else None
    elif case["op"] == "act":
        state["x"] = _rows((case["m"], 2 * case["i"]), t, gen, outliers=False)
    else:
        m, h = case["m"], case["h"]
        state["x"] = _rows((m, h), t, gen)
        state["residual"] = _rows((m, h), _TYPES[case["residual"]], gen, 4.0)
        centre = 1.0 - case["offset"]
        for name in ("w", "w2"):
            state[name] = (centre + 0.1 * torch.randn(h, device="cuda", generator=gen)).to(t)
        for name in ("b", "b2"):
            state[name] = (0.1 * torch.randn(h, device="cuda", generator=gen)).to(t) if case["kind"] == "layer" else None
        gate = {"none": None, "channel": (h,), "token": (m, 1), "full": (m, h)}[case["gate"]]
        state["gate"] = None if gate is None else torch.rand(gate, device="cuda", generator=gen).to(t)
    return state


# ------------------------------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    F, c = _package(), s["case"]
    if c["op"] == "linear":
        return F.fp8_block_linear(s["x"], s["w"], s["ws"], s["bias"], x_scale=s["xs"])
    if c["op"] == "act":
        return F.gated_activation(s["x"], c["kind"], swiglu_alpha=1.702, swiglu_limit=7.0, quantize=c["quantize"])
    common = dict(residual=s["residual"], gate=s["gate"], residual_scale=c["scale"], kind=c["kind"], weight_offset=c["offset"])
    if c["form"] == "before":
        return F.norm_before_block(s["x"], s["w"], bias=s["b"], quantize=c["quantize"], **common)
    if c["form"] == "after":
        return F.norm_after_block(s["x"], s["w"], bias=s["b"], **common)
    return F.norm_after_block(s["x"], s["w"], bias=s["b"], next_weight=s["w2"], next_bias=s["b2"], quantize=c["quantize"], **common)


# ------------------------------------------------------------------------------------------------- the plain form
def _normed(v, w, b, c):
    if c["kind"] == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * (c["offset"] + w.float())
    return v if b is None else v + b.float()


def _plain_act(g, u, kind):
    if kind == "silu":
        return g / (1.0 + torch.exp(-g)) * u
    if kind == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5))) * u
    g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
    return g / (1.0 + torch.exp(-1.702 * g)) * (u + 1.0)


def _run_plain(s):
    c = s["case"]
    if c["op"] == "linear":
        n, k = s["w"].shape
        xq, xs = (s["x"], s["xs"]) if s["xs"] is not None else _quantised(s["x"])
        w = s["w"].float() * _spread(s["ws"], k).repeat_interleave(128, dim=0)[:n]
        out = torch.matmul(xq.float() * _spread(xs, k), w.t())
        if s["bias"] is not None:
            out = out + s["bias"]
        return out.to(_TYPES[c["x"]])
    if c["op"] == "act":
        x = s["x"].float()
        y = _plain_act(x[:, :c["i"]], x[:, c["i"]:], c["kind"])
        return _quantised(y) if c["quantize"] else y.to(s["x"].dtype)
    z = s["x"].float()
    if c["form"] != "before":
        z = _normed(z, s["w"], s["b"], c)
    if s["gate"] is not None:
        z = z * s["gate"].float()
    h = s["residual"].float() + c["scale"] * z
    hidden = h.to(s["residual"].dtype)
    if c["form"] == "after":
        return hidden
    y = _normed(h, *((s["w"], s["b"]) if c["form"] == "before" else (s["w2"], s["b2"])), c)
    return (_quantised(y) if c["quantize"] else y.to(s["x"].dtype)), hidden


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------- work and 64-bit results
def work(case):
    b = _BYTES[case["x"]]
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        gk = -(-k // 128)
        scales = 4 * (gk * -(-n // 128) + (m * gk if case["x"] == "fp8" else 0))
        out = 2 * m * n + (4 * n if case["bias"] else 0)
        return {"bytes": n * k + b * m * k + scales + out, "flops": 2 * m * n * k}
    if case["op"] == "act":
        m, i = case["m"], case["i"]
        return {"bytes": m * (2 * i * b + (i + 4 * -(-i // 128) if case["quantize"] else i * b)), "flops": 8 * m * i}
    m, h = case["m"], case["h"]
    vectors = (1 + (case["kind"] == "layer")) * (1 + (case["form"] == "between"))
    gate = {"none": 0, "channel": h, "token": m, "full": m * h}[case["gate"]]
    out = 0 if case["form"] == "after" else h + 4 * -(-h // 128) if case["quantize"] else h * b
    return {"bytes": m * (h * b + 2 * h * _BYTES[case["residual"]] + out) + b * (h * vectors + gate),
            "flops": m * h * (6 + 6 * (case["form"] == "between"))}


def _exact_groups(y):
    """Scales and e4m3 values of 64-bit rows; a scale is what the format holds, a 32-bit number."""
    q, scales = torch.empty_like(y), []
    for g0 in range(0, y.shape[1], 128):
        part = y[:, g0:g0 + 128]
        scale = (part.abs().max(1).values.clamp(min=1e-10) / 448).float().double()
        q[:, g0:g0 + 128] = torch.clip(part / scale[:, None], -448, 448).to(_FP8).double()
        scales.append(scale)
    return q, torch.stack(scales, 1)


def _exact_norm(v, weight, bias, case):
    mean = v.sum(1, keepdim=True) / v.shape[1] if case["kind"] == "layer" else 0.0
    out = (v - mean) / torch.sqrt(((v - mean) ** 2).sum(1, keepdim=True) / v.shape[1] + 1e-6)
    out = out * (weight.double() + case["offset"])
    return out + bias.double() if bias is not None else out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        k = case["k"]
        q, scale = (s["x"].double(), s["xs"].double()) if s["xs"] is not None else _exact_groups(s["x"].double())
        out = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
        rows = torch.arange(case["n"], device="cuda") // 128
        for g, k0 in enumerate(range(0, k, 128)):
            part = q[:, k0:k0 + 128] @ s["w"][:, k0:k0 + 128].double().t()
            out.addcmul_(part, scale[:, g:g + 1] * s["ws"][rows, g].double()[None])
        return out + s["bias"].double() if s["bias"] is not None else out
    if case["op"] == "act":
        g, u = s["x"].double().split(case["i"], dim=1)
        if case["kind"] == "swiglu_oai":
            g, u = g.clip(max=7), u.clip(-7, 7) + 1
        if case["kind"] == "gelu":
            y = g * torch.special.ndtr(g) * u
        else:
            y = g * torch.sigmoid((1.702 if case["kind"] == "swiglu_oai" else 1) * g) * u
        return _exact_groups(y) if case["quantize"] else y
    h = s["x"].double()
    if case["form"] in ("after", "between"):
        h = _exact_norm(h, s["w"], s["b"], case)
    h = s["residual"].double() + h * case["scale"] * (1.0 if s["gate"] is None else s["gate"].double())
    if case["form"] == "after":
        return h
    weight, bias = (s["w2"], s["b2"]) if case["form"] == "between" else (s["w"], s["b"])
    y = _exact_norm(h, weight, bias, case)
    return (_exact_groups(y) if case["quantize"] else y), h
