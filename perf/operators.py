"""What is timed of the operators that surround the attention call of a transformer block: the residual
addition with a root-mean-square norm (16/32-bit output, or e4m3 with one scale per token), the dynamic
per-token quantiser, and the matrix product whose epilogue adds the bias, applies the activation, the
gate and the residual (16-bit operands, or e4m3 operands with their scales).

`own = False`: elementary torch operations in 32 bits.  `own = True`: the framework's entry points.
Token counts are those of the package's workloads (21x30x52 = 32760 and 21x45x80 = 75600 latent tokens),
widths are 12 and 40 heads of 128 channels, the feed-forward is four times as wide.
"""
import math
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6
_E4M3_MAX = 448.0


def _framework():
    """The package lies in a folder that is no Python name, so its parent goes on the path first."""
    if "mindie-sd_b200" not in sys.path:
        sys.path.insert(0, "mindie-sd_b200")
    import mindiesd
    return mindiesd


def listed():
    norm = {"op": "norm", "weight": "same"}
    quant = {"op": "norm_quant", "weight": "same"}
    lin = {"op": "linear", "bias": True, "act": "none", "residual": False, "gate": 0}
    lin8 = {"op": "linear_e4m3", "bias": True, "act": "none", "residual": False, "gate": 0}
    return [
        # One token of each of two prompts through a block's norm: what a step costs where nothing is large.
        {"name": "norm_2x5120_bf16", **norm, "rows": 2, "dim": 5120, "type": "bf16", "residual": "same"},
        # Query or key norm over the channels of each head, every token of a 21x30x52 grid, 12 heads.
        {"name": "norm_393120x128_fp16", **norm, "rows": 393120, "dim": 128, "type": "fp16", "residual": "none"},
        # The residual stream of a whole 21x45x80 clip, 40 heads wide.
        {"name": "norm_75600x5120_bf16", **norm, "rows": 75600, "dim": 5120, "type": "bf16", "residual": "same"},
        # A short ragged piece of text with an uneven width, quantised for an e4m3 product.
        {"name": "norm_quant_333x1004_fp16", **quant, "rows": 333, "dim": 1004, "type": "fp16", "residual": "none"},
        # The stream of the whole clip again, normalised and quantised for the e4m3 projections.
        {"name": "norm_quant_75600x5120_bf16", **quant, "rows": 75600, "dim": 5120, "type": "bf16", "residual": "same"},
        # First layer of a timestep embedding: one row.
        {"name": "linear_1x256x5120_silu", **lin, "m": 1, "k": 256, "n": 5120, "type": "bf16", "act": "silu"},
        # The modulation vectors of a block (six of them) for two prompts: the weights are all there is to read.
        {"name": "linear_2x5120x30720", **lin, "m": 2, "k": 5120, "n": 30720, "type": "bf16"},
        # A text encoder's 512 tokens brought to the model's width.
        {"name": "linear_512x4096x5120_gelu", **lin, "m": 512, "k": 4096, "n": 5120, "type": "fp16", "act": "gelu_tanh"},
        # Second linear of the feed-forward at 12 heads' width, two clips of 4681 tokens, gate and residual.
        {"name": "linear_9362x6144x1536_gate", **lin, "m": 9362, "k": 6144, "n": 1536, "type": "bf16", "residual": True,
         "gate": 2},
        # First linear of the feed-forward at 40 heads' width over a 21x30x52 grid.
        {"name": "linear_32760x5120x20480_gelu", **lin, "m": 32760, "k": 5120, "n": 20480, "type": "bf16",
         "act": "gelu_tanh"},
        # A projection of a short prompt with an output width that no vector divides.
        {"name": "linear_e4m3_300x1536x1001", **lin8, "m": 300, "k": 1536, "n": 1001, "type": "bf16"},
        # Second linear of the feed-forward over the 21x30x52 grid in e4m3, gate and residual.
        {"name": "linear_e4m3_32760x20480x5120_gate", **lin8, "m": 32760, "k": 20480, "n": 5120, "type": "bf16",
         "residual": True, "gate": 1},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_quant", "linear", "linear_e4m3"])
    if op in ("norm", "norm_quant"):
        dim = _log_int(rng, 64, 8192)
        if rng.random() < 0.75:
            dim = (dim + 7) // 8 * 8
        kind = rng.choice(["bf16", "fp16", "bf16", "fp32"] if op == "norm" else ["bf16", "fp16"])
        rows = min(_log_int(rng, 1, 393120), 37800 * 5120 // dim)
        return {"op": op, "rows": rows, "dim": dim, "type": kind, "residual": rng.choice(["none", "same", "fp32"]),
                "weight": rng.choice(["none", "same", "fp32"])}
    m, k, n = _log_int(rng, 1, 32760), _log_int(rng, 64, 20480), _log_int(rng, 16, 20480)
    step = 16 if op == "linear_e4m3" else 8
    if op == "linear_e4m3" or rng.random() < 0.9:
        k = (k + step - 1) // step * step
    if rng.random() < 0.75:
        n = (n + 7) // 8 * 8
    m = max(1, min(m, 32760 * 5120 * 20480 // (k * n)))
    gate = rng.choice([0, 0, 1, 2])
    if gate:
        m = (m + gate - 1) // gate * gate
    return {"op": op, "m": m, "k": k, "n": n, "type": rng.choice(["bf16", "fp16"]), "bias": rng.random() < 0.7,
            "act": rng.choice(["none", "none", "silu", "gelu", "gelu_tanh"]), "residual": gate > 0 or rng.random() < 0.3,
            "gate": gate}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(g, rows, dim, dtype):
    """Hidden states: unit normals, one channel in a hundred eight times as large."""
    loud = torch.where(torch.rand(dim, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    out = torch.empty(rows, dim, dtype=dtype, device="cuda")
    step = max(1, (1 << 28) // dim)
    for at in range(0, rows, step):
        part = out[at:at + step]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * loud)
    return out


def prepare(case, seed):
    g = _generator(seed)
    t = _TYPES[case["type"]]
    if case["op"] in ("norm", "norm_quant"):
        x = _activations(g, case["rows"], case["dim"], t)
        residual = None
        if case["residual"] != "none":
            residual = _activations(g, case["rows"], case["dim"], t if case["residual"] == "same" else torch.float32)
        weight = None
        if case["weight"] != "none":
            weight = 1 + 0.2 * torch.randn(case["dim"], generator=g, device="cuda")
            weight = weight.to(t if case["weight"] == "same" else torch.float32)
        return {"op": case["op"], "x": x, "residual": residual, "weight": weight}
    m, k, n = case["m"], case["k"], case["n"]
    s = {"op": case["op"], "type": t, "act": case["act"], "bias": None, "residual": None, "gate": None,
         "x_scale": None, "weight_scale": None}
    x = _activations(g, m, k, t)
    w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
    if case["op"] == "linear_e4m3":
        s["x_scale"] = (x.abs().amax(1, keepdim=True).float() / _E4M3_MAX).clamp_min(1e-12)
        s["weight_scale"] = (w.abs().amax(1) / _E4M3_MAX).clamp_min(1e-12)
        s["x"] = (x.float() / s["x_scale"]).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
        s["w"] = (w / s["weight_scale"][:, None]).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
    else:
        s["x"], s["w"] = x, w.to(t)
    if case["bias"]:
        s["bias"] = (0.1 * torch.randn(n, generator=g, device="cuda")).to(t)
    if case["residual"]:
        s["residual"] = _activations(g, m, n, t)
    if case["gate"]:
        # Two clips in one batch have a gate each; modulation vectors are kept in 32 bits.
        s["gate"] = 0.5 * torch.randn(case["gate"], 1, n, generator=g, device="cuda")
        s["x"] = s["x"].view(case["gate"], m // case["gate"], k)
        s["residual"] = s["residual"].view(case["gate"], m // case["gate"], n)
        if s["x_scale"] is not None:
            s["x_scale"] = s["x_scale"].view(case["gate"], m // case["gate"], 1)
    return s


def _plain_act(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain_norm(s):
    v = s["x"].float()
    if s["residual"] is not None:
        v = v + s["residual"].float()
    y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS)
    if s["weight"] is not None:
        y = y * s["weight"].float()
    return v, y


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "norm":
        v, y = _plain_norm(s)
        out = {"y": y.to(s["x"].dtype)}
        if s["residual"] is not None:
            out["residual"] = v.to(s["residual"].dtype)
        return out
    if s["op"] == "norm_quant":
        v, y = _plain_norm(s)
        amax = y.abs().amax(-1, keepdim=True)
        scale = torch.where(amax == 0, 1.0, (amax / _E4M3_MAX).clamp_min(2.0 ** -126))
        out = {"q": (y / scale).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn), "scale": scale}
        if s["residual"] is not None:
            out["residual"] = v.to(s["residual"].dtype)
        return out
    v = torch.matmul(s["x"].float(), s["w"].float().t())
    if s["x_scale"] is not None:
        v = v * s["x_scale"] * s["weight_scale"]
    if s["bias"] is not None:
        v = v + s["bias"].float()
    v = _plain_act(v, s["act"])
    if s["gate"] is not None:
        v = v * s["gate"].float()
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return {"out": v.to(s["type"])}


def _run_own(s):
    sd = _framework()
    if s["op"] == "norm":
        got = sd.add_rms_norm(s["x"], s["weight"], s["residual"], _EPS)
        return {"y": got} if s["residual"] is None else {"y": got[0], "residual": got[1]}
    if s["op"] == "norm_quant":
        got = sd.add_rms_norm_quant(s["x"], s["weight"], s["residual"], _EPS)
        out = {"q": got[0], "scale": got[1]}
        if s["residual"] is not None:
            out["residual"] = got[2]
        return out
    return {"out": sd.linear_forward(s["x"], s["w"], s["bias"], activation=s["act"], residual=s["residual"], gate=s["gate"],
                                     x_scale=s["x_scale"], weight_scale=s["weight_scale"], out_dtype=s["type"])}


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    t = size[case["type"]]
    if case["op"] in ("norm", "norm_quant"):
        cells = case["rows"] * case["dim"]
        out = t * cells if case["op"] == "norm" else cells + 4 * case["rows"]
        r = {"none": 0, "same": t, "fp32": 4}[case["residual"]]
        w = {"none": 0, "same": t, "fp32": 4}[case["weight"]]
        return {"bytes": t * cells + 2 * r * cells + out + w * case["dim"], "flops": 6 * cells}
    m, k, n = case["m"], case["k"], case["n"]
    e = 1 if case["op"] == "linear_e4m3" else 2
    extra = 4 * (m + n) if e == 1 else 0
    if case["bias"]:
        extra += t * n
    if case["residual"]:
        extra += t * m * n
    return {"bytes": e * (m * k + n * k) + t * m * n + extra + 4 * case["gate"] * n, "flops": 2 * m * n * k}


def exact(case, seed):
    """The operators' definitions in 64 bits, a slab of rows at a time."""
    s = prepare(case, seed)
    lead = s["x"].shape[:-1]
    x = s["x"].reshape(-1, s["x"].shape[-1])
    rows = x.shape[0]
    if case["op"] in ("norm", "norm_quant"):
        dim = case["dim"]
        w = torch.ones(dim, dtype=torch.float64, device="cuda") if s["weight"] is None else s["weight"].double()
        y = torch.empty(rows, dim, dtype=torch.float64, device="cuda")
        total = None if s["residual"] is None else torch.empty_like(y)
        scale = torch.empty(rows, 1, dtype=torch.float64, device="cuda")
        for at in range(0, rows, 8192):
            cut = slice(at, at + 8192)
            h = x[cut].double()
            if total is not None:
                h += s["residual"][cut].double()
                total[cut] = h
            h = h / torch.sqrt((h.pow(2).sum(1, keepdim=True) / dim) + _EPS) * w
            top = h.abs().max(1, keepdim=True).values
            scale[cut] = torch.where(top == 0, torch.ones_like(top), top / 448)
            y[cut] = h
        if case["op"] == "norm":
            return {"y": y} if total is None else {"y": y, "residual": total}
        got = {"q": y.div_(scale), "scale": scale}
        return got if total is None else {**got, "residual": total}
    n = case["n"]
    wt = s["w"].double()
    if s["weight_scale"] is not None:
        wt = wt * s["weight_scale"].double().unsqueeze(1)
    res = torch.empty(rows, n, dtype=torch.float64, device="cuda")
    for at in range(0, rows, 8192):
        cut = slice(at, min(rows, at + 8192))
        a = x[cut].double()
        if s["x_scale"] is not None:
            a = a * s["x_scale"].reshape(-1, 1)[cut].double()
        h = a @ wt.T
        if s["bias"] is not None:
            h += s["bias"].double()
        if case["act"] == "silu":
            h = h * torch.special.expit(h)
        elif case["act"] == "gelu":
            h = h * torch.special.ndtr(h)
        elif case["act"] == "gelu_tanh":
            h = h * torch.special.expit(2 * math.sqrt(2 / math.pi) * (h + 0.044715 * h ** 3))
        if s["gate"] is not None:
            per = rows // case["gate"]
            index = torch.arange(cut.start, cut.stop, device="cuda") // per
            h = h * s["gate"].reshape(case["gate"], n).double()[index]
        if s["residual"] is not None:
            h = h + s["residual"].reshape(rows, n)[cut].double()
        res[cut] = h
    return {"out": res.view(*lead, n)}
