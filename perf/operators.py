"""The block norms and the 4-bit-weight operators as measured work: cases, inputs, calls.

Four operators of a served transformer feed-forward block:
  norm      the norms around a block with its gate and residual scales:
            r = x_scale x + y_scale gate Npost(y), h = Npre(r); N is LayerNorm, RMS norm or none
  quantize  weights [K, N] to 4-bit codes with group scales (and zero points), and read back
  linear    act(x W + b) on 4-bit weights W = s (q - z), from one row to a prompt's rows
  mlp       a chain of 4-bit layers with a (residual +) LayerNorm tail

Where `own` is false, `run` computes them with elementary torch operations in 32 bits; where it is
true, through the package's public calls.
"""
import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16}
_ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}
_NORMS = {"none": 0, "layer": 1, "rms": 2}


def _norm(name, m, h, dtype, post, pre, **kw):
    """One norm call. stream: the residual stream's type ("16" or "32" bits); gates: gate rows (0:
    no gate, 1: one row for all, G: one row for each of G equal runs of rows); x / y / r: which of
    the stream in, the block's output and the stream out the call has."""
    c = dict(op="norm", m=m, h=h, dtype=dtype, post=post, pre=pre, stream="16", gates=0,
             x=True, y=True, r=True, beta=True, x_scale=1.0, y_scale=1.0, eps=1e-5)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def _quant(name, k, n, dtype, group, zeros):
    c = dict(op="quantize", k=k, n=n, dtype=dtype, group=group, zeros=zeros)
    if name:
        c["name"] = name
    return c


def _linear(name, m, k, n, dtype, group, zeros, act, bias):
    c = dict(op="linear", m=m, k=k, n=n, dtype=dtype, group=group, zeros=zeros, act=act, bias=bias)
    if name:
        c["name"] = name
    return c


def _mlp(name, m, widths, dtype, group, zeros, act, tail, eps):
    c = dict(op="mlp", m=m, widths="-".join(str(w) for w in widths), dtype=dtype, group=group,
             zeros=zeros, act=act, tail=tail, eps=eps)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one token of a block with a norm on both sides: latency
        _norm("norm_token", 1, 4096, "bf16", "rms", "rms", beta=False, eps=1e-6),
        # the post-norm of the BERT-large FFN configuration, 32 sequences of 512: LN(x + y)
        _norm("norm_bert", 16384, 1024, "bf16", "none", "layer", r=False, eps=1e-12),
        # a prompt batch: 8 sequences with a gate row each, norms before and after, scaled
        _norm("norm_prompt", 8192, 8192, "f16", "rms", "rms", gates=8, beta=False, y_scale=0.5),
        # ragged rows and width, stream kept in 32 bits, LayerNorm on both sides, one gate
        _norm("norm_ragged", 4099, 1096, "bf16", "layer", "layer", stream="32", gates=1,
              x_scale=1.25, y_scale=0.7),
        # one layer's weights (BERT-large FFN's first layer), small groups
        _quant("quantize_layer", 1024, 4096, "bf16", 64, False),
        # a large layer with zero points
        _quant("quantize_large", 8192, 28672, "f16", 128, True),
        # one token through the BERT-large FFN's first layer
        _linear("linear_token", 1, 1024, 4096, "bf16", 128, False, "gelu", True),
        # one token through a large layer: the weights' bytes are the time
        _linear("linear_large", 1, 8192, 28672, "f16", 128, False, "none", False),
        # a decode batch, odd sizes, zero points, the smallest groups
        _linear("linear_ragged", 13, 5128, 11003, "bf16", 32, True, "silu", True),
        # a prompt through an up projection
        _linear("linear_prompt", 512, 4096, 14336, "f16", 128, False, "silu", False),
        # one token through the whole BERT-large FFN block: LN(x + W2 gelu(W1 x + b1) + b2)
        _mlp("mlp_token", 1, (1024, 4096, 1024), "bf16", 128, False, "gelu", "residual", 1e-12),
        # a decode batch of 16 through a larger block
        _mlp("mlp_batch", 16, (4096, 14336, 4096), "f16", 128, False, "silu", "residual", 1e-5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "mlp"])
    dtype = rng.choice(["f16", "bf16"])
    group = rng.choice([32, 64, 128])
    zeros = rng.random() < 0.5
    if op == "norm":
        while True:
            m, h = _log(rng, 1, 32768), 8 * _log(rng, 8, 2048)
            if m * h <= 8192 * 8192 // 2:
                break
        post, pre = rng.choice([("none", "layer"), ("none", "rms"), ("rms", "rms"), ("layer", "layer"),
                                ("rms", "none"), ("layer", "rms")])
        y = post != "none" or rng.random() < 0.7
        gates = 0
        if y and rng.random() < 0.6:
            gates = rng.choice([1, 1, 4, 16])
            m = -(-m // gates) * gates
        return _norm(None, m, h, dtype, post, pre, stream=rng.choice(["16", "32"]), gates=gates, y=y,
                     r=y and (pre == "none" or rng.random() < 0.8), beta=rng.random() < 0.5,
                     x_scale=rng.choice([1.0, 1.25]) if y else 1.0,
                     y_scale=rng.choice([1.0, 0.5, 0.7]) if y else 1.0, eps=rng.choice([1e-5, 1e-6]))
    if op == "quantize":
        while True:
            k, n = 8 * _log(rng, 8, 2048), _log(rng, 16, 28672)
            if k * n <= 8192 * 14336:
                return _quant(None, k, n, dtype, group, zeros)
    act = rng.choice(["none", "relu", "gelu", "silu", "sigmoid"])
    if op == "linear":
        while True:
            m, k, n = _log(rng, 1, 1024), 8 * _log(rng, 8, 2048), _log(rng, 16, 28672)
            if k * n <= 8192 * 14336 and m * k * n <= 512 * 4096 * 14336:
                return _linear(None, m, k, n, dtype, group, zeros, act, rng.random() < 0.5)
    while True:
        m, k, f = _log(rng, 1, 256), 8 * _log(rng, 16, 1024), 8 * _log(rng, 16, 2048)
        if k * f <= 4096 * 14336 and m * k * f <= 256 * 4096 * 4096:
            break
    widths = rng.choice([(k, f, k), (k, f, k), (k, f, f // 16 * 8 + 8, k)])
    return _mlp(None, m, widths, dtype, group, zeros, act, rng.choice(["none", "layer", "residual"]), 1e-5)


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _codes(w, group, zeros):
    """Codes (uint8 [K, N]), group scales [ceil(K / group), N] in w's type, zero points (uint8) of
    a 16-bit weight matrix. Largest magnitude to 7 (symmetric, zero point 8), or the range with
    zero to 15."""
    k, n = w.shape
    ng = -(-k // group)
    wf = torch.zeros(ng * group, n, dtype=torch.float32, device=w.device)
    wf[:k] = w.float()
    g = wf.view(ng, group, n)
    if zeros:
        lo, hi = g.amin(1).clamp(max=0.0), g.amax(1).clamp(min=0.0)
        s = ((hi - lo) / 15.0).to(w.dtype)
    else:
        s = (g.abs().amax(1) / 7.0).to(w.dtype)
    sf = s.float()
    inv = torch.where(sf > 0, sf, torch.ones_like(sf))
    if zeros:
        z = torch.where(sf > 0, torch.round(-lo / inv).clamp(0, 15), torch.zeros_like(sf))
        q = (torch.round(g / inv[:, None]) + z[:, None]).clamp(0, 15)
    else:
        z = torch.full_like(sf, 8.0)
        q = (torch.round(g / inv[:, None]).clamp(-8, 7) + 8)
    q = torch.where(sf[:, None] > 0, q, z[:, None].expand_as(q))
    q = q.view(ng * group, n)[:k].to(torch.uint8).contiguous()
    return q, s.contiguous(), (z.to(torch.uint8).contiguous() if zeros else None)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    return g


def _rand(g, shape, dtype, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale + shift).to(dtype)


def _inputs(case, seed):
    """The tensors of a case, made from the seed alone (no weights packed yet)."""
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    if case["op"] == "norm":
        m, h = case["m"], case["h"]
        sd = torch.float32 if case["stream"] == "32" else dt
        t = {"x": _rand(g, (m, h), sd, 1.5, 0.1)}
        # a few channels of a residual stream are far larger than the rest
        hot = torch.randint(0, h, (max(1, h // 256),), generator=g, device="cuda")
        t["x"][:, hot] *= 16
        t["y"] = _rand(g, (m, h), dt, 0.8) if case["y"] else None
        t["gate"] = None
        if case["gates"]:
            shape = (h,) if case["gates"] == 1 else (case["gates"], h)
            t["gate"] = _rand(g, shape, dt, 0.3, 0.5)
        for side in ("post", "pre"):
            has = case[side] != "none"
            t[side + "_gamma"] = _rand(g, (h,), dt, 0.1, 1.0) if has else None
            t[side + "_beta"] = _rand(g, (h,), dt, 0.1) if has and case["beta"] and case[side] == "layer" else None
        return t
    if case["op"] == "quantize":
        # a trained matrix: normal, with output columns of different sizes
        col = torch.exp(_rand(g, (case["n"],), torch.float32, 0.3))
        return {"w": (_rand(g, (case["k"], case["n"]), torch.float32, 0.02) * col).to(dt)}
    if case["op"] == "linear":
        widths = (case["k"], case["n"])
    else:
        widths = tuple(int(v) for v in case["widths"].split("-"))
    t = {"x": _rand(g, (case["m"], widths[0]), dt), "layers": []}
    for k, n in zip(widths[:-1], widths[1:]):
        w = _rand(g, (k, n), dt, 1.0 / math.sqrt(k))
        bias = _rand(g, (n,), dt, 0.1) if case.get("bias", True) else None
        t["layers"].append(_codes(w, case["group"], case["zeros"]) + (bias,))
        del w
    if case["op"] == "mlp":
        n = widths[-1]
        normed = case["tail"] != "none"
        t["gamma"] = _rand(g, (n,), dt, 0.1, 1.0) if normed else None
        t["beta"] = _rand(g, (n,), dt, 0.1) if normed else None
    return t


def _package():
    import __graft_entry__
    __graft_entry__.load_package()
    from gpu_pipes_b200 import cuda_ext
    return cuda_ext


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own and case["op"] in ("linear", "mlp"):
        # a serving program packs its weights once, when it loads them
        ext = _package()
        state["packed"] = [ext.w4_pack(q, s, z, group=case["group"]) for q, s, z, _ in state["layers"]]
        state["bias"] = [layer[3] for layer in state["layers"]]
        state["layers"] = None
    return state


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _act32(name, v):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-v))
    return v


def _norm32(kind, v, gamma, beta, eps):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    if gamma is not None:
        v = v * gamma.float()
    if beta is not None:
        v = v + beta.float()
    return v


def _weights32(q, s, z, group):
    k = q.shape[0]
    w = q.float()
    zf = z.float().repeat_interleave(group, 0)[:k] if z is not None else 8.0
    return (w - zf) * s.float().repeat_interleave(group, 0)[:k]


def _plain(state):
    case = state["case"]
    dt = _DT[case["dtype"]]
    if case["op"] == "norm":
        r = state["x"].float() * case["x_scale"]
        if state["y"] is not None:
            v = _norm32(case["post"], state["y"].float(), state["post_gamma"], state["post_beta"], case["eps"])
            v = v * case["y_scale"]
            gate = state["gate"]
            if gate is not None:
                gf = gate.float()
                if gf.dim() == 2:
                    v = (v.view(gf.shape[0], -1, gf.shape[1]) * gf[:, None]).view(v.shape)
                else:
                    v = v * gf
            r = r + v
        out = []
        if case["r"]:
            out.append(r.to(state["x"].dtype))
        if case["pre"] != "none":
            out.append(_norm32(case["pre"], r, state["pre_gamma"], state["pre_beta"], case["eps"]).to(dt))
        return out
    if case["op"] == "quantize":
        q, s, z = _codes(state["w"], case["group"], case["zeros"])
        return [_weights32(q, s, z, case["group"]).to(dt), s]
    v = state["x"].float()
    for i, (q, s, z, bias) in enumerate(state["layers"]):
        v = v @ _weights32(q, s, z, case["group"])
        if bias is not None:
            v = v + bias.float()
        if case["op"] == "linear" or i + 1 < len(state["layers"]):
            v = _act32(case["act"], v)
    if case["op"] == "mlp" and case["tail"] != "none":
        if case["tail"] == "residual":
            v = v + state["x"].float()
        v = _norm32("layer", v, state["gamma"], state["beta"], case["eps"])
    return [v.to(dt)]


# ------------------------------------------------------------------------------------------------
# the package's calls
# ------------------------------------------------------------------------------------------------
def _own(state):
    ext = _package()
    case = state["case"]
    if case["op"] == "norm":
        r, h = ext.block_norm(state["x"], state["y"], post=_NORMS[case["post"]], pre=_NORMS[case["pre"]],
                              gate=state["gate"], post_gamma=state["post_gamma"],
                              post_beta=state["post_beta"], pre_gamma=state["pre_gamma"],
                              pre_beta=state["pre_beta"], x_scale=case["x_scale"],
                              y_scale=case["y_scale"], post_eps=case["eps"], pre_eps=case["eps"],
                              dtype=_DT[case["dtype"]], want_r=case["r"])
        return [t for t in (r, h) if t is not None]
    if case["op"] == "quantize":
        w4 = ext.w4_quantize(state["w"], group=case["group"], zero_points=case["zeros"])
        return [ext.w4_dequantize(w4), w4.scales()]
    if case["op"] == "linear":
        return [ext.w4_linear(state["x"], state["packed"][0], state["bias"][0], act=_ACTS[case["act"]])]
    n = len(state["packed"])
    tail = {"none": 0, "layer": 1, "residual": 2}[case["tail"]]
    return [ext.w4_mlp(state["x"], state["packed"], state["bias"], acts=[_ACTS[case["act"]]] * (n - 1) + [0],
                       tail=tail, gamma=state["gamma"], beta=state["beta"], ln_eps=case["eps"])]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        m, h = case["m"], case["h"]
        sb = 4 if case["stream"] == "32" else 2
        per = sb + (2 if case["y"] else 0) + (sb if case["r"] else 0) + (2 if case["pre"] != "none" else 0)
        rows = case["gates"] + sum(case[s] != "none" for s in ("post", "pre")) * (1 + int(case["beta"]))
        return {"bytes": m * h * per + 2 * h * rows, "flops": 12 * m * h}
    if case["op"] == "quantize":
        k, n = case["k"], case["n"]
        ng = -(-k // case["group"])
        # weights in, values and scales out
        return {"bytes": 4 * k * n + 2 * ng * n, "flops": 5 * k * n}
    if case["op"] == "linear":
        widths = (case["k"], case["n"])
    else:
        widths = tuple(int(v) for v in case["widths"].split("-"))
    total = 2 * case["m"] * (widths[0] + widths[-1])
    flops = 0
    for k, n in zip(widths[:-1], widths[1:]):
        ng = -(-k // case["group"])
        total += k * n // 2 + ng * n * (3 if case["zeros"] else 2)
        total += 2 * n if case.get("bias", True) else 0
        flops += 2 * case["m"] * k * n
    if case["op"] == "mlp" and case["tail"] != "none":
        total += 4 * widths[-1]
    return {"bytes": total, "flops": flops}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _ln64(v, kind, gamma, beta, eps):
    if kind == "none":
        return v
    centre = v.sum(1, keepdim=True) / v.shape[1] if kind == "layer" else 0.0
    d = v - centre
    d = d * torch.rsqrt(d.square().sum(1, keepdim=True) / v.shape[1] + eps)
    d = d if gamma is None else d * gamma.double()
    return d if beta is None else d + beta.double()


def _act64(name, v):
    return {"none": lambda t: t, "relu": lambda t: t.clamp(min=0.0), "silu": lambda t: t * torch.sigmoid(t),
            "sigmoid": torch.sigmoid,
            "gelu": lambda t: t * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (t + 0.044715 * t ** 3))}[name](v)


def _times64(v, layer, group):
    """v [m, K] times s (q - z), group by group."""
    q, s, z, bias = layer
    k = q.shape[0]
    out = torch.zeros(v.shape[0], q.shape[1], dtype=torch.float64, device=v.device)
    step = 8 * group  # several groups at a time
    for k0 in range(0, k, step):
        part = q[k0:k0 + step].double()
        rows = torch.arange(k0, k0 + part.shape[0], device=v.device) // group
        part -= 8.0 if z is None else z.index_select(0, rows).double()
        part *= s.index_select(0, rows).double()
        out += v[:, k0:k0 + step] @ part
    return out if bias is None else out + bias.double()


def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "norm":
        m, h = case["m"], case["h"]
        rs, hs = [], []
        step = max(1, (1 << 24) // h)  # rows at a time
        gates = case["gates"]
        for r0 in range(0, m, step):
            v = case["x_scale"] * t["x"][r0:r0 + step].double()
            if t["y"] is not None:
                y = _ln64(t["y"][r0:r0 + step].double(), case["post"], t["post_gamma"], t["post_beta"], case["eps"])
                if gates:
                    rows = torch.arange(r0, r0 + y.shape[0], device=y.device) // (m // gates)
                    y = y * t["gate"].double().view(gates, h).index_select(0, rows)
                v = v + case["y_scale"] * y
            rs.append(v if case["r"] else None)
            if case["pre"] != "none":
                hs.append(_ln64(v, case["pre"], t["pre_gamma"], t["pre_beta"], case["eps"]))
        out = [torch.cat(rs)] if case["r"] else []
        return out + ([torch.cat(hs)] if hs else [])
    if case["op"] == "quantize":
        w, g, n = t["w"].double(), case["group"], case["n"]
        scales = []
        for k0 in range(0, case["k"], g):
            part = w[k0:k0 + g]
            if case["zeros"]:
                lo, hi = part.min(0).values.clamp(max=0.0), part.max(0).values.clamp(min=0.0)
                s = ((hi - lo) / 15.0).to(t["w"].dtype).double()
            else:
                s = (torch.maximum(part.max(0).values, -part.min(0).values) / 7.0).to(t["w"].dtype).double()
            safe = torch.where(s > 0, s, 1.0)
            if case["zeros"]:
                z = (-lo / safe).round().clamp(0, 15)
                part.div_(safe).round_().add_(z).clamp_(0, 15).sub_(z).mul_(s)
            else:
                part.div_(safe).round_().clamp_(-8, 7).mul_(s)
            scales.append(s)
        return [w, torch.stack(scales)]
    v = t["x"].double()
    for i, layer in enumerate(t["layers"]):
        v = _times64(v, layer, case["group"])
        if case["op"] == "linear" or i + 1 < len(t["layers"]):
            v = _act64(case["act"], v)
    if case["op"] == "mlp" and case["tail"] != "none":
        v = v + t["x"].double() if case["tail"] == "residual" else v
        v = _ln64(v, "layer", t["gamma"], t["beta"], case["eps"])
    return [v]
