"""Measured cases of the gated residual block's operators: the gated feed-forward unit, the row norms fused with gate and
residual scale, and the 8-bit block-scaled products.  ``run`` computes them in plain torch operations, or, with ``own`` set,
through the framework's entry points."""
import math

import torch

own = False

ACTS = ("silu", "gelu", "relu", "sigmoid")
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
BLOCK = 128
E4M3_MAX = 448.0

# cost caps of a drawn case: those of the largest listed case of its kind
FFN_CAP = 65536 * 1000 * 2000
NORM_CAP = 65536 * 1000
FP8_CAP = 131072 * 1000 * 2000


def listed():
    return [
        # one profile answered by the config's 1000-wide network with a feed-forward width of twice that: latency
        dict(name="ffn_one_row_bf16", op="ffn", rows=1, dim=1000, hidden=2000, act="silu", dtype="bf16", bias=True, train=False),
        # encoder rows of one batch of 4096 profiles in the framework's default fp32 accuracy
        dict(name="ffn_encoder_fp32", op="ffn", rows=4096, dim=1000, hidden=2000, act="silu", dtype="fp32", bias=True, train=False),
        # decoder rows of a training step: 4096 profiles x 16 draws, bf16 mode; the largest
        dict(name="ffn_train_bf16", op="ffn", rows=65536, dim=1000, hidden=2000, act="silu", dtype="bf16", bias=True, train=True),
        # the shipped batch of 1024 profiles x 16 draws in fp32 accuracy
        dict(name="ffn_train_fp32", op="ffn", rows=16384, dim=1000, hidden=2000, act="gelu", dtype="fp32", bias=True, train=True),
        # a ragged last batch of a small network: no size a multiple of anything
        dict(name="ffn_train_odd_fp32", op="ffn", rows=1537, dim=203, hidden=531, act="sigmoid", dtype="fp32", bias=False, train=True),
        # the block's norms around one profile
        dict(name="norm_one_row_bf16", op="norm", rows=1, gates=1, dim=1000, norm="rms", dtype="bf16", scale="number", train=False),
        # decoder rows of a training step, one gate row for each profile shared by its 16 draws
        dict(name="norm_train_bf16", op="norm", rows=65536, gates=4096, dim=1000, norm="rms", dtype="bf16", scale="number", train=True),
        # a ragged batch, layer norm with a scale for each channel
        dict(name="norm_train_odd_fp32", op="norm", rows=4611, gates=1537, dim=203, norm="layer", dtype="fp32", scale="channel", train=True),
        # one profile through an 8-bit layer: latency
        dict(name="fp8_one_row", op="fp8", rows=1, dim=1000, out=2000, dtype="bf16", bias=True),
        # scoring rows: draws x profiles of one chunk
        dict(name="fp8_scoring", op="fp8", rows=131072, dim=1000, out=2000, dtype="bf16", bias=True),
        # a ragged chunk of a small network with fp32 activations
        dict(name="fp8_odd_fp32", op="fp8", rows=777, dim=203, out=531, dtype="fp32", bias=True),
        # the whole gated unit in 8 bits over a scoring chunk
        dict(name="fp8_ffn_scoring", op="fp8_ffn", rows=65536, dim=1000, hidden=2000, act="silu", dtype="bf16", bias=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("ffn", "ffn", "norm", "fp8", "fp8_ffn"))
    dtype = rng.choice(("fp32", "bf16"))
    if op == "norm":
        dim = _log_int(rng, 24, 4096)
        gates = _log_int(rng, 1, 4096)
        share = _log_int(rng, 1, 64)
        rows = gates * share
        while rows * dim > NORM_CAP:
            share = max(1, share // 2)
            gates = gates if share > 1 else gates // 2
            rows = gates * share
        return dict(op="norm", rows=rows, gates=gates, dim=dim, norm=rng.choice(("rms", "layer")), dtype=dtype,
                    scale=rng.choice(("number", "channel")), train=rng.random() < 0.6)
    dim, hidden = _log_int(rng, 24, 1400), _log_int(rng, 24, 4096)
    bias = rng.random() < 0.5
    if op == "fp8":
        rows = min(_log_int(rng, 1, 131072), FP8_CAP // (dim * hidden))
        return dict(op="fp8", rows=rows, dim=dim, out=hidden, dtype=dtype, bias=bias)
    rows = min(_log_int(rng, 1, 65536), FFN_CAP // (dim * hidden))
    act = rng.choice(ACTS)
    if op == "fp8_ffn":                # bf16 only: an 8-bit rounding between the products leaves fp32 outputs no more digits
        return dict(op="fp8_ffn", rows=rows, dim=dim, hidden=hidden, act=act, dtype="bf16", bias=bias)
    train = rng.random() < 0.6
    if dtype == "fp32" and train:      # costs several times the bf16 form
        rows = min(rows, max(1, 16384 * 1000 * 2000 // (dim * hidden)))
    return dict(op="ffn", rows=rows, dim=dim, hidden=hidden, act=act, dtype=dtype, bias=bias, train=train)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    m, d = case["rows"], case["dim"]
    if case["op"] == "norm":
        gates = case["gates"] * d * size
        if case["train"]:
            return {"bytes": 8 * m * d * size + 2 * gates, "flops": 40 * m * d}
        return {"bytes": 4 * m * d * size + gates, "flops": 12 * m * d}
    if case["op"] == "fp8":
        return {"bytes": m * (d + case["out"]) * size + d * case["out"], "flops": 2 * m * d * case["out"]}
    f = case["hidden"]
    if case["op"] == "fp8_ffn":
        return {"bytes": 2 * m * d * size + 3 * d * f, "flops": 6 * m * d * f}
    if case["train"]:
        return {"bytes": (4 * m * d + 6 * d * f) * size, "flops": 18 * m * d * f}
    return {"bytes": (2 * m * d + 3 * d * f) * size, "flops": 6 * m * d * f}


# ------------------------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    m, d = case["rows"], case["dim"]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    def uniform(*shape, fan):          # the initial weights of a Linear layer
        return (torch.rand(*shape, generator=g, device="cuda") * 2 - 1) / math.sqrt(fan)

    t = {}
    if case["op"] == "norm":
        t["residual"] = normal(m, d).to(dt)
        t["branch"] = normal(m, d, scale=0.5).to(dt)
        t["gate"] = (1 + normal(case["gates"], d, scale=0.2)).to(dt)
        t["scale"] = 0.5 if case["scale"] == "number" else 0.5 + normal(d, scale=0.05)
        for k in ("post_weight", "pre_weight"):
            t[k] = 1 + normal(d, scale=0.1)
        if case["norm"] == "layer":
            for k in ("post_bias", "pre_bias"):
                t[k] = normal(d, scale=0.1)
        if case["train"]:
            t["d_stream"] = normal(m, d, scale=1.0 / m).to(dt)
            t["d_normed"] = normal(m, d, scale=1.0 / m).to(dt)
        return t
    t["x"] = normal(m, d).to(dt)
    if case["op"] == "fp8":
        t["weight"] = uniform(case["out"], d, fan=d).to(dt)
        t["bias"] = uniform(case["out"], fan=d) if case["bias"] else None
        return t
    f = case["hidden"]
    t["w_gate"], t["w_up"], t["w_down"] = uniform(f, d, fan=d).to(dt), uniform(f, d, fan=d).to(dt), uniform(d, f, fan=f).to(dt)
    for k, n, fan in (("b_gate", f, d), ("b_up", f, d), ("b_down", d, f)):
        b = uniform(n, fan=fan) if case["bias"] else None
        t[k] = b if b is None or case["op"] == "fp8_ffn" else b.to(dt)
    if case.get("train"):
        t["dy"] = normal(m, d, scale=1.0 / m).to(dt)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, **t}
    if own:
        from behavio_temporal_vae_amd import block_ops as B
        if case["op"] == "fp8":        # 8-bit weights are laid out once and kept
            state["packed"] = B.fp8_weight(t["weight"])
        elif case["op"] == "fp8_ffn":
            state["packed"] = B.fp8_gated_weights(t["w_gate"], t["w_up"], t["w_down"], t["b_gate"], t["b_up"], t["b_down"])
        elif case["train"]:
            for k, v in t.items():
                if torch.is_tensor(v) and k not in ("dy", "d_stream", "d_normed"):
                    v.requires_grad_(True)
    else:
        if case["op"] == "fp8":
            state["packed"] = _quantize_blocks(t["weight"].float())
        elif case["op"] == "fp8_ffn":
            state["packed"] = {k: _quantize_blocks(t[k].float()) for k in ("w_gate", "w_up", "w_down")}
    return state


# ------------------------------------------------------------------------------------------------ plain forms (32 bits)
def _act(name, a):
    """act(a) and its derivative."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-a))
        return a * s, s * (1 + a * (1 - s))
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(a * math.sqrt(0.5)))
        return a * phi, phi + a * torch.exp(-0.5 * a * a) * (1 / math.sqrt(2 * math.pi))
    if name == "relu":
        return torch.clamp(a, min=0), (a > 0).to(a.dtype)
    s = 1 / (1 + torch.exp(-a))
    return s, s * (1 - s)


def _power(amax):
    """Exponent of a block's scale: the smallest e >= -126 with amax <= 448 * 2^e (0 for a block of zeros)."""
    mant, exp = torch.frexp(amax)
    e = torch.where(mant > 0.875, exp - 8, exp - 9).clamp(min=-126)
    return torch.where(amax > 0, e, torch.zeros_like(e))


def _quantize_rows(x):
    """Values of x [M, K] held as e4m3 with one power-of-two scale for each row and 128 columns."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    p = torch.zeros(m, kb * BLOCK, device=x.device)
    p[:, :k] = x
    p = p.view(m, kb, BLOCK)
    e = _power(p.abs().amax(dim=2, keepdim=True))
    q = torch.ldexp(p, -e).to(torch.float8_e4m3fn).float()
    return torch.ldexp(q, e).view(m, -1)[:, :k]


def _quantize_blocks(w):
    """Values of w [N, K] held as e4m3 with one power-of-two scale for each 128 x 128 block."""
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    p = torch.zeros(nb * BLOCK, kb * BLOCK, device=w.device)
    p[:n, :k] = w
    p = p.view(nb, BLOCK, kb, BLOCK)
    e = _power(p.abs().amax(dim=3, keepdim=True).amax(dim=1, keepdim=True))
    q = torch.ldexp(p, -e).to(torch.float8_e4m3fn).float()
    return torch.ldexp(q, e).reshape(nb * BLOCK, kb * BLOCK)[:n, :k]


def _norm(kind, t, weight, bias, eps):
    """Normalised rows, their affine image, and 1 / deviation."""
    if kind == "layer":
        t = t - t.mean(dim=1, keepdim=True)
    r = 1 / torch.sqrt((t * t).mean(dim=1, keepdim=True) + eps)
    hat = t * r
    out = hat * weight
    return hat, (out + bias if bias is not None else out), r


def _norm_back(kind, d, hat, weight, r):
    g = d * weight
    out = g - hat * (g * hat).mean(dim=1, keepdim=True)
    if kind == "layer":
        out = out - g.mean(dim=1, keepdim=True)
    return out * r


EPS = 1e-6


def _plain_ffn(s, case):
    dt = s["x"].dtype
    f = {k: (v.float() if torch.is_tensor(v) else v) for k, v in s.items()}
    a, b = f["x"] @ f["w_gate"].t(), f["x"] @ f["w_up"].t()
    if case["bias"]:
        a, b = a + f["b_gate"], b + f["b_up"]
    v, dv = _act(case["act"], a)
    h = v * b
    y = h @ f["w_down"].t()
    if case["bias"]:
        y = y + f["b_down"]
    if not case["train"]:
        return [y.to(dt)]
    dy = f["dy"]
    dh = dy @ f["w_down"]
    da, db = dh * b * dv, dh * v
    out = [y, da @ f["w_gate"] + db @ f["w_up"], da.t() @ f["x"], db.t() @ f["x"], dy.t() @ h]
    if case["bias"]:
        out += [da.sum(0), db.sum(0), dy.sum(0)]
    return [t.to(dt) for t in out]


def _plain_norm(s, case):
    dt, kind = s["residual"].dtype, case["norm"]
    res, br, gate = s["residual"].float(), s["branch"].float(), s["gate"].float()
    share = case["rows"] // case["gates"]
    full = gate.repeat(share, 1)
    hat1, u, r1 = _norm(kind, br, s["post_weight"], s.get("post_bias"), EPS)
    v = res + s["scale"] * full * u
    hat2, n, r2 = _norm(kind, v, s["pre_weight"], s.get("pre_bias"), EPS)
    out = [v.to(dt), n.to(dt)]
    if not case["train"]:
        return out
    dn = s["d_normed"].float()
    dv = s["d_stream"].float() + _norm_back(kind, dn, hat2, s["pre_weight"], r2)
    du = s["scale"] * full * dv
    dgate = (s["scale"] * u * dv).view(share, case["gates"], -1).sum(0)
    out += [dv.to(dt), _norm_back(kind, du, hat1, s["post_weight"], r1).to(dt), dgate.to(dt)]
    if case["scale"] == "channel":
        out.append((full * u * dv).sum(0))
    out += [(du * hat1).sum(0), (dn * hat2).sum(0)]
    if kind == "layer":
        out += [du.sum(0), dn.sum(0)]
    return out


def _plain_fp8(s, case):
    y = _quantize_rows(s["x"].float()) @ s["packed"].t()
    if case["bias"]:
        y = y + s["bias"]
    return [y.to(s["x"].dtype)]


def _plain_fp8_ffn(s, case):
    w = s["packed"]
    x = _quantize_rows(s["x"].float())
    a, b = x @ w["w_gate"].t(), x @ w["w_up"].t()
    if case["bias"]:
        a, b = a + s["b_gate"], b + s["b_up"]
    y = _quantize_rows(_act(case["act"], a)[0] * b) @ w["w_down"].t()
    if case["bias"]:
        y = y + s["b_down"]
    return [y.to(s["x"].dtype)]


# ------------------------------------------------------------------------------------------------ the framework's operators
def _own(s, case):
    from behavio_temporal_vae_amd import block_ops as B
    op = case["op"]
    if op == "ffn":
        y = B.gated_feed_forward(s["x"], s["w_gate"], s["w_up"], s["w_down"], s["b_gate"], s["b_up"], s["b_down"], activation=case["act"])
        if not case["train"]:
            return [y]
        leaves = [s[k] for k in ("x", "w_gate", "w_up", "w_down")] + ([s[k] for k in ("b_gate", "b_up", "b_down")] if case["bias"] else [])
        return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]
    if op == "norm":
        keys = ["residual", "branch", "gate"] + (["scale"] if case["scale"] == "channel" else []) + ["post_weight", "pre_weight"]
        keys += ["post_bias", "pre_bias"] if case["norm"] == "layer" else []
        v, n = B.norm_gate_residual(s["residual"], s["branch"], gate=s["gate"], scale=s["scale"], post_norm=case["norm"],
                                    post_weight=s["post_weight"], post_bias=s.get("post_bias"), pre_norm=case["norm"],
                                    pre_weight=s["pre_weight"], pre_bias=s.get("pre_bias"), eps=EPS)
        if not case["train"]:
            return [v, n]
        return [v.detach(), n.detach(), *torch.autograd.grad([v, n], [s[k] for k in keys], [s["d_stream"], s["d_normed"]])]
    if op == "fp8":
        return [B.fp8_linear(s["x"], s["packed"], s["bias"])]
    return [B.fp8_gated_feed_forward(s["x"], s["packed"], activation=case["act"])]


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return {"ffn": _plain_ffn, "norm": _plain_norm, "fp8": _plain_fp8, "fp8_ffn": _plain_fp8_ffn}[case["op"]](state, case)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _round_e4m3(v):
    """Nearest e4m3 value (ties to even) of |v| <= 448: steps of 2^-3 of the value's binade, of 2^-9 below 2^-6."""
    binade = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(binade - 3)
    return torch.round(v / step) * step


def _exact_blocks(t, rows, cols):
    """t [A, B] in 64 bits as e4m3 values with a power-of-two scale for each rows x cols block."""
    a, b = t.shape
    out = torch.nn.functional.pad(t, (0, -b % cols, 0, -a % rows))
    blocks = out.unfold(0, rows, rows).unfold(1, cols, cols)            # [A/rows, B/cols, rows, cols]
    amax = blocks.abs().flatten(2).max(dim=2).values
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.full_like(amax, E4M3_MAX)) / E4M3_MAX)).clamp(min=-126)
    s = torch.exp2(e).repeat_interleave(rows, 0).repeat_interleave(cols, 1)
    return (_round_e4m3(out / s) * s)[:a, :b]


def _exact_act(name, a):
    if name == "silu":
        return a * torch.sigmoid(a)
    if name == "gelu":
        return a * torch.special.ndtr(a)
    return torch.relu(a) if name == "relu" else torch.sigmoid(a)


def _exact_norm(kind, t, w, c):
    if kind == "layer":
        var, mean = torch.var_mean(t, dim=-1, correction=0, keepdim=True)
        t = (t - mean) * torch.rsqrt(var + EPS) * w
    else:
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * w
    return t if c is None else t + c


def exact(case, seed):
    d = {k: (v.double() if torch.is_tensor(v) else v) for k, v in _inputs(case, seed).items()}
    op = case["op"]
    if op == "fp8":
        y = _exact_blocks(d["x"], 1, BLOCK) @ _exact_blocks(d["weight"], BLOCK, BLOCK).T
        return [y if d["bias"] is None else y + d["bias"]]
    if op == "fp8_ffn":
        add = (lambda t, k: t) if not case["bias"] else (lambda t, k: t + d[k])
        x = _exact_blocks(d["x"], 1, BLOCK)
        w = {k: _exact_blocks(d[k], BLOCK, BLOCK) for k in ("w_gate", "w_up", "w_down")}
        h = _exact_act(case["act"], add(x @ w["w_gate"].T, "b_gate")) * add(x @ w["w_up"].T, "b_up")
        return [add(_exact_blocks(h, 1, BLOCK) @ w["w_down"].T, "b_down")]
    if op == "ffn":
        keys = ["x", "w_gate", "w_up", "w_down"] + (["b_gate", "b_up", "b_down"] if case["bias"] else [])
        if case["train"]:
            for k in keys:
                d[k].requires_grad_(True)
        lin = torch.nn.functional.linear
        h = _exact_act(case["act"], lin(d["x"], d["w_gate"], d["b_gate"])) * lin(d["x"], d["w_up"], d["b_up"])
        y = lin(h, d["w_down"], d["b_down"])
        if not case["train"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, [d[k] for k in keys], d["dy"])]
    keys = ["residual", "branch", "gate"] + (["scale"] if case["scale"] == "channel" else []) + ["post_weight", "pre_weight"]
    keys += ["post_bias", "pre_bias"] if case["norm"] == "layer" else []
    if case["train"]:
        for k in keys:
            d[k].requires_grad_(True)
    u = _exact_norm(case["norm"], d["branch"], d["post_weight"], d.get("post_bias"))
    gate = d["gate"].repeat(case["rows"] // case["gates"], 1)
    v = d["residual"] + d["scale"] * gate * u
    n = _exact_norm(case["norm"], v, d["pre_weight"], d.get("pre_bias"))
    if not case["train"]:
        return [v, n]
    return [v.detach(), n.detach(), *torch.autograd.grad([v, n], [d[k] for k in keys], [d["d_stream"], d["d_normed"]])]
