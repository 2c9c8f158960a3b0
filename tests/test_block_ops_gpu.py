"""GPU: the gated residual block's operators against their definitions in 64 bits.

Tolerances.  u(t) = finfo(t).eps / 2 is the largest relative error of one rounding to t.  A float32 sum of n products picks up
about sqrt(n) roundings of the size of its partial sums: its Frobenius error is held to 2^-24 (4 + sqrt(n)) of the result's norm,
chains of products to the sum of their terms (times the factor by which cancellation shrinks a result, stated where there is one).
bfloat16 results are held element by element to bounds that count every rounding: with |.| the product of magnitudes,
an operand rounded to bfloat16 contributes u |.| and the result's own rounding u |result|; float32 sums add n 2^-24 |.|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from behavio_temporal_vae_amd import _native as nv  # noqa: E402
from behavio_temporal_vae_amd import block_ops as B  # noqa: E402

BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -8          # bfloat16
E = 2.0 ** -24         # float32


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    d = torch.device("cuda:0")
    nv.ensure_device(d)
    return d


def rnd(dev, *shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(dev)


def d64(t):
    return None if t is None else t.detach().double()


def frob(got, ref, tol, what):
    assert got.shape == ref.shape, what
    err, norm = (got.detach().double() - ref).norm().item(), ref.norm().item()
    assert err <= tol * norm + 1e-300, f"{what}: relative error {err / (norm + 1e-300):.3e} > {tol:.3e}"


def within(got, ref, lim, what):
    err = (got.detach().double() - ref).abs()
    bad = ~(err <= lim + 1e-300)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst ratio {(err / (lim + 1e-300)).max().item():.2f}"


def act64(name, a):
    if name == "silu":
        return a * torch.sigmoid(a)
    if name == "gelu":
        return 0.5 * a * torch.special.erfc(-a / math.sqrt(2))
    return torch.relu(a) if name == "relu" else torch.sigmoid(a)


def ffn64(t, act):
    a = t["x"] @ t["wg"].t()
    b = t["x"] @ t["wu"].t()
    if t["bg"] is not None:
        a, b = a + t["bg"], b + t["bu"]
    h = act64(act, a) * b
    y = h @ t["wd"].t()
    return a, b, h, y if t["bd"] is None else y + t["bd"]


def ffn_case(dev, M, K, F, N, dtype, bias, seed=1):
    t = dict(x=rnd(dev, M, K, seed=seed, dtype=dtype), wg=rnd(dev, F, K, seed=seed + 1, scale=1 / math.sqrt(K), dtype=dtype),
             wu=rnd(dev, F, K, seed=seed + 2, scale=1 / math.sqrt(K), dtype=dtype), wd=rnd(dev, N, F, seed=seed + 3, scale=1 / math.sqrt(F), dtype=dtype))
    for k, n, s in (("bg", F, 4), ("bu", F, 5), ("bd", N, 6)):
        t[k] = rnd(dev, n, seed=seed + s, scale=0.3, dtype=dtype) if bias else None
    return t


def call_ffn(t, act):
    return B.gated_feed_forward(t["x"], t["wg"], t["wu"], t["wd"], t["bg"], t["bu"], t["bd"], activation=act)


def check_ffn_forward(y, t, act):
    r = {k: d64(v) for k, v in t.items()}
    a, b, h, ref = ffn64(r, act)
    K, F = t["x"].shape[1], t["wg"].shape[0]
    if t["x"].dtype == F32:
        # two projections meet in h (a 1-Lipschitz-like activation: |act'| <= 1.13), one more product follows
        frob(y, ref, E * (2.3 * (4 + math.sqrt(K)) + 4 + math.sqrt(F)) * max(1.0, h.norm().item() * r["wd"].norm().item() / math.sqrt(F) / ref.norm().item()), "y")
        return
    xs = r["x"].abs()
    ea = (K + 4) * E * (xs @ r["wg"].abs().t()) + 2 ** -20 * a.abs()          # float32 sums; the fast exp and reciprocal
    eb = (K + 4) * E * (xs @ r["wu"].abs().t())
    eh = 1.13 * ea * b.abs() + act64(act, a).abs() * (eb + 2 ** -20 * b.abs()) + U * h.abs()
    lim = eh @ r["wd"].abs().t() + (F + 4) * E * (h.abs() @ r["wd"].abs().t()) + U * ref.abs()
    within(y, ref, lim * 1.01, "y")


SIZES = [(1, 8, 8, 8), (1, 1000, 2000, 1000), (3, 7, 5, 1), (17, 203, 531, 96), (32, 24, 40, 72), (33, 203, 531, 203), (129, 64, 333, 65), (300, 1000, 264, 48), (700, 40, 1001, 31)]


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("M,K,F,N", SIZES)
def test_ffn_forward(dev, M, K, F, N, dtype):
    for i, act in enumerate(B.ACTIVATIONS):
        t = ffn_case(dev, M, K, F, N, dtype, bias=i % 2 == 0, seed=10 * i)
        check_ffn_forward(call_ffn(t, act), t, act)
        y, _ = B.gated_feed_forward_tape(t["x"], t["wg"], t["wu"], t["wd"], t["bg"], t["bu"], t["bd"], activation=act)
        check_ffn_forward(y, t, act)


def ffn_grads(t, act, dy):
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in t.items() if v is not None}
    y = call_ffn({**{k: None for k in t}, **leaves}, act)
    return y, dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))


def ffn_grads64(t, act, dy):
    leaves = {k: d64(v).requires_grad_(True) for k, v in t.items() if v is not None}
    y = ffn64({**{k: None for k in t}, **leaves}, act)[3]
    return dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy.double())))


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("M,K,F,N", [(1, 8, 8, 8), (2, 7, 5, 1), (31, 203, 531, 96), (257, 64, 333, 65), (1037, 200, 264, 200), (2500, 40, 1001, 31)])
def test_ffn_backward(dev, M, K, F, N, dtype):
    for i, act in enumerate(B.ACTIVATIONS):
        t = ffn_case(dev, M, K, F, N, dtype, bias=i % 2 == 1, seed=100 + 10 * i)
        dy = rnd(dev, M, N, seed=99, dtype=dtype)
        y, got = ffn_grads(t, act, dy)
        check_ffn_forward(y, t, act)
        ref = ffn_grads64(t, act, dy)
        if dtype == F32:
            # products in the chain before a gradient: projections (K), dh (N), then its own (2F or M); sums over rows may cancel: times
            # the ratio of what is added to what is left, at most sqrt(terms) for independent terms of one size
            for k, v in got.items():
                n = {"x": 2 * F}.get(k, M)
                frob(v, ref[k], 3 * E * ((4 + math.sqrt(K)) + (4 + math.sqrt(N)) + (4 + math.sqrt(n))), f"d{k} ({act})")
            continue
        r = {k: d64(v) for k, v in t.items()}
        a, b, h, _ = ffn64(r, act)
        a = a.detach().requires_grad_(True)
        v = act64(act, a)
        d1 = torch.autograd.grad(v.sum(), a, create_graph=act != "relu")[0]
        d2 = torch.autograd.grad(d1.sum(), a)[0] if act != "relu" else torch.zeros_like(a)
        a, v, d1 = a.detach(), v.detach(), d1.detach()
        dy64 = dy.double()
        dh = dy64 @ r["wd"]
        s = (K + N + 8) * E * 4 + 2 ** -18                     # float32 sums and the fast exp, generously
        eh = U * h.abs() + s * (h.abs() + a.abs() * b.abs() + b.abs())
        # the kept a and b are rounded; act' may move over u |a| by as much as its slope nearby allows (1.2 |a| u covers curvature: |act''| <= 1.2)
        shift = U * a.abs() + s * (r["x"].abs() @ r["wg"].abs().t())
        curve = torch.maximum(d2.abs(), torch.full_like(a, 0.1)) * 2 * shift if act != "relu" else (a.abs() <= 2 * shift).double()
        slope = d1.abs() + curve
        da, db = dh * b * d1, dh * v
        dhs = s * (dy64.abs() @ r["wd"].abs())
        eda = dh.abs() * (U * b.abs() * slope + b.abs() * curve) + dhs * b.abs() * slope + U * da.abs() + s * dh.abs() * (b.abs() + 1)
        edb = dh.abs() * slope * 2 * shift + dhs * v.abs() + U * db.abs() + s * dh.abs()
        eda, edb = 1.1 * eda, 1.1 * edb
        x, wg, wu = r["x"], r["wg"], r["wu"]
        lim = {"x": eda @ wg.abs() + edb @ wu.abs(), "wg": eda.t() @ x.abs(), "wu": edb.t() @ x.abs(), "wd": dy64.abs().t() @ eh,
               "bg": eda.sum(0), "bu": edb.sum(0), "bd": (M + 4) * E * dy64.abs().sum(0)}
        mag = {"x": da.abs() @ wg.abs() + db.abs() @ wu.abs(), "wg": da.abs().t() @ x.abs(), "wu": db.abs().t() @ x.abs(), "wd": dy64.abs().t() @ h.abs(),
               "bg": da.abs().sum(0), "bu": db.abs().sum(0), "bd": dy64.abs().sum(0)}
        for k, g in got.items():
            within(g, ref[k], 1.01 * (lim[k] + (2 * F + M + 8) * E * mag[k] + U * ref[k].abs()), f"d{k} ({act})")


def test_ffn_backward_matches_differences(dev):
    """Directional derivative of the float32 forward, taken in 64 bits from the definition at x +- s v: the gradient's inner product
    with v is the difference quotient up to O(s^2)."""
    t = ffn_case(dev, 70, 24, 40, 16, F32, True, seed=7)
    dy = rnd(dev, 70, 16, seed=8)
    _, got = ffn_grads(t, "gelu", dy)
    s = 1e-4
    for k in got:
        v = rnd(dev, *t[k].shape, seed=9).double()
        f = []
        for sign in (1, -1):
            r = {q: d64(w) for q, w in t.items()}
            r[k] = r[k] + sign * s * v
            f.append((ffn64(r, "gelu")[3] * dy.double()).sum().item())
        quotient, inner = (f[0] - f[1]) / (2 * s), (got[k].double() * v).sum().item()
        scale = (got[k].double().abs() * v.abs()).sum().item()
        assert abs(quotient - inner) <= 2e-6 * scale, (k, quotient, inner)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
def test_ffn_strides_and_shapes(dev, dtype):
    """Inputs that are views: padded rows, transposed storage, odd offsets, leading dimensions."""
    t = ffn_case(dev, 96, 40, 56, 24, dtype, True, seed=3)
    base = call_ffn(t, "silu")
    wide = torch.full((96, 48), float("nan"), dtype=dtype, device=dev)
    wide[:, :40] = t["x"]
    odd = torch.full((96 * 43 + 1,), float("nan"), dtype=dtype, device=dev)[1:].view(96, 43)
    odd[:, :40] = t["x"]
    for x in (wide[:, :40], odd[:, :40], t["x"].t().contiguous().t(), t["x"].view(4, 24, 40)):
        y = call_ffn({**t, "x": x}, "silu")
        assert y.shape == (*x.shape[:-1], 24) and torch.equal(y.reshape(96, 24), base)
    wt = {**t, "wg": t["wg"].t().contiguous().t(), "wd": torch.cat([t["wd"], t["wd"]], 1)[:, :56]}
    assert torch.equal(call_ffn(wt, "silu"), base)
    few = {**t, "x": odd[:5, :40]}
    check_ffn_forward(call_ffn(few, "silu"), few, "silu")
    dy = rnd(dev, 24, 96, dtype=dtype).t()                     # a gradient that is a transposed view
    _, got = ffn_grads(t, "silu", dy)
    _, ref = ffn_grads(t, "silu", dy.contiguous())
    for k in got:
        assert torch.equal(got[k], ref[k]), k


def test_ffn_empty_and_no_grad_paths(dev):
    t = ffn_case(dev, 0, 40, 56, 24, F32, True)
    y, got = ffn_grads(t, "silu", torch.empty(0, 24, device=dev))
    assert y.shape == (0, 24) and got["x"].shape == (0, 40)
    for k in ("wg", "wu", "wd", "bg", "bu", "bd"):
        assert not got[k].any(), k
    t = ffn_case(dev, 50, 40, 56, 24, F32, False)
    wd = t["wd"].clone().requires_grad_(True)                  # only one gradient asked for
    call_ffn({**t, "wd": wd}, "silu").sum().backward()
    assert wd.grad is not None
    x = t["x"].clone().requires_grad_(True)
    gx, = torch.autograd.grad(call_ffn({**t, "x": x}, "silu").sum(), x)
    assert gx.shape == x.shape


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("M", [20, 200])
def test_ffn_non_finite_rows_stay_alone(dev, M, dtype):
    t = ffn_case(dev, M, 72, 96, 40, dtype, True, seed=5)
    base = call_ffn(t, "silu")
    x = t["x"].clone()
    x[3, 71] = float("nan")
    x[7, 0] = float("inf")
    y = call_ffn({**t, "x": x}, "silu")
    keep = [i for i in range(M) if i not in (3, 7)]
    assert torch.equal(y[keep], base[keep]) and y[3].isnan().all() and not y[7].isfinite().all()


def test_ffn_graph_replays_and_streams(dev):
    """Tapes captured into two graphs, replayed in turn with eager work between: every replay equals the eager result."""
    t = ffn_case(dev, 300, 64, 96, 64, BF, True, seed=6)
    dy = rnd(dev, 300, 64, seed=1, dtype=BF)
    args = (t["wg"], t["wu"], t["wd"], t["bg"], t["bu"], t["bd"])

    def step(x):
        y, tape = B.gated_feed_forward_tape(x, *args)
        return (y, *tape.backward(dy))

    xs = [t["x"].clone(), t["x"].clone()]
    step(xs[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x))
        graphs.append(g)
    for rep in range(4):
        for i in (0, 1):
            xs[i].copy_(rnd(dev, 300, 64, seed=20 + 2 * rep + i, dtype=BF))
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            for a, b in zip(outs[i], step(xs[i].clone())):
                assert torch.equal(a, b), (rep, i)
    side = torch.cuda.Stream()
    want = step(t["x"])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(t["x"])
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    x = t["x"].clone().requires_grad_(True)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="tape"):
        with torch.cuda.graph(g):
            call_ffn({**t, "x": x}, "silu")


def test_planes_are_exact(dev):
    """x times the identity comes back bit for bit from the three-plane product; so does the identity's transposed product."""
    M, K = 200, 72
    x = rnd(dev, M, K, seed=4) * torch.exp(rnd(dev, M, K, seed=5) * 8)
    x[0, 0], x[1, 1], x[2, 2] = 3.4e38, -3.4028234e38, 1e-30
    eye = torch.eye(K, device=dev)
    X, I = B._operand(x, 3, K), B._operand(eye, 3, M)
    out = torch.empty(M, K, device=dev)
    assert torch.equal(B._product(X, I, None, out, 3, M, K, X.width), x)
    lib = nv.lib()
    eyem = torch.eye(M, device=dev)
    Im = B._operand(eyem, 3, K)
    ws = torch.empty(lib.btvae_block_wgrad_ws(M, K, M, 3), device=dev)
    out2 = torch.empty(M, K, device=dev)
    nv.call("btvae_block_wgrad", Im.ptr(), Im.ld, X.ptr(), X.ld, ws.data_ptr(), ws.numel(), out2.data_ptr(), M, None, 0, 0, K, 0, 0, 3, M, K, M)
    assert torch.equal(out2, x)


@pytest.mark.parametrize("planes", [1, 3])
@pytest.mark.parametrize("M,N,K", [(256, 256, 32), (300, 260, 1000), (1000, 77, 40), (64, 16, 4096), (4100, 2056, 64)])
def test_block_product(dev, planes, M, N, K):
    dt = F32 if planes == 3 else BF
    a, b, bias = rnd(dev, M, K, seed=1, dtype=dt), rnd(dev, N, K, seed=2, dtype=dt), rnd(dev, N, seed=3)
    A, W = B._operand(a, planes, N), B._operand(b, planes, M)
    ref = a.double() @ b.double().t() + bias.double()
    frob(B._product(A, W, bias, torch.empty(M, N, device=dev), planes, M, N, A.width), ref, E * (4 + math.sqrt(K)), "fp32 result")
    got = B._product(A, W, bias, torch.empty(M, N, dtype=BF, device=dev), planes, M, N, A.width)
    within(got, ref, U * ref.abs() * 1.01 + (K + 4) * E * (a.double().abs() @ b.double().abs().t()) + E, "bf16 result")
    pad = torch.full((M, N + 3), 7.0, device=dev)
    B._product(A, W, bias, pad[:, :N], planes, M, N, A.width)
    assert (pad[:, N:] == 7.0).all()


@pytest.mark.parametrize("planes", [1, 3])
@pytest.mark.parametrize("R", [0, 1, 31, 32, 33, 1000, 5000])
@pytest.mark.parametrize("M,N", [(8, 8), (130, 264), (333, 65), (1062, 203)])
def test_block_wgrad(dev, planes, R, M, N):
    dt = F32 if planes == 3 else BF
    a, b = rnd(dev, R, M, seed=1, dtype=dt), rnd(dev, R, N, seed=2, dtype=dt)
    A, X = B._operand(a, planes, N), B._operand(b, planes, M)
    lib = nv.lib()
    ws = torch.empty(lib.btvae_block_wgrad_ws(M, N, R, planes), device=dev)
    h = M // 3
    o0, o1 = torch.full((h, N), 2.0, device=dev), torch.full((M - 2 * h, N), 3.0, device=dev)
    for acc in (1, 0):
        nv.call("btvae_block_wgrad", A.ptr(), A.ld, X.ptr(), X.ld, ws.data_ptr(), ws.numel(), o0.data_ptr(), h, o1.data_ptr(), 2 * h, M - 2 * h, N, 0, acc, planes, M, N, R)
        ref = a.double().t() @ b.double()
        tol = E * (4 + math.sqrt(max(R, 1)))
        frob(o0, ref[:h] + 2.0 * acc, tol + 2 * E, "first rows")
        frob(o1, ref[2 * h:] + 3.0 * acc, tol + 2 * E, "last rows")


# ------------------------------------------------------------------------------------------------ norms
def norm64(t, kind, w, c, eps):
    if kind is None:
        return t
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
    t = t if w is None else t * w
    return t if c is None else t + c


def block64(r, post, pre, scale, eps):
    v = r["residual"]
    if r["branch"] is not None:
        u = norm64(r["branch"], post, r["post_weight"], r["post_bias"], eps)
        if r["gate"] is not None:
            u = u * r["gate"].repeat(v.shape[0] // r["gate"].shape[0], 1)
        v = v + (scale if r["scale"] is None else r["scale"]) * u
    return v, None if pre is None else norm64(v, pre, r["pre_weight"], r["pre_bias"], eps)


def norm_case(dev, M, N, G, rt, bt, post, pre, vec_scale, affine, seed=1):
    t = dict(residual=rnd(dev, M, N, seed=seed, dtype=rt), branch=rnd(dev, M, N, seed=seed + 1, dtype=bt),
             gate=(1 + rnd(dev, G, N, seed=seed + 2, scale=0.3)).to(bt) if G else None,
             scale=0.5 + rnd(dev, N, seed=seed + 3, scale=0.1) if vec_scale else None)
    for k, on in (("post", post), ("pre", pre)):
        t[k + "_weight"] = 1 + rnd(dev, N, seed=seed + 4, scale=0.2) if affine and on else None
        t[k + "_bias"] = rnd(dev, N, seed=seed + 5, scale=0.2) if affine and on else None
    return t


def call_norm(t, post, pre, eps=1e-6):
    return B.norm_gate_residual(t["residual"], t["branch"], gate=t["gate"], scale=0.7 if t["scale"] is None else t["scale"], post_norm=post, post_weight=t["post_weight"],
                                post_bias=t["post_bias"], pre_norm=pre, pre_weight=t["pre_weight"], pre_bias=t["pre_bias"], eps=eps)


def rounding(t):
    return U if t.dtype == BF else E


NORM_CASES = [  # M, N, G, residual type, branch type, post, pre, scale vector, affine
    (1, 1, 1, F32, F32, "rms", "rms", False, True),
    (1, 1000, 1, BF, BF, "rms", "rms", False, True),
    (5, 7, 0, F32, F32, "layer", "layer", True, True),
    (12, 203, 3, F32, F32, "layer", "rms", True, True),
    (64, 512, 64, F32, BF, "rms", "layer", False, False),
    (130, 520, 65, BF, BF, None, "rms", True, True),
    (96, 1000, 32, BF, BF, "layer", "layer", True, True),
    (40, 1001, 1, F32, BF, "rms", None, False, True),
    (4096, 48, 1, F32, F32, "rms", "rms", True, True),
    (9000, 96, 3000, BF, BF, "rms", "rms", False, True),
    (33, 2049, 11, F32, F32, "rms", "layer", False, True),
    (30, 4096, 10, BF, BF, "layer", "rms", True, True),
    (14, 8192, 7, F32, F32, "layer", "layer", True, True),
    (6, 5003, 2, F32, BF, "layer", "rms", False, True),
]


@pytest.mark.parametrize("case", NORM_CASES, ids=lambda c: f"{c[0]}x{c[1]}g{c[2]}")
def test_norm_gate_residual(dev, case):
    M, N, G, rt, bt, post, pre, vec, affine = case
    t = norm_case(dev, *case)
    eps = 1e-6
    names = [k for k, v in t.items() if v is not None]
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items() if v is not None}
    v, n = call_norm({**{k: None for k in t}, **leaves}, post, pre)
    with torch.no_grad():
        v2, n2 = call_norm(t, post, pre)
    assert torch.equal(v, v2) and (n is None or torch.equal(n, n2))
    r = {k: (d64(w).requires_grad_(True) if w is not None else None) for k, w in t.items()}
    rv, rn = block64(r, post, pre, 0.7, eps)
    # forward: a dozen float32 roundings of terms no larger than these, sums of N in a tree, the result's own rounding
    f = (16 + math.log2(N)) * E
    full = None if t["gate"] is None else t["gate"].double().repeat(M // G, 1).abs()
    su = (rv - r["residual"]).abs().detach()
    post_out = norm64(r["branch"], post, r["post_weight"], None, eps).abs().detach() * (1 if full is None else full) * (0.7 if t["scale"] is None else t["scale"].double().abs())
    shift = 1.0
    if post == "layer":
        shift = 1 + (t["branch"].double().mean(-1, keepdim=True).abs() / t["branch"].double().std(-1, keepdim=True).clamp(min=1e-3) if N > 1 else 1e3)
    ev = f * shift * (r["residual"].abs().detach() + 4 * post_out + 4 * su) + f * shift
    within(v, rv.detach(), ev + rounding(v) * rv.abs().detach(), "stream")
    if n is not None:
        q = 1 / torch.sqrt((rv * rv).mean(-1, keepdim=True) + eps) if pre == "rms" else 1 / torch.sqrt(rv.var(-1, correction=0, keepdim=True) + eps)
        w = 1 if r["pre_weight"] is None else r["pre_weight"].abs()
        en = (2 * (ev + ev.amax(-1, keepdim=True)) * q * w + 16 * f * rn.abs() + f * (1 + (rv.abs().amax(-1, keepdim=True) * q) * w)).detach()
        within(n, rn.detach(), en * (1 + (rv.abs().amax(-1, keepdim=True) * q).detach() * 0 + 2) + rounding(n) * rn.abs().detach(), "normed")
    dv = rnd(dev, M, N, seed=50, dtype=v.dtype)
    dn = rnd(dev, M, N, seed=51, dtype=n.dtype) if n is not None else None
    outs = [v] + ([n] if n is not None else [])
    ups = [dv] + ([dn] if dn is not None else [])
    got = dict(zip(names, torch.autograd.grad(outs, [leaves[k] for k in names], ups)))
    routs = [rv] + ([rn] if rn is not None else [])
    ref = dict(zip(names, torch.autograd.grad(routs, [r[k] for k in names], [u.double() for u in ups])))
    # gradients: float32 inside; the stream is kept in its type (a rounding of it moves its norm's gradient by as much), the
    # result is rounded once; column sums add M terms
    cond = 8.0 if N > 4 else 1e4            # one or a few columns: the norm's gradient cancels to nearly nothing
    for k in names:
        tol = rounding(got[k]) + cond * rounding(t["residual"]) + cond * E * (8 + math.sqrt(M) + math.sqrt(N))
        scale = max(1.0, math.sqrt(M * N) * 0.1 / (ref[k].norm().item() + 1e-30)) if N <= 4 else 1.0
        frob(got[k], ref[k], tol * scale, f"d{k}")


def test_norm_parts(dev):
    """Pre norm alone, no norm at all, partial gradients, leading dimensions, an infinite row, no rows."""
    x = rnd(dev, 6, 5, 40, seed=1)
    s, n = B.norm_gate_residual(x, pre_norm="layer")
    assert s is x and n.shape == x.shape
    frob(n, norm64(x.double(), "layer", None, None, 1e-6), 20 * E, "layer norm")
    y = rnd(dev, 6, 5, 40, seed=2)
    s, n = B.norm_gate_residual(x, y, scale=2.0, pre_norm=None)
    assert n is None
    within(s, x.double() + 2 * y.double(), 2 * E * (x.double().abs() + 2 * y.double().abs()), "sum")
    xg, yg = x.clone().requires_grad_(True), y.clone().requires_grad_(True)
    s, n = B.norm_gate_residual(xg, yg, post_norm="rms")
    gs, = torch.autograd.grad(s.sum(), xg, retain_graph=True)
    assert torch.equal(gs, torch.ones_like(x))
    gn, = torch.autograd.grad((n * y).sum(), yg)
    xr, yr = x.double().requires_grad_(True), y.double().requires_grad_(True)
    nr = norm64(xr + norm64(yr, "rms", None, None, 1e-6), "rms", None, None, 1e-6)
    frob(gn, torch.autograd.grad((nr * y.double()).sum(), yr)[0], 200 * E, "gradient through normed alone")
    xi = x.reshape(30, 40).clone()
    base = B.norm_gate_residual(xi, y.reshape(30, 40))[1]
    xi[4, 3], xi[9, 0] = float("inf"), float("nan")
    out = B.norm_gate_residual(xi, y.reshape(30, 40))[1]
    keep = [i for i in range(30) if i not in (4, 9)]
    assert torch.equal(out[keep], base[keep]) and not out[4].isfinite().all() and out[9].isnan().all()
    w = torch.ones(40, device=dev, requires_grad=True)
    e = torch.empty(0, 40, device=dev, requires_grad=True)
    s, n = B.norm_gate_residual(e, torch.empty(0, 40, device=dev), pre_weight=w)
    ge, gw = torch.autograd.grad(n.sum() + s.sum(), [e, w])
    assert ge.shape == (0, 40) and not gw.any()
    z = torch.zeros(3, 40, device=dev)
    assert not B.norm_gate_residual(z, z, post_norm="rms")[1].any()          # rows of zeros: finite, zero


def test_norm_gradients_match_differences(dev):
    t = norm_case(dev, 24, 40, 8, F32, F32, "layer", "rms", True, True, seed=3)
    names = list(t)
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    v, n = call_norm(leaves, "layer", "rms")
    dv, dn = rnd(dev, 24, 40, seed=5), rnd(dev, 24, 40, seed=6)
    got = dict(zip(names, torch.autograd.grad([v, n], [leaves[k] for k in names], [dv, dn])))
    s = 1e-4
    for k in names:
        d = rnd(dev, *t[k].shape, seed=7).double()
        f = []
        for sign in (1, -1):
            r = {q: d64(w) for q, w in t.items()}
            r[k] = r[k] + sign * s * d
            a, b = block64(r, "layer", "rms", None, 1e-6)
            f.append((a * dv.double()).sum().item() + (b * dn.double()).sum().item())
        quotient, inner = (f[0] - f[1]) / (2 * s), (got[k].double() * d).sum().item()
        assert abs(quotient - inner) <= 5e-6 * (got[k].double().abs() * d.abs()).sum().item() + 1e-6, k


def test_norm_graph_replays(dev):
    t = norm_case(dev, 96, 200, 32, BF, BF, "rms", "rms", True, True, seed=8)
    dv, dn = rnd(dev, 96, 200, seed=1, dtype=BF), rnd(dev, 96, 200, seed=2, dtype=BF)

    def step(res):
        v, n, tape = B.norm_gate_residual_tape(res, t["branch"], gate=t["gate"], scale=t["scale"], post_norm="rms", post_weight=t["post_weight"],
                                               post_bias=t["post_bias"], pre_norm="rms", pre_weight=t["pre_weight"], pre_bias=t["pre_bias"])
        return (v, n, *tape.backward(dv, dn))

    res = t["residual"].clone()
    step(res)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(res)
    for rep in range(4):
        res.copy_(rnd(dev, 96, 200, seed=30 + rep, dtype=BF))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step(res.clone())):
            assert torch.equal(a, b), rep


# ------------------------------------------------------------------------------------------------ 8-bit products
def e4m3_64(t, rows, cols):
    """Values of t in 64 bits as e4m3 with a power-of-two scale for each rows x cols block, from the definition."""
    t = t.double()
    a, b = t.shape
    p = torch.zeros(-(-a // rows) * rows, -(-b // cols) * cols, dtype=torch.float64, device=t.device)
    p[:a, :b] = t
    k = p.view(p.shape[0] // rows, rows, p.shape[1] // cols, cols)
    amax = k.abs().amax(dim=(1, 3), keepdim=True)
    e = torch.where(amax > 0, torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448)), torch.zeros_like(amax)).clamp(min=-126)
    v = k / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step * torch.exp2(e)).reshape(p.shape)[:a, :b]


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 128), (7, 129), (130, 203), (64, 1000), (257, 4100)])
def test_fp8_quantize(dev, M, K, dtype):
    x = (rnd(dev, M, K, seed=1) * torch.exp(3 * rnd(dev, M, 1, seed=2))).to(dtype)
    x[0, 0] = 448.0
    if K > 130:
        x[0, 128:] = 0
        x[-1, :128] *= 2.0 ** -100
        x[-1, 128:] = (x[-1, 128:].float() * 2.0 ** -124).to(dtype)
    assert torch.equal(B.fp8_quantize(x).dequantize().double(), e4m3_64(x, 1, 128))
    assert torch.equal(B.fp8_weight(x).dequantize().double(), e4m3_64(x, 128, 128))
    assert torch.equal(B.fp8_quantize(x.t().contiguous().t()).dequantize(), B.fp8_quantize(x).dequantize())


def test_fp8_quantize_ties_and_non_finite(dev):
    grid = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()     # every finite value from 0 to 448
    mid = (grid[:-1] + grid[1:]) / 2
    x = torch.zeros(4, 256)
    x[0, :127], x[0, 127] = grid, 448.0
    x[1, :126], x[1, 127] = mid, 448.0                         # ties: to even
    x[2, :126], x[2, 127] = -mid, 448.0
    x[3, :126], x[3, 127] = torch.nextafter(mid, torch.tensor(1e9)), 448.0
    x = x.to(dev)
    assert torch.equal(B.fp8_quantize(x).dequantize().double(), e4m3_64(x, 1, 128))
    y = rnd(dev, 2, 256, seed=1)
    ref = B.fp8_quantize(torch.where(torch.arange(256, device=dev) == 5, torch.zeros((), device=dev), y)).dequantize()
    for bad in (float("inf"), float("-inf"), float("nan")):
        z = y.clone()
        z[0, 5] = bad
        got = B.fp8_quantize(z).dequantize()
        assert got[0, 5].isnan() and got.isnan().sum() == 1
        got[0, 5] = 0
        assert torch.equal(got[0], ref[0])


FP8_SIZES = [(1, 1, 1), (1, 1000, 2000), (5, 203, 531), (32, 4100, 70), (33, 128, 128), (200, 203, 531), (300, 1000, 264), (64, 20000, 96), (4100, 264, 2056), (1000, 72, 77)]


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("M,K,N", FP8_SIZES)
def test_fp8_linear(dev, M, K, N, dtype):
    x = (rnd(dev, M, K, seed=1) * torch.exp(2 * rnd(dev, M, 1, seed=4))).to(dtype)
    w, bias = rnd(dev, N, K, seed=2, scale=1 / math.sqrt(K), dtype=dtype), rnd(dev, N, seed=3)
    W = B.fp8_weight(w)
    xq, wq = e4m3_64(x, 1, 128), e4m3_64(w, 128, 128)
    ref = xq @ wq.t() + bias.double()
    lim = (K + 8) * E * (xq.abs() @ wq.abs().t()) + 2 * E * ref.abs()
    got = B.fp8_linear(x, W, bias, out_dtype=F32)
    within(got, ref, lim, "fp32 result")
    frob(got, ref, E * (4 + math.sqrt(K)), "fp32 result")
    # bfloat16 results of more than 32 rows: the 8-bit pipe cuts each product it adds to a multiple of a unit that follows the largest of its
    # group.  Over 128 products of normal values its error is 2^-16 of a result (rms): as the result's rms is sqrt(128) times a
    # product's, and the largest product is about 9 times a product's rms, a cut of at most 2^-15 of the largest product each;
    # K independent cuts add to sqrt(K) 2^-15 of it, and 4 of those deviations are sqrt(K) 2^-13
    pipe = math.sqrt(K) * 2.0 ** -13 * xq.abs().amax(1, keepdim=True) * wq.abs().amax(1)
    within(B.fp8_linear(x, W, bias, out_dtype=BF), ref, lim + pipe * (M > 32) + U * ref.abs() * 1.01, "bf16 result")
    within(B.fp8_linear(B.fp8_quantize(x), W, bias), ref, lim, "from quantised rows")
    assert B.fp8_linear(x, W).dtype == dtype
    within(B.fp8_linear(x, W, out_dtype=F32), xq @ wq.t(), lim, "without a bias")


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("M,K,F,N", [(1, 1000, 2000, 1000), (4, 7, 5, 3), (32, 203, 531, 96), (33, 203, 531, 96), (300, 1000, 264, 48), (5000, 72, 1001, 40)])
def test_fp8_gated_feed_forward(dev, M, K, F, N, dtype):
    for i, act in enumerate(B.ACTIVATIONS):
        t = ffn_case(dev, M, K, F, N, dtype, bias=i % 2 == 0, seed=40 + i)
        P = B.fp8_gated_weights(t["wg"], t["wu"], t["wd"], t["bg"], t["bu"], t["bd"])
        y = B.fp8_gated_feed_forward(t["x"], P, activation=act, out_dtype=F32)
        r = {k: d64(v) for k, v in t.items()}
        r["x"], r["wg"], r["wu"] = e4m3_64(t["x"], 1, 128), e4m3_64(t["wg"], 128, 128), e4m3_64(t["wu"], 128, 128)
        wd = e4m3_64(t["wd"], 128, 128)
        a, b, h, _ = ffn64({**r, "wd": wd}, act)
        hq = e4m3_64(h, 1, 128)
        ref = hq @ wd.t() + (0 if r["bd"] is None else r["bd"])
        # h comes from float32 sums: where it lies that close to a border between two e4m3 values (or its block's maximum to a
        # border between two scales) it may take the other one, a step of at most 2^-3 of |h|
        xs = r["x"].abs()
        ea = (K + 8) * E * 2 * (xs @ r["wg"].abs().t()) + 2 ** -19 * a.abs()
        eb = (K + 8) * E * 2 * (xs @ r["wu"].abs().t())
        eh = 1.13 * ea * b.abs() + act64(act, a).abs() * (eb + 2 ** -19 * b.abs()) + 2 ** -19 * h.abs()
        lo, hi = e4m3_64(h - eh, 1, 128), e4m3_64(h + eh, 1, 128)
        step = torch.maximum((lo - hq).abs(), (hi - hq).abs())
        amax = h.abs().reshape(M, F)
        for k0 in range(0, F, 128):                            # a block whose maximum is near a border of its scale: every value may move by a step
            blk, err = amax[:, k0:k0 + 128].amax(1), eh[:, k0:k0 + 128].amax(1)
            near = torch.ceil(torch.log2((blk + err).clamp(min=1e-300) / 448)) != torch.ceil(torch.log2((blk - err).clamp(min=1e-300) / 448))
            step[near, k0:k0 + 128] = torch.maximum(step[near, k0:k0 + 128], hq[near, k0:k0 + 128].abs() * 2 ** -3 + blk[near, None] * 2 ** -15)
        lim = step @ wd.abs().t() + (F + 8) * E * (hq.abs() @ wd.abs().t()) + 2 * E * ref.abs()
        within(y, ref, lim, f"y ({act})")
        # bfloat16: projections and result from the 8-bit pipe (its error above), so more of h may move by a step; which, the pipe decides:
        # every value of h is given a step's chance in proportion to its error over the step, summed in squares (independent), 6 deviations
        got = B.fp8_gated_feed_forward(t["x"], P, activation=act, out_dtype=BF)
        if M <= 32:
            within(got, ref, lim + U * ref.abs() * 1.01, f"bf16 y ({act})")
            continue
        pipe = math.sqrt(K) * 2.0 ** -15
        pa, pb = (pipe * r["x"].abs().amax(1, keepdim=True) * r[k].abs().amax(1) for k in ("wg", "wu"))
        eh = 1.13 * pa * b.abs() + act64(act, a).abs() * pb + eh
        st = torch.maximum(hq.abs() * 2 ** -3, h.abs().amax(1, keepdim=True) * 2.0 ** -15)
        var = (st * torch.minimum(st, eh) + 1e-300) @ (wd * wd).t()
        pipe = 4 * pipe * math.sqrt(F / K) * hq.abs().amax(1, keepdim=True) * wd.abs().amax(1)
        frob(got, ref, (var.sqrt().norm() * 3 + pipe.norm()).item() / ref.norm().item() + U, f"bf16 y ({act})")


def test_fp8_non_finite_rows_stay_alone(dev):
    for M in (20, 200):
        t = ffn_case(dev, M, 200, 96, 40, BF, True, seed=5)
        P, W = B.fp8_gated_weights(t["wg"], t["wu"], t["wd"], t["bg"], t["bu"], t["bd"]), B.fp8_weight(t["wg"])
        x = t["x"].clone()
        x[3, 71], x[7, 0] = float("nan"), float("inf")
        keep = [i for i in range(M) if i not in (3, 7)]
        for f in (lambda z: B.fp8_linear(z, W), lambda z: B.fp8_gated_feed_forward(z, P)):
            base, y = f(t["x"]), f(x)
            assert torch.equal(y[keep], base[keep]) and y[3].isnan().all() and y[7].isnan().all()


def test_fp8_graph_replays_and_empty(dev):
    t = ffn_case(dev, 100, 200, 264, 40, BF, True, seed=5)
    P = B.fp8_gated_weights(t["wg"], t["wu"], t["wd"], t["bg"], t["bu"], t["bd"])
    x = t["x"].clone()
    B.fp8_gated_feed_forward(x, P)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = B.fp8_gated_feed_forward(x, P)
    for rep in range(4):
        x.copy_(rnd(dev, 100, 200, seed=60 + rep, dtype=BF))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, B.fp8_gated_feed_forward(x.clone(), P)), rep
    assert B.fp8_gated_feed_forward(x[:0], P).shape == (0, 40) and B.fp8_linear(x[:0], P.gate).shape == (0, 264)


def test_block_run_together(dev):
    """Two residual blocks as they are used: norm, feed-forward, norm + gate + residual + next norm; trained in float32 against
    64-bit gradients, and evaluated in 8 bits."""
    M, G, H, F = 192, 48, 72, 136
    p = {}
    for i in range(2):
        t = ffn_case(dev, 1, H, F, H, F32, True, seed=200 + 20 * i)
        p.update({f"{k}{i}": t[k] for k in ("wg", "wu", "wd", "bg", "bu", "bd")})
        p[f"post{i}"] = 1 + rnd(dev, H, seed=300 + i, scale=0.1)
    for i in range(3):
        p[f"pre{i}"] = 1 + rnd(dev, H, seed=310 + i, scale=0.1)
    p["x"], p["gate"] = rnd(dev, M, H, seed=320), 1 + rnd(dev, G, H, seed=321, scale=0.2)

    def run(q, ffn, norm):
        stream, n = norm(q["x"], None, None, 1.0, None, q["pre0"])
        for i in range(2):
            stream, n = norm(stream, ffn(n, i), q["gate"], 0.5, q[f"post{i}"], q[f"pre{i + 1}"])
        return n

    def own(q):
        def norm(res, y, gate, s, w1, w2):
            if y is None:
                return B.norm_gate_residual(res, pre_norm="rms", pre_weight=w2)
            return B.norm_gate_residual(res, y, gate=gate, scale=s, post_norm="rms", post_weight=w1, pre_norm="rms", pre_weight=w2)
        return run(q, lambda n, i: B.gated_feed_forward(n, *[q[f"{k}{i}"] for k in ("wg", "wu", "wd", "bg", "bu", "bd")]), norm)

    def ref(q):
        def norm(res, y, gate, s, w1, w2):
            v = res if y is None else res + s * gate.repeat(M // G, 1) * norm64(y, "rms", w1, None, 1e-6)
            return v, norm64(v, "rms", w2, None, 1e-6)
        return run(q, lambda n, i: ffn64({"x": n, **{k: q[f"{k}{i}"] for k in ("wg", "wu", "wd", "bg", "bu", "bd")}}, "silu")[3], norm)

    leaves = {k: v.clone().requires_grad_(True) for k, v in p.items()}
    refs = {k: v.double().requires_grad_(True) for k, v in p.items()}
    d = rnd(dev, M, H, seed=330)
    y, yr = own(leaves), ref(refs)
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), d)))
    want = dict(zip(refs, torch.autograd.grad(yr, list(refs.values()), d.double())))
    depth = 2 * (2 * (4 + math.sqrt(H)) + 4 + math.sqrt(F) + 16) * E
    frob(y, yr.detach(), depth, "two blocks")
    for k in got:
        frob(got[k], want[k], 8 * depth + 4 * E * math.sqrt(M), f"d{k}")
    with torch.no_grad():
        packed = [B.fp8_gated_weights(*[p[f"{k}{i}"] for k in ("wg", "wu", "wd", "bg", "bu", "bd")]) for i in range(2)]
        stream, n = B.norm_gate_residual(p["x"], pre_weight=p["pre0"])
        for i in range(2):
            stream, n = B.norm_gate_residual(stream, B.fp8_gated_feed_forward(n, packed[i]), gate=p["gate"], scale=0.5, post_norm="rms", post_weight=p[f"post{i}"], pre_weight=p[f"pre{i + 1}"])
    # e4m3 rounds to 2^-4 of a value (rms about a third of it): five roundings meet in a unit's result, damped by the residual sum
    frob(n, yr.detach(), 2 * math.sqrt(5) * 2.0 ** -4, "two blocks in 8 bits")


def test_norm_normed_dtype(dev):
    """A bfloat16 normed of a float32 residual without a branch: the float32 result rounded once; gradients from a bfloat16 one."""
    M, N = 37, 72
    x, w = rnd(dev, M, N, seed=91).requires_grad_(), rnd(dev, N, seed=92).requires_grad_()
    s, n = B.norm_gate_residual(x, pre_weight=w, normed_dtype=BF)
    assert s is x and n.dtype == BF
    assert torch.equal(n, B.norm_gate_residual(x, pre_weight=w)[1].to(BF))
    d = rnd(dev, M, N, seed=93, dtype=BF)
    got = torch.autograd.grad(n, [x, w], d)
    want = torch.autograd.grad(B.norm_gate_residual(x, pre_weight=w)[1], [x, w], d.float())
    for g, r in zip(got, want):
        assert torch.equal(g, r)


# ---- the gated layers of a network -----------------------------------------------------------------------------------------
class Cdim:
    def __init__(self, c):
        self.cond_dim = c


def conditions(prec):
    """Width of the conditions: bf16 mode wants network inputs of whole groups of four columns."""
    return 4 if prec == "bf16" else 5


def gated_model(dev, prec, hidden, gated, bn=True, eval_fp8=False, act="silu", width=40):
    from behavio_temporal_vae_amd.vae_models import CVAE
    common = dict(num_neurons=width, num_hidden_layers=hidden, dropout=False, batch_normalization=bn, gated_layers=gated, gated_hidden=72, gated_activation=act,
                  gated_eval_fp8=eval_fp8)
    cfg = {"latent_dim": 8, "gemm_precision": prec, "distribution_dict": {
        "posterior": {"dist_type": "normal", "sigma_lim": 0.05, "mu_upper_lim": 5.0, "mu_lower_lim": -5.0, **common},
        "likelihood": {"dist_type": "normal", "sigma_lim": 0.05, "mu_upper_lim": 5.0, "mu_lower_lim": -5.0, **common}}}
    torch.manual_seed(17)
    return CVAE(input_dim=24, conditioner=Cdim(conditions(prec)), **cfg).to(dev)


def net64(net, x, train, wide=None):
    """A network's raw head outputs in 64 bits from its parameters ``wide`` (name -> tensor) by plain formulas."""
    blocks = net.parameterizer.block_dict
    names = {id(p): k for k, p in net.named_parameters()}
    P = lambda p: wide[names[id(p)]]

    def unit(seq, h, residual):
        y = torch.relu(h @ P(seq[0].weight).t() + P(seq[0].bias))
        for m in list(seq)[1:]:
            if isinstance(m, torch.nn.BatchNorm1d):
                mean, var = (y.mean(0), y.var(0, unbiased=False)) if train else (m.running_mean.double(), m.running_var.double())
                y = (y - mean) / torch.sqrt(var + m.eps) * P(m.weight) + P(m.bias)
        return y + h if residual else y

    t = blocks["input"]
    h = unit(t.input_layer, x, False)
    for seq in t.middle_layers:
        h = unit(seq, h, True)
    for g in getattr(t, "gated_layers", []):
        n = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * P(g.norm)
        y = act64(g.activation, n @ P(g.gate.weight).t() + P(g.gate.bias)) * (n @ P(g.up.weight).t() + P(g.up.bias))
        h = h + P(g.scale) * (y @ P(g.down.weight).t() + P(g.down.bias))
    h = unit(t.output_layer, h, False)
    out = {}
    for name in ("mu", "sigma"):
        b = blocks[name]
        v = unit(b.input_layer, h, False)
        out[name] = v @ P(b.output_layer[0].weight).t() + P(b.output_layer[0].bias)
    lo, hi = net.head_specs()["mu"][1:]
    lo2, hi2 = net.head_specs()["sigma"][1:]
    return {"mu": out["mu"].clamp(lo, hi), "sigma": torch.nn.functional.softplus(out["sigma"]).clamp(lo2, hi2)}


# Tolerances of a whole network.  Its products, six to nine of them one behind another, each add the operators' own errors (float32:
# 2^-24 (4 + sqrt(K)) with K <= 72, 13 2^-24) times the amplification of the layers behind, which for these widths and initial weights
# stays under 10, and BatchNorm's division by a column's deviation: float32 modes are held to 2000 2^-24 = 1.2e-4 of a tensor's norm.
# bf16 mode rounds every product's operands (2^-8 relative each, in Frobenius norm sqrt(2) 2^-9 a product at least): 40 2^-8 of the norm
# over all gradients together.
@pytest.mark.parametrize("prec,hidden,gated,bn,act", [("fp32", 1, 1, True, "silu"), ("fp32_split", 0, 2, True, "gelu"), ("fp32_split2", 2, 1, False, "relu"),
                                                      ("bf16", 1, 2, True, "silu")])
@pytest.mark.parametrize("M", [20, 130])
def test_network_with_gated_layers(dev, prec, hidden, gated, bn, act, M):
    """Head outputs and every parameter's gradient of a decoder with gated layers against formulas in 64 bits."""
    m = gated_model(dev, prec, hidden, gated, bn, act=act).train()
    m._check_arena()
    net = m.decoder
    x = rnd(dev, M, 8 + conditions(prec), seed=51).requires_grad_()
    wmu, wsg = rnd(dev, M, 24, seed=52), rnd(dev, M, 24, seed=53)
    try:
        for p in net.parameters():
            p.grad.zero_()
        out = net(x)
        ((out["mu"] * wmu).sum() + (out["sigma"] * wsg).sum()).backward()
        wide = {k: p.detach().double().requires_grad_() for k, p in net.named_parameters()}
        x64 = x.detach().double().requires_grad_()
        ref = net64(net, x64, True, wide)
        ((ref["mu"] * wmu.double()).sum() + (ref["sigma"] * wsg.double()).sum()).backward()
        tol = 40 * U if prec == "bf16" else 2000 * E
        for k in ("mu", "sigma"):
            frob(out[k], ref[k].detach(), tol, k)
        whole = math.sqrt(sum(float(w.grad.norm()) ** 2 for w in wide.values()))
        for k, p in net.named_parameters():
            assert ((p.grad.double() - wide[k].grad).norm().item()) <= tol * whole, k
        frob(x.grad, x64.grad, tol, "input gradient") if prec != "bf16" else None
        assert any("gated_layers" in k for k, _ in net.named_parameters())
    finally:
        nv.set_gemm_precision("fp32")


@pytest.mark.parametrize("prec", ["fp32_split2", "bf16"])
@pytest.mark.parametrize("M", [1, 20, 300])
@pytest.mark.parametrize("fp8", [False, True])
def test_network_with_gated_layers_eval(dev, prec, M, fp8):
    """Eval mode: few rows and many, float32 and bf16, and the 8-bit form (which differs from the plain one by the e4m3 roundings
    of both operands, 2^-4 each, in the branches that the scale 0.1 adds: an order below them)."""
    m = gated_model(dev, prec, 1, 2, eval_fp8=fp8).eval()
    net = m.decoder
    x = rnd(dev, M, 8 + conditions(prec), seed=61)
    try:
        m._check_arena()
        with torch.no_grad():
            out = net(x)
        wide = {k: p.detach().double() for k, p in net.named_parameters()}
        ref = net64(net, x.double(), False, wide)
        tol = 2.0 ** -4 if fp8 else 40 * U if prec == "bf16" else 2000 * E
        for k in ("mu", "sigma"):
            frob(out[k], ref[k], tol, k)
        if fp8:
            for g in net.parameterizer.block_dict["input"].gated_layers:
                g.eval_fp8 = False
            with torch.no_grad():
                plain = net(x)
            assert not torch.equal(plain["mu"], out["mu"])            # the 8-bit form ran
    finally:
        nv.set_gemm_precision("fp32")


@pytest.mark.parametrize("prec", ["fp32_split2", "bf16"])
def test_training_steps_with_gated_layers_captured(dev, monkeypatch, prec):
    """Training steps replayed from captured graphs change the weights bit for bit as eager steps do; a state dict goes round."""
    x, c, eps = rnd(dev, 60, 24, seed=71), rnd(dev, 60, conditions(prec), seed=72), rnd(dev, 2, 60, 8, seed=73)
    runs = []
    try:
        for mode in ("0", "1"):
            monkeypatch.setenv("BTVAE_STEP_GRAPH", mode)
            m = gated_model(dev, prec, 1, 1).train()
            m.train_kwargs = {"num_mc_samples": 2, "beta": 0.8, "gradient_clipping": True, "gradient_clipping_kwargs": {"max_norm": 1.0}}
            opt = m.get_optimizer(lr=1e-3, weight_decay=1e-5)
            for i in range(7):
                out = m._train_step(x, c, opt, eps=eps)
                out["loss"].item()
                (x * 2).sum().item()                                   # eager work between the replays
            runs.append({k: v.detach().clone() for k, v in m.state_dict().items()})
            assert bool(m.__dict__.get("_step_graphs")) == (mode == "1")
        for k, v in runs[0].items():
            assert torch.equal(v, runs[1][k]), k
        fresh = gated_model(dev, prec, 1, 1)
        before = {k: v.clone() for k, v in fresh.state_dict().items()}
        assert any(not torch.equal(before[k], runs[0][k]) for k in before if "gated_layers" in k and "scale" in k)
        fresh.load_state_dict(runs[0])
        m.eval(), fresh.eval()
        z = x[:, :8 + conditions(prec)].contiguous()
        with torch.no_grad():
            assert torch.equal(fresh.decoder(z)["mu"], m.decoder(z)["mu"])
    finally:
        nv.set_gemm_precision("fp32")


def test_gated_layers_argument_checks(dev):
    with pytest.raises(ValueError, match="gated_activation"):
        gated_model(dev, "fp32", 1, 1, act="tanh")


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF, F32), (BF, BF)])
def test_ffn_tape_outs(dev, dtype, out):
    """Gradients written to, and added to, given tensors: the first pass is the tape's own result (rounded once more where that was
    float32), the second one twice that, exactly, in float32.  What does not fit is refused before anything is launched."""
    M, K, F, N = 150, 40, 72, 24
    t = ffn_case(dev, M, K, F, N, dtype, True, seed=31)
    dy = rnd(dev, M, N, seed=33, dtype=dtype)
    args = [t[k] for k in ("x", "wg", "wu", "wd", "bg", "bu", "bd")]
    y, tape = B.gated_feed_forward_tape(*args)
    own = tape.backward(dy)
    outs = [torch.full(a.shape, float("nan"), dtype=out, device=dev) for a in args[1:]]
    got = tape.backward(dy, outs=outs)
    for g, o, w in zip(got[1:], outs, own[1:]):
        assert g is o
        assert torch.equal(o, w) if out == dtype else torch.equal(o.to(dtype), w)
    once = [o.clone() for o in outs]
    tape.backward(dy, outs=outs, accumulate=True)
    for o, w in zip(outs, once):
        if out == F32:
            assert torch.equal(o, 2 * w)
        else:                                      # the sum of a rounded value and an unrounded one, rounded: two roundings of 2^-8
            within(o, 2 * d64(w), (2 * U + U) * 2 * d64(w).abs() + 2.0 ** -130, "accumulated")
    dx = tape.backward(dy, need_weights=False)
    assert dx[1:] == (None,) * 6 and torch.equal(dx[0], own[0])
    bad = lambda i, o: [o if k == i else v for k, v in enumerate(outs)]
    for wrong, error, words in ((outs[:5], ValueError, "six"), (bad(0, None), ValueError, "w_gate is missing"), (bad(2, outs[0]), ValueError, "w_down must have shape"),
                                (bad(1, torch.empty(K, F, dtype=out, device=dev).t()), ValueError, "contiguous"), (bad(3, outs[3].half()), TypeError, "b_gate"),
                                (bad(4, outs[4].to(BF if out == F32 else F32)), TypeError, "one type"), (bad(5, outs[5].cpu()), RuntimeError, "on cpu")):
        with pytest.raises(error, match=words):
            tape.backward(dy, outs=wrong)
    for wrong, error in ((dy.half(), TypeError), (dy[:-1], ValueError), (dy[:, :-1], ValueError), (dy.cpu(), RuntimeError)):
        with pytest.raises(error):
            tape.backward(wrong)
    assert tape.backward(dy, outs=bad(3, None))[4] is None


def test_networks_gradients_accumulate(dev):
    """Two backward passes through a network with gated layers add up in its parameters' gradients, exactly."""
    m = gated_model(dev, "fp32", 1, 1).train()
    m._check_arena()
    net, x, w = m.decoder, rnd(dev, 40, 13, seed=81), rnd(dev, 40, 24, seed=82)
    grads = []
    for passes in (1, 2):
        for p in net.parameters():
            p.grad.zero_()
        for _ in range(passes):
            (net(x)["mu"] * w).sum().backward()
        grads.append({k: p.grad.clone() for k, p in net.named_parameters() if "gated_layers" in k})
    assert grads[0]
    for k, g in grads[0].items():
        assert torch.equal(grads[1][k], 2 * g), k


@pytest.mark.parametrize("planes", [1, 3])
@pytest.mark.parametrize("R,shapes", [(1537, ((104, 203), (203, 53))), (70, ((1, 1), (9, 260))), (0, ((8, 8), (16, 5))), (3000, ((2000, 1000), (130, 40)))])
def test_block_wgrad_pair(dev, planes, R, shapes):
    """Two weight gradients in one call (one launch when both are small, two when not): each as by itself, to float32's accuracy, the
    memory behind the workspace untouched, sums added to what was there."""
    lib = nv.lib()
    dtype = BF if planes == 1 else F32
    mats, jobs, outs, refs = [], [], [], []
    for i, (M, N) in enumerate(shapes):
        a, b = rnd(dev, R, M, seed=101 + i, dtype=dtype), rnd(dev, R, N, seed=111 + i, dtype=dtype)
        A, X = (B._operand(a, planes, 1 << 30), B._operand(b, planes, 1 << 30)) if R else (None, None)
        out = torch.full((M, N), 2.0, device=dev)
        mats += [A, X]
        jobs += [A.ptr() if R else 0, A.ld if R else 0, X.ptr() if R else 0, X.ld if R else 0, out.data_ptr(), M, 0, 0, 0, N, 0, M, N]
        outs.append(out)
        refs.append(2.0 + d64(a).t() @ d64(b))
    need = lib.btvae_block_wgrad_pair_ws(*shapes[0], *shapes[1], R, planes)
    ws = torch.full((need + 64,), 7.0, device=dev)
    nv.call("btvae_block_wgrad_pair", (nv.ctypes.c_longlong * 26)(*jobs), ws.data_ptr(), need, planes, R, 1)
    for o, r, (M, N) in zip(outs, refs, shapes):
        frob(o, r, E * (6 + math.sqrt(max(R, 1))), f"{M} x {N}")
    assert bool((ws[need:] == 7.0).all())
    with pytest.raises(RuntimeError, match="workspace"):
        nv.call("btvae_block_wgrad_pair", (nv.ctypes.c_longlong * 26)(*jobs), ws.data_ptr(), need - 1, planes, R, 1)


@pytest.mark.parametrize("dtype,K", [(F32, 40), (BF, 64), (BF, 40), (BF, 41)])
def test_ffn_saved_tensor_hooks_and_lifetime(dev, dtype, K):
    """Saved tensors that a hook moves (as offloading does) give the same gradients to the last bit; they are let go with the backward pass; a
    second pass over a kept graph repeats the first."""
    M, F, N = 90, 48, 24
    t = ffn_case(dev, M, K, F, N, dtype, True, seed=61)
    dy = rnd(dev, M, N, seed=63, dtype=dtype)
    leaves = [t[k].requires_grad_() for k in ("x", "wg", "wu", "wd", "bg", "bu", "bd")]
    y = B.gated_feed_forward(*leaves)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy)
    moved = []

    def pack(s):
        moved.append(s.numel())
        return s.detach().cpu().clone()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda s: s.to(dev)):
        y2 = B.gated_feed_forward(*leaves)
    junk = [torch.randn(1 << 16, device=dev) for _ in range(8)]         # reuse what the hook let go
    got = torch.autograd.grad(y2, leaves, dy)
    for a, b, c in zip(want, again, got):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert len(moved) == 8 and junk
    x2 = rnd(dev, 4096, 256, seed=64, dtype=dtype).requires_grad_()
    big = [rnd(dev, 512, 256, seed=65, dtype=dtype), rnd(dev, 512, 256, seed=66, dtype=dtype), rnd(dev, 256, 512, seed=67, dtype=dtype)]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y3 = B.gated_feed_forward(x2, *big)
    held = torch.cuda.memory_allocated() - before
    torch.autograd.grad(y3, x2, torch.ones_like(y3))
    assert torch.cuda.memory_allocated() - before <= held - 4096 * 512 * 3   # the kept projections, at least, are gone with y3 alive


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_results_stored_past_l2(out):
    """More than 128 MiB of results, the last tile of rows and of columns ragged: sampled rows (the last among them) against 64 bits.  A result is off by
    its own rounding (bf16: half a step, 2^-8) and by the sums': 2^-16 of the sum of magnitudes on the 8-bit pipe, K 2^-24 in fp32."""
    M, K, N = 70001, 136, 1001
    torch.manual_seed(5)
    x = torch.randn(M, K, device="cuda")
    w = B.fp8_weight(torch.randn(N, K, device="cuda") * K ** -0.5)
    q = B.fp8_quantize(x)
    y = B.fp8_linear(q, w, out_dtype=out)
    rows = torch.cat([torch.arange(0, M, 997, device="cuda"), torch.arange(M - 130, M, device="cuda")])
    a, b = q.dequantize()[rows].double(), w.dequantize().double()
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -16 * size if out == torch.bfloat16 else 2.0 ** -24 * want.abs() + K * 2.0 ** -24 * size
    assert ((y[rows].double() - want).abs() <= bound).all()


@pytest.mark.gpu
def test_unit_whose_results_pass_l2():
    """A bf16 unit with more than 128 MiB of h and of projection gradients, ragged in rows and columns, both ways against the same unit on 24,577 of
    its rows, too few for that and enough that no reduction is split: y and dx of a row depend on that row alone, so they are equal."""
    M, K, F, m = 68001, 64, 1010, 24577
    torch.manual_seed(6)
    make = lambda *s: torch.randn(*s, device="cuda").bfloat16()
    x, dy, wg, wu, wd = make(M, K), make(M, 64), make(F, K) * 0.125, make(F, K) * 0.125, make(64, F) * 0.03
    y, tape = B.gated_feed_forward_tape(x, wg, wu, wd)
    dx = tape.backward(dy)[0]
    y2, tape2 = B.gated_feed_forward_tape(x[-m:].contiguous(), wg, wu, wd)
    dx2 = tape2.backward(dy[-m:].contiguous())[0]
    assert torch.equal(y[-m:], y2) and torch.equal(dx[-m:], dx2)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
def test_norm_gradients_of_no_rows(dev, dtype):
    """A batch without rows: the gradients of what its rows would share, gate rows and channel scale among them, are zeros, whatever the allocator's
    memory held before."""
    N, G = 40, 3
    w = lambda: torch.ones(N, device=dev, requires_grad=True)
    none = torch.empty(0, N, dtype=dtype, device=dev)
    gate = torch.ones(G, N, dtype=dtype, device=dev, requires_grad=True)
    shared = [gate, w(), w(), w(), w(), w()]
    stream, normed = B.norm_gate_residual(none, none, gate=gate, scale=shared[1], post_norm="layer", post_weight=shared[2], post_bias=shared[3], pre_norm="layer",
                                          pre_weight=shared[4], pre_bias=shared[5])
    junk = [torch.full((G, N), float("nan"), dtype=dtype, device=dev) for _ in range(64)] + [torch.full((N,), float("nan"), device=dev) for _ in range(64)]
    del junk
    for t, g in zip(shared, torch.autograd.grad(stream.sum() + normed.sum(), shared)):
        assert g.shape == t.shape and torch.equal(g, torch.zeros_like(t))
    tape = B.norm_gate_residual_tape(none, none, gate=gate.detach())[2]
    junk = [torch.full((G, N), float("nan"), dtype=dtype, device=dev) for _ in range(64)]
    del junk
    assert torch.equal(tape.backward(none, none)[2], torch.zeros_like(gate))


@pytest.mark.parametrize("prec", ["fp32_split2", "bf16"])
@pytest.mark.parametrize("M", [20, 130])
def test_gated_layers_of_a_training_network_without_gradients(dev, prec, M):
    """A network in training mode has one forward pass: under no_grad it gives the head outputs and the BatchNorm statistics of the pass that
    gradients are taken of, to the last bit; ``gated_eval_fp8`` changes neither, and changes the outputs in eval mode."""
    runs = []
    try:
        for fp8, grad in ((False, True), (True, True), (True, False)):
            m = gated_model(dev, prec, 1, 1, eval_fp8=fp8).train()
            m._check_arena()
            x = rnd(dev, M, 8 + conditions(prec), seed=91)
            with torch.set_grad_enabled(grad):
                out = m.decoder(x)
            runs.append(({k: v.detach().clone() for k, v in out.items()}, {k: v.clone() for k, v in m.decoder.state_dict().items() if "running" in k}))
        assert runs[0][1]
        for got in runs[1:]:
            for a, b in zip(runs[0], got):
                for k in a:
                    assert torch.equal(a[k], b[k]), k
    finally:
        nv.set_gemm_precision("fp32")


def test_norm_of_more_rows_than_half_the_numbers(dev):
    """2^30 + 3 rows of one column: the statistics' four rows lie further apart than 32-bit indices reach.  The first, some middle and the last rows, both
    ways, against 64 bits: a dozen float32 roundings (the bound of 16 2^-24 of what is added), each result rounded once, the stream's own rounding in front of its
    norm's gradient (which the backward pass recomputes unrounded)."""
    M, eps = 2 ** 30 + 3, 1.0
    need = 20 * 2 * M + 16 * M
    free = torch.cuda.mem_get_info()[0]
    assert free > need, f"{need >> 30} GiB of device memory are needed, {free >> 30} are free"
    torch.cuda.empty_cache()
    base = torch.arange(M, dtype=torch.int32, device=dev)

    def values(k):                                             # (bf16 holds them: 7 bits and a sign)
        v = torch.empty(M, 1, dtype=BF, device=dev)
        v[:, 0] = (base + k) % 251 - 125
        return v.mul_(2.0 ** -5)

    res, branch = values(0), values(77)
    stream, normed, tape = B.norm_gate_residual_tape(res, branch, scale=0.5, post_norm="rms", pre_norm="rms", eps=eps)
    dv, dn = values(13), values(101)
    dres, dbranch = tape.backward(dv, dn, need=(True, True) + (False,) * 6)[:2]
    at = torch.cat([torch.arange(0, 300), torch.arange(M // 2 - 150, M // 2 + 150), torch.arange(M - 300, M)]).to(dev)
    r, y = (t[at].double().requires_grad_(True) for t in (res, branch))
    norm = lambda t: t / torch.sqrt(t * t + eps)
    rv = r + 0.5 * norm(y)
    rn = norm(rv)
    gr, gy = torch.autograd.grad([rv, rn], [r, y], [dv[at].double(), dn[at].double()])
    f = 16 * E
    within(stream[at], rv.detach(), U * rv.detach().abs() + f * (r.detach().abs() + 1), "stream")
    within(normed[at], rn.detach(), U * rn.detach().abs() + 4 * f, "normed")
    size = dv[at].double().abs() + dn[at].double().abs()
    within(dres[at], gr, U * gr.abs() + 4 * f * size, "d residual")
    within(dbranch[at], gy, U * gy.abs() + 4 * f * size, "d branch")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M", [5, 60])
def test_ffn_activation_of_large_values(dev, M, act):
    """Gate pre-activations up to the largest finite magnitudes, float32: silu and gelu are 0 (their slope too) far below zero, the identity (slope 1) far above.
    One up projection of 1 and a down weight of 1 hand act(a) and act'(a) out as they are: a product of one pair of values, exact but for three pieces' last bits.
    Bounds: eight float32 roundings of the value, and what a sigmoid below the smallest normal number, 2^-126, loses: that times |a|, which is at most 104 before
    e^a is no number at all."""
    big = [88.0, 89.5, 1e2, 1e4, 1e10, 1e20, 1e30, 1e35, 1e37, 3e38]
    vals = torch.tensor([-v for v in big] + big + [0.0, 1.0, -1.0, -20.0, 20.0] * 2 + [-87.0, 87.0] * 10 + [0.5] * 10, device=dev)[:, None]
    vals = vals[:M] if M < 10 else vals
    one = torch.ones(1, 1, device=dev)
    zero, bu = torch.zeros(1, 1, device=dev), torch.ones(1, device=dev)
    leaves = vals.clone().requires_grad_(True)
    with torch.no_grad():
        y = B.gated_feed_forward(vals, one, zero, one, None, bu, None, activation=act)
    yg = B.gated_feed_forward(leaves, one, zero, one, None, bu, None, activation=act)
    g, = torch.autograd.grad(yg.sum(), leaves)
    a = vals.double().requires_grad_(True)
    if act == "silu":
        ref = a / (1 + torch.exp(-a))
    else:
        ref = torch.where(a < 0, 0.5 * a * torch.special.erfc(-a / math.sqrt(2)), a * (1 - 0.5 * torch.special.erfc(a / math.sqrt(2))))
    s = torch.sigmoid(a.detach())
    if act == "silu":
        slope = s * (1 + torch.where(a.detach() > 700, torch.zeros_like(s), a.detach() * torch.sigmoid(-a.detach())))
    else:
        phi = torch.exp(-0.5 * a.detach() ** 2) / math.sqrt(2 * math.pi)
        slope = 0.5 * torch.special.erfc(-a.detach() / math.sqrt(2)) + torch.where(phi == 0, phi, a.detach() * phi)
    ref = ref.detach()
    tiny = 2.0 ** -126 * 104
    # erfc and exp are good to 1.2e-7 of a value of at most 1, the slope's terms are of size 1
    within(y, ref, 8 * E * ref.abs() + 4 * E * (a.detach().abs() < 20) * (a.detach().abs() + 1) + tiny, "act, no graph")
    within(yg, ref, 8 * E * ref.abs() + 4 * E * (a.detach().abs() < 20) * (a.detach().abs() + 1) + tiny, "act")
    within(g, slope, 16 * E + 8 * E * slope.abs(), "slope")


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
def test_ffn_rows_far_apart(dev, dtype):
    """x, the result's gradient and a weight whose rows are 8 MiB and more apart (the last position of every long sequence, a slice of a large buffer): the
    results of the same values side by side, to the last bit."""
    M, K, F, N = 40, 64, 48, 64
    t = ffn_case(dev, M, K, F, N, dtype, True, seed=17)
    dy = rnd(dev, M, N, seed=18, dtype=dtype)
    pitch = 2 ** 22 + 64                                       # elements: past 8 MiB in bf16, 16 MiB in fp32
    room = torch.empty(48, pitch, dtype=dtype, device=dev)     # (F rows, the most of the three)
    want_y, want = ffn_grads(t, "silu", dy)
    with torch.no_grad():
        plain = call_ffn(t, "silu")
    for k in ("x", "dy", "wg", "wd"):
        src = dy if k == "dy" else t[k]
        far = room[:src.shape[0], :src.shape[1]] if src.shape[0] <= 48 else torch.empty(src.shape[0], pitch, dtype=dtype, device=dev)[:, :src.shape[1]]
        far.copy_(src)
        u = t if k == "dy" else {**t, k: far}
        with torch.no_grad():
            assert torch.equal(call_ffn(u, "silu"), plain), k
        y, tape = B.gated_feed_forward_tape(u["x"], u["wg"], u["wu"], u["wd"], u["bg"], u["bu"], u["bd"])
        assert torch.equal(y, want_y), k
        for name, g in zip(("x", "wg", "wu", "wd", "bg", "bu", "bd"), tape.backward(far if k == "dy" else dy)):
            assert torch.equal(g, want[name]), (k, name)


@pytest.mark.parametrize("M", [3, 20])
@pytest.mark.parametrize("big,small", [(1e35, 2.0 ** -20), (2.0 ** -110, 2.0 ** 70)])
def test_fp8_few_rows_of_large_and_small_values(dev, M, big, small):
    """Rows and weights whose scales are far from 1 in opposite directions: a block's sum times one scale alone would leave float32's range, the result does
    not.  Few rows are held to the float32 sums of their definition, as many rows are."""
    K, N = 256, 40
    x, w = rnd(dev, M, K, seed=1).abs() * big, rnd(dev, N, K, seed=2).abs() * small
    xq, wq = e4m3_64(x, 1, 128), e4m3_64(w, 128, 128)
    ref = xq @ wq.t()
    W = B.fp8_weight(w)
    lim = (K + 8) * E * (xq.abs() @ wq.abs().t()) + 2 * E * ref.abs()
    assert ref.abs().max() < 1e38
    within(B.fp8_linear(x, W), ref, lim, "few rows")
    within(B.fp8_linear(x.repeat(40, 1), W)[:M], ref, lim, "many rows")


def test_fp8_bias_that_wants_a_gradient_is_refused(dev):
    """Also beside rows that are quantised already: a result without a graph would drop the bias's gradient in silence."""
    W, bias = B.fp8_weight(rnd(dev, 12, 8)), torch.zeros(12, device=dev, requires_grad=True)
    q = B.fp8_quantize(rnd(dev, 40, 8))
    for x in (q, rnd(dev, 40, 8)):
        with pytest.raises(RuntimeError, match="no backward pass"):
            B.fp8_linear(x, W, bias)
    with torch.no_grad():
        assert B.fp8_linear(q, W, bias).shape == (40, 12)


# ---- kernels that only large sizes, or widths between the others, reach --------------------------------------------------------
@pytest.mark.parametrize("planes", [1, 3])
@pytest.mark.parametrize("M,N,R", [(2050, 1001, 9001), (1062, 203, 66000), (4001, 4100, 1025)])
def test_block_wgrad_large_tiles(dev, planes, M, N, R):
    """Weight gradients that fill the chip with 256 x 256 tiles (tiles times rows / 1024 of 256 and more), ragged in columns and rows, every element against
    64 bits; sums added to what was there."""
    assert -(-M // 256) * -(-N // 256) * (R // 1024) >= 256
    dt = F32 if planes == 3 else BF
    a, b = rnd(dev, R, M, seed=1, dtype=dt), rnd(dev, R, N, seed=2, dtype=dt)
    A, X = B._operand(a, planes, 1 << 30), B._operand(b, planes, 1 << 30)
    need = nv.lib().btvae_block_wgrad_ws(M, N, R, planes)
    ws = torch.full((need + 64,), 7.0, device=dev)
    out = torch.full((M, N), 2.0, device=dev)
    ref = a.double().t() @ b.double()
    for acc in (1, 0):
        nv.call("btvae_block_wgrad", A.ptr(), A.ld, X.ptr(), X.ld, ws.data_ptr(), need, out.data_ptr(), M, None, 0, 0, N, 0, acc, planes, M, N, R)
        frob(out, ref + 2.0 * acc, E * (6 + math.sqrt(R)), "sum" if acc else "result")
        # no element is further off than its own terms allow: R roundings of partial sums below the sum of magnitudes
        within(out, ref + 2.0 * acc, (4 + math.sqrt(R)) * 4 * E * (a.double().abs().t() @ b.double().abs()) / math.sqrt(R) + 8 * E * (ref.abs() + 2), "element")
    assert bool((ws[need:] == 7.0).all())


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
def test_ffn_of_many_tiles(dev, dtype):
    """A unit whose gated products, forward and backward, are several tiles to every workgroup, and whose weight gradients take the large tiles: the result and
    every gradient against 64 bits.  float32: the bounds of the small sizes.  bfloat16: the operands' roundings (h, da, db: 2^-8 each) and the result's own are
    independent from element to element, so a gradient's Frobenius error stays below 2^-8 of its terms' root sum of squares, which for sums of
    independent terms is the result's norm: 2^-8 for each of at most three roundings."""
    M, K, F, N = 8200, 264, 2010, 264
    t = ffn_case(dev, M, K, F, N, dtype, True, seed=23)
    dy = rnd(dev, M, N, seed=24, dtype=dtype)
    y, got = ffn_grads(t, "silu", dy)
    assert -(-M // 128) * -(-F // 128) > 2 * 512 and -(-2 * F // 256) * -(-K // 256) * (M // 1024) >= 256 and -(-N // 256) * -(-F // 256) * (M // 1024) < 256
    ref = ffn_grads64(t, "silu", dy)
    yr = ffn64({k: d64(v) for k, v in t.items()}, "silu")[3]
    if dtype == F32:
        check_ffn_forward(y, t, "silu")
        for k, v in got.items():
            n = {"x": 2 * F}.get(k, M)
            frob(v, ref[k], 3 * E * ((4 + math.sqrt(K)) + (4 + math.sqrt(N)) + (4 + math.sqrt(n))), f"d{k}")
        return
    frob(y, yr, 2 * U, "y")
    for k, v in got.items():
        frob(v, ref[k], 3 * U, f"d{k}")


@pytest.mark.parametrize("case", [(70, 1025, 35, F32, F32, "layer", "rms", True, True), (96, 1032, 32, BF, BF, "layer", "layer", True, True), (40, 1500, 1, F32, BF, "rms", "layer", False, True),
                                  (2500, 2048, 500, BF, BF, "rms", "rms", False, True), (33, 2047, 11, F32, F32, "rms", "rms", False, False), (24, 1288, 0, F32, BF, None, "rms", True, True),
                                  (9, 1096, 3, F32, F32, "layer", None, False, True)], ids=lambda c: f"{c[0]}x{c[1]}g{c[2]}")
def test_norm_of_four_waves_a_row(dev, case):
    """Widths from 1025 to 2048, where a row belongs to four waves: vector and scalar, all types, both kinds of column sums."""
    test_norm_gate_residual(dev, case)


def test_ffn_kept_projections_hold_24_bits(dev):
    """bfloat16: the projections kept for the backward pass are good to 2^-15, not only to a bfloat16 rounding.  With one row that has a gradient the bias
    gradients are that row's da and db as they were before any rounding, in float32: db = dh act(a), da = dh b act'(a), off by 2^-15 of a and of b through
    the functions' slopes (|act''| <= 0.5 for silu), and by float32's sums and the fast exp (2^-18, generously).  A kept bfloat16 would be off by up to 2^-8 of a."""
    M, K, F, N = 40, 64, 300, 24
    t = ffn_case(dev, M, K, F, N, BF, True, seed=29)
    dy = torch.zeros(M, N, dtype=BF, device=dev)
    dy[33] = rnd(dev, N, seed=30, dtype=BF)
    y, tape = B.gated_feed_forward_tape(*[t[k] for k in ("x", "wg", "wu", "wd", "bg", "bu", "bd")])
    outs = [torch.empty(v.shape, device=dev) for v in (t["wg"], t["wu"], t["wd"], t["bg"], t["bu"], t["bd"])]
    tape.backward(dy, outs=outs)
    r = {k: d64(v)[33:34] if k == "x" else d64(v) for k, v in t.items()}
    a, b, _, _ = ffn64(r, "silu")
    a, b = a[0], b[0]
    s = torch.sigmoid(a)
    v, d = a * s, s * (1 + a * (1 - s))
    dh = dy[33].double() @ r["wd"]
    cut, small = 2.0 ** -15, 2.0 ** -18
    sums = (K + 4) * E * (r["x"][0].abs() @ r["wg"].abs().t() + r["x"][0].abs() @ r["wu"].abs().t() + 1) + small
    dhe = (N + 4) * E * (dy[33].double().abs() @ r["wd"].abs()) + small * dh.abs()
    within(outs[4], dh * v, dh.abs() * (cut * a.abs() * 1.1 + 1.1 * sums) + dhe * (v.abs() + 1), "db")
    within(outs[3], dh * b * d, dh.abs() * ((cut * a.abs() * 0.5 + 1.1 * sums) * b.abs() + (cut * b.abs() + sums) * 1.1) + dhe * (1.1 * b.abs() + 1), "da")


@pytest.mark.parametrize("prec,width,bn", [("fp32_split2", 50, True), ("fp32_split2", 41, True), ("fp32_split", 41, False), ("fp32", 50, True), ("bf16", 50, True)])
@pytest.mark.parametrize("M", [20, 200])
def test_network_with_gated_layers_of_odd_widths(dev, prec, width, bn, M):
    """Trunks whose rows are no whole groups of four or eight columns: head outputs and every gradient against 64 bits, bounds as above."""
    m = gated_model(dev, prec, 1, 1, bn, width=width).train()
    m._check_arena()
    net = m.decoder
    x = rnd(dev, M, 8 + conditions(prec), seed=51)
    wmu, wsg = rnd(dev, M, 24, seed=52), rnd(dev, M, 24, seed=53)
    try:
        for p in net.parameters():
            p.grad.zero_()
        out = net(x)
        ((out["mu"] * wmu).sum() + (out["sigma"] * wsg).sum()).backward()
        wide = {k: p.detach().double().requires_grad_() for k, p in net.named_parameters()}
        ref = net64(net, x.double(), True, wide)
        ((ref["mu"] * wmu.double()).sum() + (ref["sigma"] * wsg.double()).sum()).backward()
        tol = 40 * U if prec == "bf16" else 2000 * E
        for k in ("mu", "sigma"):
            frob(out[k], ref[k].detach(), tol, k)
        whole = math.sqrt(sum(float(w.grad.norm()) ** 2 for w in wide.values()))
        for k, p in net.named_parameters():
            assert ((p.grad.double() - wide[k].grad).norm().item()) <= tol * whole, k
    finally:
        nv.set_gemm_precision("fp32")


@pytest.mark.parametrize("N", [3, 60])
def test_scoring_of_a_model_with_gated_layers(dev, N):
    """Importance-weighted log-likelihoods through encoder and decoder with gated layers, few rows and many, against 64 bits.  Both networks' errors
    (2000 2^-24 of a tensor's norm) enter a row's log-density times its residual over the deviation (sums of 24 terms of a few units each): 0.1 of a row's
    terms' size at most is allowed for, relative 2^-10."""
    from behavio_temporal_vae_amd.testing_lib import iw_loglikelihood_device
    K, L, D = 7, 8, 24
    m = gated_model(dev, "fp32_split2", 1, 1).eval()
    x, c, eps = rnd(dev, N, D, seed=1, scale=0.3), rnd(dev, N, conditions("fp32_split2"), seed=2), rnd(dev, K, N, L, seed=3)
    try:
        with torch.no_grad():
            ll, rlls, _ = iw_loglikelihood_device(m, x, c, K, mc_sample_batch_size=4, eps=eps, return_rlls=True)
        wide = lambda net: {k: p.detach().double() for k, p in net.named_parameters()}
        q = net64(m.encoder, torch.cat([x, c], 1).double(), False, wide(m.encoder))
        z = q["mu"] + q["sigma"] * eps.double()
        p = net64(m.decoder, torch.cat([z.reshape(K * N, L), c.double().repeat(K, 1)], 1), False, wide(m.decoder))
        normal = lambda t, mu, sd: (-0.5 * ((t - mu) / sd) ** 2 - torch.log(sd) - 0.5 * math.log(2 * math.pi)).sum(-1)
        r = normal(x.double().repeat(K, 1), p["mu"], p["sigma"]).view(K, N)
        ref = torch.logsumexp(r + normal(z, torch.zeros_like(z), torch.ones_like(z)) - normal(z, q["mu"], q["sigma"]), 0) - math.log(K)
        size = ((x.double().repeat(K, 1) - p["mu"]) / p["sigma"]).pow(2).sum(-1).view(K, N) + 60
        within(rlls, r, size * 2.0 ** -10, "log-densities")
        within(ll, ref, size.amax(0) * 2.0 ** -10, "scores")
    finally:
        nv.set_gemm_precision("fp32")


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_results_under_another_default_type(dev, default):
    """A program that builds its model under torch.set_default_dtype calls the operators under it too: the same results, nothing written past its memory."""
    out = []
    for kind in (F32, default):
        t = {d: ffn_case(dev, M, 136, 264, 72, d, True, seed=41) for M, d in ((9, F32), (10, BF))}
        t |= {(M, d): ffn_case(dev, M, 136, 264, 72, d, True, seed=43) for M in (60,) for d in (F32, BF)}
        n = norm_case(dev, 24, 40, 8, F32, F32, "layer", "rms", True, True, seed=3)
        ups = rnd(dev, 24, 40, seed=5)
        torch.set_default_dtype(kind)
        try:
            got = []
            for c in t.values():
                P, W = B.fp8_gated_weights(c["wg"], c["wu"], c["wd"], c["bg"], c["bu"], c["bd"]), B.fp8_weight(c["wg"])
                y, tape = B.gated_feed_forward_tape(*[c[k] for k in ("x", "wg", "wu", "wd", "bg", "bu", "bd")])
                got += [call_ffn(c, "silu"), y, *tape.backward(y), B.fp8_linear(c["x"], W), B.fp8_linear(c["x"], W, out_dtype=F32), B.fp8_gated_feed_forward(c["x"], P),
                        B.fp8_gated_feed_forward(c["x"], P, out_dtype=F32), W.dequantize(), B.fp8_quantize(c["x"]).dequantize()]
            s, v, tape = B.norm_gate_residual_tape(n["residual"], n["branch"], gate=n["gate"], scale=n["scale"], post_norm="layer", post_weight=n["post_weight"],
                                                   post_bias=n["post_bias"], pre_weight=n["pre_weight"], pre_bias=n["pre_bias"])
            got += [s, v, *tape.backward(ups, ups)]
        finally:
            torch.set_default_dtype(F32)
        out.append(got)
    for a, b in zip(*out):
        assert a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("planes", [1, 3])
@pytest.mark.parametrize("M,N,K", [(9000, 2056, 8), (70000, 72, 24)])
def test_block_product_of_short_reductions(dev, planes, M, N, K):
    """One stage to a tile and several tiles to a workgroup: every copy is for a later tile."""
    dt = F32 if planes == 3 else BF
    a, b, bias = rnd(dev, M, K, seed=1, dtype=dt), rnd(dev, N, K, seed=2, dtype=dt), rnd(dev, N, seed=3)
    A, W = B._operand(a, planes, N), B._operand(b, planes, 1 << 30)
    ref = a.double() @ b.double().t() + bias.double()
    size = a.double().abs() @ b.double().abs().t() + bias.double().abs()
    within(B._product(A, W, bias, torch.empty(M, N, device=dev), planes, M, N, A.width), ref, (K + 4) * E * size, "fp32 result")


@pytest.mark.parametrize("M,K,F,N", [(9000, 8, 2010, 8), (40000, 16, 300, 24)])
def test_ffn_of_short_reductions(dev, M, K, F, N):
    """The same for the gated products both ways: one or two stages to a tile."""
    t = ffn_case(dev, M, K, F, N, F32, True, seed=23)
    dy = rnd(dev, M, N, seed=24)
    y, got = ffn_grads(t, "gelu", dy)
    check_ffn_forward(y, t, "gelu")
    ref = ffn_grads64(t, "gelu", dy)
    for k, v in got.items():
        n = {"x": 2 * F}.get(k, M)
        frob(v, ref[k], 3 * E * ((4 + math.sqrt(K)) + (4 + math.sqrt(N)) + (4 + math.sqrt(n))), f"d{k}")
    b16 = {k: v.to(BF) for k, v in t.items()}
    check_ffn_forward(call_ffn(b16, "gelu"), b16, "gelu")


def test_fp8_linear_of_short_reductions(dev):
    M, K, N = 40000, 8, 600
    x, w = rnd(dev, M, K, seed=1), rnd(dev, N, K, seed=2)
    W = B.fp8_weight(w)
    xq, wq = e4m3_64(x, 1, 128), e4m3_64(w, 128, 128)
    ref = xq @ wq.t()
    lim = (K + 8) * E * (xq.abs() @ wq.abs().t()) + 2 * E * ref.abs()
    within(B.fp8_linear(x, W), ref, lim, "fp32 result")
    pipe = math.sqrt(K) * 2.0 ** -13 * xq.abs().amax(1, keepdim=True) * wq.abs().amax(1)
    within(B.fp8_linear(x, W, out_dtype=BF), ref, lim + pipe + U * ref.abs() * 1.01, "bf16 result")


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
def test_one_dimension_and_the_same_tensor_twice(dev, dtype):
    """A single row without leading dimensions; one tensor in two places, whose gradient is the sum of both places'."""
    K, F = 40, 56
    t = ffn_case(dev, 1, K, F, K, dtype, True, seed=3)
    x = t["x"][0]
    for grad in (False, True):
        y = call_ffn({**t, "x": x.clone().requires_grad_(grad)}, "silu")
        assert y.shape == (K,)
        check_ffn_forward(y[None], t, "silu")
    s, n = B.norm_gate_residual(x, y.detach(), gate=t["bd"], post_norm="rms")
    s2, n2 = B.norm_gate_residual(t["x"], y.detach()[None], gate=t["bd"][None], post_norm="rms")
    assert s.shape == n.shape == (K,) and torch.equal(s, s2[0]) and torch.equal(n, n2[0])
    W = B.fp8_weight(t["wg"])
    assert B.fp8_linear(x, W).shape == (F,) and torch.equal(B.fp8_linear(x, W), B.fp8_linear(t["x"], W)[0])
    for M in (7, 60):
        a, w, wd = (rnd(dev, *sh, seed=i, scale=0.2, dtype=dtype) for i, sh in enumerate(((M, K), (F, K), (K, F))))
        dy = rnd(dev, M, K, seed=5, dtype=dtype)
        wl = w.clone().requires_grad_()
        tied, = torch.autograd.grad(B.gated_feed_forward(a, wl, wl, wd), wl, dy)
        w1, w2 = w.clone().requires_grad_(), w.clone().requires_grad_()
        g1, g2 = torch.autograd.grad(B.gated_feed_forward(a, w1, w2, wd), (w1, w2), dy)
        assert torch.equal(tied, g1 + g2)
        al = a.clone().requires_grad_()
        both, = torch.autograd.grad(B.norm_gate_residual(al, al, post_norm="rms")[1], al, dy)
        a1, a2 = a.clone().requires_grad_(), a.clone().requires_grad_()
        g1, g2 = torch.autograd.grad(B.norm_gate_residual(a1, a2, post_norm="rms")[1], (a1, a2), dy)
        assert torch.equal(both, g1 + g2)


def test_two_threads_and_streams_at_once(dev):
    """Forward and backward passes, norms and 8-bit units from two threads on streams of their own, at the same time: every result is the one of the
    same call alone."""
    import threading
    cases = [(ffn_case(dev, M, 136, 264, 72, d, True, seed=s), rnd(dev, M, 72, seed=s, dtype=d)) for M, d, s in ((300, F32, 1), (300, BF, 2), (9, BF, 3), (2000, F32, 4))]
    packs = [B.fp8_gated_weights(*[t[k] for k in ("wg", "wu", "wd", "bg", "bu", "bd")]) for t, _ in cases]

    def work(t, dy, P):
        y, g = ffn_grads(t, "silu", dy)
        s, n = B.norm_gate_residual(dy, y.detach(), gate=dy[:1], post_norm="rms")
        return [y.detach(), *g.values(), s, n, B.fp8_gated_feed_forward(t["x"], P)]

    alone = [work(*c, P) for c, P in zip(cases, packs)]
    torch.cuda.synchronize()
    errors = []

    def run(first):
        try:
            torch.cuda.set_device(dev)
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for rep in range(6):
                    i = (first + rep) % len(cases)
                    got = work(*cases[i], packs[i])
                    st.synchronize()
                    for a, b in zip(got, alone[i]):
                        assert torch.equal(a, b), (first, rep)
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in (0, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_forms_for_few_rows_are_captured(dev):
    """The forms for up to 32 rows in a graph: replays after new inputs equal the eager results."""
    for dtype in (F32, BF):
        t = ffn_case(dev, 7, 136, 264, 72, dtype, True, seed=5)
        P = B.fp8_gated_weights(t["wg"], t["wu"], t["wd"], t["bg"], t["bu"], t["bd"])
        x = t["x"].clone()

        def step(x):
            y = B.gated_feed_forward(x, t["wg"], t["wu"], t["wd"], t["bg"], t["bu"], t["bd"])
            return [y, *B.norm_gate_residual(y, y, post_norm="layer"), B.fp8_gated_feed_forward(x, P), B.fp8_linear(x, P.gate)]

        step(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(x)
        for rep in range(4):
            x.copy_(rnd(dev, 7, 136, seed=60 + rep, dtype=dtype))
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, step(x.clone())):
                assert torch.equal(a, b), rep


def test_weight_gradients_of_a_unit_whose_results_pass_l2(dev):
    """The weight and bias gradients of a bfloat16 unit with more than 128 MiB of h and of projection gradients against 64 bits: three operand roundings of
    2^-8 at most, independent from element to element (the bound of a unit of many tiles)."""
    M, K, F, N = 68001, 64, 1010, 64
    t = ffn_case(dev, M, K, F, N, BF, True, seed=47)
    dy = rnd(dev, M, N, seed=48, dtype=BF)
    y, tape = B.gated_feed_forward_tape(*[t[k] for k in ("x", "wg", "wu", "wd", "bg", "bu", "bd")])
    got = dict(zip(("x", "wg", "wu", "wd", "bg", "bu", "bd"), tape.backward(dy)))
    ref = ffn_grads64(t, "silu", dy)
    for k, v in got.items():
        frob(v, ref[k], 3 * U, f"d{k}")
