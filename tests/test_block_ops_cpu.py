"""What the gated residual block's operators refuse, without a GPU: every case ends in an exception (Python) or a non-zero status
with a message (C entry points) before anything could be launched."""
import ctypes

import pytest
import torch

from behavio_temporal_vae_amd import _native as nv
from behavio_temporal_vae_amd import block_ops as B

BF = torch.bfloat16
M, K, F, N = 5, 8, 12, 6


def ffn(**kw):
    t = dict(x=torch.zeros(M, K), w_gate=torch.zeros(F, K), w_up=torch.zeros(F, K), w_down=torch.zeros(N, F), b_gate=None, b_up=None, b_down=None)
    act = kw.pop("activation", "silu")
    t.update(kw)
    return lambda fn: fn(*t.values(), activation=act)


@pytest.mark.parametrize("fn", [B.gated_feed_forward, B.gated_feed_forward_tape])
@pytest.mark.parametrize("call,error,words", [
    (ffn(), RuntimeError, "MI355X only"),
    (ffn(activation="tanh"), ValueError, "unknown activation"),
    (ffn(activation=["silu"]), ValueError, "unknown activation"),
    (ffn(x=[[0.0]]), TypeError, "x must be a tensor"),
    (ffn(x=torch.zeros(M, K, dtype=torch.float16)), TypeError, "x must be float32 or bfloat16"),
    (ffn(x=torch.zeros(M, K, dtype=torch.float64)), TypeError, "x must be"),
    (ffn(x=torch.tensor(1.0)), ValueError, "at least one dimension"),
    (ffn(x=torch.zeros(M, 0), w_gate=torch.zeros(F, 0), w_up=torch.zeros(F, 0)), ValueError, "no columns"),
    (ffn(x=torch.zeros(1, K).expand(2 ** 31 - 2 ** 20, K)), ValueError, "too large"),
    (ffn(x=torch.zeros(M, K + 1)), ValueError, "w_gate must have shape"),
    (ffn(x=torch.zeros(M, K, dtype=BF)), TypeError, "w_gate must be bfloat16"),
    (ffn(w_gate=torch.zeros(0, K), w_up=torch.zeros(0, K), w_down=torch.zeros(N, 0)), ValueError, "w_gate must be a matrix"),
    (ffn(w_gate=torch.zeros(F)), ValueError, "w_gate must be a matrix"),
    (ffn(w_up=torch.zeros(F + 1, K)), ValueError, "w_up must have shape"),
    (ffn(w_down=torch.zeros(N, F + 1)), ValueError, "w_down must have shape"),
    (ffn(w_down=torch.zeros(0, F)), ValueError, "w_down must be a matrix"),
    (ffn(w_down=torch.zeros(N, F, dtype=BF)), TypeError, "w_down must be float32"),
    (ffn(w_up=torch.zeros(F, K, device="meta")), RuntimeError, "w_up is on meta"),
    (ffn(b_gate=torch.zeros(F + 1)), ValueError, "b_gate must have shape"),
    (ffn(b_up=torch.zeros(1, F)), ValueError, "b_up must have shape"),
    (ffn(b_down=torch.zeros(N, dtype=BF)), TypeError, "b_down must be float32"),
    (ffn(x=torch.zeros(M, K, requires_grad=True)), RuntimeError, "MI355X only"),
])
def test_ffn_refusals(fn, call, error, words):
    with pytest.raises(error, match=words):
        call(fn)


def norm(**kw):
    t = dict(residual=torch.zeros(M, N), branch=torch.zeros(M, N))
    t.update(kw)
    return lambda fn: fn(**t)


@pytest.mark.parametrize("fn", [B.norm_gate_residual, B.norm_gate_residual_tape])
@pytest.mark.parametrize("call,error,words", [
    (norm(), RuntimeError, "MI355X only"),
    (norm(post_norm="batch"), ValueError, "unknown norm"),
    (norm(pre_norm=3), ValueError, "unknown norm"),
    (norm(residual=torch.zeros(M, N, dtype=torch.float16)), TypeError, "residual must be"),
    (norm(residual=torch.zeros(M, N, dtype=BF)), TypeError, "bfloat16 residual needs a bfloat16 branch"),
    (norm(residual=torch.zeros(M, 0), branch=torch.zeros(M, 0)), ValueError, "no columns"),
    (norm(residual=torch.zeros(1, 8193), branch=torch.zeros(1, 8193)), ValueError, "up to 8192 columns"),
    (norm(eps=-1.0), ValueError, "eps"),
    (norm(eps=float("nan")), ValueError, "eps"),
    (norm(branch=torch.zeros(M, N + 1)), ValueError, "branch must have shape"),
    (norm(branch=torch.zeros(M + 1, N)), ValueError, "branch must have shape"),
    (norm(branch=None, scale=2.0), ValueError, "need a branch"),
    (norm(branch=None, gate=torch.zeros(1, N)), ValueError, "need a branch"),
    (norm(branch=None, post_norm="rms"), ValueError, "need a branch"),
    (norm(branch=None, pre_norm=None), ValueError, "nothing to compute"),
    (norm(gate=torch.zeros(2, N)), ValueError, "a multiple of G"),
    (norm(gate=torch.zeros(0, N)), ValueError, "a multiple of G"),
    (norm(gate=torch.zeros(M, N - 1)), ValueError, "gate must be"),
    (norm(gate=torch.zeros(M, N, dtype=BF)), TypeError, "gate must be float32"),
    (norm(scale=torch.zeros(N + 1)), ValueError, "scale must have shape"),
    (norm(scale=torch.zeros(N, dtype=BF)), TypeError, "scale must be float32"),
    (norm(post_weight=torch.ones(N)), ValueError, "need a post norm"),
    (norm(pre_norm=None, pre_bias=torch.ones(N)), ValueError, "need a pre norm"),
    (norm(pre_weight=torch.ones(N - 1)), ValueError, "pre_weight must have shape"),
    (norm(post_norm="layer", post_bias=torch.ones(N, dtype=BF)), TypeError, "post_bias must be float32"),
    (norm(normed_dtype=BF), TypeError, "normed_dtype must be float32"),
    (norm(branch=None, normed_dtype=torch.float16), TypeError, "normed_dtype must be float32 or bfloat16"),
    (norm(residual=torch.zeros(M, N, dtype=BF), branch=None, normed_dtype=torch.float32), TypeError, "normed_dtype must be bfloat16"),
    (norm(branch=torch.zeros(M, N, device="meta")), RuntimeError, "branch is on meta"),
])
def test_norm_refusals(fn, call, error, words):
    with pytest.raises(error, match=words):
        call(fn)


def weight(n=N, k=K):
    kb = -(-k // 128)
    return B.Fp8Weight(torch.zeros(n, kb * 128, dtype=torch.uint8), torch.zeros(-(-n // 128), 4 * (-(-kb // 4)), dtype=torch.uint8), (n, k))


@pytest.mark.parametrize("call,error,words", [
    (lambda: B.fp8_quantize(torch.zeros(M, K)), RuntimeError, "MI355X only"),
    (lambda: B.fp8_quantize(torch.zeros(M, K, dtype=torch.float16)), TypeError, "x must be"),
    (lambda: B.fp8_quantize(torch.zeros(M, 0)), ValueError, "no columns"),
    (lambda: B.fp8_quantize(torch.zeros(M, K, requires_grad=True)), RuntimeError, "no backward pass"),
    (lambda: B.fp8_weight(torch.zeros(N, K)), RuntimeError, "MI355X only"),
    (lambda: B.fp8_weight(torch.zeros(N)), ValueError, "must be a matrix"),
    (lambda: B.fp8_weight(torch.zeros(0, K)), ValueError, "must be a matrix"),
    (lambda: B.fp8_weight(torch.zeros(N, K, dtype=torch.int8)), TypeError, "the weight must be"),
    (lambda: B.fp8_linear(torch.zeros(M, K), torch.zeros(N, K)), TypeError, "fp8_weight"),
    (lambda: B.fp8_linear(torch.zeros(M, K + 1), weight()), ValueError, "x must have 8 columns"),
    (lambda: B.fp8_linear(torch.tensor(0.0), weight()), ValueError, "x must have 8 columns"),
    (lambda: B.fp8_linear(weight(), weight()), TypeError, "x must be a tensor"),
    (lambda: B.fp8_linear(torch.zeros(M, K), weight(), torch.zeros(N + 1)), ValueError, "bias must have shape"),
    (lambda: B.fp8_linear(torch.zeros(M, K), weight(), torch.zeros(N, requires_grad=True)), RuntimeError, "no backward pass"),
    (lambda: B.fp8_linear(torch.zeros(M, K, requires_grad=True), weight()), RuntimeError, "no backward pass"),
    (lambda: B.fp8_linear(torch.zeros(M, K), weight(), out_dtype=torch.float16), TypeError, "out_dtype"),
    (lambda: B.fp8_linear(torch.zeros(M, K, device="meta"), weight()), RuntimeError, "the weight is on cpu"),
    (lambda: B.fp8_linear(torch.zeros(M, K), weight()), RuntimeError, "MI355X only"),
    (lambda: B.fp8_gated_weights(torch.zeros(F, K), torch.zeros(F, K), torch.zeros(N, F)), RuntimeError, "MI355X only"),
    (lambda: B.fp8_gated_feed_forward(torch.zeros(M, K), weight()), TypeError, "fp8_gated_weights"),
    (lambda: B.fp8_gated_feed_forward(torch.zeros(M, K), gated(), "softplus"), ValueError, "unknown activation"),
    (lambda: B.fp8_gated_feed_forward(torch.zeros(M, K + 1), gated()), ValueError, "x must have 8 columns"),
    (lambda: B.fp8_gated_feed_forward(torch.zeros(M, K), gated(), out_dtype=torch.int8), TypeError, "out_dtype"),
    (lambda: B.fp8_gated_feed_forward(torch.zeros(M, K, requires_grad=True), gated()), RuntimeError, "no backward pass"),
    (lambda: B.fp8_gated_feed_forward(torch.zeros(M, K), gated()), RuntimeError, "MI355X only"),
])
def test_fp8_refusals(call, error, words):
    with pytest.raises(error, match=words):
        call()


def gated():
    return B.Fp8GatedWeights(weight(F, K), weight(F, K), weight(N, F), None, None, None)


def test_c_entry_points_refuse():
    """Sizes, layouts and workspaces that the kernels do not take come back as a status, with a message."""
    lib = nv.lib()
    a = 1 << 20                                    # an address that is never followed: every call is refused first

    def refused(name, words, *args):
        assert getattr(lib, name)(*args, None) != 0, (name, args)
        assert words in nv.last_error(), (words, nv.last_error())

    def pack(words, **kw):
        j = dict(src=a, bf16=0, ld=64, dst=a, planes=1, dld=128, rows=4, cols=64, dst_cols=64, t=0)
        j.update(kw)
        refused("btvae_block_pack", words, (ctypes.c_longlong * 10)(*j.values()), 1)

    pack("planes", planes=2)
    pack("source", cols=0)
    pack("source", rows=-1)
    pack("source", ld=63)
    pack("source", rows=1 << 31)
    pack("destination", dst_cols=60)
    pack("destination", dst=a + 8)
    pack("destination", dld=120)
    pack("destination", planes=3)                  # a row of 64 columns is 384 bytes
    pack("destination", t=1, rows=80)              # 80 columns do not fit in 64
    pack("null", src=0)
    refused("btvae_block_pack", "four", None, 1)
    refused("btvae_block_pack", "four", (ctypes.c_longlong * 50)(), 5)

    refused("btvae_gated_proj_fwd", "planes", a, 128, a, a, 128, None, None, 0, a, 128, None, 2, 0, 4, 64, 64)
    refused("btvae_gated_proj_fwd", "sizes", a, 128, a, a, 128, None, None, 0, a, 128, None, 1, 0, 4, 64, 60)
    refused("btvae_gated_proj_fwd", "activation", a, 128, a, a, 128, None, None, 0, a, 128, None, 1, 4, 4, 64, 64)
    refused("btvae_gated_proj_fwd", "operand", a, 112, a, a, 128, None, None, 0, a, 128, None, 1, 0, 4, 64, 64)
    refused("btvae_gated_proj_fwd", "layout of H", a, 128, a, a, 128, None, None, 0, a, 112, None, 1, 0, 4, 64, 64)
    refused("btvae_gated_proj_fwd", "kept", a, 128, a, a, 128, None, None, 0, a, 128, a + 8, 1, 0, 4, 64, 64)
    refused("btvae_gated_proj_bwd", "kept", a, 128, a, 128, None, a, 256, None, 1, 0, 4, 64, 64)
    refused("btvae_gated_proj_bwd", "gradients", a, 128, a, 128, a, a, 128, None, 1, 0, 4, 64, 64)
    refused("btvae_block_product", "sizes", a, 128, a, 128, None, 0, a, 60, 0, None, 0, 1, 4, 64, 64)
    refused("btvae_block_product", "operand", a, 128, a + 4, 128, None, 0, a, 64, 0, None, 0, 1, 4, 64, 64)
    need = lib.btvae_block_product_ws(64, 64, 4096, 1)
    assert need > 0
    refused("btvae_block_product", "workspace", a, 8192, a, 8192, None, 0, a, 64, 0, a, need - 1, 1, 64, 64, 4096)
    refused("btvae_block_wgrad", "sizes", a, 128, a, 128, a, 1, a, 65, None, 0, 0, 64, 0, 0, 1, 64, 64, 4)
    refused("btvae_block_wgrad", "row ranges", a, 128, a, 128, a, 1, a, 32, a, 16, 32, 64, 0, 0, 1, 64, 64, 4)
    refused("btvae_block_wgrad", "workspace", a, 128, a, 128, a, 0, a, 64, None, 0, 0, 64, 0, 0, 1, 64, 64, 4)
    refused("btvae_block_colsum", "workspace", a, 0, 64, None, 0, a, 0, 0, 4, 64)
    refused("btvae_block_strip_sums", "sizes", a, -1, 64, a, a, 0, 0)
    rows = lib.btvae_few_rows_max()
    refused("btvae_few_rows", "sizes", a, 0, 64, a, None, 0, 64, None, None, a, 0, 64, 0, rows + 1, 64, 64)
    refused("btvae_few_rows", "types", a, 1, 64, a, None, 0, 64, None, None, a, 0, 64, 0, 1, 64, 64)
    refused("btvae_few_rows", "types", a, 0, 64, a, a, 1, 64, None, None, a, 0, 64, 0, 1, 64, 64)
    refused("btvae_fp8_few_rows", "layout", a, 0, 64, a, a, None, None, 64, 4, None, None, a, 64, 0, 0, 1, 64, 64)
    refused("btvae_fp8_quantize", "layout", a, 0, 64, a, 64, a, 4, 4, 64)
    refused("btvae_fp8_product", "operand", a, 128, a, 3, a, 128, a, 4, None, a, 64, 0, None, 0, 4, 64, 64)
    limit = lib.btvae_norm_max_columns()
    none = [None] * 3

    def nfwd(words, M=4, N=64, types=0, post=0, pre=1, eps=1e-6, branch=a, gate=None, G=0, out=a, normed=a):
        refused("btvae_norm_gate_residual_fwd", words, a, branch, gate, G, 1.0, None, *none, None, post, pre, eps, out, normed, None, types, M, N)

    nfwd("columns", N=limit + 1)
    nfwd("columns", N=0)
    nfwd("rows", M=2 ** 31 - 2 ** 20)
    nfwd("bf16 branch", types=1)
    nfwd("bad norm", post=3)
    nfwd("bad norm", eps=-1.0)
    nfwd("outputs", out=None)
    nfwd("outputs", normed=None)
    nfwd("gate rows", gate=a, G=3)


def test_workspace_sizes_of_nothing():
    """The sizes of empty (or nonsensical) problems are numbers, not crashes."""
    lib = nv.lib()
    for m in (-1, 0, 1):
        for n in (-1, 0, 1):
            for k in (-1, 0, 1, 5000):
                for planes in (1, 3):
                    assert lib.btvae_block_product_ws(m, n, k, planes) >= 0
                    assert lib.btvae_block_wgrad_ws(m, n, k, planes) >= 0 or m * n < 0
                    lib.btvae_block_wgrad_pair_ws(m, n, n, m, k, planes)
                lib.btvae_fp8_product_ws(m, n, k)
            lib.btvae_block_colsum_ws(m, max(n, 0))
            assert lib.btvae_gated_kept_bytes(max(m, 0), max(n, 0), 1) >= 0


def unit(**kw):
    u = dict(x=1 << 20, x16=0, ldx=8, M=5, K=8, F=12, N=6, wg=1 << 20, ldg=8, wu=1 << 20, ldu=8, wd=1 << 20, ldd=12, w16=0, bg=0, bu=0, bd=0, b16=0, planes=3, act=0)
    u.update(kw)
    return (ctypes.c_longlong * 20)(*u.values())


def test_gated_unit_entry_points():
    """Sizes of the whole unit's memory, and what its entry points refuse."""
    lib = nv.lib()
    sizes = (ctypes.c_longlong * 3)()
    assert lib.btvae_gated_unit_bytes(unit(), 1, sizes) == 0
    store, scratch, in_place = sizes
    assert in_place == 0 and store >= 5 * 192 + 5 * 192 + lib.btvae_gated_kept_bytes(5, 12, 3) and scratch > 0
    assert lib.btvae_gated_unit_bytes(unit(), 0, sizes) == 0 and sizes[0] == 0 and sizes[1] > scratch
    assert lib.btvae_gated_unit_bytes(unit(x16=1, w16=1, planes=1, ldd=16, F=16), 1, sizes) == 0 and sizes[2] == 1
    assert lib.btvae_gated_unit_bytes(unit(M=0), 1, sizes) == 0 and sizes[0] == 0
    for bad, words in ((dict(K=0), "sizes"), (dict(M=-1), "sizes"), (dict(F=1 << 31), "sizes"), (dict(M=2 ** 31 - 2 ** 20), "sizes"), (dict(ldx=7), "overlap"), (dict(ldd=11), "overlap"), (dict(planes=2), "planes"),
                       (dict(act=9), "activation"), (dict(wu=0), "null"), (dict(x=0), "null")):
        assert lib.btvae_gated_unit_bytes(unit(**bad), 1, sizes) != 0
        assert words in nv.last_error(), (bad, nv.last_error())
    a = 1 << 20
    assert lib.btvae_gated_unit_fwd(unit(), a, 6, 0, a, store - 1, a, scratch, None) != 0 and "workspace" in nv.last_error()
    assert lib.btvae_gated_unit_fwd(unit(), a, 6, 0, a, store, a, scratch - 1, None) != 0 and "workspace" in nv.last_error()
    g = lambda **kw: (ctypes.c_longlong * 15)(*{**dict(dy=a, dy16=0, lddy=6, dx=a, dwg=a, dwu=a, dwd=a, dbg=0, dbu=0, dbd=0, w16=0, d16=0, b16=0, bd16=0, acc=0), **kw}.values())
    need = lib.btvae_gated_unit_bwd_bytes(unit(), g())
    assert need > 0 and lib.btvae_gated_unit_bwd_bytes(unit(), g(dwg=0, dwu=0, dwd=0, dx=0)) < need
    assert lib.btvae_gated_unit_bwd_bytes(unit(), g(lddy=5)) == -1 and "gradient" in nv.last_error()
    assert lib.btvae_gated_unit_bwd_bytes(unit(), g(dwu=0)) == -1 and "all weights" in nv.last_error()
    assert lib.btvae_gated_unit_bwd(unit(), g(), a, store, a, need - 1, None) != 0 and "workspace" in nv.last_error()
    assert lib.btvae_gated_unit_bwd(unit(), g(), None, 0, a, need, None) != 0 and "workspace" in nv.last_error()


def test_norm_gradient_of_absent_gate_is_refused():
    assert nv.lib().btvae_norm_gate_residual_bwd(None, None, None, None, None, 3, 1.0, None, None, None, None, 0, 1, None, None, None, 1 << 20, None, None, None, None, None, None, 0, 0, 0, 8, None) != 0
    assert "absent gate" in nv.last_error()


def test_ffn_outs_that_share_memory_are_refused():
    """Gradients that one launch writes: tied weights, or slices of one buffer that overlap, would race."""
    w = [torch.zeros(8, 8) for _ in range(3)]
    tape = B.GatedTape(torch.zeros(5, 8), w, [torch.zeros(8)] * 3, None, None, False)
    outs = lambda: [torch.zeros(8, 8) for _ in range(3)] + [torch.zeros(8) for _ in range(3)]
    tape._check_outs(outs())
    whole = torch.zeros(6 * 64)
    tape._check_outs([whole[64 * i:64 * i + 64].view(8, 8) for i in range(3)] + [whole[192 + 8 * i:200 + 8 * i] for i in range(3)])
    for i, j in ((0, 1), (0, 2), (1, 2), (3, 4), (3, 5), (4, 5)):
        o = outs()
        o[j] = o[i]
        with pytest.raises(ValueError, match="share memory"):
            tape._check_outs(o)
    o = outs()
    room = torch.zeros(100)
    o[0], o[1] = room[:64].view(8, 8), room[36:].view(8, 8)
    with pytest.raises(ValueError, match="w_gate and w_up share memory"):
        tape._check_outs(o)
    o = outs()
    o[4] = o[0].view(-1)[60:64].repeat(2)                      # (a copy)
    tape._check_outs(o)
    o[4] = o[0].view(-1)[56:]
    with pytest.raises(ValueError, match="w_gate and b_up share memory"):
        tape._check_outs(o)


def test_fp8_bias_that_wants_a_gradient_is_refused_beside_quantised_rows():
    rows = B.Fp8Rows(torch.zeros(M, 128, dtype=torch.uint8), torch.zeros(M, 4, dtype=torch.uint8), (M, K))
    with pytest.raises(RuntimeError, match="no backward pass"):
        B.fp8_linear(rows, weight(), torch.zeros(N, requires_grad=True))
    with torch.no_grad(), pytest.raises(RuntimeError, match="MI355X only"):
        B.fp8_linear(rows, weight(), torch.zeros(N, requires_grad=True))
    with pytest.raises(TypeError, match="x must be a tensor"):
        B.fp8_linear([1.0], weight(), torch.zeros(N, requires_grad=True))


@pytest.mark.parametrize("config,words", [(dict(gated_layers=-1), "gated_layers"), (dict(gated_layers=1.5), "gated_layers"), (dict(gated_layers="2"), "gated_layers"),
                                          (dict(gated_layers=1, gated_hidden=-4), "gated_hidden"), (dict(gated_layers=1, gated_hidden=2.5), "gated_hidden"),
                                          (dict(gated_layers=1, num_neurons=8193), "up to 8192 neurons"), (dict(gated_layers=2, gated_activation="tanh"), "gated_activation")])
def test_gated_layers_of_a_configuration_are_checked(config, words):
    """What the layers cannot be is refused where the network is built, not in its first forward pass."""
    from behavio_temporal_vae_amd.submodels import GaussianNN, NNBlock
    common = dict(num_neurons=16, num_hidden_layers=0, **config) if "num_neurons" not in config else dict(num_hidden_layers=0, **config)
    with pytest.raises(ValueError, match=words):
        NNBlock(3, 4, **common)
    with pytest.raises(ValueError, match=words):
        GaussianNN(3, 4, **common)


def test_gated_layers_of_a_configuration():
    from behavio_temporal_vae_amd.submodels import NNBlock
    for none in (0, None):
        assert not hasattr(NNBlock(3, 4, num_neurons=16, gated_layers=none), "gated_layers")
    block = NNBlock(3, 4, num_neurons=16, gated_layers=2)
    assert [tuple(g.gate.weight.shape) for g in block.gated_layers] == [(32, 16)] * 2
    assert NNBlock(3, 4, num_neurons=16, gated_layers=1, gated_hidden=5).gated_layers[0].down.weight.shape == (16, 5)


def test_tensors_are_made_with_a_type_of_their_own():
    """Memory that kernels write as float32 is not made with torch's default type, which a program may have set to bfloat16."""
    import ast
    import inspect
    makers = {"empty", "zeros", "ones", "full", "tensor", "arange"}
    for call in ast.walk(ast.parse(inspect.getsource(B))):
        if isinstance(call, ast.Call) and isinstance(call.func, ast.Attribute) and call.func.attr in makers and ast.unparse(call.func.value) == "torch":
            assert any(k.arg == "dtype" for k in call.keywords), ast.unparse(call)
