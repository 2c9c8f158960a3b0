"""Operators of a gated residual block, for networks that want more than Linear+ReLU+BatchNorm units (the reference's
only kind, src/submodels.py:6-35): a gated feed-forward unit, row norms fused with the block's gate, residual scale and
addition, and the 8-bit forms of the products for evaluation.

    a = x Wg^T + bg;  b = x Wu^T + bu;  h = act(a) * b;  y = h Wd^T + bd              ``gated_feed_forward``
    u = post(branch);  stream = residual + scale * gate * u;  normed = pre(stream)    ``norm_gate_residual``
    y = x W^T + b with x and W held as e4m3 and a power-of-two scale a block          ``fp8_linear``, ``fp8_gated_feed_forward``

Matrices are float32 or bfloat16, rows last dimension first; float32 products are float32-accurate (three bf16 planes a
value), bfloat16 products accumulate in float32.  Every call runs on the current stream of the tensors' device, which must
be the current device; scratch memory comes from torch's allocator call by call, so captured graphs and streams share none of it.
Autograd nodes are not captured into graphs: inside one, use the tapes (``gated_feed_forward_tape``,
``norm_gate_residual_tape``), whose ``backward`` launches the gradient kernels directly.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native as nv

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}
NORMS = {None: 0, "none": 0, "rms": 1, "layer": 2}
FP8_BLOCK = 128
_FLOATS = (torch.float32, torch.bfloat16)
MAX_ROWS = 2 ** 31 - 2 ** 21            # row numbers, and those a few tiles or splits past them, are 32 bits


# ------------------------------------------------------------------------------------------------ checks and layout
def _name(table, key, what):
    try:
        return table[key]
    except (KeyError, TypeError):
        raise ValueError(f"unknown {what} {key!r}; choose from {[k for k in table if k is not None]}") from None


def _tensor(t, what, dtypes=_FLOATS):
    if not torch.is_tensor(t):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {str(t.dtype)[6:]}")
    return t


def _matrix(t, what, shape, dtype, device):
    _tensor(t, what, (dtype,))
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must have shape {list(shape)}, got {list(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{what} is on {t.device}, the input on {device}")
    return t


def _vector(t, what, n, dtypes, device):
    if t is None:
        return None
    _tensor(t, what, dtypes)
    if tuple(t.shape) != (n,):
        raise ValueError(f"{what} must have shape [{n}], got {list(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{what} is on {t.device}, the input on {device}")
    return t


def _rows(t, what):
    """[rows, width] view of a tensor whose last dimension is the width; a copy when its rows are not contiguous."""
    if t.dim() < 1:
        raise ValueError(f"{what} needs at least one dimension")
    if t.shape[-1] == 0:
        raise ValueError(f"{what} has no columns")
    rows = 1
    for n in t.shape[:-1]:
        rows *= n
    if rows > MAX_ROWS or t.shape[-1] >= 2 ** 30:
        raise ValueError(f"{what} is too large: {list(t.shape)}")
    if t.dim() != 2:
        t = t.reshape(rows, t.shape[-1])
    if t.stride(1) != 1 or (rows > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _shaped(t, shape):
    return t if t.shape == shape else t.view(shape)          # a view is one more autograd node


def _pitch(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _up(n, m):
    return -(-n // m) * m


def _p(t):
    return None if t is None else t.data_ptr()


def _refuse_capture(what):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: autograd nodes are not captured into a graph; use the operator's tape inside one")


class _Operand:
    """A matrix as the products read it: bf16 (``planes`` 1), or float32 values as three bf16 pieces each, 96 bytes for every 16
    columns (``planes`` 3); ``ld`` bytes to a row, rows on 16 bytes, ``width`` columns of which those beyond the matrix's own are zeros."""
    __slots__ = ("at", "ld", "width", "t")

    def __init__(self, at, ld, width, t=None):
        self.at, self.ld, self.width, self.t = at, ld, width, t      # `t` holds the memory at address `at`

    def ptr(self):
        return self.at


def _operand(t, planes, reads=0) -> _Operand:
    """``t`` laid out as an operand of the products that are called one by one (a whole unit lays out its own), or where it is: a bf16 matrix
    with whole 16-byte pieces that is read against few others."""
    rows, cols = t.shape
    if planes == 1 and t.dtype == torch.bfloat16 and cols % 8 == 0 and _pitch(t) % 8 == 0 and t.data_ptr() % 16 == 0 and reads < 2048 and 2 * _pitch(t) < 2 ** 23:
        return _Operand(t.data_ptr(), 2 * _pitch(t), cols, t)
    ld = _up(cols, 32) * 6 if planes == 3 else _up(cols, 64) * 2
    buf = torch.empty(rows * ld, dtype=torch.uint8, device=t.device)
    nv.call("btvae_block_pack", (ctypes.c_longlong * 10)(t.data_ptr(), t.dtype == torch.bfloat16, _pitch(t), buf.data_ptr(), planes, ld, rows, cols, _up(cols, 32), 0), 1)
    return _Operand(buf.data_ptr(), ld, _up(cols, 8), buf)


def _workspace(floats, device):
    return torch.empty(floats, dtype=torch.float32, device=device) if floats else None


def _product(a: _Operand, b: _Operand, bias, out, planes, M, N, K):
    ws = _workspace(nv.lib().btvae_block_product_ws(M, N, K, planes) if M else 0, out.device)
    nv.call("btvae_block_product", a.ptr(), a.ld, b.ptr(), b.ld, _p(bias), int(bias is not None and bias.dtype == torch.bfloat16),
            _p(out), _pitch(out), int(out.dtype == torch.bfloat16), _p(ws), ws.numel() if ws is not None else 0, planes, M, N, K)
    return out


# ------------------------------------------------------------------------------------------------ gated feed-forward unit
_Numbers = {n: ctypes.c_longlong * n for n in (3, 15, 20)}


def _at(t):
    return 0 if t is None else t.data_ptr()


def _weight_numbers(weights):
    g, u, d = weights
    return (g.data_ptr(), _pitch(g), u.data_ptr(), _pitch(u), d.data_ptr(), _pitch(d), g.dtype == torch.bfloat16)


class GatedTape:
    """What the backward pass of one ``gated_feed_forward`` needs: the inputs, and (``store``) x and h as operands and both projections."""

    def __init__(self, x, weights, biases, unit, store, in_place):
        self.x, self.weights, self.biases, self.unit, self.store, self.in_place = x, weights, biases, unit, store, in_place

    def _check_outs(self, outs):
        if len(outs) != 6:
            raise ValueError(f"outs must be six tensors, got {len(outs)}")
        names = ("w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")
        for o, t, what in zip(outs, (*self.weights, *self.biases), names):
            if t is None or o is None:
                if o is not None or what[0] == "w":
                    raise ValueError(f"outs: {what} " + ("is absent" if t is None else "is missing"))
                continue
            _matrix(_tensor(o, f"outs: {what}"), f"outs: {what}", t.shape, o.dtype, self.x.device)
            if not o.is_contiguous():
                raise ValueError(f"outs: {what} must be contiguous")
        for a, b in ((0, 1), (3, 4)):
            if outs[a] is not None and outs[b] is not None and outs[a].dtype != outs[b].dtype:
                raise TypeError(f"outs: {names[a]} and {names[b]} must be of one type")
        spans = sorted((o.data_ptr(), o.data_ptr() + o.numel() * o.element_size(), what) for o, what in zip(outs, names) if o is not None)
        for (_, end, a), (start, _, b) in zip(spans, spans[1:]):
            if start < end:                                    # one launch writes several of them
                raise ValueError(f"outs: {a} and {b} share memory")

    def backward(self, dy, need_input=True, need_weights=True, outs=None, accumulate=False):
        """Gradients (x, w_gate, w_up, w_down, b_gate, b_up, b_down) for the gradient ``dy`` of the result; entries that are
        not wanted, or belong to an absent bias, are None.  ``outs``: six tensors (float32 or bfloat16, contiguous, None for
        biases that are absent or not wanted; no two in the same memory) that the weights' and biases' gradients are written to, or added to
        with ``accumulate``."""
        x, weights = self.x, self.weights
        dev, (M, K), N = x.device, x.shape, weights[2].shape[0]
        nv.ensure_device(dev)
        dy = _rows(_tensor(dy, "the gradient"), "the gradient")
        _matrix(dy, "the gradient", (M, N), dy.dtype, dev)
        if outs is not None:
            self._check_outs(outs)
        elif need_weights:
            accumulate = False
            outs = [None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format) for t in (*weights, *self.biases)]
        if not need_weights:
            outs = (None,) * 6
        dx = torch.empty(M, K, dtype=x.dtype, device=dev) if need_input else None
        types = [o is not None and o.dtype == torch.bfloat16 for o in outs]
        grads = _Numbers[15](dy.data_ptr(), dy.dtype == torch.bfloat16, max(_pitch(dy), N), _at(dx), *[_at(o) for o in outs],
                             types[0], types[2], types[3] or types[4], types[5], accumulate)
        unit = _Numbers[20](*self.unit)
        unit[7:14] = _weight_numbers(weights)
        if self.in_place and (x.data_ptr(), _pitch(x)) != (unit[0], unit[2]):
            # not the tensor of the forward pass but what a hook on saved tensors made of it: rows that can be read in place again
            moved = torch.empty(M, _up(K, 64), dtype=x.dtype, device=dev)[:, :K]
            moved.copy_(x)
            unit[0], unit[2] = moved.data_ptr(), _pitch(moved)
        lib = nv.lib()
        size = lib.btvae_gated_unit_bwd_bytes(unit, grads)
        if size < 0:
            raise RuntimeError(f"btvae_gated_unit_bwd_bytes: {nv.last_error()}")
        scratch = torch.empty(size, dtype=torch.uint8, device=dev)
        nv.call("btvae_gated_unit_bwd", unit, grads, self.store.data_ptr(), self.store.numel(), scratch.data_ptr(), size)
        return (dx, *outs)


def _ffn_inputs(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation):
    act = _name(ACTIVATIONS, activation, "activation")
    _tensor(x, "x")
    _tensor(w_gate, "w_gate")
    if w_gate.dim() != 2 or w_gate.shape[0] == 0:
        raise ValueError(f"w_gate must be a matrix [hidden, {x.shape[-1] if x.dim() else '?'}], got {list(w_gate.shape)}")
    x2 = _rows(x, "x")
    F, K = w_gate.shape[0], x2.shape[1]
    _matrix(w_gate, "w_gate", (F, K), x.dtype, x.device)
    _matrix(w_up, "w_up", (F, K), x.dtype, x.device)
    _tensor(w_down, "w_down")
    if w_down.dim() != 2 or w_down.shape[0] == 0:
        raise ValueError(f"w_down must be a matrix [out, {F}], got {list(w_down.shape)}")
    _matrix(w_down, "w_down", (w_down.shape[0], F), x.dtype, x.device)
    for b, n, what in ((b_gate, F, "b_gate"), (b_up, F, "b_up"), (b_down, w_down.shape[0], "b_down")):
        _vector(b, what, n, (x.dtype,), x.device)
    nv.ensure_device(x.device)
    weights = [_rows(w, "weight") for w in (w_gate, w_up, w_down)]
    biases = [None if b is None else b.contiguous() for b in (b_gate, b_up, b_down)]
    return x2, weights, biases, act


def _ffn_forward(x2, weights, biases, act, planes, out_dtype, keep):
    """(y [M, N], tape or None): the tile kernels."""
    dev, (M, K), (F, _), N = x2.device, x2.shape, weights[0].shape, weights[2].shape[0]
    bias16 = any(b is not None and b.dtype == torch.bfloat16 for b in biases)
    unit = _Numbers[20](x2.data_ptr(), x2.dtype == torch.bfloat16, _pitch(x2), M, K, F, N, *_weight_numbers(weights), *[_at(b) for b in biases], bias16, planes, act)
    sizes = _Numbers[3]()
    if nv.lib().btvae_gated_unit_bytes(unit, keep, sizes):
        raise RuntimeError(f"btvae_gated_unit_bytes: {nv.last_error()}")
    y = torch.empty(M, N, dtype=out_dtype, device=dev)
    store = torch.empty(sizes[0], dtype=torch.uint8, device=dev) if keep else None
    scratch = torch.empty(sizes[1], dtype=torch.uint8, device=dev)
    nv.call("btvae_gated_unit_fwd", unit, y.data_ptr(), N, out_dtype == torch.bfloat16, _p(store), sizes[0], scratch.data_ptr(), sizes[1])
    return y, GatedTape(x2, weights, biases, unit, store, sizes[2]) if keep else None


def _ffn_few(x2, weights, biases, act):
    w_gate, w_up, w_down = weights
    (M, K), F, N = x2.shape, w_gate.shape[0], w_down.shape[0]
    if _pitch(w_up) != _pitch(w_gate):
        w_gate, w_up = w_gate.contiguous(), w_up.contiguous()
    bf = int(x2.dtype == torch.bfloat16)
    h = torch.empty(M, F, dtype=torch.float32, device=x2.device)         # few rows cost nothing to keep unrounded
    y = torch.empty(M, N, dtype=x2.dtype, device=x2.device)
    nv.call("btvae_few_rows", _p(x2), bf, _pitch(x2), _p(w_gate), _p(w_up), bf, _pitch(w_gate), _p(biases[0]), _p(biases[1]), _p(h), 0, F, act, M, F, K)
    nv.call("btvae_few_rows", _p(h), 0, F, _p(w_down), None, bf, _pitch(w_down), _p(biases[2]), None, _p(y), bf, N, act, M, N, F)
    return y


def _planes(x2):
    """Operands of a unit that keeps what its backward pass needs: float32 accuracy, or bfloat16 for more than a few bfloat16 rows.  Few
    rows are a host's time: there neither h nor the projections' gradients are rounded on their way (error of two rows' gradients
    1.7e-3, the rounding of the results, against 3.3e-3)."""
    return 3 if x2.dtype == torch.float32 or x2.shape[0] <= nv.lib().btvae_few_rows_max() else 1


class _GatedNode(torch.autograd.Function):
    @staticmethod
    def forward(ctx, act, x2, w_gate, w_up, w_down, b_gate, b_up, b_down):
        planes = _planes(x2)
        y, tape = _ffn_forward(x2, [w_gate, w_up, w_down], [b_gate, b_up, b_down], act, planes, x2.dtype, True)
        ctx.save_for_backward(x2, w_gate, w_up, w_down, b_gate, b_up, b_down, tape.store)
        ctx.unit, ctx.in_place = tape.unit, tape.in_place
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_capture("gated_feed_forward")
        x2, w_gate, w_up, w_down, b_gate, b_up, b_down, store = ctx.saved_tensors
        need = ctx.needs_input_grad
        tape = GatedTape(x2, (w_gate, w_up, w_down), (b_gate, b_up, b_down), ctx.unit, store, ctx.in_place)
        return (None, *tape.backward(dy, need_input=need[1], need_weights=any(need[2:])))


def gated_feed_forward(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu"):
    """y = (act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down.

    ``x`` [..., K], ``w_gate`` and ``w_up`` [F, K], ``w_down`` [N, F], all float32 or all bfloat16; result [..., N] of that type.
    ``activation``: "silu", "gelu" (erf form), "relu" or "sigmoid".  Differentiable in every tensor; for up to 32 rows without
    a graph the weights are streamed once (the form for single profiles).  bfloat16: h, and in the backward pass the gradients of
    both projections, are rounded to bfloat16 as operands of the next product, but not for up to 32 rows.  In float32 a row with an infinite input, or
    whose hidden values pass float32's range, may come out as NaN where float32 arithmetic would give an infinity."""
    x2, weights, biases, act = _ffn_inputs(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation)
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w_gate, w_up, w_down, b_gate, b_up, b_down))
    if grad:
        _refuse_capture("gated_feed_forward")
        y = _GatedNode.apply(act, x2, *weights, *biases)
    elif x2.shape[0] <= nv.lib().btvae_few_rows_max():
        y = _ffn_few(x2, weights, biases, act)
    else:
        y, _ = _ffn_forward(x2, weights, biases, act, 3 if x.dtype == torch.float32 else 1, x.dtype, False)
    return _shaped(y, (*x.shape[:-1], y.shape[1]))


@torch.no_grad()
def gated_feed_forward_tape(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu"):
    """``gated_feed_forward`` without autograd: (y, tape), ``tape.backward(dy)`` returns the gradients.  May be captured into a graph."""
    x2, weights, biases, act = _ffn_inputs(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation)
    y, tape = _ffn_forward(x2, weights, biases, act, _planes(x2), x.dtype, True)
    return _shaped(y, (*x.shape[:-1], y.shape[1])), tape


# ------------------------------------------------------------------------------------------------ norms, gate, residual
class NormTape:
    """What the backward pass of one ``norm_gate_residual`` needs."""

    def __init__(self, residual, branch, gate, scale, scale_vec, vectors, post, pre, ntype, stats):
        self.ntype = ntype
        self.residual, self.branch, self.gate, self.scale, self.scale_vec = residual, branch, gate, scale, scale_vec
        self.vectors, self.post, self.pre, self.stats = vectors, post, pre, stats

    def backward(self, d_stream=None, d_normed=None, need=(True,) * 8):
        """Gradients (residual, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias) for the gradients of stream and
        normed (None: zero), rows as [M, N]; entries not wanted or of absent tensors are None."""
        residual, branch, gate = self.residual, self.branch, self.gate
        (M, N), dev = residual.shape, residual.device
        nv.ensure_device(dev)
        if d_stream is not None:
            d_stream = _matrix(d_stream.reshape(M, N), "the gradient of stream", (M, N), residual.dtype, dev).contiguous()
        ntype = self.ntype
        if d_normed is not None:
            if not self.pre:
                raise ValueError("a gradient of normed, which was not asked for")
            d_normed = _matrix(d_normed.reshape(M, N), "the gradient of normed", (M, N), ntype, dev).contiguous()
        like = (residual, branch, gate, self.scale_vec, *self.vectors)
        outs = [torch.empty_like(t) if t is not None and w else None for t, w in zip(like, need)]
        if d_normed is None:
            for i in (6, 7):
                if outs[i] is not None:
                    outs[i].zero_()
        lib, G = nv.lib(), gate.shape[0] if gate is not None else 0
        ws = _workspace(lib.btvae_norm_gate_residual_ws(M, N, G), dev)
        w1, c1, w2, _ = self.vectors
        nv.call("btvae_norm_gate_residual_bwd", _p(d_stream), _p(d_normed), _p(residual), _p(branch), _p(gate), G, self.scale, _p(self.scale_vec),
                _p(w1), _p(c1), _p(w2), self.post, self.pre, _p(self.stats), *[_p(o) for o in outs], _p(ws), ws.numel() if ws is not None else 0,
                _types(residual, ntype), M, N)
        return tuple(outs)


def _types(residual, branch_type):
    return int(residual.dtype == torch.bfloat16) | (2 if branch_type == torch.bfloat16 else 0)


def _norm_forward(residual, branch, gate, scale, scale_vec, vectors, post, pre, eps, ntype, keep):
    (M, N), dev = residual.shape, residual.device
    stream = torch.empty_like(residual) if branch is not None else None
    normed = torch.empty(M, N, dtype=ntype, device=dev) if pre else None
    stats = torch.empty(4 * M, dtype=torch.float32, device=dev) if keep else None
    w1, c1, w2, c2 = vectors
    nv.call("btvae_norm_gate_residual_fwd", _p(residual), _p(branch), _p(gate), gate.shape[0] if gate is not None else 0, scale, _p(scale_vec),
            _p(w1), _p(c1), _p(w2), _p(c2), post, pre, eps, _p(stream), _p(normed), _p(stats), _types(residual, ntype), M, N)
    tape = NormTape(residual, branch, gate, scale, scale_vec, vectors, post, pre, ntype, stats) if keep else None
    return stream, normed, tape


class _NormNode(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scale, post, pre, eps, ntype, residual, branch, gate, scale_vec, *vectors):
        stream, normed, tape = _norm_forward(residual, branch, gate, scale, scale_vec, vectors, post, pre, eps, ntype, True)
        ctx.meta = (scale, post, pre, ntype, tape.stats)
        ctx.has = (branch is not None, pre != 0)
        ctx.save_for_backward(residual, branch, gate, scale_vec, *vectors)
        ctx.set_materialize_grads(False)
        return tuple(t for t in (stream, normed) if t is not None)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        _refuse_capture("norm_gate_residual")
        residual, branch, gate, scale_vec, *vectors = ctx.saved_tensors
        scale, post, pre, ntype, stats = ctx.meta
        grads = list(grads)
        d_stream = grads.pop(0) if ctx.has[0] else None
        d_normed = grads.pop(0) if ctx.has[1] else None
        if d_stream is None and d_normed is None:
            return (None,) * 13
        tape = NormTape(residual, branch, gate, scale, scale_vec, vectors, post, pre, ntype, stats)
        return (None, None, None, None, None, *tape.backward(d_stream, d_normed, need=ctx.needs_input_grad[5:]))


def _norm_inputs(residual, branch, gate, scale, post_norm, post_weight, post_bias, pre_norm, pre_weight, pre_bias, eps, normed_dtype):
    post, pre = _name(NORMS, post_norm, "norm"), _name(NORMS, pre_norm, "norm")
    _tensor(residual, "residual")
    dev = residual.device
    r2 = _rows(residual, "residual").contiguous()
    M, N = r2.shape
    if N > nv.lib().btvae_norm_max_columns():
        raise ValueError(f"norm_gate_residual supports up to {nv.lib().btvae_norm_max_columns()} columns, got {N}")
    if not (isinstance(eps, (int, float)) and eps >= 0):
        raise ValueError("eps must be a number >= 0")
    b2 = g2 = None
    if branch is not None:
        _tensor(branch, "branch")
        if residual.dtype == torch.bfloat16 and branch.dtype != torch.bfloat16:
            raise TypeError("a bfloat16 residual needs a bfloat16 branch")
        b2 = _rows(_matrix(branch, "branch", residual.shape, branch.dtype, dev), "branch").contiguous()
    elif gate is not None or post or torch.is_tensor(scale) or scale != 1.0 or post_weight is not None or post_bias is not None:
        raise ValueError("gate, scale and post norm need a branch")
    elif not pre:
        raise ValueError("nothing to compute: neither a branch nor a pre norm")
    if gate is not None:
        _tensor(gate, "gate", (branch.dtype,))
        g2 = _rows(_matrix(gate, "gate", gate.shape, branch.dtype, dev), "gate").contiguous()
        if g2.shape[1] != N or g2.shape[0] == 0 or M % g2.shape[0]:
            raise ValueError(f"gate must be [G, {N}] with {M} rows a multiple of G, got {list(gate.shape)}")
    f32 = (torch.float32,)
    vec = None
    if torch.is_tensor(scale):
        vec, scale = _vector(scale, "scale", N, f32, dev).contiguous(), 1.0
    if (post_weight is not None or post_bias is not None) and not post:
        raise ValueError("post_weight and post_bias need a post norm")
    if (pre_weight is not None or pre_bias is not None) and not pre:
        raise ValueError("pre_weight and pre_bias need a pre norm")
    vectors = [v if v is None else v.contiguous() for v in (_vector(post_weight, "post_weight", N, f32, dev), _vector(post_bias, "post_bias", N, f32, dev),
                                                            _vector(pre_weight, "pre_weight", N, f32, dev), _vector(pre_bias, "pre_bias", N, f32, dev))]
    ntype = branch.dtype if branch is not None else residual.dtype
    if normed_dtype is not None and normed_dtype != ntype:
        if branch is not None or normed_dtype != torch.bfloat16:
            raise TypeError(f"normed_dtype must be {str(ntype)[6:]}" + ("" if branch is not None or residual.dtype == torch.bfloat16 else " or bfloat16"))
        ntype = normed_dtype
    nv.ensure_device(dev)
    return r2, b2, g2, float(scale), vec, vectors, post, pre, float(eps), ntype


def norm_gate_residual(residual, branch=None, gate=None, scale=1.0, post_norm=None, post_weight=None, post_bias=None, pre_norm="rms",
                       pre_weight=None, pre_bias=None, eps=1e-6, normed_dtype=None):
    """(stream, normed): stream = residual + scale * gate * post(branch), normed = pre(stream), in one pass.

    ``residual``, ``branch`` [..., N] float32 or bfloat16 (a bfloat16 residual needs a bfloat16 branch; normed has the branch's
    type, stream the residual's); ``gate`` [G, N] of the branch's type multiplies row r with its row r % G (draw s of profile b
    is row s * B + b); ``scale`` a number or a float32 [N]; norms "rms", "layer" or None with float32 weights and biases
    (absent: 1 and 0).  Without a branch the stream is the residual itself; without a pre norm normed is None.  Up to 8192 columns.
    ``normed_dtype``: without a branch, bfloat16 gives a bfloat16 normed of a float32 residual.  Statistics and sums are float32; normed is computed from the stream before its rounding.  Differentiable in every tensor."""
    args = _norm_inputs(residual, branch, gate, scale, post_norm, post_weight, post_bias, pre_norm, pre_weight, pre_bias, eps, normed_dtype)
    r2, b2, g2, number, vec, vectors, post, pre, eps, ntype = args
    tensors = [t for t in (r2, b2, g2, vec, *vectors) if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        _refuse_capture("norm_gate_residual")
        out = list(_NormNode.apply(number, post, pre, eps, ntype, r2, b2, g2, vec, *vectors))
        stream = out.pop(0) if b2 is not None else None
        normed = out.pop(0) if pre else None
    else:
        stream, normed, _ = _norm_forward(r2, b2, g2, number, vec, vectors, post, pre, eps, ntype, False)
    return residual if stream is None else _shaped(stream, residual.shape), None if normed is None else _shaped(normed, residual.shape)


@torch.no_grad()
def norm_gate_residual_tape(residual, branch=None, gate=None, scale=1.0, post_norm=None, post_weight=None, post_bias=None, pre_norm="rms",
                            pre_weight=None, pre_bias=None, eps=1e-6, normed_dtype=None):
    """``norm_gate_residual`` without autograd: (stream, normed, tape), ``tape.backward(d_stream, d_normed)`` returns the gradients.
    May be captured into a graph."""
    r2, b2, g2, number, vec, vectors, post, pre, eps, ntype = _norm_inputs(residual, branch, gate, scale, post_norm, post_weight, post_bias, pre_norm,
                                                                          pre_weight, pre_bias, eps, normed_dtype)
    stream, normed, tape = _norm_forward(r2, b2, g2, number, vec, vectors, post, pre, eps, ntype, True)
    return residual if stream is None else _shaped(stream, residual.shape), None if normed is None else _shaped(normed, residual.shape), tape


# ------------------------------------------------------------------------------------------------ 8-bit products
class Fp8Rows:
    """Rows [M, K] as e4m3 with one power-of-two scale for each row and 128 columns (``q`` [M, padded K] bytes, ``scales`` [M, ..]
    bytes, exponent + 127)."""

    blocks = 0

    def __init__(self, q, scales, shape):
        self.q, self.scales, self.shape = q, scales, tuple(shape)

    @property
    def device(self):
        return self.q.device

    def dequantize(self):
        """The values held, as float32."""
        nv.ensure_device(self.device)
        rows, K = self.q.shape[0], self.shape[-1]
        out = torch.empty(rows, K, dtype=torch.float32, device=self.device)
        nv.call("btvae_fp8_dequantize", _p(self.q), self.q.shape[1], _p(self.scales), self.scales.shape[1], self.blocks, _p(out), rows, K)
        return out.view(self.shape)


    def _expanded(self) -> "_Operand":
        """The values as a bfloat16 operand (exactly: e4m3 times a power of two)."""
        rows, ld = self.q.shape
        out = torch.empty(rows, ld, dtype=torch.bfloat16, device=self.device)
        nv.call("btvae_fp8_expand", _p(self.q), ld, _p(self.scales), self.scales.shape[1], self.blocks, _p(out), ld, rows, self.shape[-1])
        return _Operand(out.data_ptr(), 2 * ld, ld, out)


class Fp8Weight(Fp8Rows):
    """A weight [N, K] as e4m3 with one power-of-two scale for each 128 x 128 block."""

    blocks = 1


def _fp8_buffers(rows, K, scale_rows, device):
    kb = -(-K // FP8_BLOCK)
    return torch.empty(rows, kb * FP8_BLOCK, dtype=torch.uint8, device=device), torch.empty(scale_rows, _up(kb, 4), dtype=torch.uint8, device=device)


def _no_graph(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward pass: 8-bit products are for evaluation; call it under torch.no_grad()")


def fp8_quantize(x) -> Fp8Rows:
    """Rows [..., K] (float32 or bfloat16) as e4m3: for each row and 128 columns e is the smallest integer >= -126 with
    max |x| <= 448 * 2^e, and the value x * 2^-e is rounded to the nearest e4m3, ties to even.  Non-finite values become NaN and
    take no part in their block's maximum."""
    _tensor(x, "x")
    _no_graph("fp8_quantize", x)
    x2 = _rows(x, "x")
    nv.ensure_device(x.device)
    M, K = x2.shape
    q, sc = _fp8_buffers(M, K, M, x.device)
    nv.call("btvae_fp8_quantize", _p(x2), int(x.dtype == torch.bfloat16), _pitch(x2), _p(q), q.shape[1], _p(sc), sc.shape[1], M, K)
    return Fp8Rows(q, sc, x.shape)


@torch.no_grad()
def fp8_weight(w) -> Fp8Weight:
    """A weight [N, K] as e4m3 with the scales of 128 x 128 blocks; a copy of ``w`` as it is now."""
    _tensor(w, "the weight")
    if w.dim() != 2 or w.shape[0] == 0:
        raise ValueError(f"the weight must be a matrix, got {list(w.shape)}")
    w2 = _rows(w, "the weight")
    nv.ensure_device(w.device)
    N, K = w2.shape
    q, sc = _fp8_buffers(N, K, -(-N // FP8_BLOCK), w.device)
    nv.call("btvae_fp8_quantize_blocks", _p(w2), int(w.dtype == torch.bfloat16), _pitch(w2), _p(q), q.shape[1], _p(sc), sc.shape[1], N, K)
    return Fp8Weight(q, sc, w.shape)


def _fp8_bias(bias, what, n, device):
    b = _vector(bias, what, n, _FLOATS, device)
    return None if b is None else b.detach().float().contiguous()


def _fp8_product(x: Fp8Rows, w: Fp8Weight, bias, out):
    """bfloat16 results on the 8-bit matrix pipe, whose sums are off by about 2^-16 of a result (a hundredth of its rounding:
    the products it adds together are cut to a unit that follows the largest of them); float32 results on the bfloat16
    pipe, whose sums are float32's."""
    M, N, K = x.q.shape[0], w.shape[0], w.shape[1]
    if out.dtype == torch.float32:
        X, W = x._expanded(), w._expanded()
        return _product(X, W, bias, out, 1, M, N, X.width)
    ws = _workspace(nv.lib().btvae_fp8_product_ws(M, N, K) if M else 0, out.device)
    nv.call("btvae_fp8_product", _p(x.q), x.q.shape[1], _p(x.scales), x.scales.shape[1], _p(w.q), w.q.shape[1], _p(w.scales), w.scales.shape[1], _p(bias),
            _p(out), N, int(out.dtype == torch.bfloat16), _p(ws), ws.numel() if ws is not None else 0, M, N, K)
    return out


def fp8_linear(x, weight: Fp8Weight, bias=None, out_dtype: Optional[torch.dtype] = None):
    """x weight^T + bias with x quantised by ``fp8_quantize`` (or given as ``Fp8Rows``).  ``out_dtype``: float32 or
    bfloat16, by default x's (float32 for ``Fp8Rows``).  Float32 results, and those of up to 32 rows that are quantised here, come from float32 sums; other
    bfloat16 results from the 8-bit matrix pipe, whose own sums are off by about 2^-16 of a result.  Evaluation only: no backward pass, and what
    wants a gradient is refused."""
    if not isinstance(weight, Fp8Weight):
        raise TypeError("weight must come from fp8_weight")
    packed = isinstance(x, Fp8Rows) and not isinstance(x, Fp8Weight)
    if not packed:
        _tensor(x, "x")
    _no_graph("fp8_linear", None if packed else x, bias)
    N, K = weight.shape
    if len(x.shape) < 1 or x.shape[-1] != K:
        raise ValueError(f"x must have {K} columns, got {list(x.shape)}")
    if weight.device != x.device:
        raise RuntimeError(f"the weight is on {weight.device}, the input on {x.device}")
    dtype = out_dtype or (torch.float32 if packed else x.dtype)
    if dtype not in _FLOATS:
        raise TypeError(f"out_dtype must be float32 or bfloat16, got {dtype}")
    b = _fp8_bias(bias, "bias", N, x.device)
    nv.ensure_device(x.device)
    shape = x.shape
    if not packed:
        x2 = _rows(x, "x")
        M = x2.shape[0]
        out = torch.empty(M, N, dtype=dtype, device=x.device)
        if M <= nv.lib().btvae_few_rows_max():
            nv.call("btvae_fp8_few_rows", _p(x2), int(x2.dtype == torch.bfloat16), _pitch(x2), _p(weight.q), _p(weight.scales), None, None, weight.q.shape[1],
                    weight.scales.shape[1], _p(b), None, _p(out), N, int(dtype == torch.bfloat16), 0, M, N, K)
            return out.view(*shape[:-1], N)
        x = fp8_quantize(x2)
    else:
        out = torch.empty(x.q.shape[0], N, dtype=dtype, device=x.device)
    return _fp8_product(x, weight, b, out).view(*shape[:-1], N)


class Fp8GatedWeights:
    """The weights of a gated feed-forward unit in 8 bits (``fp8_gated_weights``) and its biases in float32."""

    def __init__(self, gate, up, down, b_gate, b_up, b_down):
        self.gate, self.up, self.down, self.b_gate, self.b_up, self.b_down = gate, up, down, b_gate, b_up, b_down


def fp8_gated_weights(w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None) -> Fp8GatedWeights:
    """Quantise the weights of a gated feed-forward unit (shapes as in ``gated_feed_forward``): a copy of them as they are now."""
    gate, up, down = fp8_weight(w_gate), fp8_weight(w_up), fp8_weight(w_down)
    if up.shape != gate.shape or down.shape[1] != gate.shape[0]:
        raise ValueError(f"weights do not fit together: {list(gate.shape)}, {list(up.shape)}, {list(down.shape)}")
    if up.device != gate.device or down.device != gate.device:
        raise RuntimeError("the weights are on different devices")
    F, N = gate.shape[0], down.shape[0]
    return Fp8GatedWeights(gate, up, down, _fp8_bias(b_gate, "b_gate", F, gate.device), _fp8_bias(b_up, "b_up", F, gate.device), _fp8_bias(b_down, "b_down", N, gate.device))


def fp8_gated_feed_forward(x, weights: Fp8GatedWeights, activation="silu", out_dtype: Optional[torch.dtype] = None):
    """``gated_feed_forward`` on 8-bit operands: x is quantised, h = act(a) * b is quantised again from float32 without leaving the
    kernel that computes it; products as in ``fp8_linear``.  Result in ``out_dtype`` (x's by default).  Evaluation only."""
    act = _name(ACTIVATIONS, activation, "activation")
    if not isinstance(weights, Fp8GatedWeights):
        raise TypeError("weights must come from fp8_gated_weights")
    _tensor(x, "x")
    _no_graph("fp8_gated_feed_forward", x)
    w, dev = weights, x.device
    if w.gate.device != dev:
        raise RuntimeError(f"the weights are on {w.gate.device}, the input on {dev}")
    x2 = _rows(x, "x")
    (F, K), N, M = w.gate.shape, w.down.shape[0], x2.shape[0]
    if x2.shape[1] != K:
        raise ValueError(f"x must have {K} columns, got {list(x.shape)}")
    dtype = out_dtype or x.dtype
    if dtype not in _FLOATS:
        raise TypeError(f"out_dtype must be float32 or bfloat16, got {dtype}")
    nv.ensure_device(dev)
    y = torch.empty(M, N, dtype=dtype, device=dev)
    if M <= nv.lib().btvae_few_rows_max():
        h = torch.empty(M, F, dtype=torch.float32, device=dev)
        nv.call("btvae_fp8_few_rows", _p(x2), int(x.dtype == torch.bfloat16), _pitch(x2), _p(w.gate.q), _p(w.gate.scales), _p(w.up.q), _p(w.up.scales), w.gate.q.shape[1],
                w.gate.scales.shape[1], _p(w.b_gate), _p(w.b_up), _p(h), F, 0, act, M, F, K)
        nv.call("btvae_fp8_few_rows", _p(h), 0, F, _p(w.down.q), _p(w.down.scales), None, None, w.down.q.shape[1], w.down.scales.shape[1], _p(w.b_down), None,
                _p(y), N, int(dtype == torch.bfloat16), 0, M, N, F)
    else:
        xq = fp8_quantize(x2)
        hq, hs = _fp8_buffers(M, F, M, dev)
        if dtype == torch.float32:
            X, Wg, Wu = xq._expanded(), w.gate._expanded(), w.up._expanded()
            operands = (X.ptr(), X.width, None, 0, Wg.ptr(), None, Wu.ptr(), None, Wg.width, 0, 1)
        else:
            operands = (_p(xq.q), xq.q.shape[1], _p(xq.scales), xq.scales.shape[1], _p(w.gate.q), _p(w.gate.scales), _p(w.up.q), _p(w.up.scales),
                        w.gate.q.shape[1], w.gate.scales.shape[1], 0)
        nv.call("btvae_fp8_gated_proj", *operands, _p(w.b_gate), _p(w.b_up), _p(hq), hq.shape[1], _p(hs), hs.shape[1], act, M, F, K)
        _fp8_product(Fp8Rows(hq, hs, (M, F)), w.down, w.b_down, y)
    return y.view(*x.shape[:-1], N)
