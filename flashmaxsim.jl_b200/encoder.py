"""The token encoder in front of MaxSim: the operators of its blocks and its INT8
serving form (no reference counterpart: the reference scores features that the
caller brings).

    gated_ffn(x, w_gate, w_up, act)              h = a(x Wg^T) * (x Wu^T)
    norm_residual(x, h, w_post, w_pre, ...)      z = scale x + gate * N(h), y = N(z)
    int8_linear(x, w::Int8Index, bias)           (sx sw) * (codes_x codes_w^T) + b

Features are (..., dim), tokens as rows, on one CUDA device; the first two are
differentiable in every tensor argument.
"""
from __future__ import annotations

import torch

from . import _lib
from .autograd import needs_grad
from .errors import ArgumentError, DimensionMismatch
from .layouts import _device_of
from .quant import Int8Index, require_int8_index

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}
NORMS = {"rms": 0, "layer": 1}
NORM_MAX_DIM = 16384
_HALF = (torch.float16, torch.bfloat16)
_FLOAT = (torch.float32, torch.float16, torch.bfloat16)


def _run(name, dev, *args):
    # one short call: the raw stream, no device switch where none is needed
    fn = getattr(_lib.lib(), name)
    index = dev.index
    if torch._C._cuda_getDevice() == index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status != 0:
        _lib.check(status, name)


def _p(t):
    return None if t is None else t.data_ptr()


def _same_device(*ts):
    """The one CUDA device of the tensors (None among them is left out)."""
    index = -2
    for t in ts:
        if t is not None:
            i = t.get_device()
            if index == -2:
                index = i
            if i < 0 or i != index:
                return _device_of(*ts)  # raises with its reason
    return next(t for t in ts if t is not None).device


def _workspace(nbytes, like):
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


# --------------------------------------------------------------------------- gated feed-forward

class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act):
        ctx.save_for_backward(x, w_gate, w_up)
        ctx.act = act
        return _ffn_forward(x, w_gate, w_up, act)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up = ctx.saved_tensors
        return (*_ffn_pullback(dh, x, w_gate, w_up, ctx.act, ctx.needs_input_grad[:3]), None)


def _ffn_forward(x, w_gate, w_up, act):
    dim, hidden = x.shape[-1], w_gate.shape[0]
    x, w_gate, w_up = x.contiguous(), w_gate.contiguous(), w_up.contiguous()
    dev = x.device
    h = x.new_empty((*x.shape[:-1], hidden))
    rows = h.numel() // hidden if hidden else 0
    nb = _lib.lib().fms_gated_ffn_workspace_size(rows, dim, hidden, 0)
    ws = _workspace(nb, x)
    _run("fms_gated_ffn_fwd", dev, _lib.DTYPE_CODE[x.dtype], _p(x), _p(w_gate),
         _p(w_up), rows, dim, hidden, act, _p(h), _p(ws), nb)
    return h


def _ffn_pullback(dh, x, w_gate, w_up, act, wanted):
    dim, hidden = x.shape[-1], w_gate.shape[0]
    x, w_gate, w_up, dh = x.contiguous(), w_gate.contiguous(), w_up.contiguous(), dh.contiguous()
    dev = x.device
    rows = x.numel() // dim if dim else 0
    grads = [torch.empty_like(t) if w else None for t, w in zip((x, w_gate, w_up), wanted)]
    if rows == 0 or hidden == 0:
        return [g if g is None else g.zero_() for g in grads]
    nb = _lib.lib().fms_gated_ffn_workspace_size(rows, dim, hidden, 1)
    ws = _workspace(nb, x)
    _run("fms_gated_ffn_bwd", dev, _lib.DTYPE_CODE[x.dtype], _p(x), _p(w_gate),
         _p(w_up), _p(dh), rows, dim, hidden, act, *map(_p, grads),
         _p(ws), nb)
    return grads


def gated_ffn(x, w_gate, w_up, act="silu"):
    """The gated half of a feed-forward block: h = a(x w_gate^T) * (x w_up^T).

    x (..., dim), w_gate and w_up (hidden, dim) as torch.nn.Linear holds them, all
    float16 or all bfloat16; act is "silu", "gelu" (error function), "gelu_tanh"
    or "relu".  Returns (..., hidden).  Sums are float32; the products are not
    kept for the backward pass but computed again there."""
    if act not in ACTIVATIONS:
        raise ArgumentError(f"gated_ffn: act must be one of {sorted(ACTIVATIONS)}, got {act!r}")
    if x.dim() < 1 or w_gate.dim() != 2:
        raise DimensionMismatch("gated_ffn expects (..., dim) features and (hidden, dim) weights")
    if w_gate.shape != w_up.shape:
        raise DimensionMismatch("gated_ffn: w_gate and w_up")
    if x.shape[-1] != w_gate.shape[1]:
        raise DimensionMismatch("feature dim")
    if x.dtype not in _HALF:
        raise ArgumentError(f"gated_ffn takes float16 or bfloat16 features, got {x.dtype}")
    if w_gate.dtype != x.dtype or w_up.dtype != x.dtype:
        raise ArgumentError("gated_ffn: features and weights must share an eltype")
    _same_device(x, w_gate, w_up)
    if needs_grad(x, w_gate, w_up):
        return _GatedFFN.apply(x, w_gate, w_up, ACTIVATIONS[act])
    return _ffn_forward(x, w_gate, w_up, ACTIVATIONS[act])


# --------------------------------------------------------------------------- norms around a block

def _norm_forward(x, h, w_post, b_post, w_pre, b_pre, gate, groups, scale, kind, eps, want_stats):
    dev, dim = x.device, x.shape[-1]
    rows = x.numel() // dim
    z, y = torch.empty_like(x), torch.empty_like(x)
    stats = x.new_empty((4, rows), dtype=torch.float32) if want_stats else None
    _run("fms_norm_residual_fwd", dev, _lib.DTYPE_CODE[x.dtype], _lib.DTYPE_CODE[w_post.dtype],
         kind, _p(x), _p(h), _p(w_post), _p(b_post), _p(w_pre),
         _p(b_pre), _p(gate), groups, rows, dim, eps, scale, _p(z), _p(y),
         _p(stats))
    return z, y, stats


class _NormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, w_post, b_post, w_pre, b_pre, gate, groups, scale, kind, eps):
        z, y, stats = _norm_forward(x, h, w_post, b_post, w_pre, b_pre, gate, groups, scale, kind,
                                    eps, True)
        ctx.save_for_backward(x, h, w_post, b_post, w_pre, b_pre, gate, stats)
        ctx.geometry = (groups, scale, kind)
        ctx.set_materialize_grads(False)
        return z, y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dz, dy):
        x, h, w_post, b_post, w_pre, b_pre, gate, stats = ctx.saved_tensors
        groups, scale, kind = ctx.geometry
        dev, dim = x.device, x.shape[-1]
        rows = x.numel() // dim
        dz = None if dz is None else dz.contiguous()
        dy = None if dy is None else dy.contiguous()
        dx, dh = torch.empty_like(x), torch.empty_like(h)
        dv = [torch.empty_like(t) if t is not None and need else None for t, need in
              zip((w_post, b_post, w_pre, b_pre, gate), ctx.needs_input_grad[2:7])]
        nb = _lib.lib().fms_norm_residual_bwd_workspace_size(rows, groups, dim)
        ws = _workspace(nb, x)
        _run("fms_norm_residual_bwd", dev, _lib.DTYPE_CODE[x.dtype],
             _lib.DTYPE_CODE[w_post.dtype], kind, _p(x), _p(h), _p(w_post),
             _p(b_post), _p(w_pre), _p(gate), groups, rows, dim, scale,
             _p(stats), _p(dz), _p(dy), _p(dx), _p(dh),
             *map(_p, dv), _p(ws), nb)
        return (dx, dh, *dv, None, None, None, None)


def norm_residual(x, h, w_post, w_pre, *, gate=None, b_post=None, b_pre=None, scale=1.0,
                  kind="rms", eps=1e-6):
    """The norm after a block, its gate, the residual sum with its scale and the
    norm before the next block, in one pass:

        z = scale * x + gate * N(h; w_post, b_post),   y = N(z; w_pre, b_pre)

    x (the residual stream) and h (the block's output) are (..., dim) in float32,
    float16 or bfloat16; the vectors are (dim,) in the same type or all float32.
    kind is "rms" or "layer".  gate is None, (dim,), or for x (B, T, dim) one
    vector per sequence, (B, dim).  scale is a number.  Returns (z, y); y is the
    norm of z before z is rounded to the features' type."""
    if kind not in NORMS:
        raise ArgumentError(f"norm_residual: kind must be one of {sorted(NORMS)}, got {kind!r}")
    if x.dtype not in _FLOAT:
        raise ArgumentError(f"norm_residual: unsupported dtype {x.dtype}")
    if x.dim() < 1 or x.shape != h.shape:
        raise DimensionMismatch("norm_residual: x and h")
    if h.dtype != x.dtype:
        raise ArgumentError("norm_residual: x and h must share an eltype")
    dim = x.shape[-1]
    if not 1 <= dim <= NORM_MAX_DIM:
        raise DimensionMismatch(f"norm_residual: feature dim must be 1 to {NORM_MAX_DIM}")
    vectors = [v for v in (w_post, w_pre, b_post, b_pre, gate) if v is not None]
    vt = w_post.dtype
    if vt not in (x.dtype, torch.float32) or any(v.dtype != vt for v in vectors):
        raise ArgumentError("norm_residual: weights, biases and gate must all have the features' "
                            "eltype or all be float32")
    for v in (w_post, w_pre, b_post, b_pre):
        if v is not None and tuple(v.shape) != (dim,):
            raise DimensionMismatch("norm_residual: weights and biases must be (dim,)")
    groups = 1
    if gate is not None and tuple(gate.shape) != (dim,):
        if x.dim() != 3 or tuple(gate.shape) != (x.shape[0], dim):
            raise DimensionMismatch("norm_residual: gate must be (dim,) or (B, dim) for (B, T, dim)")
        groups = x.shape[0]
    if not eps >= 0:
        raise ArgumentError("norm_residual: eps must be >= 0")
    _same_device(x, h, *vectors)
    args = [None if t is None else t.contiguous() for t in (x, h, w_post, b_post, w_pre, b_pre, gate)]
    if needs_grad(x, h, *vectors):
        return _NormResidual.apply(*args, groups, float(scale), NORMS[kind], float(eps))
    return _norm_forward(*args, groups, float(scale), NORMS[kind], float(eps), False)[:2]


# --------------------------------------------------------------------------- INT8 linear

def int8_linear(x, w: Int8Index, bias=None, out_dtype=None):
    """Linear layer in 8-bit integers with one scale per token and one per output
    channel: y[t, c] = (sx_t * sw_c) * float(sum_k xc[t, k] * wc[c, k]) + bias_c.

    w is `quantize_int8_symmetric(weight)` of a float32 (out, dim) weight (a token
    of that index is an output channel).  x is (..., dim) float32, float16 or
    bfloat16, quantised per token inside the call (in float32 whatever its type),
    or an Int8Index of features with float32 scales.  The result (..., out) has
    the features' type, out_dtype where given (float32 for an Int8Index).  A token
    that holds an infinity or a NaN gives NaN.  Forward only."""
    require_int8_index(w)
    codes, scales = w.codes, w.scales
    if codes.dim() != 2:
        raise DimensionMismatch("int8_linear expects an (out, dim) weight index")
    if codes.dtype != torch.int8 or scales.dtype != torch.float32:
        raise ArgumentError("int8_linear: the weight index must hold int8 codes and float32 scales")
    xs = None
    if isinstance(x, Int8Index):
        require_int8_index(x)
        x, xs = x.codes, x.scales
        if x.dtype != torch.int8 or xs.dtype != torch.float32:
            raise ArgumentError("int8_linear: an index of features must hold int8 codes and float32 scales")
        xt, out_dtype = _lib.I8, out_dtype or torch.float32
    else:
        if x.dtype not in _FLOAT:
            raise ArgumentError(f"int8_linear: unsupported dtype {x.dtype}")
        xt, out_dtype = _lib.DTYPE_CODE[x.dtype], out_dtype or x.dtype
    if needs_grad(x, xs, scales, bias):
        raise ArgumentError("int8_linear is forward-only (no autograd pullback)")
    if out_dtype not in _FLOAT:
        raise ArgumentError(f"int8_linear: unsupported output dtype {out_dtype}")
    out, dim = codes.shape
    if x.dim() < 1 or x.shape[-1] != dim or dim < 1:
        raise DimensionMismatch("feature dim")
    if bias is not None:
        if tuple(bias.shape) != (out,):
            raise DimensionMismatch("int8_linear: bias must be (out,)")
        if bias.dtype != out_dtype:
            raise ArgumentError("int8_linear: bias must have the output's eltype")
        bias = bias.contiguous()
    dev = _same_device(x, xs, codes, scales, bias)
    x, codes, scales = x.contiguous(), codes.contiguous(), scales.contiguous()
    xs = None if xs is None else xs.contiguous()
    y = x.new_empty((*x.shape[:-1], out), dtype=out_dtype)
    rows = x.numel() // dim
    nb = _lib.lib().fms_int8_linear_workspace_size(xt, rows, dim, out)
    ws = _workspace(nb, x)
    _run("fms_int8_linear_fwd", dev, xt, _p(x), _p(xs), _p(codes),
         _p(scales), _p(bias), rows, dim, out, _lib.DTYPE_CODE[out_dtype], _p(y),
         _p(ws), nb)
    return y
