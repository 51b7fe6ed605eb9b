"""Fused LayerNorm (optionally with a fused residual add) -- HIP kernels on GPU.

Replaces apex ``fused_layer_norm_cuda`` (K9-K11, reference
`smp/torch/apex/normalization/fused_layer_norm.py:26-78`).  ``MixedFusedLayerNorm``
semantics (fp32 input, low-precision affine) are covered by the kernel's independent
input / weight dtypes.
"""
import math

import torch

from ..backend.exceptions import SMPInvalidArgumentError
from ._ext import ext, fused_ok
from .dropout import dropout_seed_offset
from .linear import _fusable


def _ln_bwd(dy, x, w, b, mean, rstd, need_w, need_b, dres, drop=None):
    """LayerNorm backward; dgamma/dbeta of parameters bound to the flat grad buffer are
    accumulated in place by the reduce kernel (autograd then gets None for them, and the
    params' post-accumulate hooks still fire).  ``drop = (p, seed, offset)``: also returns the
    dropout backward of dx (4th value) -- from the same kernel pass where the block kernels
    serve the width, else by a separate dropout pass."""
    dkw = {}
    if drop is not None and drop[0] > 0.0:
        dkw = dict(dropout_p=drop[0], seed=drop[1], offset=drop[2])
    if need_w and need_b and _fusable(w) and _fusable(b):
        out = ext().layernorm_bwd(dy, x, w, mean, rstd, True, True, dres, w.grad, b.grad, None, 0.0, **dkw)
        dx, dw, db = out[0], None, None
    else:
        out = ext().layernorm_bwd(dy, x, w, mean, rstd, need_w, need_b, dres, None, None, None, 0.0, **dkw)
        dx, dw, db = out[0], (out[1] if need_w else None), (out[2] if need_b else None)
    if drop is None:
        return dx, dw, db
    if len(out) > 3:
        return dx, dw, db, out[3]
    p, seed, off = drop
    return dx, dw, db, (ext().dropout_bwd(dx, p, seed, off) if p > 0.0 else dx)


class _FusedLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        shape = x.shape
        x2 = x.contiguous()
        y, mean, rstd = ext().layernorm_fwd(x2, None, weight, bias, eps)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.bias = bias
        ctx.has_w = weight is not None
        ctx.has_b = bias is not None
        return y.view(shape)

    @staticmethod
    def backward(ctx, dy):
        x, w, mean, rstd = ctx.saved_tensors
        need_w = ctx.has_w and ctx.needs_input_grad[1]
        need_b = ctx.has_b and ctx.needs_input_grad[2]
        dx, dw, db = _ln_bwd(dy.contiguous(), x, w, ctx.bias, mean, rstd, need_w, need_b, None)
        return dx, dw, db, None


class _FusedLayerNormPassthrough(torch.autograd.Function):
    """(LN(x), x) -- the second output is the residual branch.  Backward sums the two
    gradient paths of x inside the LN backward kernel (dres) instead of leaving autograd
    to add them with a separate full-size elementwise pass."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = x.contiguous()
        y, mean, rstd = ext().layernorm_fwd(x2, None, weight, bias, eps)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.bias = bias
        ctx.has_w = weight is not None
        ctx.has_b = bias is not None
        ctx.set_materialize_grads(False)
        return y.view(x.shape), x.view_as(x)

    @staticmethod
    def backward(ctx, dy, dres):
        x, w, mean, rstd = ctx.saved_tensors
        need_w = ctx.has_w and ctx.needs_input_grad[1]
        need_b = ctx.has_b and ctx.needs_input_grad[2]
        if dy is None:
            return dres, None, None, None
        dres = dres.contiguous() if dres is not None else None
        dx, dw, db = _ln_bwd(dy.contiguous(), x, w, ctx.bias, mean, rstd, need_w, need_b, dres)
        return dx.view(dy.shape), dw, db, None


class _FusedAddLayerNorm(torch.autograd.Function):
    """s = dropout(x) + r ; y = LN(s).  Returns (y, s).  Backward fuses ds into the LN
    backward; the x branch then gets dropout's backward (mask regenerated from the hash)."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, dropout_p, drawn):
        x2, r2 = x.contiguous(), residual.contiguous()
        if dropout_p <= 0.0:
            seed, off = 0, 0
        else:
            seed, off = drawn if drawn is not None else dropout_seed_offset(x.device)
        y, mean, rstd, s = ext().layernorm_fwd(x2, r2, weight, bias, eps, dropout_p, seed, off)
        ctx.save_for_backward(s, weight, mean, rstd)
        ctx.bias = bias
        ctx.has_w = weight is not None
        ctx.has_b = bias is not None
        ctx.drop = (dropout_p, seed, off)
        return y.view(x.shape), s.view(x.shape)

    @staticmethod
    def backward(ctx, dy, ds):
        s, w, mean, rstd = ctx.saved_tensors
        need_w = ctx.has_w and ctx.needs_input_grad[2]
        need_b = ctx.has_b and ctx.needs_input_grad[3]
        dres = ds.contiguous() if ds is not None else None
        # the x branch's dropout backward comes out of the LN backward kernel itself (one pass
        # writing dx and dx * keep / (1 - p)) instead of a separate read of dx
        dx, dw, db, dxin = _ln_bwd(dy.contiguous(), s, w, ctx.bias, mean, rstd, need_w, need_b, dres, drop=ctx.drop)
        return dxin, dx, dw, db, None, None, None


class _MixedLayerNorm(torch.autograd.Function):
    """apex MixedFusedLayerNorm (K10): output in the parameters' dtype, written by the kernel
    from the fp32 statistics (no input-dtype rounding before the cast)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = x.contiguous()
        y, mean, rstd = ext().layernorm_fwd(x2, None, weight, bias, eps, 0.0, 0, 0, True)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.bias = bias
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x, w, mean, rstd = ctx.saved_tensors
        need_w, need_b = ctx.needs_input_grad[1], ctx.needs_input_grad[2]
        dx, dw, db = _ln_bwd(dy.to(x.dtype).contiguous(), x, w, ctx.bias, mean, rstd, need_w, need_b, None)
        return dx.view(dy.shape), dw, db, None


def mixed_layer_norm(x, weight, bias, eps=1e-5):
    """LayerNorm whose output takes the affine parameters' dtype (input any dtype)."""
    if fused_ok(x) and weight is not None and bias is not None:
        return _MixedLayerNorm.apply(x, weight, bias, eps)
    # statistics and affine in fp32 from the unrounded input, one rounding into the parameters' dtype
    w = weight.float() if weight is not None else None
    b = bias.float() if bias is not None else None
    y = torch.nn.functional.layer_norm(x.float(), (x.shape[-1],), w, b, eps)
    return y.to(weight.dtype) if weight is not None else y.to(x.dtype)


def layer_norm(x, weight, bias, eps=1e-5):
    if fused_ok(x):
        return _FusedLayerNorm.apply(x, weight, bias, eps)
    return torch.nn.functional.layer_norm(x, (x.shape[-1],), weight, bias, eps)


def layer_norm_passthrough(x, weight, bias, eps=1e-5):
    """Returns (LN(x), x) with the two backward paths of x summed inside the LN kernel."""
    if fused_ok(x):
        return _FusedLayerNormPassthrough.apply(x, weight, bias, eps)
    return torch.nn.functional.layer_norm(x, (x.shape[-1],), weight, bias, eps), x


def add_layer_norm(x, residual, weight, bias, eps=1e-5, dropout_p=0.0, drawn=None):
    """Returns (LN(dropout(x) + residual), dropout(x) + residual).  ``drawn``: the dropout's
    (seed, offset), drawn earlier with ``dropout_seed_offset`` to keep a generator order."""
    if fused_ok(x):
        return _FusedAddLayerNorm.apply(x, residual, weight, bias, eps, float(dropout_p), drawn)
    if dropout_p > 0.0:
        x = torch.nn.functional.dropout(x, dropout_p, True)
    s = x + residual
    return torch.nn.functional.layer_norm(s, (s.shape[-1],), weight, bias, eps), s


# ------------------------------------------------- the norms before and after a block, fused
MAX_BLOCK_NORM_WIDTH = 16384
MAX_BLOCK_NORM_ROWS = 1 << 30


def _block_norm_hip(x, residual, weight, bias, post_weight, post_bias, gate, gate_rows, alpha, eps, rms):
    """[y, s] by the kernels (x None: [y], the norm of residual); parameters bound to the flat
    gradient buffer take their gradients there in place, unless they have hooks that want them.
    None where the kernels do not take the call: dual numbers, function transforms, torch.compile,
    traces, dispatch modes, tensor classes that dispatch operations themselves."""
    if torch.compiler.is_compiling():
        return None
    marks = [int(getattr(t, "_smp_fused_grad", False)) for t in (weight, bias, post_weight, post_bias, gate)]
    return ext().block_norm(x, residual, weight, bias, post_weight, post_bias, gate, gate_rows, alpha, eps, rms, marks)


def _gate_matrix(gate, shape):
    """The gate as rows of d elements, each for a run of consecutive rows of the input, and the
    length of that run.  Gates that broadcast otherwise are expanded, in fp32: autograd sums
    their gradient back, and its terms must not be rounded before they are added."""
    d = shape[-1]
    if gate.shape == (d,):
        return gate, max(math.prod(shape[:-1]), 1)
    if gate.shape[-1:] != (d,):
        gate = gate.float().expand(*gate.shape[:-1], d)
    lead = (1,) * (len(shape) - gate.dim()) + tuple(gate.shape[:-1])
    k = 0  # the leading dimensions in which the gate has its own rows; in all others it has one
    while k < len(lead) and lead[k] == shape[k]:
        k += 1
    if any(n != 1 for n in lead[k:]):
        gate, k = gate.float().expand(*shape), len(shape) - 1
    groups = math.prod(shape[:k])
    return gate, max(math.prod(shape[:-1]) // max(groups, 1), 1)  # (an input without rows has runs too)


def _norm_torch(v, weight, bias, eps, rms):
    if not rms:
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * weight.float()
    return v if bias is None else v + bias.float()


def _block_norm_torch(x, residual, weight, bias, post_weight, post_bias, gate, alpha, eps, rms):
    h = x.float() if post_weight is None else _norm_torch(x.float(), post_weight, post_bias, eps, rms)
    s = residual.float() + alpha * (h if gate is None else gate.float() * h)
    return _norm_torch(s, weight, bias, eps, rms).to(x.dtype), s.to(x.dtype)


def _check_norm(name, rows, weight, bias, dtype):
    if not torch.is_tensor(weight) or weight.shape != rows.shape[-1:] or weight.device != rows.device:
        raise SMPInvalidArgumentError(f"{name} must be a [{rows.shape[-1]}] tensor on {rows.device}")
    if weight.dtype not in (rows.dtype, torch.float32) or weight.dtype != dtype:
        raise SMPInvalidArgumentError("weights and biases must all have the input's dtype, or all be fp32")
    if bias is not None and (bias.shape != weight.shape or bias.dtype != weight.dtype or bias.device != weight.device):
        raise SMPInvalidArgumentError(f"the bias beside {name} must have its shape, dtype and device")


def _check_rows(t, name):
    if not torch.is_tensor(t) or t.dim() == 0 or t.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise SMPInvalidArgumentError(f"{name} must be a fp32 / fp16 / bf16 tensor [..., dim]")
    if not 1 <= t.shape[-1] <= MAX_BLOCK_NORM_WIDTH:
        raise SMPInvalidArgumentError(f"{name}: widths of 1 to {MAX_BLOCK_NORM_WIDTH} are supported, got {t.shape[-1]}")
    if t.numel() // t.shape[-1] > MAX_BLOCK_NORM_ROWS:
        raise SMPInvalidArgumentError(f"{name}: at most {MAX_BLOCK_NORM_ROWS} rows are supported")


def block_norm(x, residual, weight, bias=None, post_weight=None, post_bias=None, gate=None, residual_scale=1.0,
               eps=1e-5, rms=False):
    """The norms after one block and before the next, with the gated residual add between them:

        h = norm(x; post_weight, post_bias)        (h = x without post_weight)
        s = residual + residual_scale * gate * h
        y = norm(s; weight, bias)

    -> ``(y, s)``, in one kernel each way (two backward for rows above 6144).  Without a gate and a
    norm after the block it is ``add_layer_norm`` without dropout, and keeps x and the residual for
    the backward, where that keeps their sum.  ``norm`` is LayerNorm or, with ``rms``, the
    root-mean-square norm.  ``x`` and ``residual`` [..., dim] are alike; the weights and biases
    [dim] have their dtype or are fp32.  ``gate`` (that dtype or fp32) broadcasts to ``x``: one
    vector, one for each sample ([batch, 1, dim]), or one value for each element; None is 1.
    All arithmetic is fp32, and the second norm is taken of ``s`` before it is rounded.  Under
    torch.autocast, where a block's output and the residual differ in type, the residual's holds for
    the output and for a 16-bit gate; a fp32 gate stays."""
    if torch.is_tensor(x) and torch.is_tensor(residual) and torch.is_autocast_enabled(x.device.type):
        x = x.to(residual.dtype)
        if torch.is_tensor(gate) and gate.dtype != torch.float32:  # (fp32 gates go with rows of any type)
            gate = gate.to(residual.dtype)
    _check_rows(x, "x")
    if not torch.is_tensor(residual) or residual.shape != x.shape or residual.dtype != x.dtype \
            or residual.device != x.device:
        raise SMPInvalidArgumentError("residual must have x's shape, dtype and device")
    _check_norm("weight", x, weight, bias, weight.dtype if torch.is_tensor(weight) else None)
    if post_weight is not None:
        _check_norm("post_weight", x, post_weight, post_bias, weight.dtype)
    elif post_bias is not None:
        raise SMPInvalidArgumentError("post_bias needs a post_weight")
    residual_scale, eps = float(residual_scale), float(eps)
    if not math.isfinite(residual_scale) or not (math.isfinite(eps) and eps >= 0.0):
        raise SMPInvalidArgumentError(f"bad residual_scale {residual_scale} or eps {eps}")
    if gate is not None:
        if not torch.is_tensor(gate) or gate.dtype not in (x.dtype, torch.float32) or gate.device != x.device:
            raise SMPInvalidArgumentError("gate must be a tensor of x's dtype or fp32, on its device")
        lead = x.dim() - gate.dim()
        if lead < 0 or any(n not in (1, m) for n, m in zip(gate.shape, x.shape[lead:])):
            raise SMPInvalidArgumentError(f"gate {tuple(gate.shape)} does not broadcast to {tuple(x.shape)}")
    out = None
    if x.is_cuda:
        rows, run = (gate, 1) if gate is None else _gate_matrix(gate if gate.dim() else gate.reshape(1), x.shape)
        out = _block_norm_hip(x, residual, weight, bias, post_weight, post_bias, rows, run, residual_scale, eps, bool(rms))
    if out is None:
        out = _block_norm_torch(x, residual, weight, bias, post_weight, post_bias, gate, residual_scale, eps, rms)
    return tuple(out)


def rms_norm(x, weight, eps=1e-5):
    """``x / sqrt(mean(x^2) + eps) * weight``: the norm before the first block of a model whose
    blocks are joined by ``block_norm(..., rms=True)``.  ``weight`` [dim] of x's dtype or fp32."""
    _check_rows(x, "x")
    _check_norm("weight", x, weight, None, weight.dtype if torch.is_tensor(weight) else None)
    eps = float(eps)
    if not (math.isfinite(eps) and eps >= 0.0):
        raise SMPInvalidArgumentError(f"bad eps {eps}")
    out = _block_norm_hip(None, x, weight, None, None, None, None, 1, 1.0, eps, True) if x.is_cuda else None
    return _norm_torch(x.float(), weight, None, eps, True).to(x.dtype) if out is None else out[0]
