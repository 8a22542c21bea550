"""Linear and Conv2d layers on the reproducible GEMM and convolutions: the counterparts of ``_LinearFn`` /
``Linear`` and ``_ConvFn`` / ``Conv2d`` in the reference's repro_torch/repro_torch/layers.py:70-135; and the operators around them in a
language-model training step: ``linear`` / ``FusedLinear`` (bias, activation and residual in the product's epilogue, with their own bias
gradient), ``block_norm`` / ``BlockNorm``, ``linear_cross_entropy`` / ``LinearCrossEntropy``.  The optimizer is repro_optim.AdamW.

Forward  Y  = X W^T     gemm(x,  W, m, n, k, trans_a=False, trans_b=True)     (layers.py:85)
Backward dX = dY W      gemm(dy, W, m, k, n, False, False)                    (layers.py:89)
         dW = dY^T X    gemm(dy, x, n, k, m, True,  False)                    (layers.py:90)

The bias gradient of the reference is an exact superaccumulator sum from another component
(repro_sum, layers.py:92), which is not part of this library.  A layer with a bias therefore needs
the caller's column-sum function (``set_bias_grad``); without one, asking for the bias gradient
raises instead of silently falling back to a sum whose bits depend on the reduction order.
"""
import torch
from torch.autograd import forward_ad

from . import repro_conv as rc
from . import repro_gemm as rg
from . import repro_loss as rl
from . import repro_norm as rn

_slices = 3
_bias_grad = None


def set_slices(s):
    """Number of int8 slices for all layers (1..3), like the reference's set_slices (layers.py:10-13)."""
    global _slices
    if s not in (1, 2, 3):
        raise ValueError("slices must be 1, 2 or 3")
    _slices = s


def set_bias_grad(fn):
    """fn(dy[m, n]) -> db[n]: the reproducible column sum to use for bias gradients (Conv2d passes dY as
    [N * OH * OW, F] rows)."""
    global _bias_grad
    _bias_grad = fn


def _no_tangents(*tensors):
    """The fused operators read their tensors' memory, where forward-mode derivatives are not: a tangent would be lost without a word."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("forward-mode derivatives are not supported by this operator")


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(x, weight)
        m, k, n = x.shape[0], weight.shape[1], weight.shape[0]
        y = rg.gemm(x, weight, m, n, k, False, True, _slices)
        return y + bias if bias is not None else y      # one IEEE addition per element

    @staticmethod
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        dy = dy.contiguous()
        m, k, n = x.shape[0], weight.shape[1], weight.shape[0]
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = rg.gemm(dy, weight, m, k, n, False, False, _slices)
        if ctx.needs_input_grad[1]:
            dw = rg.gemm(dy, x, n, k, m, True, False, _slices)
        if ctx.needs_input_grad[2]:
            if _bias_grad is None:
                raise NotImplementedError("bias gradient needs a reproducible column sum: call set_bias_grad(fn)")
            db = _bias_grad(dy)
        return dx, dw, db


class Linear(torch.nn.Linear):
    """torch.nn.Linear whose three matrix products are bit-reproducible (2-D input [tokens, features])."""

    def forward(self, x):
        return _LinearFn.apply(x.contiguous(), self.weight, self.bias)


class _FusedLinearFn(torch.autograd.Function):
    """act(X W^T + b) + R with bias, activation and residual in the product's epilogue; backward forms dZ = dY act'(Z) and
    db in one pass, then dX and dW through the reproducible product."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        x, weight = x.contiguous(), weight.contiguous()      # the copies, where there are any, serve the backward pass too
        n, k = weight.shape
        m = x.numel() // k
        keep = activation is not None and any(ctx.needs_input_grad[:3])
        out = rg.gemm_epilogue(x, weight, m, n, k, False, True, _slices, bias, activation, residual, keep)
        y, z = out if keep else (out, None)
        ctx.save_for_backward(x, weight, z)
        ctx.how = (m, n, k, activation, _slices)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], n)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dx, dw, db = rg.linear_backward(dy, z, x, weight, *ctx.how, need_x, need_w, need_b)
        if dx is not None and x.dim() != 2:
            dx = dx.view(x.shape)
        return dx, dw, db, (dy if need_r else None), None


def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x @ weight.T + bias) + residual in one reproducible product, differentiable in every tensor.

    x [..., in], weight [out, in], bias [out], residual [..., out]; activation None, "relu", "silu", "gelu" (erf) or
    "gelu_tanh".  The bias gradient is summed in an order that depends on the sizes alone (no set_bias_grad is needed)."""
    xs, ws = x.shape, weight.shape
    if len(ws) != 2 or len(xs) < 1 or xs[-1] != ws[1]:
        raise ValueError("x must be [..., in] and weight [out, in]")
    n, k = ws
    shape = (*xs[:-1], n)
    if bias is not None and bias.shape != (n,):
        raise ValueError("bias must be [%d]" % n)
    if residual is not None and residual.shape != shape:
        raise ValueError("residual must have the output's shape")
    if k == 0 or n == 0:
        raise ValueError("weight must not be empty")
    rg._activation(activation)
    if forward_ad._current_level >= 0:
        _no_tangents(x, weight, bias, residual)
    if x.numel() == 0:                                   # no tokens: nothing to launch, gradients of zeros
        return torch.nn.functional.linear(x, weight, bias) + (0 if residual is None else residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        return _FusedLinearFn.apply(x, weight, bias, residual, activation)
    y = rg.gemm_epilogue(x, weight, x.numel() // k, n, k, False, True, _slices, bias, activation, residual)
    return y if len(xs) == 2 else y.view(shape)


class FusedLinear(torch.nn.Linear):
    """torch.nn.Linear followed by an activation and, with forward's `residual`, an addition, as one reproducible product."""

    def __init__(self, in_features, out_features, bias=True, activation=None, **kw):
        super().__init__(in_features, out_features, bias, **kw)
        rg._activation(activation)
        self.activation = activation

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, self.activation, residual)


class _ConvFn(torch.autograd.Function):
    """Y = conv(x, W), dX and dW through the three reproducible calls (layers.py:103-126 in the reference)."""

    @staticmethod
    def forward(ctx, x, weight, bias, stride, padding):
        ctx.save_for_backward(x, weight)
        n, c, h, w = x.shape
        f, _, kh, kw = weight.shape
        ctx.shape = rc.ConvShape(n, c, h, w, f, kh, kw, stride[0], stride[1], padding[0], padding[1])
        y = rc.conv2d(x, weight, ctx.shape, _slices)
        return y + bias[None, :, None, None] if bias is not None else y      # one IEEE addition per element

    @staticmethod
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        dy = dy.contiguous()
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = rc.conv2d_grad_input(dy, weight, ctx.shape, _slices)
        if ctx.needs_input_grad[1]:
            dw = rc.conv2d_grad_weight(dy, x, ctx.shape, _slices)
        if ctx.needs_input_grad[2]:
            if _bias_grad is None:
                raise NotImplementedError("bias gradient needs a reproducible column sum: call set_bias_grad(fn)")
            db = _bias_grad(dy.permute(0, 2, 3, 1).reshape(-1, dy.shape[1]))
        return dx, dw, db, None, None


class Conv2d(torch.nn.Conv2d):
    """torch.nn.Conv2d whose forward and both gradients are bit-reproducible: stride and zero padding only,
    like the reference's layer (layers.py:129-135)."""

    def forward(self, x):
        if self.groups != 1 or self.dilation != (1, 1) or isinstance(self.padding, str) or self.padding_mode != "zeros":
            raise NotImplementedError("Conv2d supports stride and zero padding only")
        return _ConvFn.apply(x.contiguous(), self.weight, self.bias, self.stride, self.padding)


class _BlockNormFn(torch.autograd.Function):
    """block_norm and its gradients (repro_norm); r is an output of its own when there is a y."""

    @staticmethod
    def forward(ctx, x, y, weight, bias, post_weight, gate, residual_scale, kind, eps):
        y = None if y is None else y.contiguous()
        r, h, stats = rn.block_norm(x, y, weight=weight, bias=bias, post_weight=post_weight, gate=gate, residual_scale=residual_scale,
                                    kind=kind, eps=eps, keep_stats=True)
        ctx.save_for_backward(r, y, stats, weight, bias, post_weight, gate)
        ctx.set_materialize_grads(False)
        ctx.how = dict(residual_scale=residual_scale, kind=kind, eps=eps)
        return h if y is None else (r, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        r, y, stats, weight, bias, post_weight, gate = ctx.saved_tensors
        dr, dh = (None, grads[0]) if y is None else grads
        if dh is None:
            if dr is None:
                return (None,) * 9
            dh = torch.zeros_like(r)                 # only the residual stream is used
        names = ("x", "y", "weight", "bias", "post_weight", "gate")
        g = rn.block_norm_backward(dh, dr, r, y, stats, weight=weight, bias=bias, post_weight=post_weight, gate=gate,
                                   wanted=[n for n, need in zip(names, ctx.needs_input_grad) if need], **ctx.how)
        return g.x, g.y, g.weight, g.bias, g.post_weight, g.gate, None, None, None


def block_norm(x, y=None, *, weight, bias=None, post_weight=None, gate=None, residual_scale=1.0, kind="rms", eps=1e-5):
    """(r, h): the residual stream r = residual_scale * x + gate * (post_weight * N(y)) behind a block with output y, and
    h = weight * N(r) + bias for the next block, differentiable in every tensor.  Without y, r is x.  See repro_norm.block_norm."""
    tensors = (x, y, weight, bias, post_weight, gate)
    if forward_ad._current_level >= 0:
        _no_tangents(*tensors)
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in tensors):
        return rn.block_norm(x, y, weight=weight, bias=bias, post_weight=post_weight, gate=gate, residual_scale=residual_scale, kind=kind, eps=eps)[:2]
    out = _BlockNormFn.apply(*tensors, residual_scale, kind, eps)
    return (x, out) if y is None else out


class BlockNorm(torch.nn.Module):
    """The parameters of block_norm for rows of `dim` values: `post` adds the norm behind the block, `gate` a learned gate for
    each channel (a gate computed elsewhere, [groups, dim], is passed to forward instead).  forward(x, y=None) -> (r, h)."""

    def __init__(self, dim, kind="rms", bias=False, post=False, gate=False, residual_scale=1.0, eps=1e-5):
        super().__init__()
        if kind not in rn.KINDS:
            raise ValueError("kind must be 'rms' or 'layer'")
        self.kind, self.residual_scale, self.eps = kind, residual_scale, eps
        self.weight = torch.nn.Parameter(torch.ones(dim))
        self.bias = torch.nn.Parameter(torch.zeros(dim)) if bias else None
        self.post_weight = torch.nn.Parameter(torch.ones(dim)) if post else None
        self.gate = torch.nn.Parameter(torch.ones(dim)) if gate else None

    def forward(self, x, y=None, gate=None):
        if gate is not None and self.gate is not None:
            raise ValueError("this module has a gate of its own")
        has_y = y is not None
        return block_norm(x, y, weight=self.weight, bias=self.bias, post_weight=self.post_weight if has_y else None,
                          gate=(self.gate if gate is None else gate) if has_y else gate, residual_scale=self.residual_scale, kind=self.kind, eps=self.eps)


class _LinearCrossEntropyFn(torch.autograd.Function):
    """Cross entropy of x W^T in pieces of the vocabulary (repro_loss): keeps two values a row for the backward pass."""

    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        x, weight, target = x.contiguous(), weight.contiguous(), target.contiguous()
        loss, stats = rl.linear_cross_entropy(x, weight, target, ignore_index, reduction, _slices)
        ctx.save_for_backward(x, weight, target, stats)
        ctx.how = (ignore_index, reduction, _slices)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, weight, target, stats = ctx.saved_tensors
        dx, dw = rl.linear_cross_entropy_backward(dloss, x, weight, target, stats, *ctx.how, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dx, dw, None, None, None


def linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean"):
    """Cross entropy of the logits x @ weight.T without storing them, differentiable in x and weight.  x [..., dim], weight
    [vocabulary, dim], target [...] int64; reduction "mean", "sum" or "none".  See repro_loss.linear_cross_entropy."""
    if forward_ad._current_level >= 0:
        _no_tangents(x, weight)
    if not torch.is_grad_enabled() or not (x.requires_grad or weight.requires_grad):
        if target.numel():
            return rl.linear_cross_entropy(x, weight, target, ignore_index, reduction, _slices)[0]
    n = rl._sizes(x, weight, target, reduction, _slices)[0]
    if n == 0:                                           # no rows: a loss of 0 (or no losses) and gradients of zeros
        logits = torch.nn.functional.linear(x, weight)
        return logits.sum(-1) if reduction == "none" else logits.sum()
    return _LinearCrossEntropyFn.apply(x, weight, target, ignore_index, reduction)


class LinearCrossEntropy(torch.nn.Module):
    """The output projection of a language model and its loss: forward(x, target).  `weight` [vocabulary, dim] may be shared with
    an embedding (assign the same Parameter)."""

    def __init__(self, dim, vocabulary, ignore_index=-100, reduction="mean"):
        super().__init__()
        if reduction not in rl.REDUCTIONS:
            raise ValueError("reduction must be 'none', 'mean' or 'sum'")
        self.ignore_index, self.reduction = ignore_index, reduction
        self.weight = torch.nn.Parameter(torch.randn(vocabulary, dim) * 0.02)

    def forward(self, x, target):
        return linear_cross_entropy(x, self.weight, target, self.ignore_index, self.reduction)
