"""Cross entropy of the logits x @ weight.T against targets in pieces of the vocabulary, on the C ABI.

The [tokens, vocabulary] logits are never stored: the forward pass keeps each row's log-sum-exp and the others' share beside its target, the
backward pass forms the probabilities of one piece of words at a time.  ``layers.linear_cross_entropy`` and
``layers.LinearCrossEntropy`` are the differentiable forms.  CUDA float32 only; there is no CPU path.
"""
import torch

from . import _lib
from .repro_gemm import ReproGemmError, _addr, _check, _extent, _on, _raise_if_incomplete, _raw_stream, _scratch, cudaSuccess

REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _sizes(x, weight, target, reduction, slices):
    if reduction not in REDUCTIONS:
        raise ValueError("reduction must be 'none', 'mean' or 'sum'")
    if slices not in (1, 2, 3):
        raise ValueError("slices must be 1, 2 or 3")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError("x must be [..., dim] and weight [vocabulary, dim]")
    if target.dtype != torch.int64:
        raise TypeError("target must be int64")
    if target.shape != x.shape[:-1]:
        raise ValueError("target must have the shape of x without its last dimension")
    if not (x.device == weight.device == target.device):
        raise ValueError("all tensors must be on one device")
    _extent(target.numel(), *weight.shape)
    return target.numel(), weight.shape[0], weight.shape[1]


def _workspace(n, v, d, slices, backward, device):
    nbytes = _lib.lib().rgb200_linear_xent_workspace(n, v, d, slices, backward)
    if nbytes == 0:
        raise ValueError("sizes not supported: %d tokens, %d words, %d values a token" % (n, v, d))
    return _scratch(nbytes, device)


def linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean", slices=3):
    """(loss, stats).  x [..., dim], weight [vocabulary, dim], target [...] int64.

    loss: a scalar ("mean" over the rows whose target is not ignore_index, at least 1; or "sum"), or with "none" the rows'
    losses: 0 where the target is ignore_index and NaN, without a gradient, where it is outside the vocabulary otherwise.
    stats: float32 [2 n + 1] for the backward call, the rows' log-sum-exp, the probability of all words
    but their target, and the weight of a row."""
    n, v, d = _sizes(x, weight, target, reduction, slices)
    shape = target.shape
    x, weight, target = _check(x, n * d, "x"), _check(weight, v * d, "weight"), target.contiguous()
    stats = torch.empty(2 * n + 1, dtype=torch.float32, device=x.device)
    nll = torch.empty(shape, dtype=torch.float32, device=x.device)
    loss = torch.empty((), dtype=torch.float32, device=x.device) if reduction != "none" else None
    at = stats.data_ptr()
    with _on(x.device):
        ws = _workspace(n, v, d, slices, 0, x.device)
        rc = _lib.lib().rgb200_linear_xent_forward(_addr(x), _addr(weight), _addr(target), ignore_index, REDUCTIONS[reduction], n, v, d, slices, _addr(loss),
                                                   _addr(nll), at, at + 4 * n, at + 8 * n, _addr(ws), ws.numel(), _raw_stream(x.device))
    if rc != cudaSuccess:
        raise ReproGemmError(rc, "linear_xent_forward")
    _raise_if_incomplete(ws, "linear_cross_entropy")
    return (nll if loss is None else loss), stats


def linear_cross_entropy_backward(dloss, x, weight, target, stats, ignore_index=-100, reduction="mean", slices=3, want_dx=True, want_dw=True):
    """(dx, dweight) from the loss's gradient (a scalar, or one value a row with reduction "none") and the forward call's stats."""
    n, v, d = _sizes(x, weight, target, reduction, slices)
    shape = x.shape
    x, weight, target = _check(x, n * d, "x"), _check(weight, v * d, "weight"), target.contiguous()
    stats = _check(stats, 2 * n + 1, "stats")
    dloss = _check(dloss, n if reduction == "none" else 1, "dloss")
    if dloss.device != x.device or stats.device != x.device:
        raise ValueError("all tensors must be on one device")
    if not (want_dx or want_dw):
        return None, None
    dx = torch.empty(shape, dtype=torch.float32, device=x.device) if want_dx else None
    dw = torch.empty((v, d), dtype=torch.float32, device=x.device) if want_dw else None
    at = stats.data_ptr()
    with _on(x.device):
        ws = _workspace(n, v, d, slices, 1, x.device)
        rc = _lib.lib().rgb200_linear_xent_backward(_addr(x), _addr(weight), _addr(target), ignore_index, REDUCTIONS[reduction], n, v, d, slices, at, at + 4 * n,
                                                    at + 8 * n, _addr(dloss), _addr(dx), _addr(dw), _addr(ws), ws.numel(), _raw_stream(x.device))
    if rc != cudaSuccess:
        raise ReproGemmError(rc, "linear_xent_backward")
    _raise_if_incomplete(ws, "linear_cross_entropy_backward")
    return dx, dw
