"""The norm of all gradients together, and clipping by it: what stands between the
backward pass of the loss and the optimizer.  The reference leaves it to
``torch.nn.utils.clip_grad_norm_``, whose definition :func:`clip_grad_norm_` has; here
it is two kernels for any number of tensors, of mixed types, and the clipped gradients
may go somewhere else (the optimizer's float32 copies) instead of staying in place.
"""
import math

import torch

from . import _lib

__all__ = ["grad_norm", "clip_grad_norm_"]

_KINDS = {1.0: _lib.NORM_1, 2.0: _lib.NORM_2, math.inf: _lib.NORM_INF}


def _table(tensors, who, what):
    """(pointers, counts, type flags, device) of dense CUDA tensors on one device; the first three are C arrays."""
    pointers, counts, types, device, at, why = _lib.tensors().describe(tensors)
    if why == "":
        return pointers, counts, types, device
    t = tensors[at]
    if why == "tensor":
        raise RuntimeError(f"{who}: expected {what} to be tensors, got {type(t).__name__}")
    if why == "type":
        raise RuntimeError(f"{who}: expected {what} to be float32, float64, bfloat16 or float16, got {t.dtype}")
    if why == "layout":
        raise RuntimeError(f"{who}: expected {what} to be dense (no gaps, no expanded dimensions), got {t.layout} of shape "
                           f"{tuple(t.shape)}")
    if why == "cpu":
        raise RuntimeError(f"{who}: CUDA tensors only (sm_100a kernels, no CPU path), got one on {t.device}")
    if why == "dual":
        raise RuntimeError(f"{who}: one of {what} carries a forward-mode tangent, and there is no forward-mode derivative: pass "
                           "its primal (torch.autograd.forward_ad.unpack_dual)")
    raise RuntimeError(f"{who}: expected {what} to be on one device, got {t.device} and {tensors[0].device}")


def _kind(norm_type, who):
    kind = _KINDS.get(float(norm_type))
    if kind is None:
        raise RuntimeError(f"{who}: norm_type must be 1, 2 or inf, got {norm_type}")
    return kind


def _call(who, tensors, norm_type, apply, max_norm, out):
    kind = _kind(norm_type, who)
    if not tensors:
        raise RuntimeError(f"{who}: no gradients were given")
    grads, counts, types, device = _table(tensors, who, "the gradients")
    outs = out_types = None
    if out is not None:
        if len(out) != len(tensors):
            raise RuntimeError(f"{who}: expected one output per gradient, got {len(out)} for {len(tensors)}")
        outs, _, out_types, out_device = _table(out, who, "the outputs")
        at = _lib.tensors().alike(tensors, out)
        if at >= 0 or out_device != device:
            raise RuntimeError(f"{who}: an output must have its gradient's shape, strides and device, got {tuple(out[at].shape)} "
                               f"on {out[at].device} for {tuple(tensors[at].shape)} on {tensors[at].device}")
    return _lib.tensors().clip(grads, counts, types, outs, out_types, tensors[0], kind, 1 if apply else 0, float(max_norm))


def _list(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def grad_norm(tensors, norm_type=2.0):
    """The norm (``norm_type`` 1, 2 or inf) of all ``tensors`` together, as if they were
    one vector: a 0-dim float32 tensor on their device.  ``tensors``: one dense CUDA
    tensor or an iterable of them, float32, float64, bfloat16 or float16, mixed as one
    likes.  Sums are taken in float64 over groups of at most 32 elements in a fixed
    order: the same inputs give the same bits.  The norm has no derivative: tensors that
    require a gradient are refused unless under ``torch.no_grad()``, forward-mode dual
    tensors always."""
    who = "grad_norm"
    tensors = _list(tensors)
    if torch.is_grad_enabled():
        at = _lib.tensors().writable(tensors)
        if at >= 0:
            raise RuntimeError(f"{who}: tensor {at} requires a gradient, and the norm has no derivative: pass detached tensors "
                               "or call it under torch.no_grad()")
    return _call(who, tensors, norm_type, False, 0.0, None)


def clip_grad_norm_(tensors, max_norm, norm_type=2.0, out=None):
    """Scales the gradients ``tensors`` by ``min(1, max_norm / (norm + 1e-6))``, the
    definition of ``torch.nn.utils.clip_grad_norm_``, and returns their norm before that
    (:func:`grad_norm`).  ``tensors`` are the gradients themselves
    (``[p.grad for p in parameters if p.grad is not None]``), or what
    ``transducer_loss_and_grad`` returns.  They are scaled in place (left untouched when
    the factor is 1), or, with ``out`` (one tensor per gradient, same shape and strides,
    any of the types), written there and left as they are.  No two tensors may overlap.
    Tensors that require a gradient are refused: unlike torch's function this one is not
    given the parameters.  The factor is taken from the norm in float64 (float64 gradients are
    scaled in float64, the others in float32); what is returned is the norm in float32.  The host
    does not wait for the device.  As in torch an infinite norm scales by 0 and a NaN one by NaN,
    and without any tensors (a step in which everything is frozen) the norm is a 0 on the CPU."""
    who = "clip_grad_norm_"
    if not float(max_norm) >= 0.0:
        raise RuntimeError(f"{who}: max_norm must not be negative or a NaN, got {max_norm}")
    tensors = _list(tensors)
    written = tensors if out is None else _list(out)
    at = _lib.tensors().writable(written)
    if at >= 0:
        raise RuntimeError(f"{who}: tensor {at} requires a gradient: pass the gradients (p.grad), not the parameters, and no "
                           "gradient that is part of a graph")
    if not tensors and not written:
        _kind(norm_type, who)
        return torch.zeros(())
    norm = _call(who, tensors, norm_type, True, max_norm, None if out is None else written)
    _lib.tensors().written(written)
    return norm
