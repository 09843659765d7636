"""The norm of all gradients together, and clipping by it: what stands between the
backward pass of the loss and the optimizer.  The reference leaves it to
``torch.nn.utils.clip_grad_norm_``, whose definition :func:`clip_grad_norm_` has; here
it is two kernels for any number of tensors, of mixed types, and the clipped gradients
may go somewhere else (the optimizer's float32 copies) instead of staying in place.
"""
import ctypes
import math

import torch

from . import _lib
from .transducer_loss import _DTYPE_FLAG, _on_device

__all__ = ["grad_norm", "clip_grad_norm_"]

_KINDS = {1.0: _lib.NORM_1, 2.0: _lib.NORM_2, math.inf: _lib.NORM_INF}


def _dense(t):
    """Whether t fills one stretch of memory, each element once (any order of its dimensions)."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((t.stride(d), t.size(d)) for d in range(t.dim()) if t.size(d) != 1):
        if stride != want:
            return False
        want *= size
    return True


def _table(tensors, who, what, device):
    """(pointers, counts, type flags) of dense CUDA tensors on one device, as ctypes arrays."""
    n = len(tensors)
    try:
        types = [_DTYPE_FLAG[t.dtype] for t in tensors]
    except KeyError as e:
        raise RuntimeError(f"{who}: expected {what} to be float32, float64, bfloat16 or float16, got {e.args[0]}") from None
    for t in tensors:
        if t.get_device() != device:
            raise RuntimeError(f"{who}: expected {what} to be CUDA tensors on one device (sm_100a kernels, no CPU path), "
                               f"got one on {t.device}")
        if t.layout != torch.strided or not (t.is_contiguous() or _dense(t)):
            raise RuntimeError(f"{who}: expected {what} to be dense (no gaps, no expanded dimensions), got "
                               f"{t.layout} of shape {tuple(t.shape)}")
    counts = [t.numel() for t in tensors]
    return ((ctypes.c_void_p * n)(*[t.data_ptr() for t in tensors]), (ctypes.c_int64 * n)(*counts),
            (ctypes.c_int32 * n)(*types))


def _call(who, tensors, norm_type, apply, max_norm, out):
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    kind = _KINDS.get(float(norm_type))
    if kind is None:
        raise RuntimeError(f"{who}: norm_type must be 1, 2 or inf, got {norm_type}")
    if not tensors:
        raise RuntimeError(f"{who}: no gradients were given")
    device = tensors[0].get_device()
    if device < 0:
        raise RuntimeError(f"{who}: CUDA tensors only (sm_100a kernels, no CPU path)")
    grads, counts, types = _table(tensors, who, "the gradients", device)
    outs = out_types = None
    if out is not None:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(out) != len(tensors):
            raise RuntimeError(f"{who}: expected one output per gradient, got {len(out)} for {len(tensors)}")
        for t, o in zip(tensors, out):
            if t.shape != o.shape or (t.stride() != o.stride() and not (t.is_contiguous() and o.is_contiguous())):
                raise RuntimeError(f"{who}: an output must have its gradient's shape and strides, got {tuple(o.shape)} "
                                   f"for {tuple(t.shape)}")
        outs, _, out_types = _table(out, who, "the outputs", device)
    lib = _lib.load()
    with _on_device(device):
        need = ctypes.c_uint64()
        _lib.check(lib.ot_b200_clip_workspace_bytes(len(tensors), ctypes.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device=tensors[0].device)
        norm = torch.empty((), dtype=torch.float32, device=tensors[0].device)
        _lib.check(lib.ot_b200_clip_gradients(
            len(tensors), grads, counts, types, outs, out_types, kind, 1 if apply else 0, float(max_norm), ws.data_ptr(),
            need.value, norm.data_ptr(), torch.cuda.current_stream(device).cuda_stream))
    return norm


def grad_norm(tensors, norm_type=2.0):
    """The norm (``norm_type`` 1, 2 or inf) of all ``tensors`` together, as if they were
    one vector: a 0-dim float32 tensor on their device.  ``tensors``: one dense CUDA
    tensor or an iterable of them, float32, float64, bfloat16 or float16, mixed as one
    likes.  Sums are taken in float64 over groups of at most 32 elements in a fixed
    order: the same inputs give the same bits."""
    return _call("grad_norm", tensors, norm_type, False, 0.0, None)


def clip_grad_norm_(tensors, max_norm, norm_type=2.0, out=None):
    """Scales the gradients ``tensors`` by ``min(1, max_norm / (norm + 1e-6))``, the
    definition of ``torch.nn.utils.clip_grad_norm_``, and returns their norm before that
    (:func:`grad_norm`).  ``tensors`` are the gradients themselves
    (``[p.grad for p in parameters if p.grad is not None]``), or what
    ``transducer_loss_and_grad`` returns.  They are scaled in place (left untouched when
    the factor is 1), or, with ``out`` (one tensor per gradient, same shape and strides,
    any of the types), written there and left as they are.  No two tensors may overlap.
    The host does not wait for the device.  As in torch an infinite norm scales by 0 and
    a NaN one by NaN."""
    who = "clip_grad_norm_"
    if not float(max_norm) >= 0.0:
        raise RuntimeError(f"{who}: max_norm must not be negative or a NaN, got {max_norm}")
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    written = tensors if out is None else ([out] if isinstance(out, torch.Tensor) else list(out))
    norm = _call(who, tensors, norm_type, True, max_norm, None if out is None else written)
    torch.autograd.graph.increment_version([t for t in written if not t.is_inference()])
    return norm
