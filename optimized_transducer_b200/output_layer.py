"""The joiner's output layer in 8-bit floating point.

:func:`joiner_logits` computes ``logits = joiner_in @ weight.T + bias`` on the
tensor cores with both operands in e4m3 and one float32 scale for every block of
128 elements along the contraction: blocks of 1 x 128 for the activations, which
are quantised inside the call, and of 128 x 128 for the weight.  It stands beside
``joiner_scores`` / ``joiner_loss`` (the same operands in bfloat16, the logits
never stored) for callers that want the logits themselves: a decoder, or a loss of
their own.  The reference has no counterpart (its loss is given the logits).

Training: ``weight`` is a tensor, quantised in the call, and gradients flow to
``joiner_in``, ``weight`` and ``bias``; both products of the backward pass run in
e4m3 too.  Serving: :class:`Fp8Weight` holds a weight that was quantised once
(:func:`quantize_weight`, or a checkpoint's bytes and scales).
"""
import ctypes

import torch

from . import _lib
from .transducer_loss import _DTYPE_FLAG, _check_mode, _on_device

__all__ = ["joiner_logits", "Fp8Weight", "quantize_weight"]

_BLOCK = 128
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _blocks(n):
    return -(-n // _BLOCK)


def _pitch(n):
    """Bytes from row to row of a quantised matrix: whole cache lines."""
    return -(-n // 128) * 128


def _stream(device):
    return torch.cuda.current_stream(device.index).cuda_stream


def _forward(x, w, pitch, scale, bias, v, out_dtype):
    """The logits of a quantised weight, (rows, V): one library call."""
    rows, d = x.shape
    dev = x.device
    lib = _lib.load()
    flags = _DTYPE_FLAG[out_dtype] | (0 if _check_mode() == "off" else _lib.REPORT_ERRORS)
    with _on_device(dev.index):
        need = ctypes.c_uint64()
        _lib.check(lib.ot_b200_joiner_logits_workspace_bytes(rows, d, v, ctypes.byref(need)))
        size = need.value
        out = torch.empty((rows, v), dtype=out_dtype, device=dev)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        rc = lib.ot_b200_joiner_logits(
            x.data_ptr(), rows, d, x.stride(0) if rows > 1 else d, _DTYPE_FLAG[x.dtype], w.data_ptr(), pitch, scale.data_ptr(), v,
            bias.data_ptr() if bias is not None else None, flags, ws.data_ptr(), size, out.data_ptr(), _stream(dev))
    if rc:
        _lib.check(rc)
    return out


def _check_weight(data, scale, who):
    """Raises the error for a quantised weight that the kernels cannot read."""
    for t, name in ((data, "data"), (scale, "scale")):
        if not isinstance(t, torch.Tensor):
            raise RuntimeError(f"{who}: expected {name} to be a tensor, got {type(t).__name__}")
    if data.dtype != torch.float8_e4m3fn or data.dim() != 2 or data.numel() == 0:
        raise RuntimeError(f"{who}: data must be a non-empty 2-D float8_e4m3fn tensor")
    if not data.is_cuda:
        raise RuntimeError(f"{who}: CUDA tensors only (sm_100a kernels, no CPU path)")
    if (data.stride(1) != 1 and data.size(1) > 1) or (data.stride(0) % 16 and data.size(0) > 1) \
            or (data.size(0) > 1 and data.stride(0) < data.size(1)) or data.data_ptr() % 16:
        raise RuntimeError(f"{who}: data must have a unit column stride, rows a multiple of 16 bytes apart "
                           f"and a 16-byte aligned base, got strides {tuple(data.stride())}")
    want = (_blocks(data.size(0)), _blocks(data.size(1)))
    if scale.dtype != torch.float32 or tuple(scale.shape) != want or not scale.is_contiguous() \
            or scale.device != data.device:
        raise RuntimeError(f"{who}: scale must be a contiguous float32 tensor of shape {want} on {data.device}")


class Fp8Weight:
    """A quantised projection weight.  ``data``: (V, D) ``torch.float8_e4m3fn``, unit
    column stride, rows a multiple of 16 bytes apart, 16-byte aligned; ``scale``:
    (ceil(V/128), ceil(D/128)) float32, contiguous.  The value of an element is its
    e4m3 value times its block's scale.  The tensors are used as they are, not copied;
    they may be written to, but a handle keeps the two that it was made with."""

    __slots__ = ("_data", "_scale")

    def __init__(self, data, scale):
        if not _lib.tensors().weight(data, scale):
            _check_weight(data, scale, "Fp8Weight")  # says what is wrong
        self._data, self._scale = data, scale

    @property
    def data(self):
        return self._data

    @property
    def scale(self):
        return self._scale

    @property
    def shape(self):
        return self.data.shape

    @property
    def device(self):
        return self.data.device

    def dequantize(self):
        """The weight's values, (V, D) float32."""
        v, d = self.shape
        s = self.scale.repeat_interleave(_BLOCK, 0)[:v].repeat_interleave(_BLOCK, 1)[:, :d]
        return self.data.float() * s


def _check_matrix(t, name, who):
    if not t.is_cuda:
        raise RuntimeError(f"{who}: CUDA tensors only (sm_100a kernels, no CPU path)")
    if t.dtype not in _FLOATS:
        raise RuntimeError(f"{who}: expected {name} to be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() != 2 or t.size(1) == 0 or (t.stride(1) != 1 and t.size(1) > 1) \
            or (t.size(0) > 1 and t.stride(0) < t.size(1)):
        raise RuntimeError(f"{who}: expected {name} to be a 2-D tensor with contiguous rows")


def _row_stride(t):
    return t.stride(0) if t.size(0) > 1 else t.size(1)


def _quantize(x, mode, sums=False):
    """((q, scale), (qT, scaleT) or None, column sums or None) of a (rows, cols) matrix; see ot_b200_fp8_quantize."""
    rows, cols = x.shape
    dev = x.device
    q = torch.empty((rows, _pitch(cols)), dtype=torch.uint8, device=dev)
    square = mode in (_lib.FP8_SQUARES, _lib.FP8_SQUARES_BOTH)
    scale = torch.empty((_blocks(rows), _blocks(cols)) if square else (_blocks(cols), rows), dtype=torch.float32, device=dev)
    qt = scale_t = part = total = None
    if mode >= _lib.FP8_ROWS_AND_SQUARES:
        qt = torch.empty((cols, _pitch(rows)), dtype=torch.uint8, device=dev)
        columns = mode == _lib.FP8_ROWS_AND_COLUMNS
        scale_t = torch.empty((_blocks(rows), cols) if columns else (_blocks(cols), _blocks(rows)), dtype=torch.float32, device=dev)
    if sums:
        part = torch.empty((_blocks(rows), cols), dtype=torch.float32, device=dev)
        total = torch.empty(cols, dtype=torch.float32, device=dev)
    with _on_device(dev.index):
        _lib.check(_lib.load().ot_b200_fp8_quantize(
            x.data_ptr(), rows, cols, _row_stride(x), _DTYPE_FLAG[x.dtype], mode, q.data_ptr(), q.size(1), scale.data_ptr(),
            qt.data_ptr() if qt is not None else None, qt.size(1) if qt is not None else 0,
            scale_t.data_ptr() if qt is not None else None, part.data_ptr() if sums else None,
            total.data_ptr() if sums else None, _stream(dev)))
    return (q, scale), ((qt, scale_t) if qt is not None else None), total


def quantize_weight(weight):
    """:class:`Fp8Weight` of a (V, D) float32, bfloat16 or float16 CUDA tensor: blocks
    of 128 x 128, each with the smallest power of two as its scale that keeps the
    block's largest magnitude within e4m3 (448)."""
    _check_matrix(weight, "weight", "quantize_weight")
    if weight.size(0) == 0:
        raise RuntimeError("quantize_weight: the weight is empty")
    (q, scale), _, _ = _quantize(weight.detach(), _lib.FP8_SQUARES)
    return Fp8Weight(q.view(torch.float8_e4m3fn)[:, :weight.size(1)], scale)


def joiner_logits(joiner_in, weight, bias=None, out_dtype=torch.bfloat16):
    """``joiner_in @ weight.T + bias`` in 8-bit floating point (e4m3), (rows, V).

    ``joiner_in`` (rows, D) float32, bfloat16 or float16 with contiguous rows;
    ``weight`` a (V, D) tensor of those types, or an :class:`Fp8Weight`; ``bias`` (V,)
    float32 or None; ``out_dtype`` float32, bfloat16 or float16.  The activations are
    quantised in blocks of 1 x 128 and a weight tensor in blocks of 128 x 128; with
    ``s`` the block's scale (between 1/448 and 1/224 of its largest magnitude) an element
    is off by at most ``max(2^-4 |x|, 2^-10 s)``, so one below ``2^-10 s`` becomes 0.  The
    sums are float32, rounded once to ``out_dtype``.  The scales of two blocks that meet are
    multiplied in float32 first: magnitudes that multiply to 2^144 and more overflow there
    even if the largest ones never meet, below 2^-132 the pair's share is lost.  A block that holds an infinity or a NaN makes its products NaN.

    With a weight tensor the call is differentiable: ``d joiner_in = q(G) q(W)`` and
    ``d weight = q(G^T) q(X)`` in e4m3 (the gradient G of the logits in blocks of 128
    along the contraction, X in blocks of 128 x 128), ``d bias`` the float32 column
    sums of G.  X and W are kept for the backward pass in e4m3 (one byte per element),
    so overwriting ``joiner_in`` afterwards does no harm.  The gradient is not itself
    differentiable (``create_graph=True`` is refused), and there is no forward-mode
    derivative (dual tensors are refused); a call whose gradients are wanted needs at least
    one row.  An :class:`Fp8Weight` has
    no gradient: ``joiner_in`` may then not require one."""
    who = "joiner_logits"
    served = isinstance(weight, Fp8Weight)
    report = 0 if _check_mode() == "off" else _lib.REPORT_ERRORS
    if served:
        usual = _lib.tensors().logits(joiner_in, weight._data, weight._scale, bias, out_dtype, report)
        if usual is not None:
            return usual
    grads = torch.is_grad_enabled() and (joiner_in.requires_grad or (bias is not None and bias.requires_grad)
                                         or (not served and weight.requires_grad))
    _check_arguments(joiner_in, weight, bias, out_dtype, served, grads, who)
    if joiner_in.size(0) == 0:
        return torch.empty((0, weight.shape[0]), dtype=out_dtype, device=joiner_in.device)
    if grads:
        return _lib.tensors().train(joiner_in, weight, bias, out_dtype, report)
    if served:
        w = weight.data
        return _forward(joiner_in, w, w.stride(0) if w.size(0) > 1 else _pitch(w.size(1)), weight.scale, bias, w.size(0), out_dtype)
    q, scale = _quantize(weight, _lib.FP8_SQUARES)[0]
    return _forward(joiner_in, q, q.size(1), scale, bias, weight.size(0), out_dtype)


def _check_arguments(joiner_in, weight, bias, out_dtype, served, grads, who):
    """Raises the error for the first argument of :func:`joiner_logits` that will not do."""
    _check_matrix(joiner_in, "joiner_in", who)
    if served:
        _check_weight(weight.data, weight.scale, who)
    else:
        _check_matrix(weight, "weight", who)
    if weight.device != joiner_in.device or weight.shape[1] != joiner_in.size(1) or weight.shape[0] == 0:
        raise RuntimeError(f"{who}: expected joiner_in (rows, D) and weight (V, D) on one device, got "
                           f"{tuple(joiner_in.shape)} on {joiner_in.device} and {tuple(weight.shape)} on {weight.device}")
    if bias is not None and (bias.dtype != torch.float32 or bias.dim() != 1 or bias.numel() != weight.shape[0]
                             or bias.device != joiner_in.device or not bias.is_contiguous()):
        raise RuntimeError(f"{who}: bias must be a contiguous float32 tensor of V entries")
    if out_dtype not in _FLOATS:
        raise RuntimeError(f"{who}: out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    operands = [joiner_in, weight.scale if served else weight, bias]
    at = _lib.tensors().tangent(operands)
    if at >= 0:
        raise RuntimeError(f"{who}: {('joiner_in', 'weight', 'bias')[at]} carries a forward-mode tangent, and there is no forward-mode "
                           "derivative: pass its primal (torch.autograd.forward_ad.unpack_dual)")
    if served and grads:
        raise RuntimeError(f"{who}: an Fp8Weight is for inference; pass the weight as a tensor to train")
    if grads and joiner_in.size(0) == 0:
        raise RuntimeError(f"{who}: joiner_in has no rows")
