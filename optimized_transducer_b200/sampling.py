"""Drawing symbols from the joiner's logits.

:func:`sample_tokens` draws one symbol per row of packed logits (the layout the
loss takes, or one row per hypothesis of a decoder) with temperature, top-k, top-p
and min-p, from uniform numbers that the caller gives, so a run can be repeated.
The reference has no counterpart (decoding lies outside its loss).
"""
import torch

from . import _lib
from .transducer_loss import _DTYPE_FLAG, _on_device

__all__ = ["sample_tokens"]

MAX_V = 262144
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _setting(value, name, dtype, logits):
    """(device pointer or None, scalar) of one setting: a number, or one value per row."""
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype or value.shape != (logits.size(0),) or not value.is_contiguous() \
                or value.device != logits.device:
            raise RuntimeError(f"sample_tokens: {name} must be a number or a contiguous {dtype} tensor with one value "
                               f"per row on {logits.device}")
        return value.data_ptr(), 0
    return None, (int(value) if dtype == torch.int32 else float(value))


def sample_tokens(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One symbol per row: ``(tokens (rows,) int32, logprobs (rows,) float32)``.

    ``logits`` (rows, V) float32, bfloat16 or float16 with contiguous rows, V up to
    262144; ``uniforms`` (rows,) float32 in [0, 1].  With
    ``w = exp((logits - max) / temperature)`` a row keeps its ``top_k`` largest logits
    (0: all), of those the ones before which less than ``top_p`` of their weight lies
    (1: all), of those the ones with ``w >= min_p`` (0: all); "before" is the order of
    falling logits, the lower index first among equal ones, and its first symbol always
    stays.  The token is the first index, in index order, at which the kept weights sum
    to more than ``uniforms`` times their total; the log-probability is that of the kept
    weights.  ``temperature=0`` takes the first symbol (log-probability 0).  Each setting
    is a number or a tensor with one value per row (float32; ``top_k`` int32).  Neither
    result carries a derivative, of either mode: the log-probabilities of drawn symbols
    that a loss needs are taken from the logits again.

    Tokens are those of 64-bit arithmetic.  ``-inf`` logits are never drawn.  A row
    without a finite maximum (everything ``-inf``, or a NaN or ``+inf`` in it), or whose
    own settings are out of range (``uniforms`` outside [0, 1], ``temperature`` outside
    [0, 1e6], a NaN), gets token -1 and log-probability NaN."""
    usual = _lib.tensors().sample(logits, uniforms, temperature, top_k, top_p, min_p)
    if usual is not None:
        return usual
    t_ptr, t = _setting(temperature, "temperature", torch.float32, logits)
    k_ptr, k = _setting(top_k, "top_k", torch.int32, logits)
    p_ptr, p = _setting(top_p, "top_p", torch.float32, logits)
    m_ptr, m = _setting(min_p, "min_p", torch.float32, logits)
    _check_arguments(logits, uniforms, t_ptr, t, k, p, m)
    rows, v = logits.shape
    device = logits.device
    tokens = torch.empty(rows, dtype=torch.int32, device=device)
    logprobs = torch.empty(rows, dtype=torch.float32, device=device)
    if rows == 0:
        return tokens, logprobs
    index = device.index
    with _on_device(index):
        rc = _lib.load().ot_b200_sample(
            logits.data_ptr(), rows, v, logits.stride(0) if rows > 1 else v, _DTYPE_FLAG[logits.dtype],
            uniforms.data_ptr(), t_ptr, t, k_ptr, k, p_ptr, p, m_ptr, m, tokens.data_ptr(), logprobs.data_ptr(),
            torch.cuda.current_stream(index).cuda_stream)
    if rc:
        _lib.check(rc)
    return tokens, logprobs


def _check_arguments(logits, uniforms, t_ptr, t, k, p, m):
    """Raises the error for the first argument of :func:`sample_tokens` that will not do."""
    who = "sample_tokens"
    if not logits.is_cuda:
        raise RuntimeError(f"{who}: CUDA tensors only (sm_100a kernels, no CPU path)")
    if logits.dtype not in _FLOATS:
        raise RuntimeError(f"{who}: expected logits to be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() != 2 or not 1 <= logits.size(1) <= MAX_V or (logits.size(1) > 1 and logits.stride(1) != 1) \
            or (logits.size(0) > 1 and logits.stride(0) < logits.size(1)):
        raise RuntimeError(f"{who}: expected logits to be (rows, V) with contiguous rows and 1 <= V <= {MAX_V}")
    if uniforms.dtype != torch.float32 or uniforms.shape != (logits.size(0),) or not uniforms.is_contiguous() \
            or uniforms.device != logits.device:
        raise RuntimeError(f"{who}: uniforms must be a contiguous float32 tensor with one value per row on {logits.device}")
    if t_ptr is None and not 0.0 <= t <= 1e6:
        raise RuntimeError(f"{who}: temperature must be in [0, 1e6], got {t}")
    if p != p or m != m:
        raise RuntimeError(f"{who}: top_p and min_p must be numbers")
    if not -(1 << 31) <= k < (1 << 31):
        raise RuntimeError(f"{who}: top_k must fit 32 bits, got {k}")
