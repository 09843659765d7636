"""What the output-layer entry points refuse, without a GPU."""
import ctypes

import pytest
import torch

import optimized_transducer_b200 as ot
from optimized_transducer_b200 import _lib


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 16), torch.zeros(3, 16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ot.joiner_logits(x, w)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ot.quantize_weight(w)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ot.Fp8Weight(w.to(torch.float8_e4m3fn), torch.ones(1, 1))
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        ot.Fp8Weight(w, torch.ones(1, 1))


def _memory():
    buf = ctypes.create_string_buffer(4096)
    return buf, (ctypes.addressof(buf) + 255) & ~255


def test_quantiser_argument_errors():
    lib = _lib.load()
    keep, p = _memory()

    def call(x=p, rows=4, cols=20, ld=20, flags=0, mode=_lib.FP8_ROWS, q=p, pitch=32, s=p, qt=None, tp=0, st=None, part=None, tot=None):
        return lib.ot_b200_fp8_quantize(x, rows, cols, ld, flags, mode, q, pitch, s, qt, tp, st, part, tot, None)

    bad = [dict(x=None), dict(rows=0), dict(cols=0), dict(rows=1 << 31), dict(ld=19), dict(flags=_lib.FP64),
           dict(flags=_lib.BF16 | _lib.FP16), dict(mode=5), dict(mode=-1), dict(q=None), dict(q=p + 8), dict(pitch=20), dict(pitch=16),
           dict(s=None), dict(mode=_lib.FP8_SQUARES_BOTH), dict(mode=_lib.FP8_SQUARES_BOTH, qt=p, tp=24, st=p),
           dict(mode=_lib.FP8_SQUARES_BOTH, qt=p, tp=144, st=p),
           dict(part=p, tot=p), dict(mode=_lib.FP8_ROWS_AND_COLUMNS, qt=p, tp=16, st=p, part=p)]
    for kw in bad:
        assert call(**kw) == _lib.ERR_ARGUMENT, kw
        assert "ot_b200_fp8_quantize" in _lib.last_error()


def test_product_argument_errors():
    lib = _lib.load()
    keep, p = _memory()

    def call(a=p, ap=32, sa=p, b=p, bp=32, sb=p, M=4, N=5, K=20, flags=0, ws=None, wb=0, out=p):
        return lib.ot_b200_fp8_matmul(a, ap, sa, b, bp, sb, None, M, N, K, flags, ws, wb, out, None)

    bad = [dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(out=None), dict(a=p + 8), dict(b=p + 1), dict(ap=24),
           dict(bp=16), dict(M=0), dict(N=0), dict(K=0), dict(M=1 << 31), dict(flags=_lib.FP64), dict(out=p + 2)]
    for kw in bad:
        assert call(**kw) == _lib.ERR_ARGUMENT, kw
    long_k = dict(M=10, N=10, K=100000, ap=100000, bp=100000)
    assert call(**long_k) == _lib.ERR_WORKSPACE
    need = ctypes.c_uint64()
    assert lib.ot_b200_fp8_matmul_workspace_bytes(10, 10, 100000, ctypes.byref(need)) == _lib.OK and need.value > 0
    assert call(**long_k, ws=p, wb=need.value - 1) == _lib.ERR_WORKSPACE
    assert lib.ot_b200_fp8_matmul_workspace_bytes(100000, 500, 512, ctypes.byref(need)) == _lib.OK and need.value == 0


def test_forward_in_one_call_argument_errors():
    lib = _lib.load()
    keep, p = _memory()
    need = ctypes.c_uint64()
    assert lib.ot_b200_joiner_logits_workspace_bytes(0, 20, 5, ctypes.byref(need)) == _lib.ERR_ARGUMENT
    assert lib.ot_b200_joiner_logits_workspace_bytes(4, 20, 5, ctypes.byref(need)) == _lib.OK and need.value >= 4 * 32 + 16

    def call(x=p, rows=4, d=20, ld=20, xf=0, w=p, wp=32, ws_=p, v=5, of=0, ws=p, wb=need.value, out=p):
        return lib.ot_b200_joiner_logits(x, rows, d, ld, xf, w, wp, ws_, v, None, of, ws, wb, out, None)

    for kw in (dict(ws=None), dict(ws=p + 16), dict(wb=need.value - 1)):
        assert call(**kw) == _lib.ERR_WORKSPACE, kw
    for kw in (dict(x=None), dict(rows=0), dict(d=0), dict(v=0), dict(ld=19), dict(xf=_lib.FP64)):
        assert call(**kw) == _lib.ERR_ARGUMENT, kw


def test_training_calls_argument_errors():
    lib = _lib.load()
    keep, p = _memory()
    n = [ctypes.c_uint64() for _ in range(3)]
    out = [ctypes.byref(x) for x in n]
    assert lib.ot_b200_joiner_train_bytes(0, 20, 5, 1, 1, 1, *out) == _lib.ERR_ARGUMENT
    assert lib.ot_b200_joiner_train_bytes(4, 20, 5, 1, 1, 1, None, *out[1:]) == _lib.ERR_ARGUMENT
    assert lib.ot_b200_joiner_train_bytes(4, 20, 5, 0, 0, 1, *out) == _lib.OK and n[0].value == 0
    assert lib.ot_b200_joiner_train_bytes(4, 20, 5, 1, 1, 1, *out) == _lib.OK and all(x.value for x in n)
    fwd = lambda x=p, rows=4, ld=20, saved=p, ws=p, o=p: lib.ot_b200_joiner_train_forward(  # noqa: E731
        x, rows, 20, ld, 0, p, 5, 20, 0, None, 0, 1, 1, saved, ws, o, None)
    assert fwd(ws=None) == _lib.ERR_WORKSPACE and fwd(saved=p + 16) == _lib.ERR_WORKSPACE
    assert fwd(rows=0) == _lib.ERR_ARGUMENT
    bwd = lambda g=p, rows=4, ld=5, saved=p, flags=0, ws=p: lib.ot_b200_joiner_train_backward(  # noqa: E731
        g, rows, 5, ld, 0, 20, saved, p, 0, p, 0, p, flags, ws, None)
    assert bwd(ws=None) == _lib.ERR_WORKSPACE and bwd(saved=None) == _lib.ERR_WORKSPACE
    assert bwd(g=None) == _lib.ERR_ARGUMENT and bwd(ld=4) == _lib.ERR_ARGUMENT and bwd(flags=_lib.BF16) == _lib.ERR_ARGUMENT


def test_a_handle_of_things_that_are_no_tensors_is_refused():
    q = torch.zeros(3, 16).to(torch.float8_e4m3fn)
    for data, scale, what in ((None, torch.ones(1, 1), "data"), (q, None, "scale"), (q, [1.0], "scale"), ("w", 3, "data")):
        with pytest.raises(RuntimeError, match=f"expected {what} to be a tensor"):
            ot.Fp8Weight(data, scale)


def test_training_calls_refuse_small_buffers():
    lib = _lib.load()
    keep, p = _memory()
    n = [ctypes.c_uint64() for _ in range(3)]
    assert lib.ot_b200_joiner_train_bytes(4, 20, 5, 1, 1, 1, *[ctypes.byref(x) for x in n]) == _lib.OK
    saved, forward, backward = (x.value for x in n)
    fwd = lambda s=saved, w=forward: lib.ot_b200_joiner_train_forward_sized(  # noqa: E731
        p, 4, 20, 20, 0, p, 5, 20, 0, None, _lib.FP64, 1, 1, p, s, p, w, p, None)
    bwd = lambda s=saved, w=backward: lib.ot_b200_joiner_train_backward_sized(  # noqa: E731
        p, 4, 5, 5, 0, 20, p, s, p, 0, p, 0, p, _lib.FP64, p, w, None)
    for call, need in ((fwd, forward), (bwd, backward)):
        for kw in (dict(s=saved - 1), dict(w=need - 1), dict(s=0), dict(w=0)):
            assert call(**kw) == _lib.ERR_WORKSPACE, kw
            assert "fewer than" in _lib.last_error()
    assert bwd() == _lib.ERR_ARGUMENT                 # past the sizes: the flag that it does not know
