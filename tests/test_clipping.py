"""What the clipping entry points refuse, without a GPU."""
import ctypes

import pytest
import torch

import optimized_transducer_b200 as ot
from optimized_transducer_b200 import _lib


def test_refusals():
    g = [torch.ones(3)]
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ot.grad_norm(g)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ot.clip_grad_norm_(g, 1.0)
    with pytest.raises(RuntimeError, match="no gradients"):
        ot.grad_norm([])
    with pytest.raises(RuntimeError, match="norm_type"):
        ot.grad_norm(g, 3.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(RuntimeError, match="max_norm"):
            ot.clip_grad_norm_(g, bad)


def test_argument_errors():
    lib = _lib.load()
    need = ctypes.c_uint64()
    assert lib.ot_b200_clip_workspace_bytes(-1, ctypes.byref(need)) == _lib.ERR_ARGUMENT
    assert lib.ot_b200_clip_workspace_bytes(2, ctypes.byref(need)) == _lib.OK and need.value > 0
    buf = ctypes.create_string_buffer(need.value + 4096)
    p = (ctypes.addressof(buf) + 255) & ~255

    def call(n=2, ptrs=(p, p + 64), counts=(4, 4), types=(0, 0), outs=None, out_types=None, kind=_lib.NORM_2, apply=1, limit=1.0,
             ws=p + 512, wb=need.value, norm=p + 256):
        array = lambda t, v: None if v is None else (t * len(v))(*v)  # noqa: E731
        return lib.ot_b200_clip_gradients(n, array(ctypes.c_void_p, ptrs), array(ctypes.c_int64, counts), array(ctypes.c_int32, types),
                                          array(ctypes.c_void_p, outs), array(ctypes.c_int32, out_types), kind, apply, limit, ws, wb, norm, None)

    bad = [dict(n=-1), dict(ptrs=None), dict(counts=None), dict(types=None), dict(norm=None), dict(kind=3), dict(limit=-1.0),
           dict(limit=float("nan")), dict(types=(0, 3)), dict(counts=(4, -1)), dict(ptrs=(p, 0)), dict(ptrs=(p, p + 66)),
           dict(ptrs=(p, p)), dict(ptrs=(p, p + 8)), dict(outs=(p + 128, p + 192)), dict(outs=(p + 128, p + 192), out_types=(0, 0), apply=0),
           dict(outs=(p + 128, p + 136), out_types=(0, 0)), dict(outs=(p + 64, p + 128), out_types=(0, 0))]
    for kw in bad:
        assert call(**kw) == _lib.ERR_ARGUMENT, kw
        assert "ot_b200_clip_gradients" in _lib.last_error()
    for kw in (dict(ws=None), dict(wb=need.value - 1), dict(ws=p + 516)):
        assert call(**kw) == _lib.ERR_WORKSPACE, kw


def test_parameters_in_place_of_their_gradients_are_refused():
    p = torch.nn.Parameter(torch.ones(3))
    with pytest.raises(RuntimeError, match="not the parameters"):
        ot.clip_grad_norm_([torch.ones(3), p], 1.0)
    with pytest.raises(RuntimeError, match="not the parameters"):
        ot.clip_grad_norm_([torch.ones(3)], 1.0, out=[p])


def test_a_norm_that_should_carry_a_gradient_is_refused():
    p = torch.nn.Parameter(torch.ones(3))
    for t in (p, 2 * p, torch.autograd.grad((p ** 3).sum(), p, create_graph=True)[0]):
        with pytest.raises(RuntimeError, match="no derivative"):
            ot.grad_norm([torch.ones(3), t])
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensors only"):   # as far as a CPU tensor comes
            ot.grad_norm([t])


def test_nothing_to_clip_is_a_norm_of_zero_as_in_torch():
    want = torch.nn.utils.clip_grad_norm_([torch.nn.Parameter(torch.ones(3))], 1.0)   # no gradient anywhere
    for got in (ot.clip_grad_norm_([], 1.0), ot.clip_grad_norm_((t for t in ()), 1.0, norm_type=float("inf")), ot.clip_grad_norm_([], 0.0, out=[])):
        assert got.shape == want.shape and got.dtype == want.dtype and got.device == want.device and float(got) == float(want) == 0.0
    with pytest.raises(RuntimeError, match="norm_type"):
        ot.clip_grad_norm_([], 1.0, norm_type=3.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        ot.clip_grad_norm_([], -1.0)
    with pytest.raises(RuntimeError, match="no gradients|one output per gradient"):
        ot.clip_grad_norm_([], 1.0, out=[torch.ones(3)])
