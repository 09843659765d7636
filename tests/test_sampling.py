"""What the sampling entry points refuse, without a GPU."""
import ctypes

import pytest
import torch

import optimized_transducer_b200 as ot
from optimized_transducer_b200 import _lib


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ot.sample_tokens(torch.zeros(2, 5), torch.zeros(2))


def test_argument_errors():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) & ~255

    def call(x=p, rows=4, v=20, ld=20, flags=0, u=p, tp=None, t=1.0, kp=None, k=0, pp=None, top_p=1.0, mp=None, min_p=0.0, tok=p, lp=p):
        return lib.ot_b200_sample(x, rows, v, ld, flags, u, tp, t, kp, k, pp, top_p, mp, min_p, tok, lp, None)

    nan = float("nan")
    bad = [dict(x=None), dict(u=None), dict(tok=None), dict(lp=None), dict(rows=0), dict(v=0), dict(v=262145, ld=262145), dict(ld=19),
           dict(flags=_lib.FP64), dict(flags=_lib.BF16 | _lib.FP16), dict(t=-0.5), dict(t=2e6), dict(t=nan), dict(top_p=nan), dict(min_p=nan)]
    for kw in bad:
        assert call(**kw) == _lib.ERR_ARGUMENT, kw
        assert "ot_b200_sample" in _lib.last_error()
