"""Waits of the 8-bit product that run out (OT_B200_WAIT_LIMIT lowers the number of polls
after which one does; 0: every wait gives up at once).  Nothing faults or hangs: a block
that gives up waits for its copies and MMAs in flight, fills its tiles with NaN, leaves the
record that the next call raises, and returns."""
import numpy as np
import pytest
import torch

import optimized_transducer_b200 as ot

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _operands(rows, d, v):
    rng = np.random.default_rng(rows + d + v)
    x = torch.from_numpy(rng.standard_normal((rows, d))).to(torch.bfloat16).to(DEV)
    w = ot.quantize_weight(torch.from_numpy(rng.standard_normal((v, d)) / np.sqrt(d)).float().to(DEV))
    return x, w, torch.from_numpy(rng.standard_normal(v)).float().to(DEV)


# fewer K blocks than the ring has stages (the producer never waits), exactly one block, more
# blocks than stages, several tiles per block; columns whose rows leave by TMA and by plain stores
SHAPES = [(8, 512, 500), (8, 100, 33), (200, 2000, 300), (5000, 300, 5000), (5000, 300, 5003)]


@pytest.mark.parametrize("shape", SHAPES)
def test_every_wait_gives_up_at_once(shape, monkeypatch):
    x, w, b = _operands(*shape)
    want = ot.joiner_logits(x, w, b)
    monkeypatch.setenv("OT_B200_WAIT_LIMIT", "0")
    for out in (torch.bfloat16, torch.float32):
        y = ot.joiner_logits(x, w, b, out_dtype=out)
        torch.cuda.synchronize()
        assert bool(torch.isnan(y).all())
        with pytest.raises(RuntimeError, match="did not complete in time"):
            ot.check_inputs(DEV)
    monkeypatch.setenv("OT_CHECKS", "0")             # nothing recorded, the results still say it
    assert bool(torch.isnan(ot.joiner_logits(x, w, b)).all())
    monkeypatch.undo()
    ot.check_inputs(DEV)
    assert torch.equal(ot.joiner_logits(x, w, b), want)


def test_products_in_pieces_give_up_too(monkeypatch):
    """The weight's gradient: a long contraction cut into pieces whose sums are joined."""
    x = torch.randn(9000, 64, device=DEV, requires_grad=True)
    w = torch.randn(40, 64, device=DEV, requires_grad=True)
    g = torch.randn(9000, 40, device=DEV, dtype=torch.bfloat16)
    y = ot.joiner_logits(x, w)
    want = torch.autograd.grad(y, (x, w), g, retain_graph=True)
    monkeypatch.setenv("OT_B200_WAIT_LIMIT", "0")
    monkeypatch.setenv("OT_CHECKS", "0")
    z = ot.joiner_logits(x, w)
    gx, gw = torch.autograd.grad(z, (x, w), g)
    assert bool(torch.isnan(z).all()) and bool(torch.isnan(gx).all()) and bool(torch.isnan(gw).all())
    monkeypatch.undo()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), g), want))


@pytest.mark.parametrize("limit", [1, 2, 4, 8, 32])
def test_waits_that_give_up_halfway(limit, monkeypatch):
    """Some blocks get through and some do not: every entry is right or a NaN, and a NaN is
    never left without a record."""
    for shape in SHAPES[2:]:
        x, w, b = _operands(*shape)
        want = ot.joiner_logits(x, w, b)
        monkeypatch.setenv("OT_B200_WAIT_LIMIT", str(limit))
        y = ot.joiner_logits(x, w, b)
        torch.cuda.synchronize()
        monkeypatch.delenv("OT_B200_WAIT_LIMIT")
        lost = torch.isnan(y)
        assert bool((lost | (y == want)).all())
        if bool(lost.any()):
            with pytest.raises(RuntimeError, match="did not complete in time"):
                ot.check_inputs(DEV)
        else:
            ot.check_inputs(DEV)
        assert torch.equal(ot.joiner_logits(x, w, b), want)


def test_a_pending_record_is_raised_before_anything_is_launched(monkeypatch):
    """The record of a failed call reaches the next call at its entry: none of that call's buffers is written."""
    import ctypes

    from optimized_transducer_b200 import _lib

    lib, rows, d, v = _lib.load(), 50, 96, 40
    x, w, b = _operands(rows, d, v)
    wt = torch.randn(v, d, device=DEV)
    g = torch.randn(rows, v, device=DEV)
    n = [ctypes.c_uint64() for _ in range(4)]
    _lib.check(lib.ot_b200_joiner_train_bytes(rows, d, v, 1, 1, 1, *[ctypes.byref(i) for i in n[:3]]))
    _lib.check(lib.ot_b200_joiner_logits_workspace_bytes(rows, d, v, ctypes.byref(n[3])))
    saved, fwd, bwd, ws = (torch.full((i.value,), 0xAB, dtype=torch.uint8, device=DEV) for i in n)
    out, gx, gw, gb = (torch.full(s, 7.0, device=DEV) for s in ((rows, v), (rows, d), (v, d), (v,)))
    buffers = (saved, fwd, bwd, ws, out, gx, gw, gb)
    stream, on = torch.cuda.current_stream().cuda_stream, _lib.REPORT_ERRORS
    calls = [
        lambda: lib.ot_b200_joiner_logits(x.data_ptr(), rows, d, d, _lib.BF16, w.data.data_ptr(), w.data.stride(0), w.scale.data_ptr(), v,
                                          b.data_ptr(), on, ws.data_ptr(), ws.numel(), out.data_ptr(), stream),
        lambda: lib.ot_b200_joiner_train_forward(x.data_ptr(), rows, d, d, _lib.BF16, wt.data_ptr(), v, d, 0, b.data_ptr(), on, 1, 1,
                                                 saved.data_ptr(), fwd.data_ptr(), out.data_ptr(), stream),
        lambda: lib.ot_b200_joiner_train_backward(g.data_ptr(), rows, v, v, 0, d, saved.data_ptr(), gx.data_ptr(), 0, gw.data_ptr(), 0,
                                                  gb.data_ptr(), on, bwd.data_ptr(), stream),
    ]
    for call in calls:
        monkeypatch.setenv("OT_B200_WAIT_LIMIT", "0")
        ot.joiner_logits(x, w, b)
        torch.cuda.synchronize()
        monkeypatch.delenv("OT_B200_WAIT_LIMIT")
        before = [t.clone() for t in buffers]
        assert call() == _lib.ERR_INPUT and "did not complete in time" in _lib.last_error()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(before, buffers))
        assert call() == _lib.OK                      # raised once; this call runs
        torch.cuda.synchronize()
    assert float((gb - g.sum(0)).abs().max()) <= 1e-4
