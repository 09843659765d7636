"""Waits of the fused projection kernels that run out (OT_B200_WAIT_LIMIT lowers the number
of polls after which one does; 0: every wait gives up at once).  Nothing faults or hangs: a
block that gives up waits for its copies and MMAs in flight, says so, and returns."""
import pytest
import torch

import optimized_transducer_b200 as ot
from test_fused_linear_gpu import DEV, _case

pytestmark = pytest.mark.gpu

# fewer K blocks than the ring has stages, more of them, several column tiles and row tiles per block
SHAPES = [(1, 3, (5, 12), (2, 6), 64, 40, False), (2, 4, (20, 40), (5, 12), 512, 500, True),
          (3, 12, (90, 120), (20, 30), 200, 1032, True)]


def _on_gpu(shape):
    x, w, b, tg, T, U, _ = _case(*shape)
    return [t.to(DEV) if t is not None else None for t in (x, w, b, *(torch.from_numpy(a) for a in (tg, T, U)))]


@pytest.mark.parametrize("limit", [0, 1, 2, 4, 8, 32])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, limit, monkeypatch):
    x, w, b, tg, T, U = _on_gpu(shape)
    want = ot.joiner_scores(x, w, b, tg, T, U, 0)
    monkeypatch.setenv("OT_B200_WAIT_LIMIT", str(limit))
    if limit == 0:
        with pytest.raises(RuntimeError, match="did not complete in time"):
            ot.joiner_scores(x, w, b, tg, T, U, 0)
    else:
        try:                                          # either every block got through or the call says so
            assert torch.equal(ot.joiner_scores(x, w, b, tg, T, U, 0), want)
        except RuntimeError as e:
            assert "did not complete in time" in str(e)
    monkeypatch.undo()
    assert torch.equal(ot.joiner_scores(x, w, b, tg, T, U, 0), want)


@pytest.mark.parametrize("limit", [0, 1, 2, 4, 8, 32])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(shape, limit, monkeypatch):
    x, w, b, tg, T, U = _on_gpu(shape)
    x.requires_grad_(True)
    loss = ot.joiner_loss(x, w, b, tg, T, U, 0)
    (want,) = torch.autograd.grad(loss, x, retain_graph=True)
    torch.cuda.synchronize()
    monkeypatch.setenv("OT_B200_WAIT_LIMIT", str(limit))
    (got,) = torch.autograd.grad(loss, x, retain_graph=True)
    torch.cuda.synchronize()
    monkeypatch.undo()
    lost = torch.isnan(got)
    assert bool((lost | (got == want)).all()) and (limit > 0 or bool(lost.all()))
    if bool(lost.any()):
        with pytest.raises(RuntimeError, match="did not complete in time"):
            ot.check_inputs(DEV)
    ot.check_inputs(DEV)
    assert torch.equal(torch.autograd.grad(loss, x)[0], want)
