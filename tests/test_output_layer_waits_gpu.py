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
