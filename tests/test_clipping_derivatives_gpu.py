"""The norm and the clipping have no derivative: what would lose one is refused."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import optimized_transducer_b200 as ot

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_gradient_that_is_part_of_a_graph():
    x = torch.full((4,), 2.0, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)    # 12 each; a penalty on its norm would be constant
    with pytest.raises(RuntimeError, match="no derivative"):
        ot.grad_norm([g])
    with pytest.raises(RuntimeError, match="part of a graph"):
        ot.clip_grad_norm_([g], 1.0)
    assert float(ot.grad_norm([g.detach()])) == 24.0
    with torch.no_grad():
        assert float(ot.grad_norm([g])) == 24.0
        assert float(ot.grad_norm(torch.nn.Parameter(torch.full((4,), 3.0, device=DEV)))) == 6.0


def test_forward_mode():
    g = torch.full((4,), 3.0, device=DEV)
    with fwd.dual_level():
        d = fwd.make_dual(g, torch.ones_like(g))
        for call in (lambda: ot.grad_norm([g, d]), lambda: ot.clip_grad_norm_([d], 1.0), lambda: ot.clip_grad_norm_([g], 1.0, out=[d])):
            with pytest.raises(RuntimeError, match="forward-mode tangent"):
                call()
        assert float(ot.grad_norm([fwd.unpack_dual(d).primal])) == 6.0
    assert torch.equal(g, torch.full((4,), 3.0, device=DEV))
