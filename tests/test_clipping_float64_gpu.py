"""Clipping of float64 gradients in 64 bits.

Tolerance, derived: the squares (one rounding each) of at most 100 000 elements are added
along chains of at most 8 per thread, 5 + 8 across a block, then 5 + 5 + 8 across the
blocks' sums: 40 roundings, and half of that in the root.  The 1e-6, the division and the
product add three: 48 * 2^-53 of the value covers all of it."""
import math

import pytest
import torch

import optimized_transducer_b200 as ot

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64


def _grads(sizes):
    g = torch.Generator().manual_seed(len(sizes))
    return [torch.randn(n, dtype=F64, generator=g) for n in sizes]


def _norm(tensors, p):
    a = torch.cat([t.reshape(-1) for t in tensors]).abs().tolist()
    return max(a) if p == math.inf else (math.fsum(a) if p == 1 else math.sqrt(math.fsum(x * x for x in a)))


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("sizes", [[1], [5, 1, 1023, 2049], [100000], [17] * 60])
def test_the_factor_keeps_53_bits(sizes, p):
    cpu = _grads(sizes)
    norm = _norm(cpu, p)
    for limit in (norm / 3, norm * (1 - 1e-9), norm * 2):
        factor = min(1.0, limit / (norm + 1e-6))
        for out_of_place in (False, True):
            grads = [t.to(DEV) for t in cpu]
            outs = [torch.empty_like(t) for t in grads] if out_of_place else None
            ot.clip_grad_norm_(grads, limit, norm_type=p, out=outs)
            for got, t in zip(outs or grads, cpu):
                assert bool(((got.cpu() - t * factor).abs() <= 48 * 2.0 ** -53 * t.abs()).all())


def test_float64_beside_other_types():
    """Each tensor is scaled in its own arithmetic, by one factor."""
    cpu = _grads([3000, 500])
    f32 = torch.randn(700, generator=torch.Generator().manual_seed(9))
    grads = [cpu[0].to(DEV), f32.to(DEV), cpu[1].to(DEV)]
    norm = _norm([cpu[0], f32.double(), cpu[1]], 2)
    ot.clip_grad_norm_(grads, norm / 7)
    factor = norm / 7 / (norm + 1e-6)
    # float32 elements are squared and added in float32 in groups of 32: 33 * 2^-24 of their part of the sum
    for got, t in ((grads[0], cpu[0]), (grads[2], cpu[1])):
        share = float((f32.double() ** 2).sum()) / norm ** 2
        tol = 48 * 2.0 ** -53 + 33 * 2.0 ** -24 * share
        assert bool(((got.cpu() - t * factor).abs() <= tol * t.abs() * factor).all())
        ratio = got.cpu() / t                        # one factor for all, to the rounding of the product and the quotient
        assert float(ratio.max() / ratio.min()) - 1 <= 4 * 2.0 ** -53


@pytest.mark.parametrize("out_type", [torch.bfloat16, torch.float16, torch.float32])
def test_float64_gradients_are_rounded_once_into_smaller_types(out_type):
    """A hair above or below the middle of two neighbours: rounded by way of float32 the hair
    is lost and the tie goes to the even one."""
    step = torch.finfo(out_type).eps                  # from 1 to its neighbour
    hair = 2.0 ** -40
    above, below = 1 + step / 2 + hair, 1 + 1.5 * step - hair
    want = {above: 1 + step, below: 1 + step, -above: -1 - step, -below: -1 - step, 1 + step / 2: 1.0, 1 + 1.5 * step: 1 + 2 * step}
    g = torch.tensor(list(want) * 40, dtype=F64)
    out = torch.empty(g.numel(), dtype=out_type, device=DEV)
    ot.clip_grad_norm_([g.to(DEV)], 1e9, out=[out])   # the factor is 1
    assert torch.equal(out.cpu().double(), torch.tensor(list(want.values()) * 40, dtype=F64))
    # odd pieces: the elements that vectors leave over
    for n in (1, 3, 7):
        ot.clip_grad_norm_([g[:n].to(DEV)], 1e9, out=[out[1:1 + n]])
        assert torch.equal(out[1:1 + n].cpu().double(), torch.tensor(list(want.values()) * 40, dtype=F64)[:n])
