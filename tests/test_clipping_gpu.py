"""``grad_norm`` and ``clip_grad_norm_`` against float64 sums.  Tolerance of the norm: at
most 32 terms are added in float32 before a sum goes to float64, so a sum is off by at
most 33 * 2^-24 of itself (squares included), the 2-norm by half of that, and the result is
rounded to float32 once: 34 * 2^-24 relative covers all three norms.  A clipped element adds
the factor's rounding to float32 and its own to the output type: (36 * 2^-24 + eps(out)/2) of itself."""
import math

import numpy as np
import pytest
import torch

import optimized_transducer_b200 as ot

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]
TOL = 34 * 2.0 ** -24


def norm64(tensors, p):
    flat = torch.cat([t.detach().double().cpu().reshape(-1) for t in tensors])
    if p == math.inf:
        return float(flat.abs().max()) if flat.numel() else 0.0
    return float((flat.abs() ** p).sum() ** (1 / p))


def tensors_of(rng, sizes, types, scale=1.0):
    return [torch.from_numpy(rng.standard_normal(n) * scale).to(types[i % len(types)]).to(DEV) for i, n in enumerate(sizes)]


SIZES = [[1], [0, 7], [5, 1, 1023, 1024, 1025], [2048, 2049, 16, 100003], [300001], [3] * 100, [17 * i + 1 for i in range(1100)]]


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("types", [[t] for t in TYPES] + [TYPES])
def test_norm_and_clipping(types, p):
    rng = np.random.default_rng(int(p) if p < 9 else 9)
    for sizes in SIZES:
        grads = tensors_of(rng, sizes, types)
        keep = [g.clone() for g in grads]
        want = norm64(grads, p)
        got = ot.grad_norm(grads, p)
        assert got.dtype == torch.float32 and got.dim() == 0
        assert abs(float(got) - want) <= TOL * want
        for limit in (0.37 * want, 2.0 * want + 1.0):
            grads = [g.clone() for g in keep]
            norm = ot.clip_grad_norm_(grads, limit, norm_type=p)
            assert torch.equal(norm, got)
            factor = min(1.0, limit / (want + 1e-6))
            for g, k in zip(grads, keep):
                if factor == 1.0:
                    assert torch.equal(g, k)
                    continue
                exact = k.double() * factor
                tol = (36 * 2.0 ** -24 + torch.finfo(g.dtype).eps / 2) * exact.abs() + torch.finfo(g.dtype).tiny
                assert bool(((g.double() - exact).abs() <= tol).all())


@pytest.mark.parametrize("out_type", TYPES)
def test_clipped_gradients_elsewhere(out_type):
    rng = np.random.default_rng(3)
    grads = tensors_of(rng, [1000, 1, 4097, 33], TYPES)
    keep = [g.clone() for g in grads]
    outs = [torch.full_like(g, 7.0, dtype=out_type) for g in grads]
    want = norm64(grads, 2.0)
    for limit in (0.5 * want, 5.0 * want):
        ot.clip_grad_norm_(grads, limit, out=outs)
        factor = min(1.0, limit / (want + 1e-6))
        for g, k, o in zip(grads, keep, outs):
            assert torch.equal(g, k)
            exact = k.double() * factor
            tol = (36 * 2.0 ** -24 + torch.finfo(out_type).eps / 2 + torch.finfo(torch.float32).eps / 2) * exact.abs() + torch.finfo(out_type).tiny
            assert bool(((o.double() - exact).abs() <= tol).all())
    # an output may be its own gradient; the others go elsewhere
    ot.clip_grad_norm_(grads, 0.5 * want, out=[grads[0], *outs[1:]])
    assert torch.equal(grads[0], (keep[0].double() * 0.5).float()) or bool((grads[0] - keep[0] * 0.5).abs().max() <= 1e-5)


def test_views_of_one_buffer_at_every_alignment():
    rng = np.random.default_rng(4)
    for dtype in TYPES:
        flat = torch.from_numpy(rng.standard_normal(60000)).to(dtype).to(DEV)
        keep = flat.clone()
        cuts = [0, 1, 4, 9, 16, 31, 2080, 5000, 5001, 23456, 59999]
        views = [flat[a:b] for a, b in zip(cuts[:-1], cuts[1:])]
        want = norm64(views, 2.0)
        norm = ot.clip_grad_norm_(views, 0.25 * want)
        assert abs(float(norm) - want) <= TOL * want
        assert torch.equal(flat[59999:], keep[59999:])          # behind the last view
        exact = keep[:59999].double() * (0.25 * want / (want + 1e-6))
        tol = (36 * 2.0 ** -24 + torch.finfo(dtype).eps / 2) * exact.abs() + torch.finfo(dtype).tiny
        assert bool(((flat[:59999].double() - exact).abs() <= tol).all())
        out = torch.zeros(59999 + 3, dtype=torch.float32, device=DEV)
        ot.clip_grad_norm_([keep[5:50000]], 1.0, out=[out[3:3 + 49995]])
        assert float(out[:3].abs().sum()) == 0 and float(out[3 + 49995:].abs().sum()) == 0


def test_extreme_values():
    big = [torch.full((1000,), 1e30, device=DEV), torch.full((10,), -1e-30, device=DEV)]
    assert abs(float(ot.grad_norm(big)) / (1e30 * math.sqrt(1000)) - 1) <= TOL + 1e-6
    small = [torch.full((1000,), 1e-30, device=DEV), torch.zeros(100, device=DEV)]
    v = float(torch.tensor(1e-30))
    assert abs(float(ot.grad_norm(small)) / (v * math.sqrt(1000)) - 1) <= TOL
    assert float(ot.grad_norm([torch.zeros(5000, device=DEV)])) == 0.0
    zeros = torch.zeros(3000, device=DEV)
    assert float(ot.clip_grad_norm_([zeros], 0.0)) == 0.0 and float(zeros.abs().sum()) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_norms_that_are_not_finite_scale_as_in_torch(p, dtype):
    for bad in (math.inf, -math.inf, math.nan):
        g = torch.ones(3000, dtype=dtype, device=DEV)
        g[1234] = bad
        ref = torch.nn.Parameter(torch.zeros(3000, dtype=dtype, device=DEV))
        ref.grad = g.clone()
        want = torch.nn.utils.clip_grad_norm_([ref], 1.0, norm_type=p)
        got = ot.clip_grad_norm_([g], 1.0, norm_type=p)
        assert math.isnan(float(got)) == math.isnan(float(want)) and (math.isnan(float(got)) or float(got) == math.inf)
        assert torch.equal(torch.isnan(g), torch.isnan(ref.grad))
        assert torch.equal(torch.nan_to_num(g), torch.nan_to_num(ref.grad))


def test_same_as_torch_on_a_model():
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(80, 300), torch.nn.Tanh(), torch.nn.Linear(300, 501)).to(DEV)
    net(torch.randn(40, 80, device=DEV)).square().sum().backward()
    grads = [p.grad.clone() for p in net.parameters()]
    want = torch.nn.utils.clip_grad_norm_(net.parameters(), 5.0)
    got = ot.clip_grad_norm_(grads, 5.0)
    assert abs(float(got) / float(want) - 1) <= 1e-5
    for g, p in zip(grads, net.parameters()):
        assert torch.allclose(g, p.grad, rtol=1e-5, atol=0)


def test_dense_tensors_in_any_order_of_dimensions():
    rng = np.random.default_rng(5)
    g = torch.from_numpy(rng.standard_normal((30, 50))).float().to(DEV)
    t = g.t()
    want = norm64([g], 2.0)
    assert abs(float(ot.grad_norm([t])) - want) <= TOL * want
    ot.clip_grad_norm_([t], want / 2)
    assert abs(norm64([g], 2.0) / want - 0.5) <= 1e-5
    with pytest.raises(RuntimeError, match="dense"):
        ot.grad_norm([g[:, ::2]])
    with pytest.raises(RuntimeError, match="dense"):
        ot.clip_grad_norm_([torch.zeros(1, 4, device=DEV).expand(3, 4)], 1.0)


def test_what_overlaps_is_refused():
    g = torch.ones(100, device=DEV)
    for grads, out in (([g, g], None), ([g[:60], g[50:]], None), ([g], [torch.ones(100, device=DEV)[:100]] * 1),):
        if out is None:
            with pytest.raises(RuntimeError, match="overlap"):
                ot.clip_grad_norm_(grads, 1.0)
        else:
            ot.clip_grad_norm_(grads, 1.0, out=out)
    h = torch.ones(100, device=DEV)
    with pytest.raises(RuntimeError, match="overlap"):
        ot.clip_grad_norm_([g[:50], g[50:]], 1.0, out=[g[50:], h[:50]])
    with pytest.raises(RuntimeError, match="overlap"):
        ot.clip_grad_norm_([g[:50], g[50:]], 1.0, out=[h[:50], h[25:75]])
    assert torch.equal(g, torch.ones(100, device=DEV))
    assert abs(float(ot.grad_norm([g, g])) - math.sqrt(200)) <= 1e-4      # only read: allowed


def test_nothing_to_sum():
    empty = torch.empty(0, device=DEV)
    assert float(ot.grad_norm([empty])) == 0.0
    assert float(ot.clip_grad_norm_([empty, torch.empty(3, 0, device=DEV)], 1.0)) == 0.0
    assert float(ot.grad_norm(torch.full((4,), 3.0, device=DEV))) == 6.0       # one tensor, not in a list


def test_the_version_counter_moves():
    g = torch.ones(10, device=DEV)
    v = g._version
    ot.clip_grad_norm_([g], 0.5)
    assert g._version > v


def test_same_bits_on_another_stream_and_in_a_captured_graph():
    rng = np.random.default_rng(6)
    grads = tensors_of(rng, [100000, 3, 70001], [torch.float32, torch.bfloat16])
    outs = [torch.empty_like(g, dtype=torch.float32) for g in grads]
    step = lambda: ot.clip_grad_norm_(grads, 3.0, out=outs)  # noqa: E731
    want = [step().clone()] + [o.clone() for o in outs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        n = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip([n] + outs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for g in grads:
        g.mul_(2)
    graph.replay()
    assert abs(float(held) / float(want[0]) - 2) <= 1e-5
    assert all(torch.allclose(a, b, rtol=1e-5) for a, b in zip(outs, want[1:]))
