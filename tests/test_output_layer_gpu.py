"""The output projection in 8-bit floating point (``joiner_logits``, ``ot_b200_fp8_*``)
against its definition in float64.

The quantiser is held to the definition bit by bit: its scales are powers of two, so
x / scale is exact and only the rounding to e4m3 is left.  The products are then
compared with float64 sums of the same quantised values.  Tolerance of one entry,
derived: a product of two e4m3 values is exact in float32; K terms are added, each
addition off by at most 2^-23 of the partial sums' magnitude (the tensor cores may
truncate), the scaling of a block adds two roundings and the bias one, so

    |error| <= (K + 8) * 2^-23 * (sum_k |a_k b_k| + |bias|)  +  eps(out type) / 2 * |y|.
"""
import numpy as np
import pytest
import torch

import optimized_transducer_b200 as ot
from optimized_transducer_b200 import _lib, output_layer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BLOCK = 128
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def e4m3(x, rows_per_block):
    """(bytes as floats, scales per block) of the definition, in numpy float64, written from the format."""
    x = np.asarray(x, np.float64)
    r, c = x.shape
    rb, cb = -(-r // rows_per_block), -(-c // BLOCK)
    pad = np.zeros((rb * rows_per_block, cb * BLOCK))
    pad[:r, :c] = x
    b = pad.reshape(rb, rows_per_block, cb, BLOCK)
    top = np.abs(b).max((1, 3))
    with np.errstate(all="ignore"):
        scale = np.exp2(np.maximum(np.ceil(np.log2(np.where(top > 0, top, 448.0) / 448.0)), -126.0))
        scale[~np.isfinite(top)] = np.nan
        y = b / scale[:, None, :, None]
        step = np.exp2(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
        q = np.rint(y / step) * step
    return q.reshape(pad.shape)[:r, :c], scale


def spread(scale, rows_per_block, shape):
    return np.repeat(np.repeat(scale, rows_per_block, 0)[:shape[0]], BLOCK, 1)[:, :shape[1]]


def value(x, rows_per_block):
    q, s = e4m3(x, rows_per_block)
    return q * spread(s, rows_per_block, q.shape)


def bound(a, b, bias, y, out_dtype):
    mass = np.abs(a) @ np.abs(b).T + (np.abs(bias) if bias is not None else 0)
    return (a.shape[1] + 8) * 2.0 ** -23 * mass + torch.finfo(out_dtype).eps / 2 * np.abs(y) + torch.finfo(out_dtype).tiny


def as_np(t):
    return t.detach().double().cpu().numpy()


def bytes_of(q, cols):
    return q[:, :cols].contiguous().view(torch.float8_e4m3fn).double().cpu().numpy()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1), (1, 130), (5, 500), (127, 128), (129, 33), (300, 260)])
def test_quantiser_bit_by_bit(shape, dtype):
    rng = np.random.default_rng(shape[0] * 1000 + shape[1])
    x = rng.standard_normal(shape) * np.exp(rng.uniform(-12, 8, shape))
    x[rng.random(shape) < 0.05] = 0.0
    x[0, 0] = 448.0 * 2.0 ** -3            # exactly the top of a scale
    if shape[0] > 4:
        x[3] = 0.0                         # a block of zeros
        x[4] = 2.0 ** -140 if dtype == "f32" else 0.0   # far below the smallest scale
    t = torch.from_numpy(x).to(TYPES[dtype]).to(DEV)
    x = as_np(t)
    for mode, plain, trans in ((_lib.FP8_ROWS, 1, 0), (_lib.FP8_SQUARES, 128, 0), (_lib.FP8_ROWS_AND_SQUARES, 1, 128),
                               (_lib.FP8_SQUARES_BOTH, 128, 128), (_lib.FP8_ROWS_AND_COLUMNS, 1, 1)):
        (q, s), qt, _ = output_layer._quantize(t, mode)
        want, scale = e4m3(x, plain)
        np.testing.assert_array_equal(bytes_of(q, shape[1]), want)
        np.testing.assert_array_equal(as_np(s), scale if plain > 1 else scale.T)
        if trans:
            want, scale = e4m3(x.T, trans)
            np.testing.assert_array_equal(bytes_of(qt[0], shape[0]), want)
            np.testing.assert_array_equal(as_np(qt[1]), scale if trans > 1 else scale.T)


SHAPES = [(3, 1, 2), (1, 16, 1), (1, 512, 500), (7, 100, 33), (64, 128, 128), (129, 129, 129), (300, 656, 500), (1000, 72, 1030),
          (40, 1111, 2000), (2500, 512, 515)]


@pytest.mark.parametrize("types", ["f32-f32", "bf16-bf16", "f16-f32", "bf16-f16", "f32-bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_logits(shape, types):
    rows, d, v = shape
    xt, out = (TYPES[t] for t in types.split("-"))
    rng = np.random.default_rng(rows + d + v)
    x = torch.from_numpy(rng.standard_normal((rows, d))).to(xt)
    w = torch.from_numpy(rng.standard_normal((v, d)) / np.sqrt(d)).to(xt)
    b = torch.from_numpy(rng.standard_normal(v)).float() if (rows + v) % 2 else None
    got = ot.joiner_logits(x.to(DEV), w.to(DEV), b.to(DEV) if b is not None else None, out_dtype=out)
    a, m, bias = value(as_np(x), 1), value(as_np(w), BLOCK), as_np(b) if b is not None else None
    want = a @ m.T + (bias if b is not None else 0)
    assert got.shape == (rows, v) and got.dtype == out and got.is_contiguous()
    assert np.all(np.abs(as_np(got) - want) <= bound(a, m, bias, want, out))
    # the handle holds the same weight: the same bits
    handle = ot.quantize_weight(w.to(DEV))
    again = ot.joiner_logits(x.to(DEV), handle, b.to(DEV) if b is not None else None, out_dtype=out)
    assert torch.equal(again, got)
    np.testing.assert_allclose(as_np(handle.dequantize()), m, rtol=2.0 ** -24)


def test_logits_from_strided_and_unaligned_operands():
    rng = np.random.default_rng(3)
    for dtype in TYPES.values():
        big = torch.from_numpy(rng.standard_normal((50, 301))).to(dtype).to(DEV)
        w = torch.from_numpy(rng.standard_normal((70, 200))).to(dtype).to(DEV)
        x = big[3:40:2, 1:201]                     # rows 602 elements apart, base at an odd element
        assert torch.equal(ot.joiner_logits(x, w), ot.joiner_logits(x.contiguous(), w))
        wv = torch.from_numpy(rng.standard_normal((140, 207))).to(dtype).to(DEV)[1::2, 5:205]
        assert torch.equal(ot.joiner_logits(x, wv), ot.joiner_logits(x, wv.contiguous()))


def test_a_checkpoints_weight_with_any_scales():
    rng = np.random.default_rng(4)
    rows, d, v = 33, 336, 300
    data = torch.from_numpy(rng.standard_normal((v, d)) * 60).float().to(torch.float8_e4m3fn)
    scale = torch.from_numpy(rng.uniform(1e-3, 3e-3, (3, 3))).float()
    x = torch.from_numpy(rng.standard_normal((rows, d))).to(torch.bfloat16)
    m = as_np(data) * spread(as_np(scale), BLOCK, (v, d))
    a = value(as_np(x), 1)
    want = a @ m.T
    weight = ot.Fp8Weight(data.to(DEV), scale.to(DEV))
    got = as_np(ot.joiner_logits(x.to(DEV), weight, out_dtype=torch.float32))
    assert np.all(np.abs(got - want) <= bound(a, m, None, want, torch.float32))
    wide = torch.zeros((v, 400), dtype=torch.uint8, device=DEV)   # rows 400 bytes apart
    wide[:, 16:16 + d] = data.view(torch.uint8).to(DEV)
    strided = ot.Fp8Weight(wide[:, 16:16 + d].view(torch.float8_e4m3fn), scale.to(DEV))
    assert np.array_equal(as_np(ot.joiner_logits(x.to(DEV), strided, out_dtype=torch.float32)), got)


def _grads(x, w, b, g, out_dtype=torch.bfloat16):
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w) + ((b,) if b is not None else ())]
    y = ot.joiner_logits(leaves[0], leaves[1], leaves[2] if b is not None else None, out_dtype=out_dtype)
    return y, torch.autograd.grad(y, leaves, g.to(DEV))


@pytest.mark.parametrize("types", ["f32-f32-f32", "bf16-f32-bf16", "bf16-bf16-bf16", "f16-f32-f32"])
@pytest.mark.parametrize("shape", [(1, 16, 5), (50, 60, 30), (129, 129, 500), (640, 200, 130), (5000, 72, 33), (4999, 160, 300)])
def test_gradients_against_the_formula(shape, types):
    rows, d, v = shape
    xt, wt, gt = (TYPES[t] for t in types.split("-"))
    rng = np.random.default_rng(rows + d + v + 1)
    x = torch.from_numpy(rng.standard_normal((rows, d))).to(xt)
    w = torch.from_numpy(rng.standard_normal((v, d)) / np.sqrt(d)).to(wt)
    b = torch.from_numpy(rng.standard_normal(v)).float()
    g = torch.from_numpy(rng.standard_normal((rows, v)) * rng.random((rows, 1)) ** 4).to(gt)
    y, (gx, gw, gb) = _grads(x, w, b, g, gt)
    assert gx.dtype == xt and gw.dtype == wt and gb.dtype == torch.float32
    gn, xn, wn = as_np(g), as_np(x), as_np(w)
    a, m = value(gn, 1), value(wn, BLOCK).T
    want = a @ m.T
    assert np.all(np.abs(as_np(gx) - want) <= bound(a, m, None, want, xt))
    a, m = value(gn.T, 1), value(xn.T, BLOCK)
    want = a @ m.T
    assert np.all(np.abs(as_np(gw) - want) <= bound(a, m, None, want, wt))
    assert np.all(np.abs(as_np(gb) - gn.sum(0)) <= (rows + 8) * 2.0 ** -24 * np.abs(gn).sum(0))
    assert torch.equal(y.detach(), ot.joiner_logits(x.to(DEV), w.to(DEV), b.to(DEV), out_dtype=gt))


def test_gradients_against_differences():
    """Small integers are e4m3 values times a power of two, so nothing is rounded: the
    logits are exactly linear in each operand, and <G, y(x + h) - y(x)> = <dX, h>."""
    rng = np.random.default_rng(6)
    rows, d, v = 70, 48, 40
    ints = lambda *s: torch.from_numpy(rng.integers(-3, 4, s)).float()  # noqa: E731
    x, w, b, g = ints(rows, d), ints(v, d), ints(v), ints(rows, v)
    hx, hw, hb = ints(rows, d), ints(v, d), ints(v)
    y, (gx, gw, gb) = _grads(x, w, b, g, torch.float32)
    f = lambda p, q, r: ot.joiner_logits(p.to(DEV), q.to(DEV), r.to(DEV), out_dtype=torch.float32).double().cpu()  # noqa: E731
    base, gd = f(x, w, b), g.double()
    assert torch.equal(base, x.double() @ w.double().T + b.double())
    assert float((gd * (f(x + hx, w, b) - base)).sum()) == float((gx.double().cpu() * hx).sum())
    assert float((gd * (f(x, w + hw, b) - base)).sum()) == float((gw.double().cpu() * hw).sum())
    assert float((gd * (f(x, w, b + hb) - base)).sum()) == float((gb.double().cpu() * hb).sum())


def test_gradients_of_some_operands_only():
    rng = np.random.default_rng(8)
    x = torch.from_numpy(rng.standard_normal((30, 40))).float().to(DEV)
    w = torch.from_numpy(rng.standard_normal((20, 40))).float().to(DEV)
    b = torch.from_numpy(rng.standard_normal(20)).float().to(DEV)
    g = torch.from_numpy(rng.standard_normal((30, 20))).float().to(torch.bfloat16).to(DEV)
    full = _grads(x.cpu(), w.cpu(), b.cpu(), g.cpu())[1]
    for i in range(3):
        ops = [t.detach().clone() for t in (x, w, b)]
        ops[i].requires_grad_(True)
        (got,) = torch.autograd.grad(ot.joiner_logits(*ops), [ops[i]], g)
        assert torch.equal(got, full[i]), i
    # a bias that other rows of a graph share too, and a gradient that is expanded
    bb = b.clone().requires_grad_(True)
    loss = ot.joiner_logits(x, w, bb, out_dtype=torch.float32).sum() + (2 * bb).sum()
    loss.backward()
    assert torch.equal(bb.grad, torch.full_like(bb, 32.0))


def test_a_second_derivative_is_refused():
    x = torch.randn(4, 16, device=DEV, requires_grad=True)
    y = ot.joiner_logits(x, torch.randn(3, 16, device=DEV), out_dtype=torch.float32)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_calls_that_are_not_the_usual_one_give_the_same():
    """Strided operands and int settings take another way through the Python layer."""
    x = torch.randn(20, 64, device=DEV)
    w = ot.quantize_weight(torch.randn(33, 64, device=DEV))
    b = torch.randn(33, device=DEV)
    wide = torch.zeros(20, 80, device=DEV)
    wide[:, :64] = x
    assert torch.equal(ot.joiner_logits(wide[:, :64], w, b), ot.joiner_logits(x, w, b))
    assert torch.equal(ot.joiner_logits(x.requires_grad_(True).detach(), w, b), ot.joiner_logits(x.detach(), w, b))
    with pytest.raises(RuntimeError, match="inference"):
        ot.joiner_logits(x, w, b)
    with torch.no_grad():
        assert not ot.joiner_logits(x, w, b).requires_grad
    for bad in (b[:5], b.double(), b.cpu(), torch.stack([b, b], 1)[:, 0]):
        with pytest.raises(RuntimeError, match="bias"):
            ot.joiner_logits(x.detach(), w, bad)
    with pytest.raises(RuntimeError, match="out_dtype"):
        ot.joiner_logits(x.detach(), w, b, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="joiner_in"):
        ot.joiner_logits(x.detach()[:, :63], w, b)


def test_what_is_not_finite_stays_in_its_block():
    rng = np.random.default_rng(9)
    x = torch.from_numpy(rng.standard_normal((6, 300))).float().to(DEV)
    w = torch.from_numpy(rng.standard_normal((200, 300))).float().to(DEV)
    base = ot.joiner_logits(x, w, out_dtype=torch.float32)
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[2, 299] = bad
        got = ot.joiner_logits(y, w, out_dtype=torch.float32)
        assert torch.isnan(got[2]).all()
        keep = [0, 1, 3, 4, 5]
        assert torch.equal(got[keep], base[keep])
        u = w.clone()
        u[150, 7] = bad                     # the block of columns 128..199
        got = ot.joiner_logits(x, u, out_dtype=torch.float32)
        assert torch.isnan(got[:, 128:]).all() and torch.equal(got[:, :128], base[:, :128])


def test_no_rows():
    w = torch.ones(5, 16, device=DEV)
    assert ot.joiner_logits(torch.empty(0, 16, device=DEV), w).shape == (0, 5)


def test_on_another_stream_and_in_a_captured_graph():
    rng = np.random.default_rng(10)
    x = torch.from_numpy(rng.standard_normal((300, 96))).to(torch.bfloat16).to(DEV).requires_grad_(True)
    w = torch.from_numpy(rng.standard_normal((130, 96))).float().to(DEV).requires_grad_(True)
    g = torch.from_numpy(rng.standard_normal((300, 130))).to(torch.bfloat16).to(DEV)

    def step():
        y = ot.joiner_logits(x, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), g))

    want = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    x.data.mul_(2)
    graph.replay()
    first = [t.clone() for t in held]
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    x.data.mul_(0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, want))
