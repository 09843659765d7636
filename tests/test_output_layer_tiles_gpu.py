"""The 8-bit products of large workloads: every tile width, unsplit and cut along the
contraction, with several tiles per block and partial tiles at both edges, rows that leave
by TMA and by plain stores, all output types, against float64 products of the quantised
values (on the GPU).  Tolerance of one entry, as derived in test_output_layer_gpu.py: a
product of two e4m3 values is exact in float32; K terms are added, each addition off by at
most 2^-23 of the partial sums' magnitude, a block's scaling adds two roundings and the
bias one; pieces of the contraction are K terms all the same."""
import ctypes

import pytest
import torch

import optimized_transducer_b200 as ot
from optimized_transducer_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BLOCK = 128
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def tiling(m, n, k):
    """(columns per tile, tiles, whether the contraction is cut, SMs) of an (m, n, k) product by the library's rule."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    up = lambda a, b: -(-a // b)  # noqa: E731
    mt, kb = up(m, 128), up(k, BLOCK)
    columns = 256
    while columns > 64 and (n <= columns // 2 or (kb < 32 and mt * up(n, columns) < sms)):
        columns //= 2
    tiles = mt * up(n, columns)
    need = ctypes.c_uint64()
    _lib.check(_lib.load().ot_b200_fp8_matmul_workspace_bytes(m, n, k, ctypes.byref(need)))
    return columns, tiles, need.value > 0, sms


def value(x, rows_per_block):
    """What x is in e4m3, float64: the smallest power of two with max|x| / s <= 448 for each block, ties to even."""
    x = x.double()
    r, c = x.shape
    rb, cb = -(-r // rows_per_block), -(-c // BLOCK)
    pad = torch.nn.functional.pad(x, (0, cb * BLOCK - c, 0, rb * rows_per_block - r)).reshape(rb, rows_per_block, cb, BLOCK)
    top = pad.abs().amax((1, 3), keepdim=True)
    m, e = torch.frexp(top)
    scale = torch.ldexp(torch.ones_like(top), torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126))
    scale = torch.where(top > 0, scale, torch.ones_like(scale))
    y = pad / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(y / step) * step * scale).reshape(rb * rows_per_block, cb * BLOCK)[:r, :c]


def check(got, a, b, bias=None, chunk=4096):
    """got = a @ b.T (+ bias), a and b float64."""
    for r in range(0, a.size(0), chunk):
        want, mass = a[r:r + chunk] @ b.T, a[r:r + chunk].abs() @ b.abs().T
        if bias is not None:
            want, mass = want + bias.double(), mass + bias.double().abs()
        tol = (a.size(1) + 8) * 2.0 ** -23 * mass + torch.finfo(got.dtype).eps / 2 * want.abs() + torch.finfo(got.dtype).tiny
        assert bool(((got[r:r + chunk].double() - want).abs() <= tol).all()), (r, float(((got[r:r + chunk].double() - want).abs() / tol).max()))


def operands(rows, d, v, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(rows + d + v + seed)
    normal = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    return normal(rows, d).to(BF16), normal(v, d) / d ** 0.5, normal(v), normal(rows, v) * torch.rand(rows, 1, device=DEV, generator=g) ** 4


# rows, D, V -> columns per tile, cut along K.  256 columns, several tiles per block: a multiple of 16
# bytes of columns and not; a partial column tile; one K block; more K blocks than stages.  128 columns
# with one and several tiles per block.  64 columns with several.
FORWARD = [((4000, 300, 5000), 256, False), ((4000, 300, 5003), 256, False), ((4000, 300, 5002), 256, False), ((19000, 200, 250), 256, False),
           ((20000, 100, 300), 256, False), ((5000, 1000, 1030), 256, False), ((19000, 200, 100), 128, False), ((19000, 131, 101), 128, False),
           ((40000, 72, 128), 128, False), ((1201, 656, 5000), 256, False), ((19000, 200, 60), 64, False), ((19000, 700, 33), 64, False)]


@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("case", FORWARD)
def test_logits(case, out):
    (rows, d, v), columns, cut = case
    c, tiles, is_cut, sms = tiling(rows, v, d)
    assert (c, is_cut) == (columns, cut) and tiles > sms
    x, w, b, _ = operands(rows, d, v)
    a, m = value(x, 1), value(w, BLOCK)
    check(ot.joiner_logits(x, w, b, out_dtype=out), a, m, b)
    if out == F32:
        check(ot.joiner_logits(x, ot.quantize_weight(w), out_dtype=out), a, m)


# dX = dY W has V as its contraction, dW = dY^T X the rows: (rows, D, V), whether dX and dW are cut
BACKWARD = [((700, 300, 5000), True, False), ((20000, 520, 5001), False, False), ((30000, 512, 700), False, True),
            ((6000, 100, 4200), False, True), ((5000, 60, 33), False, True), ((9001, 250, 9000), True, True), ((45000, 300, 4100), False, True)]


@pytest.mark.parametrize("types", [(BF16, BF16), (F32, BF16), (F16, F32)])
@pytest.mark.parametrize("case", BACKWARD)
def test_gradients(case, types):
    (rows, d, v), cut_x, cut_w = case
    x, w, b, g = operands(rows, d, v, 1)
    x, g = x.to(types[0]).requires_grad_(True), g.to(types[1])
    w.requires_grad_(True)
    b.requires_grad_(True)
    y = ot.joiner_logits(x, w, b, out_dtype=types[1])
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    xv, wv = x.detach(), w.detach()
    assert tiling(rows, d, v)[2] == cut_x and tiling(v, d, rows)[2] == cut_w
    check(y.detach(), value(xv, 1), value(wv, BLOCK), b.detach())
    check(gx, value(g, 1), value(wv, BLOCK).T)
    check(gw, value(g.T, 1), value(xv.T, BLOCK))
    # float32 sums over at most 128 rows, joined in a fixed order: (rows + 8) * 2^-24 of the magnitudes
    assert bool(((gb.double() - g.double().sum(0)).abs() <= (rows + 8) * 2.0 ** -24 * g.double().abs().sum(0)).all())


@pytest.mark.parametrize("rows_per_block", [1, BLOCK])
def test_the_stated_bound_of_the_quantiser(rows_per_block):
    """An element is off by at most max(2^-4 |x|, 2^-10 scale): the second term is that of small
    ones beside a large one, and it is needed."""
    from optimized_transducer_b200 import output_layer

    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    x = torch.randn(300, 500, device=DEV, generator=g) * torch.exp(-15 * torch.rand(300, 500, device=DEV, generator=g))
    (q, scale), _, _ = output_layer._quantize(x, _lib.FP8_ROWS if rows_per_block == 1 else _lib.FP8_SQUARES)
    s = scale.t() if rows_per_block == 1 else scale
    s = s.double().repeat_interleave(rows_per_block, 0)[:300].repeat_interleave(BLOCK, 1)[:, :500]
    error = (q[:, :500].contiguous().view(torch.float8_e4m3fn).double() * s - x.double()).abs()
    assert bool((error <= torch.maximum(x.double().abs() / 16, s / 1024)).all())
    assert bool((error > x.double().abs() / 16).any()) and bool((error == x.double().abs()).any())
