"""``sample_tokens`` against its definition in float64, row by row in numpy: the tokens
have to be the same.  The log-probability is (x - max) / temperature - log(sum): float32
rounds the two quotients and the logarithm by 2^-24 of themselves and the sum by
(3 ln V + 90) * 2^-24 at most, so it is held to (3 ln V + 100) * 2^-24 * max(1, |value|)."""
import math

import numpy as np
import pytest
import torch

import optimized_transducer_b200 as ot

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def oracle(x, u, t, k, p, m):
    """(token, log-probability) of one row; settings already float32 values."""
    x = np.asarray(x, np.float64)
    top = x.max() if not np.isnan(x).any() else np.nan
    if not np.isfinite(top) or not (0 <= t <= 1e6) or not (0 <= u <= 1) or p != p or m != m:
        return -1, math.nan
    order = np.lexsort((np.arange(x.size), -x))
    if t == 0:
        return int(order[0]), 0.0
    w = np.exp((x - top) / t)
    keep = order[:k] if k > 0 else order
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[keep])[:-1]])
        stay = before < p * w[keep].sum()
        stay[0] = True
        keep = keep[stay]
    stay = w[keep] >= m
    stay[0] = True
    keep = np.sort(keep[stay])
    c = np.cumsum(w[keep])
    hit = np.flatnonzero(c > u * c[-1])
    token = keep[hit[0]] if hit.size else keep[np.flatnonzero(w[keep] > 0)[-1]]
    return int(token), math.log(w[token] / c[-1])


def check(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """x: a CPU tensor (any type); settings: numbers or CPU tensors with one value per row."""
    dev = lambda s: s.to(DEV) if isinstance(s, torch.Tensor) else s  # noqa: E731
    tokens, logp = ot.sample_tokens(x.to(DEV) if not x.is_cuda else x, u.to(DEV), temperature=dev(t), top_k=dev(k), top_p=dev(p), min_p=dev(m))
    assert tokens.dtype == torch.int32 and logp.dtype == torch.float32 and tokens.shape == logp.shape == (x.size(0),)
    tokens, logp = tokens.cpu().numpy(), logp.double().cpu().numpy()
    xs, us = x.double().cpu().numpy(), u.double().numpy()
    of = lambda s, i, f: f(s[i].item()) if isinstance(s, torch.Tensor) else f(np.float32(s)) if f is float else s  # noqa: E731
    tol = (3 * math.log(x.size(1) + 1) + 100) * 2.0 ** -24
    for i in range(x.size(0)):
        token, lp = oracle(xs[i], us[i], of(t, i, float), of(k, i, int), of(p, i, float), of(m, i, float))
        assert tokens[i] == token, (i, tokens[i], token, us[i])
        if math.isnan(lp):
            assert math.isnan(logp[i]), i
        else:
            assert abs(logp[i] - lp) <= tol * max(1.0, abs(lp)), (i, logp[i], lp)


def rows(rng, n, v, dtype, spread=3.0):
    x = rng.standard_normal((n, v)) * spread * np.exp(0.4 * rng.standard_normal((n, 1)))
    x[:, 0] += 2
    x[rng.random((n, v)) < 0.03] = -np.inf
    x[:, v // 2] = np.where(np.isinf(x[:, v // 2]), 0.0, x[:, v // 2])
    return torch.from_numpy(x).to(TYPES[dtype])


FILTERS = [dict(), dict(t=0.7), dict(k=1), dict(k=7), dict(p=0.9), dict(p=0.3, t=1.5), dict(m=0.05), dict(k=40, p=0.8, m=0.01, t=0.8), dict(t=0.0, p=0.5)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("v", [1, 2, 31, 128, 129, 500, 512, 513, 1024, 1030, 4096, 5000, 8193, 16384])
def test_tokens_are_those_of_the_definition(v, dtype):
    rng = np.random.default_rng(v)
    n = 60 if v <= 1024 else 12
    for i, f in enumerate(FILTERS):
        check(rows(rng, n, v, dtype), torch.from_numpy(rng.random(n)).float(), **f)


@pytest.mark.parametrize("v", [16385, 40001, 65537, 131073, 262144])
def test_wide_rows(v):
    rng = np.random.default_rng(v)
    for f in (dict(), dict(k=50, p=0.9), dict(p=0.95, t=0.8, m=1e-4), dict(k=1), dict(t=0.0)):
        check(rows(rng, 3, v, "f32"), torch.from_numpy(rng.random(3)).float(), **f)
    check(rows(rng, 3, v, "bf16"), torch.from_numpy(rng.random(3)).float(), k=100, p=0.7)


@pytest.mark.parametrize("v", [60, 500, 3000, 20000])
def test_settings_of_each_row(v):
    rng = np.random.default_rng(v + 1)
    n = 40
    t = torch.from_numpy(rng.uniform(0.2, 2, n)).float()
    t[::7] = 0
    k = torch.from_numpy(rng.integers(-1, 30, n)).to(torch.int32)
    p = torch.from_numpy(rng.uniform(0, 1.1, n)).float()
    p[3] = 0.0
    m = torch.from_numpy(rng.uniform(0, 0.1, n)).float()
    m[5] = 1.0
    m[6] = 1.5
    check(rows(rng, n, v, "f32"), torch.from_numpy(rng.random(n)).float(), t, k, p, m)
    bad_t, bad_p, bad_m = t.clone(), p.clone(), m.clone()
    bad_t[1], bad_t[2], bad_t[3], bad_p[4], bad_m[8] = -1.0, float("nan"), 1e7, float("nan"), float("nan")
    u = torch.from_numpy(rng.random(n)).float()
    u[9], u[10], u[11], u[12], u[13] = -0.1, 1.1, float("nan"), 1.0, 0.0
    check(rows(rng, n, v, "f32"), u, bad_t, k, bad_p, bad_m)


@pytest.mark.parametrize("v", [10, 500, 1100, 9000, 30000])
def test_equal_logits_and_borders_that_are_hit_exactly(v):
    """Equal logits have weight 1 exactly: the sums are whole numbers, so top_p = 1/2 and
    u = j / 8 meet their borders exactly and ties go by the index."""
    n = 9
    u = torch.arange(n).float() / 8
    for f in (dict(), dict(p=0.5), dict(p=0.25), dict(k=3), dict(k=v - 1), dict(k=4, p=0.5), dict(m=1.0), dict(p=0.5, t=0.3)):
        check(torch.full((n, v), -2.5), u, **f)
    rng = np.random.default_rng(v)
    few = torch.from_numpy(rng.integers(0, 3, (n, v)) * 0.5).float()   # three values, many ties
    few[few == 0] = -0.0
    for f in (dict(p=0.5), dict(k=v // 2), dict(k=v // 3, p=0.6), dict(p=0.9, t=0.5), dict(m=0.5)):
        check(few, u, **f)
        check(few.to(torch.bfloat16), u, **f)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("v", [33, 700, 6000, 20000])
def test_masked_rows(v, dtype):
    rng = np.random.default_rng(v + 2)
    x = rows(rng, 16, v, dtype)
    low = torch.finfo(x.dtype).min
    x[0] = -math.inf                       # nothing is allowed
    x[1] = -math.inf
    x[1, v - 1] = 3.0                      # one symbol is
    x[2] = low                             # all at the type's lowest value: uniform
    x[3, 1:] = low
    x[4, v // 3] = math.nan
    x[5, v // 3] = math.inf
    x[6] = math.nan
    x[7] = -math.inf
    x[7, ::5] = low
    x[8, :] = 0.0
    x[8, 3] = torch.finfo(x.dtype).max
    u = torch.from_numpy(rng.random(16)).float()
    for f in (dict(), dict(k=5), dict(p=0.7), dict(m=0.2), dict(t=0.0), dict(t=1e-20), dict(t=1e6), dict(k=9, p=0.5, m=0.1)):
        check(x, u, **f)


def test_numbers_near_a_border_are_decided_as_in_64_bits():
    """u is put a few float32 steps around every border of the cumulative weights."""
    rng = np.random.default_rng(5)
    for v in (300, 2000):
        x = torch.from_numpy(rng.standard_normal((1, v)) * 2).float()
        w = np.exp(x.double().numpy()[0] - x.double().numpy()[0].max())
        border = (np.cumsum(w) / w.sum()).astype(np.float32)[rng.integers(0, v, 200)]
        u = np.concatenate([border, np.nextafter(border, np.float32(0)), np.nextafter(border, np.float32(2))]).clip(0, 1)
        check(x.expand(u.size, v).contiguous(), torch.from_numpy(u))
        # and top_p around the sums of the largest weights
        s = np.cumsum(np.sort(w)[::-1]) / w.sum()
        p = s.astype(np.float32)[rng.integers(0, v, 100)]
        p = np.concatenate([p, np.nextafter(p, np.float32(0)), np.nextafter(p, np.float32(2))])
        check(x.expand(p.size, v).contiguous(), torch.from_numpy(rng.random(p.size)).float(), 1.0, 0, torch.from_numpy(p))
        # and min_p at the weights themselves
        m = w.astype(np.float32)[rng.integers(0, v, 100)]
        m = np.concatenate([m, np.nextafter(m, np.float32(0)), np.nextafter(m, np.float32(2))])
        check(x.expand(m.size, v).contiguous(), torch.from_numpy(rng.random(m.size)).float(), 1.0, 0, 1.0, torch.from_numpy(m))


def test_strided_and_unaligned_rows():
    rng = np.random.default_rng(6)
    u = torch.from_numpy(rng.random(20)).float()
    for dtype in TYPES.values():
        big = torch.from_numpy(rng.standard_normal((40, 611)) * 3).to(dtype).to(DEV)
        for v, off in ((500, 3), (510, 101), (400, 4), (1, 7)):
            check(big[::2, off:off + v], u, k=20, p=0.9)


def test_values_at_every_magnitude():
    """Logits from the smallest to the largest floats in one row: the bisection ends."""
    e = np.arange(-149, 128)
    x = np.concatenate([-(2.0 ** e), [0.0], 2.0 ** e]).astype(np.float32)
    rng = np.random.default_rng(7)
    x = torch.from_numpy(rng.permuted(np.tile(x, (12, 1)), axis=1))
    u = torch.from_numpy(rng.random(12)).float()
    for f in (dict(k=250), dict(k=300), dict(k=400), dict(p=0.9), dict(p=0.999, t=1e5), dict(k=280, p=0.5)):
        check(x, u, **f)


def test_logits_whose_steps_are_coarse_beside_the_temperature():
    """Near 1e8 neighbouring float32 numbers are 8 apart: borders fall between roundings."""
    rng = np.random.default_rng(9)
    for v in (400, 3000):
        x = torch.from_numpy(1e8 + 8.0 * rng.integers(-4, 1, (20, v))).float()
        u = torch.from_numpy(rng.random(20)).float()
        for f in (dict(p=0.9), dict(p=0.999), dict(p=0.99, t=4.0), dict(k=5), dict(k=v // 2, p=0.99999), dict(p=0.9, t=1e-3)):
            check(x, u, **f)
            check(-x, u, **f)


def test_weights_below_the_normal_doubles():
    """u = 0 draws the first index of any weight at all, u = 1 the last: e^-720 still counts, e^-800 is 0."""
    for v in (40, 2000):
        x = torch.zeros(4, v)
        x[0, :5], x[1, :5] = -720.0, -800.0
        x[2, -5:], x[3, -5:] = -720.0, -800.0
        check(x, torch.tensor([0.0, 0.0, 1.0, 1.0]))


def test_refusals_on_the_gpu():
    x, u = torch.randn(4, 50, device=DEV), torch.rand(4, device=DEV)
    want = ot.sample_tokens(x, u, temperature=1.0, top_k=3)
    got = ot.sample_tokens(x, u, temperature=1, top_k=True * 3, top_p=1, min_p=0)     # ints where floats are usual
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for kw, what in ((dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
                     (dict(top_p=float("nan")), "top_p"), (dict(top_k=1 << 40), "top_k"), (dict(min_p=u[:2]), "min_p"),
                     (dict(top_k=u), "top_k"), (dict(temperature=u.cpu()), "temperature")):
        with pytest.raises(RuntimeError, match=what):
            ot.sample_tokens(x, u, **kw)
    for bad in (u[:3], u.double(), u.cpu(), torch.stack([u, u], 1)[:, 0]):
        with pytest.raises(RuntimeError, match="uniforms"):
            ot.sample_tokens(x, bad)
    for bad in (x.double(), x[:, ::2], x[0], torch.empty(2, 0, device=DEV), torch.empty(1, 262145, device=DEV)):
        with pytest.raises(RuntimeError, match="logits"):
            ot.sample_tokens(bad, u)


def test_no_rows_and_one_column():
    t, p = ot.sample_tokens(torch.empty(0, 5, device=DEV), torch.empty(0, device=DEV))
    assert t.shape == p.shape == (0,)
    check(torch.tensor([[1.5], [-math.inf]]), torch.tensor([0.3, 0.3]))


def test_many_rows_on_another_stream_and_in_a_captured_graph():
    rng = np.random.default_rng(8)
    x = (torch.randn(5001, 500, generator=torch.Generator().manual_seed(1)) * 3).to(DEV)
    u = torch.from_numpy(rng.random(5001)).float().to(DEV)
    step = lambda: ot.sample_tokens(x, u, 0.8, 30, 0.9, 0.01)  # noqa: E731
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
    u.copy_(1 - u)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, step()))


@pytest.mark.parametrize("v", [40, 700, 3000, 20000])
def test_subnormal_temperatures(v):
    """Logits a few of the smallest floats apart and a temperature of that size: the exponents
    are ordinary numbers although 1 / temperature is none in float32."""
    rng = np.random.default_rng(v + 3)
    least = 2.0 ** -149
    x = torch.from_numpy(-least * rng.integers(0, 40, (12, v))).float()
    u = torch.from_numpy(rng.random(12)).float()
    for t in (least, 3 * least, 20 * least, 1000 * least, 2.0 ** -127, 2.0 ** -126):
        for f in (dict(), dict(p=0.6), dict(p=0.95, k=30), dict(m=0.05), dict(k=9, p=0.9, m=1e-3)):
            check(x, u, t=t, **f)
    t = torch.from_numpy(rng.choice([0.0, least, 5 * least, 1e-40, 1e-38, 1.0], 12)).float()
    check(x, u, t=t, p=0.8)
