"""Workloads of the operators around the joiner's output layer and the training step:
the projection to logits in 8-bit floating point, sampling from logits, and the
global gradient norm with clipping.

``listed()`` names the fixed cases, ``draw(rng)`` makes one more of the same ranges,
``prepare`` builds the inputs of a case, ``run`` makes one pass through the operator:
with ``own`` through this package's public entry points, without it through their
plain form in elementary torch operations.  ``exact`` is the operator's definition
in 64 bits, written apart from the plain form.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 128          # elements that share one scale
E4M3_TOP = 448.0     # largest finite e4m3 value


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one step of a beam search: 8 hypotheses, the benchmark's joiner (D 512, V 500), weights quantised beforehand
        {"name": "project 8x512x500", "op": "project", "rows": 8, "d": 512, "v": 500, "x": "bf16", "out": "bf16", "bias": True},
        # the hypotheses of a batch of streams, a vocabulary of 5000, a joiner whose width is no multiple of the block
        {"name": "project 1201x656x5000", "op": "project", "rows": 1201, "d": 656, "v": 5000, "x": "f16", "out": "f32", "bias": True},
        # scoring a whole packed batch of 16 utterances with 5000 symbols
        {"name": "project 116250x512x5000", "op": "project", "rows": 116250, "d": 512, "v": 5000, "x": "bf16", "out": "bf16", "bias": True},
        # a training step of the output layer on a few utterances: logits, then the gradients of input, weight and bias
        {"name": "train 40007x512x500", "op": "train", "rows": 40007, "d": 512, "v": 500, "x": "bf16", "w": "f32", "bias": True},
        # the same on the packed batch of 16 utterances with 5000 symbols
        {"name": "train 116250x512x5000", "op": "train", "rows": 116250, "d": 512, "v": 5000, "x": "bf16", "w": "bf16", "bias": True},
        # the next symbol of one stream
        {"name": "sample 1x500", "op": "sample", "rows": 1, "v": 500, "x": "f32", "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "per_row": False},
        # the hypotheses of a batch of requests, each with its own settings
        {"name": "sample 256x5000", "op": "sample", "rows": 256, "v": 5000, "x": "bf16", "temperature": 0.9, "top_k": 40, "top_p": 0.9, "min_p": 0.02, "per_row": True},
        # alternative symbols at every lattice cell of a few packed utterances (self-training, sequence-level risks)
        {"name": "sample 80000x500", "op": "sample", "rows": 80000, "v": 500, "x": "f32", "temperature": 1.0, "top_k": 0, "top_p": 0.95, "min_p": 0.0, "per_row": False},
        # a word-level vocabulary
        {"name": "sample 16x100003", "op": "sample", "rows": 16, "v": 100003, "x": "f32", "temperature": 0.7, "top_k": 0, "top_p": 0.9, "min_p": 0.01, "per_row": False},
        # gradients of a predictor and a joiner, in place, the norm below the limit (an ordinary step)
        {"name": "clip 12 tensors", "op": "clip", "tensors": 12, "elements": 1_300_000, "x": "f32", "out": "", "norm": "2", "seed_sizes": 1},
        # a conformer encoder's gradients in bfloat16, clipped into the optimizer's float32 copies
        {"name": "clip 600 tensors", "op": "clip", "tensors": 600, "elements": 90_000_000, "x": "bf16", "out": "f32", "norm": "2", "seed_sizes": 2},
        # a large model's float32 gradients, clipped into the optimizer's buffers
        {"name": "clip 64 tensors", "op": "clip", "tensors": 64, "elements": 400_000_000, "x": "f32", "out": "f32", "norm": "2", "seed_sizes": 3},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("project", "train", "sample", "clip"))
    if op == "project":
        while True:
            rows, d, v = _log_int(rng, 1, 120000), 16 * _log_int(rng, 4, 128), _log_int(rng, 30, 8000)
            if rows * d * v <= 116250 * 512 * 5000 and rows * v <= 116250 * 5000:
                break
        return {"op": op, "rows": rows, "d": d, "v": v, "x": rng.choice(("f32", "bf16", "f16")),
                "out": rng.choice(("f32", "bf16", "f16")), "bias": rng.random() < 0.7}
    if op == "train":
        while True:
            rows, d, v = _log_int(rng, 50, 120000), _log_int(rng, 60, 1500), _log_int(rng, 30, 6000)
            if rows * d * v <= 116250 * 512 * 5000 and rows * v <= 116250 * 5000:
                break
        return {"op": op, "rows": rows, "d": d, "v": v, "x": rng.choice(("f32", "bf16", "f16")),
                "w": rng.choice(("f32", "bf16")), "bias": rng.random() < 0.7}
    if op == "sample":
        while True:
            rows, v = _log_int(rng, 1, 100000), _log_int(rng, 20, 200000)
            if rows * v <= 40_000_000:
                break
        return {"op": op, "rows": rows, "v": v, "x": rng.choice(("f32", "bf16", "f16")),
                "temperature": round(rng.uniform(0.3, 1.5), 2), "top_k": rng.choice((0, 0, rng.randint(1, 100))),
                "top_p": rng.choice((1.0, round(rng.uniform(0.3, 0.99), 3))),
                "min_p": rng.choice((0.0, round(rng.uniform(0.001, 0.2), 3))), "per_row": rng.random() < 0.3}
    return {"op": op, "tensors": _log_int(rng, 1, 800), "elements": _log_int(rng, 50_000, 300_000_000),
            "x": rng.choice(("f32", "bf16", "f16")), "out": rng.choice(("", "f32", "f32")),
            "norm": rng.choice(("2", "2", "1", "inf")), "seed_sizes": rng.randint(10, 10**6)}


def work(case):
    if case["op"] in ("project", "train"):
        r, d, v = case["rows"], case["d"], case["v"]
        blocks = -(-d // BLOCK) * -(-v // BLOCK)
        if case["op"] == "project":
            return {"bytes": r * d * SIZE[case["x"]] + v * d + 4 * blocks + r * v * SIZE[case["out"]] + 4 * v * case["bias"], "flops": 2 * r * d * v}
        return {"bytes": 2 * r * d * SIZE[case["x"]] + 2 * v * d * SIZE[case["w"]] + 2 * r * v * 2 + 8 * v * case["bias"],
                "flops": 3 * 2 * r * d * v}
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["v"] * SIZE[case["x"]] + 12), "flops": 5 * case["rows"] * case["v"]}
    written = SIZE[case["out"]] if case["out"] else 0  # in place the norm is below the limit: nothing is written
    return {"bytes": case["elements"] * (SIZE[case["x"]] + written) + 4, "flops": 2 * case["elements"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _sizes(case):
    """Element counts of the tensors of a model: matrices of very different sizes and small vectors, odd ones among them."""
    rng = np.random.RandomState(case["seed_sizes"])
    n = case["tensors"]
    share = np.exp(rng.uniform(-7, 0, n))
    sizes = np.maximum(1, (share / share.sum() * case["elements"]).astype(np.int64))
    sizes[np.argmax(sizes)] += max(0, case["elements"] - int(sizes.sum()))
    return [int(s) for s in sizes]


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    s = {"case": case}
    if case["op"] in ("project", "train"):
        r, d, v = case["rows"], case["d"], case["v"]
        # activations behind a tanh, weights of the usual scale with a few large columns
        s["x"] = torch.tanh(normal(r, d)).to(DTYPES[case["x"]])
        w = normal(v, d) * (2.0 / math.sqrt(d))
        w[:, ::37] *= 4
        s["bias"] = normal(v) if case["bias"] else None
        if case["op"] == "project":  # a checkpoint's quantised weight: bytes and one float32 scale for each block
            b = _blocked(w, BLOCK)
            scale = torch.clamp(b.abs().amax((1, 3)), min=1e-12) / 440.0
            s["w_scale"] = scale
            s["w_data"] = (b / scale[:, None, :, None]).reshape(b.size(0) * BLOCK, -1)[:v, :d].contiguous().to(torch.float8_e4m3fn)
        else:
            s["w"] = w.to(DTYPES[case["w"]]).requires_grad_(True)
            s["x"].requires_grad_(True)
            if s["bias"] is not None:
                s["bias"].requires_grad_(True)
            # the gradient that a transducer loss hands back: rows of softmax minus one-hot, weighted by the cell's occupancy
            z = torch.softmax(3 * normal(r, v), 1)
            z[torch.arange(r, device=dev), torch.randint(0, v, (r,), device=dev, generator=g)] -= 1
            z *= torch.rand(r, 1, device=dev, generator=g) ** 6
            s["grad"] = z.to(torch.bfloat16)
        return s
    if case["op"] == "sample":
        r, v = case["rows"], case["v"]
        x = normal(r, v) * torch.exp(0.4 * normal(r, 1)) * 2
        x[:, 0] += 5 + 2 * normal(r)  # the blank: the likeliest symbol of most cells
        dead = torch.rand(r, v, device=dev, generator=g) < 0.01  # symbols that a grammar forbids
        dead[:, 0] = False
        x.masked_fill_(dead, -math.inf)
        x = x.to(DTYPES[case["x"]])
        if r >= 64:
            x[5] = -math.inf                                   # nothing is allowed in this row
            x[7, 1:] = torch.finfo(x.dtype).min                # a mask that is the type's lowest value
        s["logits"] = x
        s["u"] = torch.rand(r, device=dev, generator=g)
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = case["temperature"], case["top_k"], case["top_p"], case["min_p"]
        if case["per_row"]:
            f = torch.rand(r, device=dev, generator=g)
            s["temperature"] = torch.where(f < 0.1, torch.zeros_like(f), case["temperature"] * (0.5 + f))
            s["top_k"] = (case["top_k"] * torch.rand(r, device=dev, generator=g) * 2).to(torch.int32)
            s["top_p"] = torch.clamp(case["top_p"] + 0.2 * (f - 0.5), 0.05, 1.0)
            s["min_p"] = case["min_p"] * f
        return s
    sizes = _sizes(case)
    flat = torch.randn(sum(sizes), device=dev, generator=g, dtype=torch.float32).mul_(1e-3)
    flat = flat.to(DTYPES[case["x"]])
    s["flat"], s["grads"] = flat, list(torch.split(flat, sizes))
    s["flat_out"] = torch.empty_like(flat, dtype=DTYPES[case["out"]]) if case["out"] else None
    s["outs"] = list(torch.split(s["flat_out"], sizes)) if case["out"] else None
    n = sum(sizes)
    usual = {"2": 1e-3 * math.sqrt(n), "1": 0.8e-3 * n, "inf": 6e-3}[case["norm"]]
    s["max_norm"] = 0.3 * usual if case["out"] else 3.0 * usual
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return (run_own if own else run_plain)(s)


def run_own(s):
    import optimized_transducer_b200 as ot

    case = s["case"]
    if case["op"] == "project":
        return ot.joiner_logits(s["x"], ot.Fp8Weight(s["w_data"], s["w_scale"]), s["bias"], out_dtype=DTYPES[case["out"]])
    if case["op"] == "train":
        leaves = [t for t in (s["x"], s["w"], s["bias"]) if t is not None]
        logits = ot.joiner_logits(s["x"], s["w"], s["bias"])
        return [logits.detach(), *torch.autograd.grad(logits, leaves, s["grad"])]
    if case["op"] == "sample":
        return ot.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    norm = ot.clip_grad_norm_(s["grads"], s["max_norm"], norm_type=float(case["norm"]), out=s["outs"])
    return norm, s["flat_out"] if case["out"] else s["flat"]


def run_plain(s):
    case = s["case"]
    if case["op"] == "project":
        x = _dequantised(s["x"], 1)
        w = s["w_data"].float() * _spread(s["w_scale"], s["w_data"].shape)
        y = x @ w.T
        return (y + s["bias"] if s["bias"] is not None else y).to(DTYPES[case["out"]])
    if case["op"] == "train":
        x, w, dy = s["x"].detach(), s["w"].detach(), s["grad"]
        wq = _dequantised(w, BLOCK)
        y = _dequantised(x, 1) @ wq.T
        if s["bias"] is not None:
            y = y + s["bias"].detach()
        dx = _dequantised(dy, 1) @ wq
        # along the rows: the gradient in blocks of 128 rows of one column, the input in blocks of 128 x 128
        dw = _dequantised(dy.T, 1).double() @ _dequantised(x.T, BLOCK).T.double()
        out = [y.to(torch.bfloat16), dx.to(x.dtype), dw.to(w.dtype)]
        return out + [dy.double().sum(0).float()] if s["bias"] is not None else out
    if case["op"] == "sample":
        return _sample_plain(s)
    p = float(case["norm"])
    pieces = torch.cat([g.reshape(-1) for g in s["grads"]]).double().abs()
    norm = (pieces.amax() if p == math.inf else pieces.pow(p).sum().pow(1 / p)).float()
    coef = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    if case["out"]:
        s["flat_out"].copy_(s["flat"].float() * coef)
        return norm, s["flat_out"]
    s["flat"].copy_(s["flat"].float() * coef)
    return norm, s["flat"]


def _blocked(x, rows_per_block):
    """(R, C) as (row blocks, rows_per_block, column blocks, 128), padded with zeros."""
    r, c = x.shape
    x = torch.nn.functional.pad(x, (0, -c % BLOCK, 0, -r % rows_per_block))
    return x.reshape(x.size(0) // rows_per_block, rows_per_block, -1, BLOCK)


def _spread(scale, shape):
    """One scale for each 128 x 128 block, for every element."""
    return scale.repeat_interleave(BLOCK, 0)[: shape[0]].repeat_interleave(BLOCK, 1)[:, : shape[1]]


def _dequantised(x, rows_per_block):
    """The values that x has in e4m3 with one scale for each block of rows_per_block x 128: the smallest power of
    two (2^-126 at least; 1 for a block of zeros) with which the block's largest magnitude stays within 448."""
    b = _blocked(x.float(), rows_per_block)
    top = b.abs().amax((1, 3), keepdim=True)
    m, e = torch.frexp(top)
    scale = torch.ldexp(torch.ones_like(top), torch.clamp(torch.where(m > 0.875, e - 8, e - 9), min=-126))
    scale = torch.where(top > 0, scale, torch.ones_like(scale))
    q = (b / scale).to(torch.float8_e4m3fn).float() * scale
    return q.reshape(q.size(0) * rows_per_block, -1)[: x.size(0), : x.size(1)]


def _column(v, like):
    """A setting as a column of doubles: a number goes through float32, the type the settings have."""
    return v.double()[:, None] if isinstance(v, torch.Tensor) else torch.tensor(v, device=like.device).float().double()


def _sample_plain(s):
    x = s["logits"].double()
    t, p, m = (_column(s[k], x) for k in ("temperature", "top_p", "min_p"))
    k = s["top_k"][:, None] if isinstance(s["top_k"], torch.Tensor) else torch.tensor(s["top_k"], device=x.device)
    v = x.size(1)
    top = x.amax(1, keepdim=True)
    ok = torch.isfinite(top)
    order = torch.sort(x, dim=1, descending=True, stable=True)
    rank = torch.arange(v, device=x.device)
    shifted = order.values - top
    w = torch.where(t > 0, torch.exp(shifted / t), (rank == 0).double())
    w = torch.where(ok, w, (rank == 0).double())
    keep = (rank < k) | (k <= 0)
    before = torch.nn.functional.pad(torch.cumsum(w * keep, 1), (1, -1))
    keep = keep & ((before < p * (w * keep).sum(1, keepdim=True)) | (p >= 1) | (rank == 0))
    keep = keep & ((w >= m) | (rank == 0))
    kept = torch.zeros_like(w).scatter(1, order.indices, w * keep)
    c = torch.cumsum(kept, 1)
    total = c[:, -1:]
    hit = c > s["u"].double()[:, None] * total
    last = v - 1 - (kept > 0).flip(1).int().argmax(1)
    token = torch.where(hit.any(1), hit.int().argmax(1), last)
    logp = torch.log(kept.gather(1, token[:, None]) / total)[:, 0]
    ok = ok[:, 0]
    return torch.where(ok, token, -1).to(torch.int32), torch.where(ok, logp, math.nan).float()


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "project":
        x = _e4m3_blocks(s["x"].double(), 1)
        r, c = (torch.arange(n, device=x.device) // BLOCK for n in s["w_data"].shape)
        w = s["w_data"].double() * s["w_scale"].double()[r][:, c]
        y = torch.matmul(x, w.t())
        return y if s["bias"] is None else y.add_(s["bias"].double())
    if case["op"] == "train":
        x, w, dy = s["x"].detach().double(), s["w"].detach().double(), s["grad"].double()
        wq = _e4m3_blocks(w, BLOCK)
        y = torch.matmul(_e4m3_blocks(x, 1), wq.t())
        if s["bias"] is not None:
            y += s["bias"].detach().double()
        dw = torch.matmul(_e4m3_blocks(dy.t(), 1), _e4m3_blocks(x.t(), BLOCK).t())
        out = [y, torch.matmul(_e4m3_blocks(dy, 1), wq), dw]
        return out + [dy.sum(0)] if s["bias"] is not None else out
    if case["op"] == "sample":
        return _sample_exact(case, s)
    total, p = [], float(case["norm"])
    for g in s["grads"]:
        a = g.double().abs()
        total.append(a.max() if p == math.inf else (a ** p).sum())
    total = torch.stack(total)
    norm = total.max() if p == math.inf else total.sum() ** (1 / p)
    coef = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    return norm, s["flat"].double() * coef


def _e4m3_blocks(x, rows_per_block):
    """Rounds x (doubles) to e4m3 block by block: 3 mantissa bits, exponents down to -6, ties to even."""
    r, c = x.shape
    rb, cb = -(-r // rows_per_block), -(-c // BLOCK)
    top = torch.zeros(rb * rows_per_block, cb * BLOCK, device=x.device, dtype=torch.float64)
    top[:r, :c] = x.abs()
    top = top.view(rb, rows_per_block, cb, BLOCK).amax(3).amax(1)
    top = torch.where(top > 0, top, torch.full_like(top, E4M3_TOP))
    scale = torch.exp2(torch.ceil(torch.log2(top / E4M3_TOP)).clamp(min=-126))
    scale = scale[torch.arange(r, device=x.device) // rows_per_block][:, torch.arange(c, device=x.device) // BLOCK]
    y = x / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale


def _sample_exact(case, s):
    r, v = case["rows"], case["v"]

    def per_row(name, dtype):
        a = s[name]
        return a.cpu().numpy().astype(dtype) if isinstance(a, torch.Tensor) else np.full(r, np.float32(a) if dtype == np.float64 else a, dtype)

    t, p, m, k = per_row("temperature", np.float64), per_row("top_p", np.float64), per_row("min_p", np.float64), per_row("top_k", np.int64)
    u = s["u"].double().cpu().numpy()
    token, logp = np.full(r, -1, np.int32), np.full(r, np.nan)
    logits = s["logits"]
    for i in range(r):
        if i % 4096 == 0:
            part = logits[i:i + 4096].double().cpu().numpy()
        x = part[i % 4096]
        top = x.max()
        if not np.isfinite(top):
            continue
        if t[i] == 0:
            token[i], logp[i] = int(np.argmax(x)), 0.0
            continue
        w = np.exp((x - top) / t[i])
        # candidates in order of falling weight, the lower index first among equals; those of no weight need no place
        live = np.flatnonzero(w > 0)
        at = live[np.lexsort((live, -x[live]))]
        if k[i] > 0:
            at = at[:k[i]]
        if p[i] < 1:
            c = np.cumsum(w[at])
            at = at[:1 + int(np.searchsorted(c[:-1], p[i] * c[-1], side="left"))]
        at = at[(w[at] >= m[i]) | (np.arange(at.size) == 0)]
        at.sort()
        c = np.cumsum(w[at])
        token[i] = at[min(at.size - 1, int(np.searchsorted(c, u[i] * c[-1], side="right")))]
        logp[i] = math.log(w[token[i]] / c[-1])
    return torch.from_numpy(token), torch.from_numpy(logp)
