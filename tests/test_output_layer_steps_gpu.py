"""The operators of the output layer together, as a training step and a decoding step use
them, against the same steps in torch.

Training: pack -> joiner_logits -> transducer_loss -> backward -> clip_grad_norm_.  The
8-bit products are replaced by float64 products of the same quantised values, the loss
and the packing by their own entry points on those logits, so what is compared is the
hand-over: the loss overwrites the logits with its gradient in place and that is what the
projection's backward pass receives."""
import numpy as np
import pytest
import torch

import optimized_transducer_b200 as ot
from test_output_layer_gpu import as_np, value

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BLOCK = 128


def _batch(seed, n, d, v):
    rng = np.random.default_rng(seed)
    T = rng.integers(8, 20, n).astype(np.int32)
    U = rng.integers(2, 7, n).astype(np.int32)
    enc = torch.from_numpy(rng.standard_normal((n, int(T.max()), d))).float().to(DEV)
    dec = torch.from_numpy(rng.standard_normal((n, int(U.max()) + 1, d))).float().to(DEV)
    targets = torch.from_numpy(rng.integers(1, v, (n, int(U.max()))).astype(np.int32)).to(DEV)
    w = torch.from_numpy(rng.standard_normal((v, d)) / np.sqrt(d)).float().to(DEV)
    b = torch.from_numpy(rng.standard_normal(v)).float().to(DEV)
    return rng, torch.from_numpy(T).to(DEV), torch.from_numpy(U).to(DEV), enc, dec, targets, w, b


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_training_step(out_dtype):
    n, d, v = 5, 96, 150
    rng, T, U, enc, dec, targets, w, b = _batch(1, n, d, v)
    leaves = [t.clone().requires_grad_(True) for t in (enc, dec, w, b)]
    x = ot.pack_joiner_input(leaves[0], leaves[1], T, U)
    logits = ot.joiner_logits(x, leaves[2], leaves[3], out_dtype=out_dtype)
    before = logits.detach().clone()
    loss = ot.transducer_loss(logits, targets, T, U, blank=0, from_log_softmax=False, reduction="sum")
    loss.backward()
    grads = [t.grad for t in leaves]
    norm = ot.clip_grad_norm_(grads, 2.0)
    torch.cuda.synchronize()
    # the same loss on the same logits
    z = before.clone().requires_grad_(True)
    want = ot.transducer_loss(z * 1, targets, T, U, blank=0, from_log_softmax=False, reduction="sum")
    want.backward()
    assert torch.equal(want, loss)
    g = z.grad
    wq = value(as_np(w), BLOCK)
    gx = value(as_np(g), 1) @ wq
    gw = value(as_np(g).T, 1) @ value(as_np(x).T, BLOCK).T
    gb = as_np(g).sum(0)
    packed = torch.from_numpy(gx).float().to(DEV)
    e, q = enc.clone().requires_grad_(True), dec.clone().requires_grad_(True)
    ot.pack_joiner_input(e, q, T, U).backward(packed)
    exact = [as_np(e.grad), as_np(q.grad), gw, gb]
    total = np.sqrt(sum((a ** 2).sum() for a in exact))
    # float32 sums of at most 700 terms each (the rows): 700 * 2^-23 < 1e-4 of the largest entry of a tensor
    assert abs(float(norm) / total - 1) <= 1e-4
    factor = min(1.0, 2.0 / (total + 1e-6))
    assert factor < 1.0
    for got, a in zip(grads, exact):
        assert np.abs(as_np(got) - a * factor).max() <= 1e-4 * np.abs(a).max()


def test_decoding_step():
    """Eight hypotheses: the output layer with weights quantised once, then a symbol each."""
    n, d, v = 8, 512, 500
    rng, _, _, _, _, _, w, b = _batch(2, 4, d, v)
    x = torch.from_numpy(np.tanh(rng.standard_normal((n, d)))).to(torch.bfloat16).to(DEV)
    u = torch.from_numpy(rng.random(n)).float().to(DEV)
    handle = ot.quantize_weight(w)

    def step():
        return ot.sample_tokens(ot.joiner_logits(x, handle, b), u, temperature=0.9, top_k=20, top_p=0.95)

    want = [t.clone() for t in step()]
    logits = ot.joiner_logits(x, handle, b)
    greedy, lp = ot.sample_tokens(logits, u, temperature=0.0)
    assert torch.equal(greedy.long(), logits.float().argmax(1)) and float(lp.abs().max()) == 0.0
    assert bool((want[0] >= 0).all()) and bool((want[1] <= 0).all())
    # with everything kept the log-probability is the log-softmax of the drawn symbol
    tokens, lp = ot.sample_tokens(logits, u)
    ref = torch.log_softmax(logits.double(), 1).gather(1, tokens.long()[:, None])[:, 0]
    assert float((lp.double() - ref).abs().max()) <= 1e-5 * float(ref.abs().max().clamp(min=1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    x.copy_(x.flip(0))
    u.copy_(u.flip(0))
    graph.replay()
    assert torch.equal(held[0].flip(0), want[0]) and torch.equal(held[1].flip(0), want[1])


def test_two_streams_at_once():
    """Calls on two streams share nothing: each gives the bits it gives alone."""
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((3000, 256))).to(torch.bfloat16).to(DEV)
    w = ot.quantize_weight(torch.from_numpy(rng.standard_normal((700, 256)) / 16).float().to(DEV))
    u = torch.from_numpy(rng.random(3000)).float().to(DEV)
    grads = [torch.from_numpy(rng.standard_normal(50000)).float().to(DEV) for _ in range(3)]
    outs = [[torch.empty_like(g) for g in grads] for _ in range(2)]
    alone = (ot.joiner_logits(x, w), *ot.sample_tokens(ot.joiner_logits(x, w), u, top_p=0.9), ot.clip_grad_norm_(grads, 1.0, out=outs[0]))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                y = ot.joiner_logits(x, w)
                got.append((y, *ot.sample_tokens(y, u, top_p=0.9), ot.clip_grad_norm_(grads, 1.0, out=outs[i])))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, alone))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
