"""What joiner_logits raises on the GPU beyond its argument checks."""
import pytest
import torch

import optimized_transducer_b200 as ot

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_failed_allocation_is_torchs_own_error():
    """320 GB of logits: the class that callers catch to go on with a smaller batch."""
    x = torch.zeros(2_000_000, 16, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(40_000, 16, device=DEV)
    handle = ot.quantize_weight(w)
    for weight in (handle, w, w.clone().requires_grad_(True)):
        with pytest.raises(torch.OutOfMemoryError):
            ot.joiner_logits(x, weight, out_dtype=torch.float32)
    assert float(ot.joiner_logits(x[:4], handle).abs().max()) == 0.0


def test_a_handle_keeps_its_tensors():
    handle = ot.quantize_weight(torch.randn(130, 64, device=DEV))
    data, scale = handle.data, handle.scale
    for name, new in (("data", scale), ("scale", None), ("data", 3), ("shape", (1, 1))):
        with pytest.raises(AttributeError):
            setattr(handle, name, new)
    assert handle.data is data and handle.scale is scale


def test_a_handle_whose_tensors_changed_since_is_refused():
    """Checked at every call: tensors can be resized or exchanged behind the handle's back."""
    x = torch.randn(5, 64, device=DEV)

    def handle():
        w = torch.randn(130, 64, device=DEV)
        q = ot.quantize_weight(w)
        return ot.Fp8Weight(q.data.view(torch.uint8).clone().view(torch.float8_e4m3fn), q.scale.clone())

    for change, what in ((lambda h: h.scale.resize_(1, 1), "scale"), (lambda h: h.data.resize_(130, 48), "expected joiner_in"),
                         (lambda h: h.data.resize_(0, 64), "data"), (lambda h: h.data.t_(), "data"),
                         (lambda h: setattr(h.scale, "data", torch.ones(2, 1, device=DEV, dtype=torch.float64)), "scale"),
                         (lambda h: h.scale.set_(torch.ones(2, 1).to(DEV)[:1]), "scale"),
                         (lambda h: object.__setattr__(h, "_data", None), "data"), (lambda h: object.__setattr__(h, "_scale", 1.0), "scale")):
        h = handle()
        ot.joiner_logits(x, h)
        change(h)
        with pytest.raises(RuntimeError, match=what):
            ot.joiner_logits(x, h)
    # written to in place: that is what the handle then holds
    h = handle()
    h.scale.mul_(2)
    assert torch.equal(ot.joiner_logits(x, h, out_dtype=torch.float32), 2 * ot.joiner_logits(x, ot.Fp8Weight(h.data, h.scale / 2), out_dtype=torch.float32))


def test_forward_mode_is_refused():
    """A tangent would be lost without a word."""
    import torch.autograd.forward_ad as fwd

    x, w, b = torch.randn(5, 64, device=DEV), torch.randn(33, 64, device=DEV), torch.randn(33, device=DEV)
    handle = ot.quantize_weight(w)
    want = ot.joiner_logits(x, handle, b)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args, what in (((dual(x), w, b), "joiner_in"), ((x, dual(w), b), "weight"), ((x, w, dual(b)), "bias"),
                           ((dual(x), handle, b), "joiner_in"), ((x, handle, dual(b)), "bias"), ((dual(x), handle), "joiner_in"),
                           ((dual(x), w.clone().requires_grad_(True), b), "joiner_in"),
                           ((x, ot.Fp8Weight(handle.data, dual(handle.scale)), b), "weight")):
            with pytest.raises(RuntimeError, match=f"{what} carries a forward-mode tangent"):
                ot.joiner_logits(*args)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                ot.joiner_logits(*args)
        assert torch.equal(ot.joiner_logits(fwd.unpack_dual(dual(x)).primal, handle, b), want)
    assert torch.equal(ot.joiner_logits(x, handle, b), want)
