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
