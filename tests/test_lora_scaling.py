"""A scaling for all adapters that lives on the device."""

import pytest
import torch

from tests.test_lora_linear import BF16, randn, weights

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("M", [3, 40])
def test_one_scaling_on_the_device_is_not_fetched(M):
    """Read when the graph is replayed, as one for each adapter is."""
    from linquant_b200.kernels.layer import lora_linear_fwd

    torch.manual_seed(1)
    w, ws, a, b = weights(48, 64, 8, 3, BF16)
    x, which, scaling = randn(M, 64, dtype=BF16), torch.randint(-1, 3, (M,), device="cuda").int(), torch.tensor(0.5, device="cuda")
    assert torch.equal(lora_linear_fwd(x, w, ws, a, b, which, scaling=scaling), lora_linear_fwd(x, w, ws, a, b, which, scaling=0.5))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        y = lora_linear_fwd(x, w, ws, a, b, which, scaling=scaling)
    scaling.fill_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, lora_linear_fwd(x, w, ws, a, b, which, scaling=2.0))
    assert torch.equal(lora_linear_fwd(x, w, ws, a, b, which, scaling=torch.tensor(2.0)), y)  # and one on the host
