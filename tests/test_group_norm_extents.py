"""Group norm over sequences of tens of millions of tokens."""

import pytest
import torch

from tests import layer_reference as ref

gpu = pytest.mark.gpu


@gpu
def test_tiles_of_many_tokens():
    """149 sequences leave one tile each, of 17.2 million tokens: more than 2^31 / 127. One sequence's values, repeated."""
    from linquant_b200.kernels.layer import group_norm_fwd

    torch.manual_seed(2)
    B, T, eps = 149, 17_200_000, 1e-5
    x = (torch.randn(1, T, 1, device="cuda") + 3).bfloat16()
    y = group_norm_fwd(x.expand(B, T, 1), 1, eps=eps, over_tokens=True)
    v = x.double().flatten()
    mean, inv = v.mean(), 1 / torch.sqrt(v.var(unbiased=False) + eps)
    want = (v - mean) * inv
    # a thread's mean takes in some 4200 batches, and what one of them rounds (2^-24) shrinks with its share of all: 2100 units; the squares' sum
    # likewise, half of it in the deviation; rows, tiles and the last step besides
    for b in (0, 77, 148):
        ref.check(y[b].flatten(), want, (v.abs() + mean.abs()) * inv, 3500 * 2.0**-24)
