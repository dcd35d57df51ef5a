"""Sampling gives the same token however the kernel's lists came to be ordered: repeated calls, other rows
beside a row, and its logits' order inside a slice where that decides nothing."""
import numpy as np
import pytest
import torch

from helm_amd.kernels import fused
from test_sample import check, logits


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,p,lo", [(1.0, 0, 0.9, 0.0), (0.8, 2000, 1.0, 0.0), (2.5, 0, 0.999, 0.0), (1.5, 30000, 0.97, 0.001)])
def test_a_row_s_token_is_the_same_in_every_call(cuda, t, k, p, lo):
    x = logits(1, 60000, 17, 2.0)
    u = torch.rand(300, generator=torch.Generator().manual_seed(9)).cuda()
    many = fused.sample(x.expand(300, 60000), u, t, k, p, lo)
    for _ in range(5):
        assert torch.equal(fused.sample(x.expand(300, 60000), u, t, k, p, lo), many)
    for i in (0, 7, 299):
        assert int(fused.sample(x, u[i:i + 1], t, k, p, lo)) == int(many[i])


@pytest.mark.gpu
@pytest.mark.parametrize("t", [0.002, 0.05, 1.0, 40.0])
@pytest.mark.parametrize("k,p,lo", [(0, 0.7, 0.0), (900, 1.0, 0.0), (0, 1.0, 1e-30), (900, 0.999999, 0.0)])
def test_weights_from_underflow_to_one(cuda, t, k, p, lo):
    """A border's range may hold weights of any size, all zeros among them."""
    x = torch.cat([logits(3, 9000, 2, 4.0), logits(3, 9000, 3, 0.01) + 8.0])
    check(x, np.random.default_rng(5).random(6, dtype=np.float32), t, k, p, lo, exact_ties=True)
