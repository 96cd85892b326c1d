"""Settings outside their range, as the header has them (GPU): refused as scalars, defined in arrays."""
from __future__ import annotations

import math

import pytest
import torch

from m1moe_b200 import M1MoECudaError, sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [64, 30000])
@pytest.mark.parametrize("bad", [-1.0, math.nan, -math.inf])
def test_settings_out_of_range(vocab, bad):
    g = torch.Generator(device="cuda").manual_seed(81)
    x = torch.randn((9, vocab), generator=g, device="cuda")
    x[:, 11], x[:, 7] = 20.0, 20.0  # two equal largest ones
    u = torch.linspace(0.05, 0.95, 9, device="cuda")
    first = [7] * 9
    two = [7] * 4 + [11] * 5  # at u = 1/2 the first one's weight does not exceed the half
    t = torch.full((9,), bad, device="cuda")
    assert sample(x, u, temperature=t).tolist() == first
    assert sample(x, u, top_p=t).tolist() == first
    want = sample(x, u, temperature=30.0)
    assert len(set(want.tolist())) > 2
    got = sample(x, u, temperature=30.0, min_p=t)
    assert got.tolist() == (two if math.isnan(bad) else want.tolist())
    assert sample(x, u, temperature=30.0, min_p=torch.full((9,), 1.5, device="cuda")).tolist() == two
    for kw in ({"temperature": bad}, {"top_p": bad}, {"min_p": bad}):
        with pytest.raises(M1MoECudaError):
            sample(x, u, **kw)


def test_one_token_may_have_any_stride():
    """A vocabulary of one has no stride between tokens: what the tensor says of it is not looked at."""
    x = torch.zeros((1, 5), device="cuda").t()
    assert x.stride() == (1, 5)
    assert sample(x, torch.rand(5, device="cuda")).tolist() == [0] * 5
