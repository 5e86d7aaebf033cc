"""Prompt attention over large bfloat16 values: sums stay in range where the output does."""

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import check_prompt, dev, index

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("rise", (6.0, 20.0, 30.0))
def test_values_near_the_range_of_the_type(rise, dim, causal):
    """The second block of 128 keys has 2^rise times the weights of the first."""
    lens = [300, 40]
    q = torch.randn(340, 2, dim) * 0.01
    k = torch.randn(340, 1, dim)
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[128:, :, 0] = rise * 0.6931
    q, k = q.bfloat16(), k.bfloat16()
    v = (torch.randn(340, 1, dim) * 1e33).bfloat16()
    got, lse = programs.prompt_attention(dev(q), dev(k), dev(v), index([0, 300, 340]), is_causal=causal, scale=1.0,
                                         return_lse=True)
    assert device_status() == 0 and got.isfinite().all()
    check_prompt(q, k, v, lens, lens, 1.0, causal, got, lse, torch.bfloat16)
