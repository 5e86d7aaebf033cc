"""chunk_attention's sum of exponentials: many weights far below the largest one."""

import math

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import HALF, index

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("log2_ratio", (24, 28, 31))
def test_small_weights_beside_a_large_one_are_in_the_lse(log2_ratio, dtype):
    """A key of score 0 and 2^18 of score -log2_ratio in base 2, in sequences enough that a CTA has whole ones."""
    slow = dtype == torch.float32
    batch, new, heads, dim, page, length = (2 if slow else 300), 1, (1 if slow else 4), 64, 1024, 1 << 18
    pages = length // page
    keys = torch.zeros(pages, 1, page, dim, dtype=torch.int8, device="cuda")
    keys[:, 0, :, 0] = -log2_ratio
    keys[0, 0, 0, 0] = 0
    values, ones = torch.ones_like(keys), torch.ones(pages, 1, device="cuda")
    query = torch.zeros(batch * new, heads, dim, dtype=dtype, device="cuda")
    query[:, :, 0] = 1.0
    table = index([list(range(pages))] * batch)  # all sequences have the same pages
    got, lse = programs.chunk_attention(query, keys, values, ones, ones, table, index(list(range(batch + 1))),
                                        index([length] * batch), scale=math.log(2), return_lse=True)
    assert device_status() == 0
    tail = (length - 1) * 2.0**-log2_ratio
    # what the 256 keys (CUDA cores) or 128 that are summed with the large one lose at most, each an exponential 2^-22
    # of itself off at a score that two factors of 24 bits give; the logarithm of 1 to 2, 2^-22 off, and its rounding
    limit = 256 * 2.0**-log2_ratio + tail * (2.0**-22 + 2 * log2_ratio * 2.0**-24) + 2.0**-22 + 2.0**-23
    assert ((lse.cpu().double() - math.log1p(tail)).abs() <= limit).all(), (float(lse[0, 0]), math.log1p(tail))
    # values are all 1; tensor memory's fp32 sums take 16 keys a step
    assert ((got.double() - 1).abs() <= HALF[dtype] + length / 16 * 2.0**-23 + 2.0**-20).all()
