"""Queries with one element far larger than the others, over keys that have nothing there."""

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import check_paged, dev, filled_cache, index

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, outlier", ((torch.bfloat16, 2.0**20), (torch.bfloat16, 2.0**16), (torch.float16, 60000.0)))
@pytest.mark.parametrize("code", (torch.float8_e4m3fn, torch.int8), ids=("e4m3", "int8"))
@pytest.mark.parametrize("dim", (64, 128))
def test_small_elements_beside_a_large_one_keep_their_bits(dim, code, dtype, outlier):
    """check_paged's bound goes by |q| |k|, in which the outlier meets zeros and does not count."""
    lens, heads, kv_heads = [200, 31], 4, 2
    cache = filled_cache(lens, 16, kv_heads, dim, code)
    cache.caches["key"].view(torch.int8)[..., 5] = 0
    query = torch.randn(len(lens), 1, heads, dim) * 2.0**-4
    query[..., 5] = outlier
    query = query.to(dtype)
    args = index(cache.table.tolist()), index(lens)
    got, lse = programs.paged_attention(dev(query), *cache.args, *args, scale=4.0, return_lse=True)
    assert device_status() == 0
    check_paged(query, cache, lens, 4.0, got, lse, dtype)


@pytest.mark.parametrize("size", (2.0**-126, 2.0**-110, 2.0**100, 2.0**120))
def test_rows_at_the_ends_of_bfloat16(size):
    lens, heads, dim = [70], 2, 64
    cache = filled_cache(lens, 32, 1, dim, torch.int8)
    query = (torch.randn(1, 1, heads, dim) * size).bfloat16()
    if size < 1:  # scores of about one, from scales that make up for it
        cache.scales["key"].mul_(2.0**100)
        scale = 1 / (size * 2.0**100)
    else:
        cache.scales["key"].mul_(2.0**-60)
        scale = 2.0**60 / size
    args = index(cache.table.tolist()), index(lens)
    got, lse = programs.paged_attention(dev(query), *cache.args, *args, scale=scale, return_lse=True)
    assert device_status() == 0
    check_paged(query, cache, lens, scale, got, lse, torch.bfloat16)
