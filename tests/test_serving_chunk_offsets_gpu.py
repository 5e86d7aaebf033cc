"""chunk_attention's offsets out of order: said so on every path, and nothing is written outside the tensors."""

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import INDEX_OUT_OF_RANGE, dev, filled_cache, index

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
@pytest.mark.parametrize("offsets", (
    [8, 20, 0, 8],  # a search for a token of the last sequence ends at the first
    [0, 10, 10, 3, 3],  # no token's search comes to the third
    [0] + [1] * 700 + [0] + [1] * 300,  # more sequences than rows
), ids=range(3))
def test_offsets_out_of_order_are_recorded(offsets, dtype):
    batch, tokens = len(offsets) - 1, max(offsets)
    cache = filled_cache([32], 16, 1, 64, torch.int8)
    query = torch.randn(tokens, 1, 64).to(dtype)
    table = cache.table.tolist()[:1] * batch
    out = torch.full((tokens + 2, 1, 64), 7.0, dtype=dtype, device="cuda")
    args = dev(query), *cache.args, index(table), index(offsets), index([32] * batch), out[1:-1]
    programs.chunk_attention_kernel(*args)
    assert device_status() == INDEX_OUT_OF_RANGE
    assert (out[0] == 7).all() and (out[-1] == 7).all()
    # in order, the same sequences
    good = sorted(offsets)
    programs.chunk_attention_kernel(*args[:6], index(good), *args[7:])
    assert device_status() == 0 and (out[0] == 7).all() and (out[-1] == 7).all()
