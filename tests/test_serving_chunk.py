"""Attention of chunks over the paged cache without a GPU: refusals on the host."""

import pytest
import torch

from ninetoothed_b200 import _lib, serving
from tests.test_serving import packed

BASE = {"tokens": 4, "batch": 1, "heads": 4, "dtype": 9, "index_dtype": 3, "cache.pages": 4, "cache.kv_heads": 2,
        "cache.page": 16, "cache.head_dim": 64, "cache.code_dtype": 12, "cache.key": 16, "cache.value": 16,
        "cache.key_scale": 16, "cache.value_scale": 16}


@pytest.mark.parametrize("change, code", [
    (dict(tokens=-1), 10001), (dict(batch=-1), 10001), (dict(heads=-1), 10001), (dict(table_columns=-1), 10001),
    (dict(dtype=12), 10002), (dict(index_dtype=8), 10002), ({"cache.code_dtype": 9}, 10002), ({"cache.page": 17}, 10003),
    ({"cache.head_dim": 272}, 10003), ({"heads": 3}, 10003), ({"cache.kv_heads": 0}, 10003), (dict(batch=0), 0),
    (dict(tokens=0), 0), (dict(heads=0), 0), (dict(), 10001),  # null pointers
    # a workspace that is too small, and one off the grid
    (dict(query=16, output=16, lengths=16, offsets=16, workspace=16, workspace_bytes=1000), 10001),
    (dict(query=16, output=16, lengths=16, offsets=16, workspace=24, workspace_bytes=1 << 40), 10001),
])
def test_refused_on_the_host(change, code):
    entry = _lib.library().nt_b200_chunk_attention
    assert entry(None, None) == 10001
    assert entry(packed("NtB200ChunkAttentionArgs", **(BASE | change)), None) == code


def test_shapes_are_refused_before_the_launch():
    query = torch.zeros(6, 4, 64).half()
    cache, scale = torch.zeros(3, 2, 16, 64, dtype=torch.int8), torch.zeros(3, 2)
    offsets, lengths, table = torch.tensor([0, 4, 6]), torch.tensor([9, 6]), torch.zeros(2, 1, dtype=torch.int64)
    base = dict(query=query, key_cache=cache, value_cache=cache, key_scale=scale, value_scale=scale, block_table=table,
                offsets=offsets, lengths=lengths, output=query, lse=None, scale=None)
    wide = torch.zeros(3, 2, 16, 272, dtype=torch.int8)
    for change in (
        dict(query=query[:, :3], output=query[:, :3]), dict(output=query[:5]), dict(output=query.float()),
        dict(query=query[:, :, :32], output=query[:, :, :32]), dict(offsets=offsets[:2]), dict(offsets=offsets.int()),
        dict(lengths=lengths[:1]), dict(block_table=table[:1]), dict(lse=torch.zeros(6, 3)), dict(value_cache=cache[:2]),
        dict(key_scale=scale[:2]), dict(key_cache=cache[:, :, :, ::2]), dict(value_cache=cache.view(torch.float8_e4m3fn)),
        dict(key_cache=cache[:, :, :8], value_cache=cache[:, :, :8]),
        dict(query=torch.zeros(6, 4, 272).half(), output=torch.zeros(6, 4, 272).half(), key_cache=wide, value_cache=wide),
    ):
        with pytest.raises(TypeError):
            serving._launch_chunk_attention(base | change, 0)
