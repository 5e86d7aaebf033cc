"""Pages outside the pool: their tokens take no part in paged attention, on either kernel."""

import math

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import HALF, INDEX_OUT_OF_RANGE, TINY, dev, filled_cache, index

pytestmark = pytest.mark.gpu


def check_without(query, cache, lens, bad, scale, got, lse, dtype):
    """Against 64 bits over the tokens whose page is not in `bad` {(sequence, column)};
    the bounds are those of check_paged."""
    batch, queries, heads, dim = query.shape
    kv_heads, page = cache.caches["key"].shape[1:3]
    got, lse = got.cpu().double(), lse.cpu().double()
    for b, n in enumerate(lens):
        k, v = ((codes * scales[..., None]) for codes, scales in (cache.tokens(name, b, n) for name in ("key", "value")))
        kept = torch.tensor([(b, t // page) not in bad for t in range(n)], dtype=torch.bool)
        for i in range(queries):
            seen = torch.nonzero(kept & (torch.arange(n) < n - queries + 1 + i)).flatten()
            for h in range(heads):
                g = h // (heads // kv_heads)
                if len(seen) == 0:
                    assert lse[b, i, h] == -math.inf and not got[b, i, h].any()
                    continue
                row, keys, values = query[b, i, h].double(), k[seen, g], v[seen, g]
                s = keys @ row * scale
                want_lse = torch.logsumexp(s, 0)
                want = torch.exp(s - want_lse) @ values
                score = (dim + 8) * 2.0**-24 * float((keys.abs() @ row.abs()).max()) * scale
                assert abs(lse[b, i, h] - want_lse) <= 2 * score + 2.0**-20 * (1 + abs(want_lse)), (b, i, h)
                weight = 2 * score + (2.0**-11 if dtype != torch.float32 else 0) + 2.0**-20
                limit = HALF[dtype] * want.abs() + TINY[dtype] + weight * float(values.abs().max())
                assert ((got[b, i, h] - want).abs() <= limit).all(), (b, i, h)


@pytest.mark.parametrize("code", (torch.float8_e4m3fn, torch.int8), ids=("e4m3", "int8"))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("page", (16, 32, 48))
def test_tokens_of_a_page_outside_the_pool_are_not_seen(page, dtype, code):
    lens, queries, heads, kv_heads, dim = [2 * page + 5, 700, 3 * page, page + 9, 30], 3, 4, 2, 64
    cache = filled_cache(lens, page, kv_heads, dim, code)
    query = torch.randn(len(lens), queries, heads, dim).to(dtype)
    # the middle of a sequence, pages of a long one, a beginning, the end, and all of one
    bad = {(0, 1), (1, 2), (1, 3), (1, 10), (2, 0), (3, 1)} | {(4, c) for c in range(-(-30 // page))}
    table = cache.table.clone()
    for at, (b, c) in enumerate(sorted(bad)):
        table[b, c] = (-1, cache.caches["key"].shape[0], 2**31 - 1)[at % 3]
    scale = dim**-0.5
    got, lse = programs.paged_attention(dev(query), *cache.args, index(table.tolist()), index(lens), scale=scale,
                                        return_lse=True)
    assert device_status() == INDEX_OUT_OF_RANGE and device_status() == 0
    check_without(query, cache, lens, bad, scale, got, lse, dtype)
