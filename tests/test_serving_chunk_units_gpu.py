"""chunk_attention where a CTA goes through many units: values that are not numbers among them."""

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import dev, filled_cache, index

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", (
    # sequences, most new tokens, most cached ones, heads, kv_heads, dim, one sequence in so many with NaN
    (100, 32, 300, 32, 8, 128, 3),  # units of one tile throughout: the second one is idle
    (100, 32, 300, 32, 8, 64, 1),
    (150, 90, 400, 16, 4, 128, 2),  # units of one tile beside units of two
    (600, 2, 60, 8, 2, 64, 5),
    (3, 700, 900, 64, 16, 64, 1),
), ids=range(5))
def test_nan_values_of_many_units_reach_only_who_sees_them(case):
    batch, most_new, most, heads, kv_heads, dim, every = case
    gen = torch.Generator().manual_seed(batch + dim)

    def below(n, count=None):
        return torch.randint(0, n, (count or 1,), generator=gen).tolist()

    news = [1 + n for n in below(most_new, batch)]
    lens = [n + x for n, x in zip(news, below(most - most_new, batch))]
    cache = filled_cache(lens, 16, kv_heads, dim, torch.float8_e4m3fn)
    offsets = [sum(news[:i]) for i in range(batch + 1)]
    query = torch.randn(sum(news), heads, dim, generator=gen).half()
    args = (*cache.args, index(cache.table.tolist()), index(offsets), index(lens))
    clean, lse = programs.chunk_attention(dev(query), *args, return_lse=True)
    slow, slow_lse = programs.chunk_attention(dev(query.float()), *args, return_lse=True)
    # scores: fp32 sums of dim products on both sides, of magnitudes that sum to 40 or less
    score = 2 * (dim + 8) * 2.0**-24 * 40
    # weights of 11 bits and that error of theirs, and an fp16 result, of values of 448 * 2 * 6 / 448 or less
    assert ((clean.float() - slow).abs() <= (2 * 2.0**-11 + 2 * score) * 12).all()
    assert torch.allclose(lse, slow_lse, rtol=1e-6, atol=score)

    want = torch.zeros(query.shape, dtype=torch.bool)
    codes = cache.caches["value"].view(torch.int8)
    for s in range(0, batch, every):
        for _ in range(3):
            (token,), (group,), (element,) = below(lens[s]), below(kv_heads), below(dim)
            codes[int(cache.table[s, token // 16]), group, token % 16, element] = 127 if token % 2 else -1
            limit = lens[s] - news[s] + 1 + torch.arange(news[s])
            per = heads // kv_heads
            want[offsets[s] : offsets[s + 1], group * per : (group + 1) * per, element] |= (limit > token)[:, None]
    for _ in range(3):
        got, got_lse = programs.chunk_attention(dev(query), *args, return_lse=True)
        assert device_status() == 0
        assert torch.equal(got.isnan().cpu(), want)
        assert torch.equal(got.nan_to_num(0.0), clean.masked_fill(want.cuda(), 0.0)) and torch.equal(got_lse, lse)
    assert torch.equal(programs.chunk_attention(dev(query.float()), *args).isnan().cpu(), want)
