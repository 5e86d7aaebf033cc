"""Weights of paged attention keep their bits beside values of a far larger scale."""

import pytest
import torch

from ninetoothed_b200 import programs
from tests.test_serving_gpu import HALF, TINY, Pages, dev, index

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", (torch.float8_e4m3fn, torch.int8), ids=("e4m3", "int8"))
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("page", (16, 32))
@pytest.mark.parametrize("lead", (10.0, 20.0))
def test_small_weights_on_large_values(lead, page, dtype, code):
    """A block whose value scale is 2^lead larger and whose probabilities are
    about 2^-lead contributes as much as the others: each weight's error is
    bounded by its own p |v|, which probabilities rounded to fp16 by themselves
    would pass by far."""
    length, dim, heads = 4 * page, 64, 4
    cache = Pages([length], page, 1, dim, code)
    top = 100
    shape = (cache.caches["key"].shape[0], 1, page, dim)
    for name in ("key", "value"):
        codes = (torch.randn(shape) * top / 4).clamp(-top, top).round()
        if name == "key":
            codes[..., 0] = 0
        cache.caches[name].copy_(codes.to(code).cuda())
        cache.scales[name].fill_(1 / 64)
    large = [int(cache.table[0, 1]), int(cache.table[0, 3])]
    cache.scales["value"][large] = 2.0**lead / 64
    # element 0 of the other blocks' keys lifts their scores by ln 2^lead
    query = torch.randn(1, 1, heads, dim) * 0.05
    query[..., 0] = 1.0
    for j in (0, 2):
        cache.caches["key"][int(cache.table[0, j]), :, :, 0] = torch.tensor(float(top)).to(code).cuda()
    query = query.to(dtype)
    scale = 0.6931471805599453 * lead * 64 / top
    got = programs.paged_attention(dev(query), *cache.args, index(cache.table.tolist()), index([length]), scale=scale)
    k, v = ((codes * scales[..., None]) for codes, scales in (cache.tokens(n, 0, length) for n in ("key", "value")))
    naive_fails = False
    for h in range(heads):
        row = query[0, 0, h].double()
        s = k[:, 0] @ row * scale
        p = torch.exp(s - s.max())
        total = p.sum()
        want = p @ v[:, 0] / total
        # scores: fp32 sums of dim exact products times a factor of a few roundings;
        # a weight: twice its score's error (its own and the sum's), half a step of
        # fp16, and a few roundings of exponentials; what falls among fp16's
        # subnormals, relative to the largest weight: half a step of 2^-24 a token
        score = (dim + 8) * 2.0**-24 * float((k[:, 0].abs() @ row.abs()).max()) * scale
        weight = 2 * score + 2.0**-11 + 2.0**-20
        sums = (p @ v[:, 0].abs()) / total
        scales = cache.tokens("value", 0, length)[1][:, 0]
        tiny = length * 2.0**-25 * top * float((p * scales).max()) / total
        limit = HALF[dtype] * want.abs() + TINY[dtype] + weight * sums + tiny
        assert ((got[0, 0, h].cpu().double() - want).abs() <= limit).all()
        # probabilities rounded to fp16 against the largest probability
        naive = p.half().double() @ v[:, 0] / total
        naive_fails |= bool(((naive - want).abs() > limit).any())
    assert naive_fails or lead < 20.0  # at 2^-20 fp16 keeps four bits and less
