"""One key that takes nearly all of the weight, and a long tail of equal values."""

import math

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import HALF, index

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("queries", (1, 12))
def test_tail_of_a_paged_sequence(dim, queries):
    """65536 tokens with 2^-25.5 of the first one's weight, which is all that has a
    value, in one warp's share (as many sequences as warps, all of the same pages)."""
    length, page, batch = 65536, 4096, 2048 // queries
    caches = [torch.zeros(length // page, 1, page, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
    caches[0][0, 0, 0, 0] = 64
    caches[1].fill_(100)
    caches[1][0, 0, 0] = 0
    scales = [torch.full((length // page, 1), 1 / 64, device="cuda") for _ in range(2)]
    query = torch.zeros(batch, queries, 1, dim, dtype=torch.float16, device="cuda")
    query[..., 0] = 25.5
    table = index([list(range(length // page))]).expand(batch, -1)
    got, lse = programs.paged_attention(query, *caches, *scales, table, index([length] * batch), scale=math.log(2.0),
                                        return_lse=True)
    assert device_status() == 0
    for i in (0, queries - 1):
        n = length - queries + 1 + i
        tail = (n - 1) * 2.0**-25.5
        want = tail * 100 / 64 / (1 + tail)
        # relative to the output: a tail weight that is kept 2^9 above the largest is
        # 2^-16.5, where half a step of fp16 is 2^-25; 2 n / 32 sums of 16 terms, each
        # off by two units in the last of 24 bits; the output's half step
        limit = (2.0**-8.5 + 2 * n / 32 * 2.0**-22 + 2.0**-11) * want
        assert float((got[:, i].double() - want).abs().max()) <= limit
        # the lanes' sums: n / 8 terms, in blocks of 256, of which the first's tail is lost
        assert float((lse[:, i].double() - math.log(1 + tail) - 25.5 * math.log(2.0)).abs().max()) <= 2.0**-16


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("dim", (64, 128))
def test_tail_of_a_prompt(dim, dtype):
    """The same over the last four queries of 131072 keys."""
    length, queries = 131072, 4
    q = torch.zeros(queries, 2, dim, dtype=dtype, device="cuda")
    q[..., 0] = 25.5
    k, v = torch.zeros(length, 1, dim), torch.full((length, 1, dim), 100 / 64)
    k[0, 0, 0], v[0] = 1.0, 0.0
    got, lse = programs.prompt_attention(q, k.to(dtype).cuda(), v.to(dtype).cuda(), index([0, queries]), index([0, length]),
                                         scale=math.log(2.0), return_lse=True)
    assert device_status() == 0
    for i in range(queries):
        n = length - queries + 1 + i
        tail = (n - 1) * 2.0**-25.5
        want = tail * 100 / 64 / (1 + tail)
        # as above; bfloat16 weights keep 8 bits wherever they are
        half = 2.0**-8.5 if dtype == torch.float16 else 2.0**-9
        limit = (half + n / 16 * 2.0**-22 + HALF[dtype]) * want
        assert float((got[i].double() - want).abs().max()) <= limit
        # n / 128 blocks are added to the sum one by one
        assert float((lse[i].double() - math.log(1 + tail) - 25.5 * math.log(2.0)).abs().max()) <= 2.0**-14 + 2.0**-18


@pytest.mark.parametrize("dim", (64, 160))
@pytest.mark.parametrize("paged", (True, False))
def test_tail_in_float32(paged, dim):
    """On CUDA cores, with a value at the first key too: a thread's sums go over to
    others every 256 keys."""
    n = 65536
    q = torch.zeros(1, 1, 2, dim, device="cuda")
    q[..., 0] = 25.5
    if paged:
        caches = [torch.zeros(n // 4096, 1, 4096, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
        caches[0][0, 0, 0, 0] = 64
        caches[1].fill_(100)
        caches[1][0, 0, 0] = 1
        scales = [torch.full((n // 4096, 1), 1 / 64, device="cuda") for _ in range(2)]
        got, lse = programs.paged_attention(q, *caches, *scales, index([list(range(n // 4096))]), index([n]),
                                            scale=math.log(2.0), return_lse=True)
    else:
        k, v = torch.zeros(n, 1, dim, device="cuda"), torch.full((n, 1, dim), 100 / 64, device="cuda")
        k[0, 0, 0], v[0] = 1.0, 1 / 64
        got, lse = programs.prompt_attention(q[0], k, v, index([0, 1]), index([0, n]), scale=math.log(2.0), return_lse=True)
    assert device_status() == 0
    tail = (n - 1) * 2.0**-25.5
    want = (1 / 64 + tail * 100 / 64) / (1 + tail)
    # 256 terms, then n / 256 sums; scores of 25.5 in base 2 with a few roundings, in each weight
    weight = (256 + n / 256) * 2.0**-24 + 8 * 2.0**-24 * 25.5
    assert float((got.double() - want).abs().max()) <= 2 * weight * want
    assert float((lse.double() - math.log(1 + tail) - 25.5 * math.log(2.0)).abs().max()) <= weight + 2.0**-19


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_lse_of_one_key_is_its_score(dtype):
    """However small: what P is kept above the maximum does not show."""
    q, k = (torch.randn(200, 1, 64).to(dtype).cuda() * 0.1 for _ in range(2))
    _, lse = programs.prompt_attention(q, k, k, index(list(range(201))), return_lse=True)
    score = (q.double() * k.double()).sum(-1) / 8
    # 64 exact products added in fp32, a factor of a few roundings
    limit = 72 * 2.0**-24 * (q.double() * k.double()).abs().sum(-1) / 8
    assert device_status() == 0 and ((lse.double() - score).abs() <= limit).all()
