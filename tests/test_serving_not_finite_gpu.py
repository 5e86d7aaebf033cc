"""Infinities and NaN in values reach the queries that see them and nobody else,
whatever is packed beside a sequence, at the cost of a second pass at most."""

import math

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import index

pytestmark = pytest.mark.gpu


def offsets_of(lens, first=0):
    return index([first + sum(lens[:i]) for i in range(len(lens) + 1)])


CASES = [
    # query lengths, key lengths (None: the same), heads, kv_heads, dim
    ([1, 5, 300], None, 4, 2, 128),
    ([130, 127, 128], None, 2, 2, 64),
    ([257, 60], None, 8, 1, 96),
    ([200], None, 3, 1, 40),  # rows of a tile that hold no query
    ([70, 9], None, 100, 2, 64),  # two queries a tile
    ([5, 60, 0, 33], [300, 60, 7, 140], 6, 3, 128),  # later parts of prompts
    ([140, 9], [10, 0], 4, 2, 64),  # queries before the first key
]


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float32))
@pytest.mark.parametrize("case", CASES, ids=range(len(CASES)))
def test_who_sees_what_is_not_finite(case, dtype, causal):
    """Exactly the elements whose query sees such a value are not finite; all others
    are bit for bit those of a run in which these values are 0."""
    q_lens, k_lens, heads, kv_heads, dim = case
    k_lens = k_lens or q_lens
    tokens = sum(k_lens)
    q = torch.randn(sum(q_lens), heads, dim).to(dtype).cuda()
    k, v = (torch.randn(tokens + 200, kv_heads, dim).to(dtype) for _ in range(2))
    bad = torch.zeros(v.shape, dtype=torch.bool)
    bad[tokens:] = True  # tokens of no sequence
    some = torch.rand(v.shape) < 2.0 / tokens  # a few in each element's column
    bad |= some & (torch.rand(v.shape[-1]) < 0.5)  # half of the columns have none
    kinds = torch.tensor([math.inf, -math.inf, math.nan])[torch.randint(0, 3, v.shape)].to(dtype)
    args = q, k.cuda()
    rest = offsets_of(q_lens), offsets_of(k_lens), causal
    clean, clean_lse = programs.prompt_attention(*args, v.masked_fill(bad, 0).cuda(), *rest, return_lse=True)
    got, lse = programs.prompt_attention(*args, torch.where(bad, kinds, v).cuda(), *rest, return_lse=True)
    assert device_status() == 0 and torch.equal(lse, clean_lse)
    got, clean = got.cpu(), clean.cpu()
    q0 = k0 = 0
    for nq, nk in zip(q_lens, k_lens):
        limit = nk - nq + 1 + torch.arange(nq) if causal else torch.full((nq,), nk)
        limit = limit.clamp(0, nk)
        for h in range(heads):
            g = h // (heads // kv_heads)
            met = torch.cat((torch.zeros(1, dim), bad[k0 : k0 + nk, g].cumsum(0)))[limit] > 0
            x, want = got[q0 : q0 + nq, h], clean[q0 : q0 + nq, h]
            assert not x[met].isfinite().any() and torch.equal(x[~met], want[~met]), (nq, h)
        q0, k0 = q0 + nq, k0 + nk


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_sign_of_an_infinite_value(dtype):
    """In the last keys, which not all rows see: one infinity keeps its sign, two of
    different signs are NaN."""
    n, dim = 100, 64
    q, k, v = (torch.randn(n, 1, dim).to(dtype) for _ in range(3))
    v[60, 0, 3], v[70, 0, 4], v[50, 0, 5], v[80, 0, 5], v[90, 0, 3] = math.inf, -math.inf, math.inf, -math.inf, math.inf
    got = programs.prompt_attention(q.cuda(), k.cuda(), v.cuda(), index([0, n])).cpu()[:, 0]
    assert (got[60:, 3] == math.inf).all() and (got[70:, 4] == -math.inf).all()
    assert (got[50:80, 5] == math.inf).all() and got[80:, 5].isnan().all()
    assert got[:60, 3].isfinite().all() and got[:70, 4].isfinite().all() and got[:50, 5].isfinite().all()


def best_of(call, times=20):
    """The least device time of a call, in us."""
    out, best = call(), math.inf
    for _ in range(times):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        b.synchronize()
        best = min(best, 1e3 * a.elapsed_time(b))
    return out, best


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("tokens, heads, kv_heads", ((4096, 8, 2), (32768, 2, 1)))
def test_long_prompts_beside_values_that_are_not_finite(tokens, heads, kv_heads, causal):
    """In tokens of no sequence right after the first, and in an early value of the
    second: the first's output is the clean one's, and no item of work is taken more
    than twice."""
    lens, gap, dim = [tokens - 100, tokens], 300, 128
    total = sum(lens) + gap
    q, k, v = (torch.randn(total, n, dim, device="cuda").bfloat16() for n in (heads, kv_heads, kv_heads))
    # the gap as a sequence of keys without queries
    q_offsets = index([0, lens[0], lens[0], lens[0] + lens[1]])
    k_offsets = index([0, lens[0], lens[0] + gap, total])

    def call(values):
        return lambda: programs.prompt_attention(q, k, values, q_offsets, k_offsets, causal)

    clean, clean_time = best_of(call(v))
    bad = v.clone()
    bad[lens[0] : lens[0] + gap : 2] = math.nan
    bad[lens[0] + 1 : lens[0] + gap : 2] = math.inf
    start = lens[0] + gap
    bad[start, 0, 7] = math.inf
    got, time = best_of(call(bad))
    assert device_status() == 0
    first = slice(0, lens[0])
    assert torch.equal(got[first], clean[first])
    second = slice(lens[0], lens[0] + lens[1])
    group = heads // kv_heads
    met = torch.zeros((heads, dim), dtype=torch.bool, device="cuda")
    met[:group, 7] = True  # element 7 of the first group's heads, which all of the second's queries see
    assert not got[second][:, met].isfinite().any() and torch.equal(got[second][:, ~met], clean[second][:, ~met])
    print(f"{tokens} tokens, causal {causal}: clean {clean_time:.0f} us, beside values that are not finite {time:.0f} us")
    assert time <= 2.5 * clean_time  # two passes, and the search for what to take out in the second
