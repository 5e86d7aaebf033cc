"""Attention of chunks over the paged cache on the GPU against a 64-bit implementation."""

import math

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import HALF, INDEX_OUT_OF_RANGE, TINY, dev, filled_cache, index

pytestmark = pytest.mark.gpu


def check_chunk(query, cache, news, lens, scale, got, lse, dtype, first=0):
    """Every row of `got` against softmax(scale q k) v in 64 bits."""
    got, lse = got.cpu().double(), lse.cpu().double()
    heads, dim = query.shape[1:]
    kv_heads = cache.caches["key"].shape[1]
    at = first
    for b, (new, length) in enumerate(zip(news, lens)):
        rows = slice(at, at + new)
        at += new
        if new == 0:
            continue
        k, v = ((codes * scales[..., None]) for codes, scales in (cache.tokens(name, b, length) for name in ("key", "value")))
        limit = length - new + 1 + torch.arange(new)
        unseen = torch.arange(length)[None, :] >= limit[:, None]
        for h in range(heads):
            g = h // (heads // kv_heads)
            q = query[rows, h].double()
            none = limit <= 0
            assert (lse[rows, h][none] == -math.inf).all() and not got[rows, h][none].any()
            if none.all():
                continue
            s = (q @ k[:, g].T * scale).masked_fill(unseen, -math.inf)[~none]
            want_lse = torch.logsumexp(s, dim=1)
            want = torch.exp(s - want_lse[:, None]) @ v[:, g]
            # scores: fp32 sums of dim products of exact factors, times a factor of a few roundings
            product = ((q.abs() @ k[:, g].abs().T * scale).masked_fill(unseen, 0.0)[~none]).amax(dim=1)
            score = (dim + 8) * 2.0**-24 * product
            assert ((lse[rows, h][~none] - want_lse).abs() <= 2 * score + 2.0**-20 * (1 + want_lse.abs())).all(), (b, h)
            # each weight: the score's error, half a step of fp16 (half precision inputs), and fp32 sums over the keys
            weight = 2 * score + (2.0**-11 if dtype != torch.float32 else 0) + 2.0**-20 + length * 2.0**-24
            limits = HALF[dtype] * want.abs() + TINY[dtype] + weight[:, None] * v[:, g].abs().max()
            wrong = (got[rows, h][~none] - want).abs() > limits
            assert not wrong.any(), (b, h, wrong.nonzero()[:5], got[rows, h][~none][wrong][:5], want[wrong][:5])


def offsets_of(news, first=0):
    return [first + sum(news[:i]) for i in range(len(news) + 1)]


CHUNKS = [
    # new tokens, cached tokens, page, heads, kv_heads, dim
    ([1], [1], 16, 1, 1, 16),
    ([3, 0, 40], [17, 5, 300], 16, 8, 2, 128),
    ([100, 1, 64, 300], [257, 1, 64, 1000], 64, 8, 1, 64),
    ([5, 2, 0, 130], [3, 1, 0, 700], 32, 4, 2, 128),
    ([200, 3], [513, 3], 48, 6, 2, 96),
    ([333, 12], [1300, 12], 128, 20, 4, 80),
    ([4] * 33 + [7, 250], [40] * 33 + [777, 1200], 16, 3, 3, 112),
    ([31, 33], [31, 133], 16, 2, 1, 48),
    ([150], [3000], 16, 5, 1, 128),
    ([70], [9000], 64, 8, 2, 128),
    ([20, 0, 0, 1], [500, 70, 0, 2], 4096, 130, 1, 32),
    ([6, 9], [100, 50], 32, 4, 2, 192),
]


@pytest.mark.parametrize("code", (torch.float8_e4m3fn, torch.int8), ids=("e4m3", "int8"))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("case", CHUNKS, ids=range(len(CHUNKS)))
def test_chunk_attention(case, dtype, code):
    news, lens, page, heads, kv_heads, dim = case
    cache = filled_cache(lens, page, kv_heads, dim, code, spread=4.0)
    query = (torch.randn(sum(news), heads, dim) * 2).to(dtype)
    wide = torch.int64 if page == 64 else torch.int32
    scale = 0.7 * dim**-0.5
    args = (dev(query), *cache.args, index(cache.table.tolist(), wide), index(offsets_of(news), wide), index(lens, wide))
    got, lse = programs.chunk_attention(*args, scale=scale, return_lse=True)
    assert device_status() == 0 and got.dtype == dtype and got.shape == query.shape and lse.shape == query.shape[:2]
    check_chunk(query, cache, news, lens, scale, got, lse, dtype)
    assert torch.equal(programs.chunk_attention(*args, scale), got)


def test_chunk_attention_of_the_last_tokens_equals_paged_attention():
    lens = [300, 45, 8]
    cache = filled_cache(lens, 16, 2, 64, torch.int8)
    query = torch.randn(3, 5, 8, 64).half()
    tables = index(cache.table.tolist()), index(lens)
    want, want_lse = programs.paged_attention(dev(query), *cache.args, *tables, return_lse=True)
    got, lse = programs.chunk_attention(dev(query.flatten(0, 1)), *cache.args, tables[0], index([0, 5, 10, 15]), tables[1],
                                        return_lse=True)
    # weights of 11 bits in both
    assert ((got.view_as(want).float() - want.float()).abs() <= 2.0**-9 * 6).all()
    assert torch.allclose(lse.view_as(want_lse), want_lse, rtol=1e-5, atol=1e-5)


def test_chunk_attention_strides_and_rows_of_no_sequence():
    news, lens, heads, kv_heads, dim = [50, 90], [100, 700], 6, 3, 64
    cache = filled_cache(lens, 32, kv_heads, dim, torch.int8)
    qkv = torch.randn(3 + 140 + 4, heads + 2 * kv_heads, 2 * dim).half()
    offsets = index(offsets_of(news, 3))
    tables = index(cache.table.tolist()), offsets, index(lens)
    for query in (dev(qkv)[:, :heads, ::2], dev(qkv)[:, :heads, :dim], dev(qkv)[:, 1 : heads + 1, 3 : dim + 3],
                  dev(qkv)[:, :heads, :dim].transpose(0, 1).contiguous().transpose(0, 1)):
        spread = torch.full((heads, 147, dim + 5), 7.0, dtype=torch.float16, device="cuda")
        lse = torch.full((heads, 147), 7.0, device="cuda").t()
        out = spread.permute(1, 0, 2)[..., 5:]
        programs.chunk_attention_kernel(query, *cache.args, *tables, out, lse)
        check_chunk(query.cpu(), cache, news, lens, dim**-0.5, out, lse, torch.float16, first=3)
        assert (spread[..., :5] == 7).all()
        for rows in (slice(0, 3), slice(143, 147)):
            assert (out[rows] == 7).all() and (lse[rows] == 7).all()
    part = programs.chunk_attention(dev(qkv)[:, 2:4, :dim], *(x[:, 1:2] for x in cache.args), *tables)
    whole = programs.chunk_attention(dev(qkv)[:, :heads, :dim], *cache.args, *tables)
    assert torch.allclose(part[3:143], whole[3:143, 2:4], rtol=2.0**-9, atol=2.0**-9)
    assert device_status() == 0


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_chunk_attention_scales_far_apart(dtype):
    """Weights value_scale * p from pages of very different scales keep their bits."""
    news, lens, dim = [30], [1500], 64
    cache = filled_cache(lens, 16, 1, dim, torch.float8_e4m3fn, spread=14.0)
    query = torch.randn(30, 4, dim).to(dtype)
    cache.scales["key"].fill_(0.02)
    args = dev(query), *cache.args, index(cache.table.tolist()), index([0, 30]), index(lens)
    got, lse = programs.chunk_attention(*args, return_lse=True)
    check_chunk(query, cache, news, lens, dim**-0.5, got, lse, dtype)
    # pages of zeros with the least scale beside the others, and of scale 0, of keys too
    block = int(cache.table[0, 3])
    cache.caches["value"].view(torch.int8)[block] = 0
    cache.scales["value"][block] = 2.0**-126
    cache.scales["value"][int(cache.table[0, 5])] = 0
    cache.scales["key"][int(cache.table[0, 93])] = 0
    cache.scales["key"][int(cache.table[0, 7])] = 0
    got, lse = programs.chunk_attention(*args, return_lse=True)
    check_chunk(query, cache, news, lens, dim**-0.5, got, lse, dtype)


def test_chunk_attention_large_and_small_queries():
    """Rows are scaled to fp16 by powers of two: bfloat16's range, and elements beside an outlier."""
    news, lens, dim = [64], [400], 128
    cache = filled_cache(lens, 16, 1, dim, torch.int8)
    query = torch.randn(64, 2, dim)
    query[10:20] *= 2.0**100
    query[20:30] *= 2.0**-100
    query[30:40, :, 3] = 60000.0
    query[40:50] = 0.0
    cache.caches["key"][:, :, :, 3] = 0  # the outlier meets zeros: the others decide
    query = query.bfloat16()
    args = dev(query), *cache.args, index(cache.table.tolist()), index([0, 64]), index(lens)
    for scale, rows in ((dim**-0.5, [r for r in range(64) if not 10 <= r < 20]), (2.0**-100, list(range(10, 20)))):
        got, lse = programs.chunk_attention(*args, scale=scale, return_lse=True)
        k, v = ((c * s[..., None])[:, 0] for c, s in (cache.tokens(name, 0, 400) for name in ("key", "value")))
        for r in rows:
            s = query[r].double() @ k[: 337 + r].T * scale
            want = torch.softmax(s, dim=1) @ v[: 337 + r]
            size = (query[r, :, :3].double().abs() @ k[: 337 + r, :3].abs().T * scale).max() + s.abs().max()
            limit = 2.0**-8 * want.abs() + (2 * 136 * 2.0**-24 * float(size) * 40 + 2.0**-10) * v.abs().max()
            assert ((got[r].cpu().double() - want).abs() <= limit).all(), (scale, r)


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
@pytest.mark.parametrize("shape", ((200, 330), (4, 70), (130, 4000)))
def test_chunk_attention_nan_values_reach_only_who_sees_them(shape, dtype):
    new, length = shape
    for heads in (2, 8):
        cache = filled_cache([length], 16, 2, 128, torch.float8_e4m3fn)
        query = torch.randn(new, heads, 128).to(dtype)
        args = dev(query), *cache.args, index(cache.table.tolist()), index([0, new]), index([length])
        clean = programs.chunk_attention(*args)
        want = torch.zeros(new, heads, 128, dtype=torch.bool)
        limit = length - new + 1 + torch.arange(new)
        for token, group, element, code in ((length - 2, 0, 5, 127), (length - new // 2, 1, 100, 255), (length - new // 3, 1, 100, 127)):
            at = int(cache.table[0, token // 16])
            cache.caches["value"].view(torch.int8)[at, group, token % 16, element] = code if code < 128 else code - 256
            want[limit > token, group * heads // 2 : (group + 1) * heads // 2, element] = True
        got = programs.chunk_attention(*args).cpu()
        assert torch.equal(got.isnan(), want)
        assert torch.equal(got.nan_to_num(0.0), clean.cpu().masked_fill(want, 0.0))
    assert device_status() == 0


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
def test_chunk_attention_nan_keys_and_scales_reach_only_who_sees_them(dtype):
    new, length = 150, 600
    cache = filled_cache([length], 16, 1, 64, torch.float8_e4m3fn)
    query = torch.randn(new, 2, 64).to(dtype)
    args = dev(query), *cache.args, index(cache.table.tolist()), index([0, new]), index([length])
    clean = programs.chunk_attention(*args).cpu()
    limit = length - new + 1 + torch.arange(new)
    at = int(cache.table[0, 560 // 16])
    cache.caches["key"].view(torch.int8)[at, 0, 560 % 16, 5] = 127
    got = programs.chunk_attention(*args).cpu()
    assert got[limit > 560].isnan().all() and torch.equal(got[limit <= 560], clean[limit <= 560])
    cache.caches["key"].view(torch.int8)[at, 0, 560 % 16, 5] = 1
    for name in ("key", "value"):
        scales = cache.scales[name].clone()
        cache.scales[name][at] = math.nan
        got = programs.chunk_attention(*args).cpu()
        assert got[limit > 560].isnan().all() and torch.equal(got[limit <= 560], clean[limit <= 560])
        cache.scales[name].copy_(scales)


def test_chunk_attention_pages_outside_the_pool_are_not_seen():
    news, lens, dim = [140], [700], 64
    cache = filled_cache(lens, 16, 1, dim, torch.int8)
    query = torch.randn(140, 4, dim).half()
    table = cache.table.clone()
    table[0, 3], table[0, 41] = -1, 10**6
    got, lse = programs.chunk_attention(dev(query), *cache.args, index(table.tolist()), index([0, 140]), index(lens),
                                        return_lse=True)
    assert device_status() == INDEX_OUT_OF_RANGE
    k, v = ((c * s[..., None])[:, 0] for c, s in (cache.tokens(name, 0, 700) for name in ("key", "value")))
    for r in range(140):
        keep = [t for t in range(561 + r) if t // 16 not in (3, 41)]
        s = query[r].double() @ k[keep].T * dim**-0.5
        assert ((got[r].cpu().double() - torch.softmax(s, 1) @ v[keep]).abs() <= 2.0**-9 * v.abs().max()).all()
        assert ((lse[r].cpu().double() - torch.logsumexp(s, 1)).abs() <= 1e-5 * (1 + s.abs().max())).all()


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
def test_chunk_attention_bad_offsets_and_lengths(dtype):
    cache = filled_cache([64, 64], 16, 1, 64, torch.int8)
    query = torch.randn(20, 2, 64).to(dtype)
    table = index(cache.table.tolist())
    want = programs.chunk_attention(dev(query), *cache.args, table, index([0, 10, 20]), index([64, 64]))
    assert device_status() == 0
    for offsets, lengths, same in (
        ([0, 10, 30], [64, 64], slice(0, 10)),  # tokens that are not there
        ([-5, 10, 20], [64, 64], slice(10, 20)),
        ([0, 10, 5], [64, 64], slice(0, 5)),
        ([0, 10, 20], [64, 10**6], slice(0, 10)),  # more tokens than the block table holds
        ([0, 10, 20], [-3, 64], slice(10, 20)),
    ):
        out = torch.full_like(want, 7.0)
        programs.chunk_attention_kernel(dev(query), *cache.args, table, index(offsets), index(lengths), out)
        assert device_status() == INDEX_OUT_OF_RANGE
        assert torch.equal(out[same], want[same])


def test_chunk_attention_long_tail():
    """Many small weights beside a large one are not lost."""
    length, new, dim = 65536, 3, 64
    cache = filled_cache([length], 64, 1, dim, torch.int8)
    cache.caches["key"].zero_()
    cache.caches["key"][int(cache.table[0, 0]), 0, 0, 0] = 1
    cache.caches["value"].fill_(100)
    cache.caches["value"][int(cache.table[0, 0]), 0, 0] = 0
    for name in ("key", "value"):
        cache.scales[name].fill_(0.01)
    query = torch.zeros(new, 2, dim).half()
    query[:, :, 0] = 1.0
    for log2_ratio in (10.0, 17.0, 25.5):
        scale = log2_ratio * math.log(2) * 100
        got, lse = programs.chunk_attention(dev(query), *cache.args, index(cache.table.tolist()), index([0, new]),
                                            index([length]), scale=scale, return_lse=True)
        for r in range(new):
            tail = (length - new + r) * 2.0**-log2_ratio
            assert torch.allclose(got[r].cpu().double(), torch.tensor(tail / (1 + tail)).double(), rtol=2.0**-9)
            assert torch.allclose(lse[r].cpu().double(), torch.tensor(math.log(1 + tail) + log2_ratio * math.log(2)).double(),
                                  rtol=2e-5)


def test_chunk_attention_offsets_past_32_bits():
    """A pool of more than 2^32 bytes: pages at its end."""
    pages, page, dim = 70000, 64, 128
    keys = torch.zeros(pages, 8, page, dim, dtype=torch.int8, device="cuda")  # 4.6 GB
    keys[-3:] = torch.randint(-127, 128, (3, 8, page, dim), dtype=torch.int8)
    scales = torch.full((pages, 8), 0.01, device="cuda")
    query = torch.randn(30, 16, dim).half().cuda()
    table = index([[pages - 1, pages - 3, pages - 2]], torch.int64)
    got = programs.chunk_attention(query, keys, keys, scales, scales, table, index([0, 30], torch.int64),
                                   index([170], torch.int64))
    small = keys[-3:].clone()
    want = programs.chunk_attention(query, small, small, scales[:3], scales[:3], index([[2, 0, 1]]), index([0, 30]), index([170]))
    assert device_status() == 0 and torch.equal(got, want)


@pytest.mark.parametrize("scale", (0.0, -0.3))
def test_chunk_attention_scale_not_positive(scale):
    news, lens = [30], [200]
    cache = filled_cache(lens, 16, 1, 64, torch.int8)
    query = torch.randn(30, 2, 64).half()
    got, lse = programs.chunk_attention(dev(query), *cache.args, index(cache.table.tolist()), index([0, 30]), index(lens),
                                        scale=scale, return_lse=True)
    k, v = ((c * s[..., None])[:, 0] for c, s in (cache.tokens(name, 0, 200) for name in ("key", "value")))
    for r in range(30):
        s = query[r].double() @ k[: 171 + r].T * scale
        assert ((got[r].cpu().double() - torch.softmax(s, 1) @ v[: 171 + r]).abs() <= 2.0**-9 * v.abs().max()).all()


def test_chunk_attention_many_sequences():
    gen = torch.Generator().manual_seed(1)
    news = torch.randint(0, 4, (700,), generator=gen).tolist()
    lens = [n + int(x) for n, x in zip(news, torch.randint(0, 60, (700,), generator=gen))]
    cache = filled_cache(lens, 16, 2, 64, torch.int8)
    query = torch.randn(sum(news), 4, 64).half()
    got, lse = programs.chunk_attention(dev(query), *cache.args, index(cache.table.tolist()), index(offsets_of(news)),
                                        index(lens), return_lse=True)
    check_chunk(query, cache, news, lens, 0.125, got, lse, torch.float16)


def test_chunk_attention_empty_and_refusals():
    cache = filled_cache([20], 16, 2, 64, torch.int8)
    query = torch.randn(4, 4, 64).half().cuda()
    table, offsets, lengths = index(cache.table.tolist()), index([0, 4]), index([20])
    good = dict(query=query, key_cache=cache.args[0], value_cache=cache.args[1], key_scale=cache.args[2],
                value_scale=cache.args[3], block_table=table, offsets=offsets, lengths=lengths)
    out, lse = programs.chunk_attention(**(good | dict(query=query[:0])), return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    none = programs.chunk_attention(**(good | dict(block_table=table[:0], offsets=offsets[:1], lengths=lengths[:0])))
    assert none.shape == query.shape
    for bad in (dict(query=query[:, :3]), dict(query=query[:, :, :32]), dict(query=query.double()), dict(offsets=index([0])),
                dict(offsets=index([0, 4], torch.int64)), dict(lengths=index([20, 20])), dict(block_table=table[0]),
                dict(key_scale=cache.args[2][:1]), dict(value_cache=cache.args[1].float()), dict(query=query.cpu()),
                dict(key_cache=cache.args[0][:, :, ::2])):
        with pytest.raises(TypeError):
            programs.chunk_attention(**(good | bad))


def test_pieces_of_prompts_through_the_cache():
    """Appending a prompt piece by piece and attending for each piece gives what the whole prompt gives."""
    heads, kv_heads, dim, page = 8, 2, 64, 16
    pieces = [[40, 0, 7], [1, 90, 7], [130, 33, 0], [29, 2, 300]]
    totals = [sum(p[s] for p in pieces) for s in range(3)]
    qkv = [torch.randn(n, heads + 2 * kv_heads, dim).half() for n in totals]
    cos, sin = (t.cuda() for t in programs.rotary_tables(512, dim))
    blocks = [-(-n // page) for n in totals]
    order = torch.randperm(sum(blocks))
    table = torch.zeros(3, max(blocks), dtype=torch.int32)
    for s in range(3):
        table[s, : blocks[s]] = order[sum(blocks[:s]) : sum(blocks[: s + 1])]
    shape = (sum(blocks), kv_heads, page, dim)
    caches = [torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(shape[:2], device="cuda") for _ in range(2)]
    past, outs = [0, 0, 0], [[], [], []]
    for piece in pieces:
        packed = torch.cat([qkv[s][past[s] : past[s] + n] for s, n in enumerate(piece)]).cuda()
        q, k, v = packed.split((heads, kv_heads, kv_heads), dim=1)
        offsets = index(offsets_of(piece))
        query, _ = programs.paged_append(k, v, offsets, index(past), table.cuda(), *caches, *scales, query=q, cos=cos, sin=sin)
        past = [a + b for a, b in zip(past, piece)]
        out = programs.chunk_attention(query, *caches, *scales, table.cuda(), offsets, index(past))
        for s, part in enumerate(out.split(piece)):
            outs[s].append(part)
    packed = torch.cat(qkv).cuda()
    q, k, v = packed.split((heads, kv_heads, kv_heads), dim=1)
    offsets = index(offsets_of(totals))
    positions = torch.cat([torch.arange(n) for n in totals]).int().cuda()
    want = programs.prompt_attention(programs.rotary(q.contiguous(), cos, sin, positions),
                                     programs.rotary(k.contiguous(), cos, sin, positions), v, offsets)
    got = torch.cat([torch.cat(x) for x in outs])
    assert device_status() == 0
    # int8 codes are half a step (1/254 of a page's largest element, some 4) off
    assert float((got.float() - want.float()).abs().max()) < 0.1


def test_chunk_attention_streams_graphs_and_used_workspaces():
    news, lens = [70, 3, 200], [700, 3, 2000]
    cache = filled_cache(lens, 32, 2, 128, torch.float8_e4m3fn)
    tables = index(cache.table.tolist()), index(offsets_of(news)), index(lens)
    query = torch.randn(273, 8, 128).half().cuda()

    def call(q):
        return programs.chunk_attention(q, *cache.args, *tables)

    want = call(query)
    junk = torch.full((60 << 20,), 255, dtype=torch.uint8, device="cuda")  # what the next workspace may lie in
    del junk
    assert torch.equal(call(query), want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        side = [call(query) for _ in range(3)]
    both = [call(query) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in side + both)
    held = query.clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(held)
            twice = call(out)
        graphs.append((graph, out, twice))
    for factor in (1.0, -2.0):
        held.copy_(query * factor)
        first = call(held)
        second = call(first)
        for graph, out, twice in graphs:
            graph.replay()
            assert torch.equal(out, first) and torch.equal(twice, second)
    assert device_status() == 0
