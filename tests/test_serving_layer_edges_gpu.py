"""The layer's operators: workspaces of any contents, host threads, offsets past 32 bits, a whole layer in a graph."""

import threading

import pytest
import torch

from ninetoothed_b200 import _lib, device_status, programs
from tests.test_serving_gpu import dev, filled_cache, index

pytestmark = pytest.mark.gpu


def chunk_case(news=(70, 3, 200, 0, 1), lens=(700, 3, 2000, 50, 4000), heads=8, kv_heads=2, dim=128):
    cache = filled_cache(list(lens), 32, kv_heads, dim, torch.float8_e4m3fn)
    query = torch.randn(sum(news), heads, dim).half().cuda()
    offsets = index([sum(news[:i]) for i in range(len(news) + 1)])
    return query, (*cache.args, index(cache.table.tolist()), offsets, index(list(lens)))


@pytest.mark.parametrize("fill", (0, 255, 0x3F, 0x7F))
def test_chunk_workspace_contents_do_not_matter(fill):
    query, rest = chunk_case()
    want = programs.chunk_attention(query, *rest)
    out = torch.empty_like(want)
    nbytes = _lib.library().nt_b200_chunk_attention_workspace_size()
    workspace = torch.full((nbytes,), fill, dtype=torch.uint8, device="cuda")
    key, value, ks, vs, table, offsets, lengths = rest
    args = _lib.pack_args(
        key.data_ptr(), value.data_ptr(), ks.data_ptr(), vs.data_ptr(), *key.shape, 12, *key.stride()[:3],
        *value.stride()[:3], *ks.stride(), *vs.stride(), query.data_ptr(), offsets.data_ptr(), lengths.data_ptr(),
        table.data_ptr(), out.data_ptr(), 0, workspace.data_ptr(), nbytes, query.shape[0], lengths.shape[0],
        query.shape[1], table.shape[1], *query.stride(), *out.stride(), 0, 0, 1, 1, *table.stride(), 8, 2,
        scale=query.shape[-1] ** -0.5)
    for _ in range(3):  # the last call's leavings too
        out.zero_()
        assert _lib.library().nt_b200_chunk_attention(args, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out, want)


def test_repeated_calls_are_bit_identical():
    query, rest = chunk_case()
    x, weight = torch.randn(30, 4096).half().cuda(), torch.rand(4096).half().cuda()
    w = [dev(t) for t in programs.int4_quantize(torch.randn(500, 4096).half(), 64, symmetric=False)]

    def calls():
        codes, scale = programs.rms_norm(x, weight, code_dtype=torch.int8)
        return programs.chunk_attention(query, *rest), codes, scale, programs.int4_matmul(codes, *w, scale), \
            programs.int4_matmul(x[:3], *w)

    first = calls()
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(first, calls()))
    assert device_status() == 0


def test_calls_from_several_host_threads():
    query, rest = chunk_case()
    x, weight = torch.randn(9, 1024).bfloat16().cuda(), torch.rand(1024).bfloat16().cuda()
    w = [dev(t) for t in programs.int4_quantize(torch.randn(130, 1024).bfloat16(), 128, symmetric=False)]

    def work():
        y, total = programs.rms_norm(x, weight, residual=x)
        return programs.chunk_attention(query, *rest), y, total, programs.int4_matmul(y, *w)

    want = work()
    torch.cuda.synchronize()
    results, errors, start = {}, [], threading.Barrier(4)

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                start.wait()
                outs = [work() for _ in range(8)]
            stream.synchronize()
            results[i] = outs
        except Exception as error:  # reported below
            errors.append(repr(error))

    pool = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in pool:
        t.start()
    for t in pool:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for outs in results.values():
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert device_status() == 0


def test_offsets_past_32_bits():
    outer, inner = 1_100_000, 8192  # 4.5 GB of codes
    codes = torch.zeros(outer, inner // 2, dtype=torch.uint8, device="cuda")
    codes[-40:] = torch.randint(0, 256, (40, inner // 2), dtype=torch.uint8, device="cuda")
    scales = torch.ones(outer, 64, dtype=torch.float16, device="cuda")
    scales[-40:] = torch.rand(40, 64, device="cuda").half()
    x = torch.randn(3, inner).half().cuda()
    got = programs.int4_matmul(x, codes, scales)
    want = programs.int4_matmul(x, codes[-40:].clone(), scales[-40:].clone())
    # another split of the columns: other sums of 8192 products
    assert torch.allclose(got[:, -40:].float(), want.float(), rtol=2.0**-9, atol=0.05)
    del codes, scales, got
    rows = torch.zeros(70_000, 32_768, dtype=torch.float16, device="cuda")  # 4.6 GB
    rows[-2:] = torch.randn(2, 32_768, device="cuda").half()
    weight = torch.rand(32_768, device="cuda").half()
    out = torch.empty_like(rows)
    programs.rms_norm_kernel(rows, weight, out)
    assert torch.equal(out[-2:], programs.rms_norm(rows[-2:].clone(), weight)) and not out[: 70_000 - 2].any()
    spread = rows.t()[:20_000]  # an element stride of 65536 bytes: 1.3 GB from a row's start to its end
    got = programs.rms_norm(spread[:, -9:], weight[:9])
    assert torch.equal(got, programs.rms_norm(spread[:, -9:].clone(), weight[:9]))


def test_a_layer_in_a_graph():
    """Norm, 4-bit projection, cache, attention of pieces, 4-bit projection, norm with the residual: captured and eager."""
    heads, kv_heads, dim, page = 4, 2, 64, 16
    width = heads * dim
    news, past = [20, 1, 7], [5, 40, 0]
    x = torch.randn(sum(news), width).half().cuda()
    weight = torch.rand(width).half().cuda()
    qkv4 = [dev(t) for t in programs.int4_quantize(torch.randn((heads + 2 * kv_heads) * dim, width).half() * width**-0.5, 64, False)]
    out4 = [dev(t) for t in programs.int4_quantize(torch.randn(width, width).half() * width**-0.5, 64, False)]
    cos, sin = (t.cuda() for t in programs.rotary_tables(64, dim))
    table = torch.randperm(9).view(3, 3).int().cuda()
    offsets = index([0, 20, 21, 28])
    before, lengths = index(past), index([a + b for a, b in zip(past, news)])
    start = [torch.randint(-90, 90, (9, kv_heads, page, dim), dtype=torch.int8).cuda() for _ in range(2)]
    scale0 = [torch.full((9, kv_heads), 0.01, device="cuda") for _ in range(2)]

    def layer(x, caches, scales):
        codes, scale = programs.rms_norm(x, weight, code_dtype=torch.float8_e4m3fn)
        qkv = programs.int4_matmul(codes, *qkv4, scale).view(-1, heads + 2 * kv_heads, dim)
        q, k, v = qkv.split((heads, kv_heads, kv_heads), dim=1)
        q, _ = programs.paged_append(k, v, offsets, before, table, *caches, *scales, query=q, cos=cos, sin=sin)
        attended = programs.chunk_attention(q, *caches, *scales, table, offsets, lengths)
        return programs.rms_norm(programs.int4_matmul(attended.flatten(1), *out4), weight, residual=x)

    def copies(tensors):
        return [t.clone() for t in tensors]

    held, caches, scales = x.clone(), copies(start), copies(scale0)
    layer(held, copies(start), copies(scale0))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, total = layer(held, caches, scales)
    for factor in (1.0, -0.5, 3.0):
        held.copy_(x * factor)
        for to, t in zip(caches + scales, start + scale0):
            to.copy_(t)
        graph.replay()
        want_caches, want_scales = copies(start), copies(scale0)
        want, want_total = layer(held, want_caches, want_scales)
        assert torch.equal(out, want) and torch.equal(total, want_total)
        assert all(torch.equal(a, b) for a, b in zip(caches + scales, want_caches + want_scales))
    assert out.isfinite().all() and device_status() == 0
