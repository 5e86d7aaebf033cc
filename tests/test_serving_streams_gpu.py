"""Serving operators on other streams, in CUDA graphs and over workspaces of any contents."""

import pytest
import torch

from ninetoothed_b200 import _lib, device_status, programs
from tests.test_serving_gpu import dev, filled_cache, index

pytestmark = pytest.mark.gpu


def paged_case(lens=(1500, 3, 700), heads=8, kv_heads=2, dim=128):
    cache = filled_cache(list(lens), 16, kv_heads, dim, torch.float8_e4m3fn)
    query = torch.randn(len(lens), 1, heads, dim).half().cuda()
    return query, (*cache.args, index(cache.table.tolist()), index(list(lens)))


def prompt_case(lens=(300, 77, 1), heads=8, kv_heads=2, dim=64):
    qkv = torch.randn(sum(lens), heads + 2 * kv_heads, dim).half().cuda()
    offsets = index([sum(lens[:i]) for i in range(len(lens) + 1)])
    return (*qkv.split((heads, kv_heads, kv_heads), 1), offsets)


def test_replayed_graph_equals_eager_calls():
    query, rest = paged_case()
    prompt = prompt_case()
    cos, sin = programs.rotary_tables(64, 64)
    tables = dev(cos), dev(sin), torch.arange(query.shape[0], device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        programs.paged_attention(query, *rest), programs.prompt_attention(*prompt)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            turned = programs.rotary(query[:, 0], *tables)
            paged = programs.paged_attention(turned[:, None], *rest)
            attended = programs.prompt_attention(*prompt)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(4):
        query.copy_(torch.randn_like(query))
        prompt[0].copy_(torch.randn_like(prompt[0]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(paged, programs.paged_attention(programs.rotary(query[:, 0], *tables)[:, None], *rest))
        assert torch.equal(attended, programs.prompt_attention(*prompt))
    assert device_status() == 0


def test_streams_side_by_side():
    """Calls on several streams at once, each with its own workspace."""
    cases = [(paged_case(lens), prompt_case()) for lens in ((1500, 3), (40, 2000, 7), (900,))]
    want = [(programs.paged_attention(q, *rest), programs.prompt_attention(*p)) for (q, rest), p in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(10):
        for stream, ((q, rest), p), out in zip(streams, cases, got):
            with torch.cuda.stream(stream):
                out.append((programs.paged_attention(q, *rest), programs.prompt_attention(*p)))
    torch.cuda.synchronize()
    for expected, out in zip(want, got):
        for a, b in out:
            assert torch.equal(a, expected[0]) and torch.equal(b, expected[1])
    assert device_status() == 0


@pytest.mark.parametrize("fill", (0, 255, 0x3F))
def test_workspace_contents_do_not_matter(fill):
    """The join counters take whatever the workspace held, the last call's leavings too."""
    query, rest = paged_case()
    want = programs.paged_attention(query, *rest)
    out = torch.empty_like(want)
    nbytes = _lib.library().nt_b200_paged_attention_workspace_size()
    workspace = torch.full((nbytes,), fill, dtype=torch.uint8, device="cuda")
    key, value, ks, vs, table, lengths = rest
    args = _lib.pack_args(
        key.data_ptr(), value.data_ptr(), ks.data_ptr(), vs.data_ptr(), *key.shape, 12, *key.stride()[:3],
        *value.stride()[:3], *ks.stride(), *vs.stride(), query.data_ptr(), lengths.data_ptr(), table.data_ptr(),
        out.data_ptr(), 0, workspace.data_ptr(), nbytes, *query.shape[:3], table.shape[1], *query.stride(),
        *out.stride(), 0, 0, 0, 1, *table.stride(), 8, 2, scale=query.shape[-1] ** -0.5)
    for _ in range(3):
        out.zero_()
        stream = torch.cuda.current_stream().cuda_stream
        assert _lib.library().nt_b200_paged_attention(args, stream) == 0
        assert torch.equal(out, want)


def test_repeated_calls_are_bit_identical():
    """Sums are taken in a fixed order however the CTAs come to their ends."""
    query, rest = paged_case((3000, 1, 0, 2999), heads=12, kv_heads=3, dim=64)
    prompt = prompt_case((700, 3, 260))
    first = programs.paged_attention(query, *rest), programs.prompt_attention(*prompt)
    for _ in range(20):
        assert torch.equal(programs.paged_attention(query, *rest), first[0])
        assert torch.equal(programs.prompt_attention(*prompt), first[1])
