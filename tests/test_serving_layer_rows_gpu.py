"""int4_matmul of more than 16 rows: weights in tensor memory, parts of the columns, units that follow one another."""

import math

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import dev
from tests.test_serving_layer_gpu import product, product_limit, weights

pytestmark = pytest.mark.gpu

SHAPES = [
    # rows, inner, outer, group
    (17, 1024, 1, 128), (18, 1152, 127, 384), (31, 1280, 38_000, 256), (32, 8192, 128, 128), (33, 4096, 129, 1024),
    (64, 2176, 300, 128), (65, 1408, 7, 1408), (100, 1024, 11_000, 512), (300, 1536, 513, 768),
]


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("shape", SHAPES)
def test_rows(shape, dtype):
    rows, inner, outer, group = shape
    x = torch.randn(rows, inner).to(dtype)
    for zeros, scale_dtype in ((False, dtype), (True, torch.float32)):
        codes, scales, zero = weights(outer, inner, group, zeros, scale_dtype)
        args = dev(x), dev(codes), dev(scales), None if zero is None else dev(zero)
        got = programs.int4_matmul(*args)
        want, size = product(x, codes, scales, zero)
        wrong = (got.cpu().double() - want).abs() > product_limit(want, size, dtype, inner, group)
        assert not wrong.any(), (zeros, wrong.nonzero()[:4], got.cpu()[wrong][:4], want[wrong][:4])
        assert torch.equal(got, programs.int4_matmul(*args))
    assert device_status() == 0


def test_an_input_scale_and_an_output_in_columns():
    rows, inner, outer, group = 40, 1536, 200, 128
    wide = dev(torch.randn(rows + 3, inner + 64).half())
    x = wide[2:-1, 32:-32]  # rows further apart than they are long
    codes, scales, zeros = weights(outer, inner, group, True, torch.float16)
    by = torch.rand(rows, 2) + 0.5
    args = x, dev(codes), dev(scales), dev(zeros), dev(by)[:, 0]
    got = programs.int4_matmul(*args)
    want, size = product(x.cpu(), codes, scales, zeros, by[:, 0])
    assert ((got.cpu().double() - want).abs() <= product_limit(want, size, torch.float16, inner, group)).all()
    columns = torch.zeros(outer + 1, 2 * rows + 1, dtype=torch.float16, device="cuda")
    programs.int4_matmul_kernel(*args[:3], columns[:outer, 1::2].t(), *args[3:])
    assert torch.equal(columns[:outer, 1::2].t(), got) and not columns[outer].any() and not columns[:, ::2].any()
    assert device_status() == 0


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_values_that_are_not_finite_stay_in_their_rows(dtype):
    x = torch.randn(36, 1152).to(dtype)
    x[1, 3], x[34, 1100] = math.nan, math.inf
    codes, scales, _ = weights(140, 1152, 128, False, dtype)
    codes[:, 550] |= 0x0F  # the infinity's weights are not 0
    scales[7], scales[130, 2] = math.nan, math.inf
    got = programs.int4_matmul(dev(x), dev(codes), dev(scales)).cpu()
    want, size = product(x, codes, scales, None)
    assert got[1].isnan().all() and got[:, 7].isnan().all()
    assert not got[34].isfinite().any() and not got[:, 130].isfinite().any()
    limit = product_limit(want, size, dtype, 1152, 128)
    rows = [m for m in range(36) if m not in (1, 34)]
    columns = [n for n in range(140) if n not in (7, 130)]
    wrong = (got.double() - want).abs() > limit
    assert not wrong[rows][:, columns].any()


def test_two_streams_a_graph_and_other_kernels_between():
    """Blocks with tensor memory of their own beside others' (a large product, a tall one of another stream)."""
    torch.manual_seed(3)
    x = dev(torch.randn(48, 4096).bfloat16())
    w = [dev(t) for t in programs.int4_quantize(torch.randn(4096, 4096).bfloat16(), 128, symmetric=False)]
    a = dev(torch.randn(1024, 1024).bfloat16())

    def step():
        y = programs.int4_matmul(x, *w)
        return y, programs.matmul(a, a), programs.int4_matmul(y[:20], *w)

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(6):
        for stream in streams:
            with torch.cuda.stream(stream):
                outs.append(step())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        outs.append([t.clone() for t in captured])
    assert all(torch.equal(p, q) for out in outs for p, q in zip(out, want))
    assert device_status() == 0


def test_offsets_past_32_bits():
    outer, inner = 1_100_000, 8192  # 4.5 GB of codes
    codes = torch.zeros(outer, inner // 2, dtype=torch.uint8, device="cuda")
    codes[-300:] = torch.randint(0, 256, (300, inner // 2), dtype=torch.uint8, device="cuda")
    scales = torch.ones(outer, 64, dtype=torch.float16, device="cuda")
    scales[-300:] = torch.rand(300, 64, device="cuda").half()
    x = torch.randn(17, inner).half()
    got = programs.int4_matmul(dev(x), codes, scales)[:, -300:].cpu()
    want, size = product(x, codes[-300:].cpu(), scales[-300:].cpu(), None)
    assert ((got.double() - want).abs() <= product_limit(want, size, torch.float16, inner, 128)).all()
    assert device_status() == 0
