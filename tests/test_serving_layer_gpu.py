"""The norm and the 4-bit products of a decoder's layer on the GPU against 64-bit implementations."""

import math

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import HALF, TINY, dev

pytestmark = pytest.mark.gpu

CODES = (torch.float8_e4m3fn, torch.int8)


# --------------------------------------------------------------------- norm
def norm_values(x, weight, residual, eps):
    """(stored sum, y as the kernel rounds it, y in 64 bits)."""
    total = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    t = total.double()
    root = 1.0 / torch.sqrt((t * t).sum(dim=1, keepdim=True) / x.shape[1] + eps)
    return total, total.float() * root.float() * weight.float(), t * root * weight.double()


def coded(y, dtype, group):
    """Codes and scales of fp32 values by the cache's rules."""
    rows, width = y.shape
    group = width if group is None else min(group, width)
    scales = []
    codes = torch.empty_like(y)
    for j in range(0, width, group):
        part = y[:, j : j + group]
        top = torch.where(part.isfinite(), part.abs(), 0.0).amax(dim=1)
        if dtype == torch.int8:
            s = torch.clamp(top * torch.tensor(1 / 127, dtype=torch.float32), min=2.0**-126)
            code = torch.nan_to_num(part * (1.0 / s)[:, None], nan=0.0, posinf=127, neginf=-127).round().clamp(-127, 127)
        else:
            fraction, exponent = torch.frexp(top)
            s = torch.ldexp(torch.ones_like(top), torch.clamp(exponent - 9 + (fraction > 0.875), min=-126))
            code = (part * (1.0 / s)[:, None]).clamp(-448, 448)
        scales.append(s)
        codes[:, j : j + group] = code
    return codes.to(dtype), torch.stack(scales, dim=1)


NORM_SHAPES = [(1, 8), (5, 16), (3, 100), (130, 128), (7, 1000), (33, 4096), (2, 4099), (3, 5120), (4, 16384), (3, 20000),
               (2, 32768), (2, 40000), (1, 131072)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_norm(shape, dtype):
    x, residual = torch.randn(shape).to(dtype), (torch.randn(shape) * 5).to(dtype)
    for weight in (torch.randn(shape[1]).to(dtype), torch.randn(shape[1])):
        for r in (None, residual):
            total, _, want = norm_values(x, weight, r, 1e-5)
            got = programs.rms_norm(dev(x), dev(weight), residual=None if r is None else dev(r), eps=1e-5)
            if r is not None:
                got, sums = got
                assert torch.equal(sums.cpu(), total)
            # r and the two products are rounded to fp32, then the result
            limit = (HALF[dtype] + 4 * 2.0**-24) * want.abs() + TINY[dtype]
            assert got.dtype == dtype and ((got.cpu().double() - want).abs() <= limit).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_norm_codes(shape, dtype, code):
    x, residual = torch.randn(shape).to(dtype), (torch.randn(shape) * 5).to(dtype)
    weight = torch.randn(shape[1]).to(dtype)
    for group in (None, 16, 48, 128, 512, 272):
        r = residual if group in (None, 48, 128) else None
        total, y, _ = norm_values(x, weight, r, 1e-5)
        got = programs.rms_norm(dev(x), dev(weight), residual=None if r is None else dev(r), eps=1e-5, code_dtype=code,
                                group=group)
        codes, scales = coded(y, code, group)
        assert len(got) == (2 if r is None else 3)
        assert got[1].shape == scales.shape and torch.equal(got[1].cpu(), scales)
        assert got[0].dtype == code and torch.equal(got[0].cpu().float(), codes.float())
        if r is not None:
            assert torch.equal(got[2].cpu(), total)


def test_norm_layouts_and_in_place():
    x, residual, weight = torch.randn(9, 640).half(), torch.randn(9, 640).half(), torch.randn(640).half()
    total, _, _ = norm_values(x, weight, residual, 1e-6)
    want = programs.rms_norm(dev(x), dev(weight), residual=dev(residual))[0]
    views = (
        lambda t: dev(t),
        lambda t: torch.cat((dev(t), dev(t)), dim=1)[:, : t.shape[1]],  # rows of a wider tensor
        lambda t: torch.cat((dev(t)[:, :1], dev(t)), dim=1)[:, 1:],  # off the 16-byte grid
        lambda t: dev(t).t().contiguous().t(),  # columns first
    )
    for view in views:
        got, sums = programs.rms_norm(view(x), torch.stack((dev(weight),) * 2, 1)[:, 0], residual=view(residual))
        assert torch.equal(got, want) and torch.equal(sums.cpu(), total)
        a, b = view(x).clone(memory_format=torch.preserve_format), view(residual)
        programs.rms_norm_kernel(a, dev(weight), a, b, b)  # over the input, the sum over the residual
        assert torch.equal(a, want) and torch.equal(b.cpu(), total)
        codes, scale, _ = programs.rms_norm(view(x), dev(weight), residual=view(residual), code_dtype=torch.int8, group=64)
        spread, other = torch.zeros(9, 1300, dtype=torch.int8, device="cuda"), torch.zeros(10, 9, device="cuda")
        programs.rms_norm_kernel(view(x), dev(weight), spread[:, 1:1281:2], view(residual), view(residual), other.t(), group=64)
        assert torch.equal(spread[:, 1:1281:2], codes) and torch.equal(other.t(), scale) and not spread[:, ::2].any()
    assert device_status() == 0


def test_norm_rows_that_are_zero_or_not_finite():
    x = torch.randn(6, 256)
    x[1] = 0.0
    x[2, 7] = math.inf
    x[3, 9] = math.nan
    x[4] *= 1e30  # squares leave fp32
    weight = torch.ones(256)
    got = programs.rms_norm(dev(x), dev(weight)).cpu()
    _, _, want = norm_values(x, weight, None, 1e-6)
    for row in (0, 1, 4, 5):
        assert ((got[row].double() - want[row]).abs() <= 5 * 2.0**-24 * want[row].abs()).all()
    assert got[2, 7].isnan() and not got[2, :7].any() and got[3].isnan().all()
    for code in CODES:
        codes, scale = programs.rms_norm(dev(x), dev(weight), code_dtype=code, group=64)
        assert not codes[1].float().any() and (scale[1] == 2.0**-126).all()
        assert (scale[3] == 2.0**-126).all()
        assert codes[3].float().isnan().all() if code != torch.int8 else not codes[3].any()
    assert programs.rms_norm(dev(x[1:2]), dev(weight), eps=0.0).isnan().all()  # 0 / 0


def test_norm_empty_and_refusals():
    x, w = torch.zeros(4, 64, device="cuda"), torch.zeros(64, device="cuda")
    assert programs.rms_norm(x[:0], w).shape == (0, 64)
    assert [t.shape for t in programs.rms_norm(x[:0], w, residual=x[:0], code_dtype=torch.int8)] == [(0, 64), (0, 1), (0, 64)]
    assert programs.rms_norm(x[:, :0], w[:0]).shape == (4, 0)
    for bad in (dict(weight=w[:32]), dict(weight=w.half()), dict(residual=x[:2]), dict(residual=x.half()), dict(group=32),
                dict(code_dtype=torch.int8, group=24), dict(code_dtype=torch.int8, group=-16), dict(code_dtype=torch.uint8),
                dict(eps=-1.0), dict(eps=math.nan), dict(weight=w.cpu()), dict(input=x[0])):
        with pytest.raises(TypeError):
            programs.rms_norm(**(dict(input=x, weight=w) | bad))
    with pytest.raises(TypeError):
        programs.rms_norm(torch.zeros(1, 131088, device="cuda"), torch.zeros(131088, device="cuda"))


# --------------------------------------------------------------------- 4-bit weights
def weights(outer, inner, group, zeros, dtype):
    codes = torch.randint(0, 256, (outer, inner // 2), dtype=torch.uint8)
    scales = (torch.rand(outer, inner // group) * 0.1 + 0.01).to(dtype)
    zero = torch.randint(0, 16, (outer, inner // group), dtype=torch.uint8) if zeros else None
    return codes, scales, zero


def product(x, codes, scales, zeros, input_scale=None):
    """(value, sum of magnitudes) in 64 bits."""
    outer, half = codes.shape
    whole = torch.stack((codes & 15, codes >> 4), dim=2).view(outer, scales.shape[1], -1).double()
    w = ((whole - (8 if zeros is None else zeros.double()[:, :, None])) * scales.double()[:, :, None]).view(outer, 2 * half)
    x = x.double() if input_scale is None else x.double() * input_scale.double().view(-1, 1)
    return x @ w.T, x.abs() @ w.abs().T


def product_limit(want, size, out, inner, group):
    # a tensor-core step adds 16 products to a sum, each cut to 24 bits of the
    # largest: 17 * 2^-24 of the magnitudes for every 16 elements of a group; then
    # one rounding a group, a part and an input scale (CUDA cores: one an element
    # of a lane, and those of its weight)
    steps = 1.1 * group + inner / group + inner / 32 + 32
    return steps * 2.0**-24 * size + HALF[out] * want.abs() + TINY[out]


INT4_SHAPES = [
    # rows, inner, outer, group
    (1, 32, 1, 32), (1, 64, 15, 64), (2, 96, 33, 96), (1, 4096, 100, 128), (3, 160, 64, 32), (5, 4128, 129, 32),
    (7, 1056, 17, 96), (8, 2048, 300, 1024), (9, 2048, 65, 64), (12, 10240, 48, 128), (16, 1536, 200, 512),
    (17, 4096, 131, 128), (32, 1024, 257, 32), (33, 512, 40, 64), (70, 768, 130, 256), (4, 4000, 5000, 32),
]


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8))
@pytest.mark.parametrize("shape", INT4_SHAPES)
def test_int4_matmul(shape, dtype):
    rows, inner, outer, group = shape
    eight = dtype in CODES
    x = torch.randn(rows, inner) * (40 if eight else 1)
    x = (x.round().clamp(-127, 127) if dtype == torch.int8 else x).to(dtype)
    for zeros in (False, True):
        scale_dtype = {torch.int8: torch.float32, torch.float8_e4m3fn: torch.float16}.get(dtype, dtype)
        if zeros and not eight:
            scale_dtype = torch.float32 if dtype == torch.float16 else torch.bfloat16
        codes, scales, zero = weights(outer, inner, group, zeros, scale_dtype)
        input_scale = torch.rand(rows) if eight and zeros else None
        got = programs.int4_matmul(dev(x), dev(codes), dev(scales), None if zero is None else dev(zero),
                                   None if input_scale is None else dev(input_scale))
        out = scales.dtype if eight else dtype
        want, size = product(x, codes, scales, zero, input_scale)
        assert got.dtype == out and got.shape == (rows, outer)
        wrong = (got.cpu().double() - want).abs() > product_limit(want, size, out, inner, group)
        assert not wrong.any(), (zeros, wrong.nonzero()[:4], got.cpu()[wrong][:4], want[wrong][:4])
        again = programs.int4_matmul(dev(x), dev(codes), dev(scales), None if zero is None else dev(zero),
                                     None if input_scale is None else dev(input_scale))
        assert torch.equal(got, again)
    assert device_status() == 0


def test_int4_layouts():
    """Weights cut out of larger ones, strides and starts off the grids, an output in columns."""
    x = torch.randn(6, 1056).half()
    codes, scales, zeros = weights(77, 1056, 32, True, torch.float16)  # 33 groups: rows of scales 2 bytes off the words
    want, size = product(x, codes, scales, zeros)
    limit = product_limit(want, size, torch.float16, 1056, 32)

    def wide(t, before=0, after=0):
        t = dev(t)
        parts = [t[:, :before], t, t[:, :after]]
        return torch.cat(parts, dim=1)[:, before : before + t.shape[1]]

    def spread(t):
        return torch.stack((dev(t), dev(t)), dim=2)[:, :, 0]

    for a, c, s, z in (
        (wide(x, 0, 8), wide(codes, 0, 16), wide(scales, 0, 3), wide(zeros, 0, 1)),
        (wide(x, 8, 0), wide(codes, 16, 0), wide(scales, 2, 0), wide(zeros, 4, 0)),
        (wide(x, 1, 0), dev(codes), dev(scales), dev(zeros)),
        (dev(x), wide(codes, 1, 2), dev(scales), dev(zeros)),
        (dev(x), dev(codes), wide(scales, 1, 0), wide(zeros, 1, 0)),
        (spread(x), spread(codes), spread(scales), spread(zeros)),
        (dev(x), dev(codes).t().contiguous().t(), dev(scales).t().contiguous().t(), dev(zeros).t().contiguous().t()),
    ):
        got = programs.int4_matmul(a, c, s, z)
        assert ((got.cpu().double() - want).abs() <= limit).all()
        columns = torch.zeros(78, 13, dtype=torch.float16, device="cuda")
        programs.int4_matmul_kernel(a, c, s, columns[:77, 1:13:2].t(), z)
        assert torch.equal(columns[:77, 1:13:2].t(), got) and not columns[77].any() and not columns[:, ::2].any()
    part = programs.int4_matmul(dev(x), dev(codes)[10:40], dev(scales)[10:40], dev(zeros)[10:40])
    assert ((part.cpu().double() - want[:, 10:40]).abs() <= limit[:, 10:40]).all()
    assert device_status() == 0


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float32))
def test_int4_values_that_are_not_finite_stay_in_their_rows(dtype):
    x = torch.randn(5, 512).to(dtype)
    x[1, 3], x[2, 500] = math.nan, math.inf
    codes, scales, _ = weights(40, 512, 64, False, dtype)
    codes[:, 250] |= 0x0F  # the infinity's weights are not 0
    scales[7] = math.nan
    got = programs.int4_matmul(dev(x), dev(codes), dev(scales)).cpu()
    want, size = product(x, codes, scales, None)
    assert got[1].isnan().all() and got[:, 7].isnan().all()
    keep = [n for n in range(40) if n != 7]
    limit = product_limit(want, size, dtype, 512, 64)
    for m in (0, 3, 4):
        assert ((got[m].double() - want[m]).abs() <= limit[m])[keep].all()
    assert not got[2].isfinite().any()


def test_int4_quantize():
    w = torch.randn(50, 512)
    w[3] = 0.0
    for dtype in (torch.float32, torch.float16):
        for group in (32, 128):
            for symmetric in (True, False):
                codes, scales, zeros = programs.int4_quantize(w.to(dtype), group, symmetric)
                assert (zeros is None) == symmetric
                eye = torch.eye(512, device="cuda")
                got = programs.int4_matmul(eye, dev(codes), dev(scales), None if symmetric else dev(zeros)).T.cpu()
                step = scales.float().repeat_interleave(group, dim=1)
                # half a step, and what the zero point's rounding and the scale's (2^-11 of 15 steps) move
                assert ((got - w.to(dtype).float()).abs() <= step * 1.02 + 1e-6).all()
                assert not got[3].any()
    for bad in (0, 48, 31, 384):
        with pytest.raises(ValueError):
            programs.int4_quantize(w, bad)


def test_int4_empty_and_refusals():
    x = torch.zeros(3, 64, dtype=torch.float16, device="cuda")
    codes, scales, zeros = (dev(t) for t in weights(5, 64, 32, True, torch.float16))
    assert programs.int4_matmul(x[:0], codes, scales).shape == (0, 5)
    assert programs.int4_matmul(x, codes[:0], scales[:0]).shape == (3, 0)
    for bad in (dict(input=x[:, :32]), dict(codes=codes[:4]), dict(scales=scales[:4]), dict(zeros=zeros[:, :1]),
                dict(zeros=zeros.to(torch.int8)), dict(input_scale=torch.zeros(2, device="cuda")), dict(input=x.double()),
                dict(codes=codes.to(torch.int8)), dict(scales=torch.zeros(5, 4, dtype=torch.float16, device="cuda")),
                dict(scales=torch.zeros(5, 0, dtype=torch.float16, device="cuda")), dict(input=x.cpu()),
                dict(input_scale=torch.zeros(3, 2, device="cuda"))):
        with pytest.raises(TypeError):
            programs.int4_matmul(**(dict(input=x, codes=codes, scales=scales) | bad))
    with pytest.raises(TypeError):
        programs.int4_matmul_kernel(x, codes, scales, torch.zeros(3, 5, device="cuda"))


# --------------------------------------------------------------------- together
def test_norm_into_4_bit_and_8_bit_products():
    """A layer's start: the norm's 8-bit rows into 4-bit weights, and into an 8-bit matrix product."""
    x, residual, weight = torch.randn(20, 512).bfloat16(), torch.randn(20, 512).bfloat16(), torch.rand(512).bfloat16()
    w = torch.randn(96, 512)
    codes4, scales4, _ = programs.int4_quantize(w, 64)
    for code in CODES:
        codes, scale, total = programs.rms_norm(dev(x), dev(weight), residual=dev(residual), code_dtype=code)
        got = programs.int4_matmul(codes, dev(codes4), dev(scales4), input_scale=scale)
        want, size = product(codes.cpu().float(), codes4, scales4, None, scale.cpu())
        assert ((got.cpu().double() - want).abs() <= product_limit(want, size, torch.float32, 512, 64)).all()
        _, _, y = norm_values(x, weight, residual, 1e-6)
        # 8 bits of each element: e4m3 2^-4 of it, int8 half of 1/127 of the row's largest
        off = 2.0**-4 * y.abs() if code != torch.int8 else y.abs().amax(dim=1, keepdim=True) / 254
        exact, _ = product(y, codes4, scales4, None)
        _, spread = product(off.expand_as(y) * 1.01 + 1e-6, codes4, scales4, None)
        assert ((got.cpu().double() - exact).abs() <= spread + 1e-3).all()
    codes, scale, _ = programs.rms_norm(dev(x), dev(weight), residual=dev(residual), code_dtype=torch.float8_e4m3fn)
    eight = w.T.contiguous().to(torch.float8_e4m3fn)
    out = torch.empty(20, 96, device="cuda")
    programs.matmul_kernel(codes, dev(eight), out)
    want = codes.cpu().double() @ eight.double()
    size = codes.cpu().double().abs() @ eight.double().abs()
    assert ((out.cpu().double() - want).abs() <= 2.0**-11 * want.abs() + 600 * 2.0**-24 * size + 2.0**-25).all()


def test_layer_products_in_a_graph_and_on_a_side_stream():
    x, weight = torch.randn(4, 1024).half().cuda(), torch.rand(1024).half().cuda()
    codes4, scales4, zeros4 = (dev(t) for t in programs.int4_quantize(torch.randn(260, 1024).half(), 64, symmetric=False))

    def layer(t):
        codes, scale = programs.rms_norm(t, weight, code_dtype=torch.int8)
        return programs.int4_matmul(codes, codes4, scales4, zeros4, scale)

    want = layer(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert torch.equal(layer(x), want)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x)
    for scale in (1.0, -3.0, 0.5):
        y = torch.randn(4, 1024).half().cuda() * scale
        expected = layer(y)
        x.copy_(y)
        graph.replay()
        assert torch.equal(out, expected)
