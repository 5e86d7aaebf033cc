"""The norm and the 4-bit products without a GPU: refusals on the host, quantization."""

import pytest
import torch

from ninetoothed_b200 import _lib, programs, serving
from tests.test_serving import packed


@pytest.mark.parametrize("struct, call, base, cases", [
    (
        "NtB200RmsNormArgs", "nt_b200_rms_norm",
        dict(rows=4, width=64, group=64, dtype=9, weight_dtype=9, output_dtype=9),
        [
            (dict(rows=-1), 10001), (dict(width=-1), 10001), (dict(group=-1), 10001), (dict(dtype=3), 10002),
            (dict(weight_dtype=8), 10002), (dict(output_dtype=10), 10002), (dict(output_dtype=13), 10002),
            (dict(rows=0), 0), (dict(width=0), 0), (dict(width=131073), 10003), (dict(output_dtype=0, group=24), 10003),
            (dict(output_dtype=12, group=0), 10003), (dict(), 10001),  # null pointers
            (dict(input=16, weight=16, output=16, residual=16), 10001),  # no room for the sum
            (dict(input=16, weight=16, output=16, output_dtype=0), 10001),  # nor for the scales
        ],
    ),
    (
        "NtB200Int4MatmulArgs", "nt_b200_int4_matmul",
        dict(rows=4, inner=64, outer=8, group=32, dtype=8, scales_dtype=8, output_dtype=8),
        [
            (dict(rows=-1), 10001), (dict(inner=-32), 10001), (dict(dtype=4), 10002), (dict(scales_dtype=0), 10002),
            (dict(output_dtype=12), 10002), (dict(rows=0), 0), (dict(outer=0), 0), (dict(group=16), 10003),
            (dict(group=0), 10003), (dict(inner=0), 10003), (dict(group=48, inner=96), 10003), (dict(inner=80), 10003),
            (dict(inner=1 << 31), 10003), (dict(), 10001),  # null pointers
        ],
    ),
])
def test_refused_on_the_host(struct, call, base, cases):
    entry = getattr(_lib.library(), call)
    assert entry(None, None) == 10001
    for change, code in cases:
        assert entry(packed(struct, **(base | change)), None) == code, change


def refused(launch, base, cases):
    for change in cases:
        with pytest.raises(TypeError):
            launch(base | change, 0)


def test_norm_shapes_are_refused_before_the_launch():
    x, w = torch.zeros(4, 64), torch.zeros(64)
    base = dict(input=x, weight=w, output=x, residual=None, total=None, scale=None, eps=1e-6, group=None)
    codes = torch.zeros(4, 64, dtype=torch.int8)
    scale = torch.zeros(4, 2)
    refused(serving._launch_rms_norm, base, (
        dict(weight=w[:32]), dict(weight=w.half()), dict(output=x[:2]), dict(output=x.half()), dict(total=x),
        dict(residual=x), dict(residual=x[:2], total=x), dict(residual=x.half(), total=x), dict(scale=scale),
        dict(output=codes), dict(output=codes, scale=scale), dict(output=codes, scale=scale, group=16),
        dict(output=codes, scale=scale, group=24), dict(output=codes, scale=scale, group=-32), dict(group=32),
        dict(eps=-1e-6), dict(eps=float("nan")),
    ))


def test_int4_shapes_are_refused_before_the_launch():
    x, codes, scales = torch.zeros(3, 64).half(), torch.zeros(5, 32, dtype=torch.uint8), torch.zeros(5, 2).half()
    base = dict(input=x, codes=codes, scales=scales, output=torch.zeros(3, 5).half(), zeros=None, input_scale=None)
    refused(serving._launch_int4_matmul, base, (
        dict(input=x[:, :32]), dict(codes=codes[:4]), dict(scales=scales[:4]), dict(output=torch.zeros(3, 5)),
        dict(output=torch.zeros(5, 3).half()), dict(zeros=torch.zeros(5, 1, dtype=torch.uint8)),
        dict(input_scale=torch.zeros(4)), dict(scales=torch.zeros(5, 4).half()), dict(scales=torch.zeros(5, 0).half()),
        dict(input=x.to(torch.int8), output=torch.zeros(3, 5)),
    ))


def test_quantized_weights_stand_for_the_weights():
    w = torch.randn(6, 128)
    for symmetric in (True, False):
        codes, scales, zeros = programs.int4_quantize(w, 32, symmetric)
        assert codes.shape == (6, 64) and codes.dtype == torch.uint8 and scales.shape == (6, 4)
        whole = torch.stack((codes & 15, codes >> 4), dim=2).view(6, 4, 32).float()
        back = (whole - (8 if symmetric else zeros.float()[:, :, None])) * scales[:, :, None]
        # half a step, and with a zero point rounded by half a step the ends another half
        off = (back.view(6, 128) - w).abs() / scales.repeat_interleave(32, dim=1)
        assert off.max() <= (0.5001 if symmetric else 1.0001)
    with pytest.raises(ValueError):
        programs.int4_quantize(w, 48)


def test_quantized_weights_of_parameters_strides_and_no_elements():
    w = torch.randn(64, 6)
    want = programs.int4_quantize(w.t().contiguous(), 32, False)
    got = programs.int4_quantize(torch.nn.Parameter(w).t(), 32, False)
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))
    for shape in ((0, 64), (5, 0), (0, 0)):
        codes, scales, zeros = programs.int4_quantize(torch.zeros(shape), 32, False)
        assert codes.shape == (shape[0], shape[1] // 2) and scales.shape == zeros.shape == (shape[0], shape[1] // 32)
    for bad in (w[0], w[None], w.to(torch.int8), w.double()):
        with pytest.raises(TypeError):
            programs.int4_quantize(bad, 32)
