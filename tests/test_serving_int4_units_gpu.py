"""int4_matmul on fragments over more weight rows than the SMs' blocks take at once."""

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import dev
from tests.test_serving_layer_gpu import CODES, product, product_limit, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float8_e4m3fn, torch.int8))
@pytest.mark.parametrize("shape", ((3, 1056, 20_000, 32), (12, 1088, 40_000, 64), (20, 800, 60_000, 32), (16, 512, 65_536, 32)))
def test_blocks_that_go_on_to_other_weight_rows(shape, dtype):
    rows, inner, outer, group = shape
    x = torch.randn(rows, inner) * (40 if dtype in CODES else 1)
    x = (x.round().clamp(-127, 127) if dtype == torch.int8 else x).to(dtype)
    scale_dtype = torch.float32 if dtype in CODES else torch.float16
    codes, scales, zeros = weights(outer, inner, group, True, scale_dtype)
    by = torch.rand(rows) + 0.5 if dtype in CODES else None
    args = dev(x), dev(codes), dev(scales), dev(zeros), None if by is None else dev(by)
    got = programs.int4_matmul(*args)
    out = scale_dtype if dtype in CODES else dtype
    want, size = product(x, codes, scales, zeros, by)
    wrong = (got.cpu().double() - want).abs() > product_limit(want, size, out, inner, group)
    assert got.dtype == out and not wrong.any(), (wrong.nonzero()[:4], got.cpu()[wrong][:4], want[wrong][:4])
    assert torch.equal(got, programs.int4_matmul(*args)) and device_status() == 0
