"""int4_matmul's zero points over their whole range, and beyond it."""

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests.test_serving_gpu import INDEX_OUT_OF_RANGE, dev
from tests.test_serving_layer_gpu import CODES, product, product_limit, weights

pytestmark = pytest.mark.gpu

SHAPES = [
    # rows, inner, outer, group: fragments of 8, 16 and 32 rows, tensor memory
    (2, 1056, 37, 32), (12, 2048, 130, 128), (20, 800, 70, 32), (24, 1536, 200, 256), (9, 1152, 20_000, 64),
]


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8))
@pytest.mark.parametrize("shape", SHAPES)
def test_zero_points_up_to_63(shape, dtype):
    rows, inner, outer, group = shape
    if dtype == torch.float32:
        outer = min(outer, 500)
    x = torch.randn(rows, inner) * (40 if dtype in CODES else 1)
    x = (x.round().clamp(-127, 127) if dtype == torch.int8 else x).to(dtype)
    scale_dtype = torch.float32 if dtype in CODES else torch.float16
    codes, scales, _ = weights(outer, inner, group, False, scale_dtype)
    zeros = torch.randint(0, 64, scales.shape, dtype=torch.uint8)
    zeros[0, 0], zeros[-1, -1] = 16, 63
    args = dev(x), dev(codes), dev(scales)
    out = scale_dtype if dtype in CODES else dtype
    got = programs.int4_matmul(*args, dev(zeros)).cpu().double()
    assert device_status() == 0
    want, size = product(x, codes, scales, zeros)
    wrong = (got - want).abs() > product_limit(want, size, out, inner, group)
    assert not wrong.any(), (wrong.nonzero()[:4], got[wrong][:4], want[wrong][:4])
    for value in (64, 128, 255):  # the first and the last of them say so
        for at in ((0, 0), (-1, -1)):
            beyond = zeros.clone()
            beyond[at] = value
            programs.int4_matmul(*args, dev(beyond))
            assert device_status() == INDEX_OUT_OF_RANGE
    # rows past the last one hold what the last call left in shared memory: nobody looks at it
    programs.int4_matmul(*args, dev(zeros))
    assert device_status() == 0
