"""int4_matmul's most rows, without a GPU."""

import pytest

from ninetoothed_b200 import _lib
from tests.test_serving import packed


@pytest.mark.parametrize("dtype, scales, output, rows", (
    (10, 10, 10, 65535 * 8 + 1),  # float32: CUDA cores
    (8, 8, 8, 65535 * 32 + 1), (12, 8, 8, 65535 * 32 + 1),  # 16 and 8 bits
))
def test_more_rows_than_a_grid_holds_are_refused(dtype, scales, output, rows):
    args = packed("NtB200Int4MatmulArgs", rows=rows, inner=64, outer=8, group=32, dtype=dtype, scales_dtype=scales,
                  output_dtype=output, input=16, codes=16, scales=16, output=16, input_strides=(64, 1),
                  codes_strides=(32, 1), scales_strides=(2, 1), output_strides=(8, 1))
    assert _lib.library().nt_b200_int4_matmul(args, None) == 10001
