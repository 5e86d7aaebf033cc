"""Head dimensions above 128, which both attentions and the append take up to 256."""

import pytest
import torch

from ninetoothed_b200 import device_status, programs
from tests import test_serving_gpu as base
from tests.test_serving_gpu import HALF, dev, index

pytestmark = pytest.mark.gpu

APPENDS = [
    # past, new, page, heads, kv_heads, dim, rotary
    ([0, 20, 31], [70, 1, 3], 16, 8, 2, 192, 192),
    ([5, 64], [130, 9], 64, 4, 1, 256, 64),
    ([7], [40], 32, 3, 3, 144, 36),
]


@pytest.mark.parametrize("code", (torch.float8_e4m3fn, torch.int8), ids=("e4m3", "int8"))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("case", APPENDS, ids=range(len(APPENDS)))
def test_paged_append(case, dtype, code):
    base.test_paged_append(case, dtype, code)


PAGED = [
    # lens, queries, page, heads, kv_heads, dim
    ([1, 0, 90], 1, 16, 4, 2, 192),
    ([257, 33], 3, 64, 4, 1, 256),
    ([70], 2, 48, 3, 3, 144),
]


@pytest.mark.parametrize("code", (torch.float8_e4m3fn, torch.int8), ids=("e4m3", "int8"))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("case", PAGED, ids=range(len(PAGED)))
def test_paged_attention(case, dtype, code):
    base.test_paged_attention(case, dtype, code)


PROMPTS = [
    # query lengths, key lengths (None: the same), heads, kv_heads, dim
    ([1, 0, 130], None, 4, 2, 192),
    ([65, 17], None, 3, 1, 256),
    ([9, 20], [40, 20], 2, 2, 144),
]


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("case", PROMPTS, ids=range(len(PROMPTS)))
def test_prompt_attention(case, dtype, causal):
    base.test_prompt_attention(case, dtype, causal)


def test_above_256_is_refused():
    x = torch.zeros(2, 1, 272, dtype=torch.float16, device="cuda")
    with pytest.raises(TypeError, match="upper bound 256"):
        programs.prompt_attention(x, x, x, index([0, 2]))
    codes, scales = torch.zeros(1, 1, 16, 272, dtype=torch.int8, device="cuda"), torch.zeros(1, 1, device="cuda")
    with pytest.raises(TypeError, match="upper bound 256"):
        programs.paged_attention(dev(x[:1, None]), codes, codes, scales, scales, index([[0]]), index([1]))
    assert device_status() == 0
