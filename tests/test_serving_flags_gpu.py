"""Flags that have no truth value raise what Python raises, through the C++ binding too."""

import pytest
import torch

from ninetoothed_b200 import _lib, device_status, programs
from tests.test_serving_gpu import filled_cache, index

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bound", (True, False), ids=("binding", "python"))
def test_flags_without_a_truth_value(bound, monkeypatch):
    if not bound:
        monkeypatch.setattr(_lib, "binding", lambda: None)
    two = torch.tensor([1, 0])
    x = torch.randn(4, 2, 64).half().cuda()
    cos, sin = (t.cuda() for t in programs.rotary_tables(8, 64))
    at = index([0, 1, 2, 3])
    cache = filled_cache([4], 16, 2, 64, torch.int8)
    table, offsets = index(cache.table.tolist()), index([0, 4])
    calls = (
        lambda: programs.rotary(x, cos, sin, at, interleaved=two),
        lambda: programs.rotary(x, cos, sin, at, adjoint=two),
        lambda: programs.paged_append(x, x, offsets, index([0]), table, *cache.args, interleaved=two),
        lambda: programs.paged_append(x, x, offsets, index([0]), table, *cache.args, return_key=two),
        lambda: programs.paged_attention(x[:1, None], *cache.args, table, index([4]), return_lse=two),
        lambda: programs.prompt_attention(x, x, x, offsets, is_causal=two),
        lambda: programs.prompt_attention(x, x, x, offsets, return_lse=two),
    )
    for call in calls:
        with pytest.raises(RuntimeError, match="ambiguous"):
            call()
    assert device_status() == 0
