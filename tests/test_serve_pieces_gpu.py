"""The serving example with prompts in pieces and with 4-bit weights."""

import pytest
import torch

from ninetoothed_b200 import device_status
from tests.test_serve_example_gpu import example

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int4", (False, True), ids=("f16", "int4"))
@pytest.mark.parametrize("code, step", ((torch.float8_e4m3fn, 2.0**-4), (torch.int8, 2.0**-7)), ids=("e4m3", "int8"))
def test_prompts_in_pieces_equal_whole_prompts(code, step, int4):
    serve = example()
    lengths = (19, 3, 130, 1, 257)
    _, whole = serve.serve(prompt_lengths=lengths, steps=1, code=code, int4=int4)
    for piece in (1000, 48, 7):
        _, got = serve.serve(prompt_lengths=lengths, steps=1, code=code, piece=piece, int4=int4)
        assert device_status() == 0
        size = float(whole.float().square().mean().sqrt())
        # keys and values differ by half a step of their codes (a factor of at most 1 +- step
        # in each element, independent): logits by that much of their size, twice (k and v)
        assert float((got.float() - whole.float()).square().mean().sqrt()) <= 2 * step * size


def test_example_runs_with_everything():
    serve = example()
    sequences, chosen = serve.serve(prompt_lengths=(40, 2), steps=5, piece=16, int4=True)
    assert [len(s) for s in sequences] == [45, 7] and chosen.isfinite().all()
    assert device_status() == 0
