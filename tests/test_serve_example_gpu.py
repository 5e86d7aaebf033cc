"""The serving example: what it decodes out of the cache is what whole prompts give."""

import importlib.util
from pathlib import Path

import pytest
import torch

from ninetoothed_b200 import device_status

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "serve.py"
    spec = importlib.util.spec_from_file_location("serve_example", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("code, step", ((torch.float8_e4m3fn, 2.0**-4), (torch.int8, 2.0**-7)), ids=("e4m3", "int8"))
def test_decoding_equals_whole_prompts(code, step):
    serve = example()
    steps = 12
    sequences, chosen = serve.serve(prompt_lengths=(19, 3, 130, 1), steps=steps, code=code)
    assert device_status() == 0
    # the same sequences as whole prompts, without a cache in between
    model = serve.Decoder()
    lengths = [len(s) for s in sequences]
    cache = serve.PagedCache(64, model.kv_heads, 16, model.head_dim, code, max(lengths), len(lengths))
    cache.reserve(lengths)
    offsets = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")
    whole = model.prompts(torch.cat(sequences), offsets, cache).float()
    size = float(whole.square().mean().sqrt())
    for s, end in enumerate(offsets[1:].tolist()):
        want = whole[end - steps - 1 : end - 1]
        got = chosen[:, s].float()
        assert torch.equal(got[0], want[0])  # chosen from the prompt's own logits
        # keys and values differ by half a step of their codes (a factor of at most 1 +- step
        # in each element, independent): logits by that much of their size, twice (k and v)
        assert float((got - want).square().mean().sqrt()) <= 2 * step * size
        assert torch.equal(got.argmax(-1), sequences[s][-steps:])
