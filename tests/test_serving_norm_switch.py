"""rms_norm for callers that switch its 8-bit output on and off."""

import pytest
import torch

from ninetoothed_b200 import programs, serving


def test_no_codes_are_no_groups(monkeypatch):
    x, weight = torch.zeros(4, 64), torch.zeros(64)
    monkeypatch.setattr(serving, "_bound", lambda name, *args: (name, *args))
    for group in (None, 16, 128):
        assert programs.rms_norm(x, weight, code_dtype=None, group=group)[4:] == (1e-6, None, None)
        assert programs.rms_norm(x, weight, code_dtype=torch.int8, group=group)[5:] == (torch.int8, group)
    assert programs.rms_norm(x, weight)[4:] == (1e-6, None, None)
    with pytest.raises(TypeError):
        programs.rms_norm(x, weight, group=32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float32))
def test_a_switch_takes_the_groups_along(dtype):
    x, weight = torch.randn(7, 200).to(dtype).cuda(), torch.rand(200).to(dtype).cuda()
    for residual in (None, x * 2):
        want = programs.rms_norm(x, weight, residual)
        for group in (32, 128):
            got = programs.rms_norm(x, weight, residual, code_dtype=None, group=group)
            pairs = zip(got, want) if isinstance(want, tuple) else ((got, want),)
            assert all(torch.equal(a, b) for a, b in pairs)
            assert len(programs.rms_norm(x, weight, residual, code_dtype=torch.int8, group=group)) == 2 + (residual is not None)
