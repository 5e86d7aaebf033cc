"""The C++ binding of the norm, the 4-bit products and the attention of chunks: the same as the Python path."""

import pytest
import torch

from ninetoothed_b200 import _lib, programs
from tests.test_serving_binding import both


def test_odd_calls_are_left_alone():
    if not torch.cuda.is_available():
        pytest.skip("the binding asks for the current CUDA device")
    binding = _lib.binding()
    assert binding.rms_norm(1) is None and binding.int4_matmul(1) is None and binding.chunk_attention(1) is None
    assert binding.rms_norm(None, None, None, 1e-6, None, None) is None
    assert binding.rms_norm(1, 1, 1, 1, 1, 1) is None
    assert binding.int4_matmul(*[None] * 5) is None
    assert binding.chunk_attention(*[None] * 10) is None


@pytest.mark.gpu
def test_binding_equals_the_python_path(monkeypatch):
    from tests.test_serving_gpu import filled_cache, index

    calls = []
    real = _lib.binding()

    class Counted:
        def __getattr__(self, name):
            def call(*args):
                result = getattr(real, name)(*args)
                calls.append((name, result is not None))
                return result

            return call

    monkeypatch.setattr(_lib, "binding", Counted)

    def same(call):
        fast, slow = both(monkeypatch, call)
        fast, slow = (x if isinstance(x, tuple) else (x,) for x in (fast, slow))
        assert len(fast) == len(slow)
        for a, b in zip(fast, slow):
            assert a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(a.float(), b.float())

    x, weight = torch.randn(9, 200).half().cuda(), torch.rand(200).half().cuda()
    for kwargs in ({}, dict(residual=x * 2), dict(code_dtype=torch.int8), dict(code_dtype=torch.float8_e4m3fn, group=48),
                   dict(code_dtype=torch.int8, group=1000, residual=x), dict(eps=0.5)):
        same(lambda: programs.rms_norm(x, weight, **kwargs))
        same(lambda: programs.rms_norm(x[:, ::2], weight.float()[:100], **{k: v[:, ::2] if k == "residual" else v
                                                                           for k, v in kwargs.items()}))
    w = programs.int4_quantize(torch.randn(33, 192).half().cuda(), 64, symmetric=False)
    for rows in (x[:, :192], x[:, :192].contiguous(), x[:, :192].float()):
        same(lambda: programs.int4_matmul(rows, w[0], w[1]))
        same(lambda: programs.int4_matmul(rows, *w))
    codes, scale = programs.rms_norm(x[:, :192].contiguous(), weight[:192], code_dtype=torch.int8)
    same(lambda: programs.int4_matmul(codes, *w, input_scale=scale))
    same(lambda: programs.int4_matmul(codes, *w, input_scale=scale[:, 0]))
    cache = filled_cache([100, 7], 16, 2, 64, torch.float8_e4m3fn)
    rest = (*cache.args, index(cache.table.tolist()), index([0, 40, 43]), index([100, 7]))
    query = torch.randn(43, 8, 64).half().cuda()
    for kwargs in ({}, dict(scale=0.3), dict(return_lse=True)):
        same(lambda: programs.chunk_attention(query, *rest, **kwargs))
    assert all(made for name, made in calls if name in ("int4_matmul", "chunk_attention", "rms_norm"))
    assert {name for name, _ in calls} >= {"int4_matmul", "chunk_attention", "rms_norm"}


@pytest.mark.gpu
def test_calls_that_the_binding_leaves_are_refused_or_made():
    x, weight = torch.randn(4, 64).half().cuda(), torch.rand(64).half().cuda()
    assert torch.equal(programs.rms_norm(x, weight, eps=0), programs.rms_norm(x, weight, eps=0.0))
    grad = x.clone().requires_grad_()
    assert not programs.rms_norm(grad, weight).requires_grad
    for bad in (dict(group=True, code_dtype=torch.int8), dict(code_dtype="int8"), dict(eps=None)):
        with pytest.raises((TypeError, ValueError)):
            programs.rms_norm(x, weight, **bad)
    assert programs.rms_norm(x, weight, code_dtype=torch.int8, group=64)[1].shape == (4, 1)
