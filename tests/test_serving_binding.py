"""The C++ binding of the serving calls: built, loaded, and the same as the Python path."""

import pytest
import torch

from ninetoothed_b200 import _lib, programs


def test_binding_is_built_and_leaves_odd_calls_alone():
    binding = _lib.binding()
    assert binding is not None
    x = torch.zeros(4, 2, 16)  # not on a CUDA device
    if not torch.cuda.is_available():
        pytest.skip("the binding asks for the current CUDA device")
    assert binding.rotary(x, x[0], x[0], x[0, 0], False, False) is None
    assert binding.rotary(x) is None
    assert binding.paged_append(*[None] * 14) is None
    assert binding.paged_attention(*[None] * 9) is None
    assert binding.prompt_attention(*[1] * 8) is None
    with pytest.raises(TypeError):
        binding.bind(1)


def both(monkeypatch, call):
    fast = call()
    with monkeypatch.context() as m:
        m.setattr(_lib, "binding", lambda: None)
        slow = call()
    return fast, slow


@pytest.mark.gpu
def test_binding_equals_the_python_path(monkeypatch):
    from tests.test_serving_gpu import filled_cache, index

    qkv = torch.randn(40, 12, 64).bfloat16().cuda()
    q, k, v = qkv.split((8, 2, 2), 1)
    cos, sin = (t.cuda() for t in programs.rotary_tables(64, 32))
    positions = torch.arange(40, device="cuda")
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
    for kwargs in ({}, dict(interleaved=True), dict(adjoint=True)):
        fast, slow = both(monkeypatch, lambda: programs.rotary(q, cos, sin, positions, **kwargs))
        assert torch.equal(fast, slow) and fast.stride() == slow.stride()
    offsets, past = index([0, 30, 40]), index([3, 0])
    table = index([[2, 0, 1], [3, 4, 5]])

    def append(**kwargs):
        caches = [torch.zeros(6, 2, 16, 64, dtype=torch.int8, device="cuda") for _ in range(2)]
        scales = [torch.ones(6, 2, device="cuda") for _ in range(2)]
        out = programs.paged_append(k, v, offsets, past, table, *caches, *scales, **kwargs)
        return *out, *caches, *scales

    for kwargs in (dict(query=q, cos=cos, sin=sin, return_key=True), dict(query=q, cos=cos, sin=sin, interleaved=True),
                   dict(cos=cos, sin=sin), {}):
        fast, slow = both(monkeypatch, lambda: append(**kwargs))
        for a, b in zip(fast, slow):
            assert (a is None and b is None) or torch.equal(a, b)
    cache = filled_cache([100, 7], 16, 2, 64, torch.float8_e4m3fn)
    rest = (*cache.args, index(cache.table.tolist()), index([100, 7]))
    query = torch.randn(2, 3, 8, 64).half().cuda()
    for kwargs in ({}, dict(scale=0.3), dict(return_lse=True)):
        for call in (lambda: programs.paged_attention(query, *rest, **kwargs),
                     lambda: programs.prompt_attention(q, k, v, offsets, **kwargs),
                     lambda: programs.prompt_attention(q, k, v, offsets, offsets, False, **kwargs)):
            fast, slow = both(monkeypatch, call)
            fast, slow = (x if isinstance(x, tuple) else (x,) for x in (fast, slow))
            assert len(fast) == len(slow) and all(torch.equal(a, b) for a, b in zip(fast, slow))
    assert {name for name, _ in calls} == {"rotary", "paged_append", "paged_attention", "prompt_attention"}
    assert all(made for _, made in calls)
    with pytest.raises(programs.KernelLaunchError):
        odd = torch.zeros(6 * 2 * 16 * 64 + 1, dtype=torch.int8, device="cuda")[1:].view(6, 2, 16, 64)
        programs.paged_append(k, v, offsets, past, table, odd, odd, *(torch.ones(6, 2, device="cuda") for _ in range(2)))
