"""paged_append at the edges of its arguments: tables without columns or rows, offsets out of order."""

import pytest
import torch

from ninetoothed_b200 import _lib, device_status, programs
from tests.test_serving_gpu import INDEX_OUT_OF_RANGE, index

pytestmark = pytest.mark.gpu


def empty_cache(pages, kv_heads=2, page=16, dim=32):
    caches = [torch.zeros(pages, kv_heads, page, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
    return *caches, *(torch.zeros(pages, kv_heads, device="cuda") for _ in range(2))


@pytest.fixture(params=(True, False), ids=("binding", "python"))
def path(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(_lib, "binding", lambda: None)


@pytest.mark.parametrize("dim", (32, 48))
@pytest.mark.parametrize("spread", (False, True))
def test_tables_without_columns_copy_the_query(path, dim, spread):
    """No rotated pairs: the query and the stored key are as they came, wherever the tokens stand."""
    q, k = torch.randn(20, 4, dim).half().cuda(), torch.randn(20, 2, dim).half().cuda()
    if spread:  # strides off the vector grid
        q = torch.stack((q, q), dim=-1)[..., 0]
    none = torch.zeros(3, 0, device="cuda")  # rows: fewer than tokens
    cache, plain = empty_cache(2, dim=dim), empty_cache(2, dim=dim)
    where = index([0, 20]), index([0]), index([[1, 0]])
    query, key = programs.paged_append(k, k, *where, *cache, query=q, cos=none, sin=none, return_key=True)
    programs.paged_append(k, k, *where, *plain)
    assert device_status() == 0
    assert torch.equal(query, q) and torch.equal(key, k)
    assert all(torch.equal(a, b) for a, b in zip(cache, plain))


def test_tables_without_rows_are_refused(path):
    """Every position is outside them: nothing may be stored as if there were no tables."""
    k = torch.randn(3, 2, 32).half().cuda()
    none = torch.zeros(0, 16, device="cuda")
    cache = empty_cache(1)
    with pytest.raises(TypeError, match="row"):
        programs.paged_append(k, k, index([0, 3]), index([0]), index([[0]]), *cache, cos=none, sin=none)
    assert not any(t.any() for t in cache)


@pytest.mark.parametrize("batch, step", ((3, 40), (80, 5)))
def test_offsets_out_of_order_are_recorded(batch, step):
    """A step back by more than two pages hides a sequence from the search by candidates."""
    k = torch.randn(400, 2, 32).half().cuda()
    good = [step * i for i in range(batch + 1)]
    table = index([[8 * s + c for c in range(8)] for s in range(batch)])  # 128 tokens each
    past = index([0] * batch)
    programs.paged_append(k, k, index(good), past, table, *empty_cache(8 * batch))
    assert device_status() == 0
    for at, value in ((1, 100), (batch - 1, good[-1] - 120), (batch, 0)):
        offsets = list(good)
        offsets[at] = value
        assert any(a > b for a, b in zip(offsets, offsets[1:])) and max(b - a for a, b in zip(offsets, offsets[1:])) <= 128
        programs.paged_append(k, k, index(offsets), past, table, *empty_cache(8 * batch))
        assert device_status() == INDEX_OUT_OF_RANGE, (at, value)
