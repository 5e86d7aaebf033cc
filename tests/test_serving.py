"""Serving operators without a GPU: tables, argument structs and refusals on the host."""

import math
import re
from pathlib import Path

import pytest
import torch

from ninetoothed_b200 import _lib, programs

HEADER = Path(__file__).resolve().parents[1] / "include" / "nt_b200.h"


def struct_fields(name):
    """(field, count) of an argument struct in the header, nested structs opened."""
    body = re.search(rf"typedef struct {name} \{{(.*?)\}} {name};", HEADER.read_text(), re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = []
    for line in filter(None, (part.strip() for part in body.split(";"))):
        kind, names = re.match(r"((?:const )?\w+)\s+(.*)", line, re.S).groups()
        for part in names.split(","):
            field, count = re.match(r"\s*\**(\w+)(?:\[(\d+)\])?\s*$", part).groups()
            if kind.startswith("NtB200"):
                fields += [(f"{field}.{inner}", n) for inner, n in struct_fields(kind)]
            else:
                fields.append((field, int(count or 1)))
    return fields


def packed(struct, **values):
    """A packed argument struct with the named fields set and the others zero."""
    out = []
    for field, count in struct_fields(struct):
        value = values.pop(field, 0)
        out += list(value) if count > 1 and value else [value] * count
    assert not values, values
    return _lib.pack_args(*out)  # a double 0.0 is eight zero bytes too


def test_rotary_tables():
    cos, sin = programs.rotary_tables(50, 16, base=100.0)
    angle = torch.arange(50, dtype=torch.float64)[:, None] * torch.tensor([100.0 ** (-i / 8) for i in range(8)]).double()
    assert cos.shape == sin.shape == (50, 8) and cos.dtype == torch.float32
    assert torch.allclose(cos.double(), angle.cos(), atol=1e-6) and torch.allclose(sin.double(), angle.sin(), atol=1e-6)
    slow, _ = programs.rotary_tables(50, 16, base=100.0, scaling="linear", factor=2.0)
    assert torch.equal(slow[::2], cos[:25])
    # ntk: the fastest pair keeps its speed, the slowest is slowed by the factor
    ntk_cos, ntk_sin = programs.rotary_tables(50, 16, base=100.0, scaling="ntk", factor=4.0)
    assert torch.equal(ntk_cos[:, 0], cos[:, 0])
    assert math.isclose(math.atan2(ntk_sin[1, 7], ntk_cos[1, 7]), 100.0 ** (-7 / 8) / 4, rel_tol=1e-6)
    # by parts: fast pairs keep their speed, slow ones are slowed by the factor
    part_cos, part_sin = programs.rotary_tables(9, 64, scaling="by_parts", factor=8.0, original_length=4096)
    size = 0.1 * math.log(8.0) + 1.0
    assert torch.allclose(part_cos**2 + part_sin**2, torch.full((9, 32), size * size), rtol=1e-6)
    assert math.isclose(math.atan2(part_sin[1, 0], part_cos[1, 0]), 1.0, rel_tol=1e-6)
    assert math.isclose(math.atan2(part_sin[1, 31], part_cos[1, 31]), 10000.0 ** (-31 / 32) / 8, rel_tol=1e-6)


@pytest.mark.parametrize("bad", (dict(rotary_dim=3), dict(rotary_dim=0), dict(factor=0.5), dict(scaling="other"),
                                 dict(scaling="by_parts", factor=2.0), dict(scaling="ntk", rotary_dim=2)))
def test_rotary_tables_refusals(bad):
    with pytest.raises(ValueError):
        programs.rotary_tables(**(dict(length=4, rotary_dim=8) | bad))


@pytest.mark.parametrize("struct, call, base, cases", [
    (
        "NtB200RotaryArgs", "nt_b200_rotary",
        dict(tokens=4, heads=2, head_dim=16, rotary_dim=8, table_rows=4, dtype=8, index_dtype=2),
        [
            (dict(tokens=-1), 10001), (dict(rotary_dim=7), 10001), (dict(dtype=3), 10002), (dict(index_dtype=1), 10002),
            (dict(rotary_dim=18), 10003), (dict(tokens=0), 0), (dict(heads=0), 0), (dict(head_dim=0, rotary_dim=0), 0),
            (dict(), 10001),  # null pointers
        ],
    ),
    (
        "NtB200PagedAppendArgs", "nt_b200_paged_append",
        {"tokens": 4, "batch": 1, "dtype": 9, "index_dtype": 3, "cache.pages": 4, "cache.kv_heads": 2, "cache.page": 16,
         "cache.head_dim": 64, "cache.code_dtype": 12},
        [
            (dict(batch=-1), 10001), (dict(dtype=11), 10002), (dict(index_dtype=10), 10002),
            ({"cache.code_dtype": 13}, 10002), ({"cache.page": 8}, 10003), ({"cache.head_dim": 40}, 10003),
            ({"cache.page": 0}, 10001), (dict(tokens=0), 0), (dict(batch=0), 0),
            (dict(), 10001),  # null pointers
            ({"cache.key": 16, "cache.value": 24, "cache.key_scale": 16, "cache.value_scale": 16}, 10001),  # off the grid
        ],
    ),
    (
        "NtB200PagedAttentionArgs", "nt_b200_paged_attention",
        {"batch": 1, "queries": 1, "heads": 4, "dtype": 9, "index_dtype": 3, "cache.pages": 4, "cache.kv_heads": 2,
         "cache.page": 16, "cache.head_dim": 64, "cache.code_dtype": 12, "cache.key": 16, "cache.value": 16,
         "cache.key_scale": 16, "cache.value_scale": 16},
        [
            (dict(queries=-1), 10001), (dict(dtype=12), 10002), (dict(index_dtype=8), 10002),
            ({"cache.code_dtype": 9}, 10002), ({"cache.page": 17}, 10003), ({"cache.head_dim": 272}, 10003),
            ({"heads": 3}, 10003), ({"cache.kv_heads": 0}, 10003), (dict(batch=0), 0), (dict(heads=0), 0),
            (dict(), 10001),  # null pointers
        ],
    ),
    (
        "NtB200PromptAttentionArgs", "nt_b200_prompt_attention",
        dict(query_tokens=4, key_tokens=4, batch=1, heads=4, kv_heads=2, head_dim=64, dtype=8, index_dtype=2),
        [
            (dict(key_tokens=-1), 10001), (dict(dtype=0), 10002), (dict(index_dtype=0), 10002), (dict(heads=3), 10003),
            (dict(kv_heads=0), 10003), (dict(head_dim=257), 10003), (dict(query_tokens=0), 0), (dict(batch=0), 0),
            (dict(heads=0), 0), (dict(head_dim=0), 0), (dict(), 10001),  # null pointers
        ],
    ),
])
def test_refused_on_the_host(struct, call, base, cases):
    entry = getattr(_lib.library(), call)
    assert entry(None, None) == 10001
    for change, code in cases:
        assert entry(packed(struct, **(base | change)), None) == code, change


def test_error_string():
    assert b"index" in _lib.library().nt_b200_error_string(10007)
    assert _lib.error_name(10007) == "NT_B200_ERR_INDEX_OUT_OF_RANGE"
