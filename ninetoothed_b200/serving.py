"""Serving operators: rotary positions, a paged 8-bit key/value cache, attention
over it, and causal attention over packed prompts.

They carry a decoder's attention from the q/k/v projection to the attention
output and follow the conventions of `programs`: `*_kernel` objects bind and
check the arguments, launch on the caller's current stream and return their
first output; the plain functions allocate the outputs.  Every call goes
through `libnt_b200.so`.

Index tensors (positions, offsets, past, lengths, block_table) are int32 or
int64 CUDA tensors, one dtype a call.  Their values are checked by the kernels:
an index outside its array is not followed and shows in
`ninetoothed_b200.device_status()` as NT_B200_ERR_INDEX_OUT_OF_RANGE.  So do
offsets out of order, with which some or all tokens of the call are left out.
"""

import math
from operator import itemgetter

import torch

from ninetoothed_b200 import _lib
from ninetoothed_b200.runtime import FLOAT_DTYPES, Kernel, KernelLaunchError, TensorArg, check_same_dtype, dtype_code

INDEX_DTYPES = (torch.int32, torch.int64)
CODE_DTYPES = (torch.float8_e4m3fn, torch.int8)
_F32 = (torch.float32,)


def _bound(name, *args):
    """The call made by the C++ binding, which checks it, allocates its outputs and
    launches it; None where there is no binding or it left the call alone (one
    that is not as it should be, for which the kernel object below says why)."""
    binding = _lib.binding()
    if binding is None:
        return None
    result = getattr(binding, name)(*args)
    if result.__class__ is int:
        raise KernelLaunchError(result)
    return result


def _check_tables(v, head_dim):
    cos, sin = v["cos"], v["sin"]
    if cos.shape != sin.shape or 2 * cos.shape[1] > head_dim:
        raise TypeError(
            f"rotary tables {tuple(cos.shape)} and {tuple(sin.shape)} must agree and cover at most the head "
            f"dimension {head_dim}."
        )
    if cos.shape[1] > 1 and (cos.stride(1) != 1 or sin.stride(1) != 1):
        raise TypeError("Kernel arguments `cos`, `sin` must have unit stride along their last dimension.")


# --------------------------------------------------------------------- rotary
def rotary_tables(length, rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=None, device=None):
    """fp32 (cos, sin) tables [length, rotary_dim / 2] of the angles
    position * base^(-2i / rotary_dim), computed in 64 bits.

    `scaling` stretches them for contexts longer than the model was trained on
    (`factor` times as long):
      "linear"   positions divided by `factor`;
      "ntk"      base * factor^(rotary_dim / (rotary_dim - 2)): the slowest pair
                 is slowed by `factor`, the fastest not at all;
      "by_parts" pairs that turn at least 32 times over `original_length` keep
                 their speed, pairs that turn at most once are slowed by
                 `factor`, those between go linearly in the number of turns;
                 cos and sin are scaled by 0.1 ln(factor) + 1.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even; got {rotary_dim}.")
    if factor < 1.0:
        raise ValueError(f"factor must be at least 1; got {factor}.")
    pair = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim
    magnitude = 1.0
    if scaling is None or scaling == "linear":
        speed = base**-pair / (factor if scaling else 1.0)
    elif scaling == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2.")
        speed = (base * factor ** (rotary_dim / (rotary_dim - 2))) ** -pair
    elif scaling == "by_parts":
        if not original_length:
            raise ValueError("by_parts scaling needs original_length.")
        speed = base**-pair
        turns = original_length * speed / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        speed = speed * (keep + (1.0 - keep) / factor)
        magnitude = 0.1 * math.log(factor) + 1.0
    else:
        raise ValueError(f"unknown scaling {scaling!r}; expected linear, ntk or by_parts.")
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * speed
    return (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()


def _launch_rotary(v, stream):
    x, cos, sin, positions, out = v["input"], v["cos"], v["sin"], v["positions"], v["output"]
    check_same_dtype(v, ("input", "output"))
    if out.shape != x.shape or positions.shape[0] != x.shape[0]:
        raise TypeError(
            f"rotary shapes {tuple(x.shape)}, positions {tuple(positions.shape)} -> {tuple(out.shape)} disagree."
        )
    _check_tables(v, x.shape[2])
    args = _lib.pack_args(
        x.data_ptr(), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), out.data_ptr(), *x.shape,
        2 * cos.shape[1], cos.shape[0], *x.stride(), *out.stride(), cos.stride(0), sin.stride(0), positions.stride(0),
        bool(v["interleaved"]), bool(v["adjoint"]), dtype_code(x.dtype), dtype_code(positions.dtype),
    )
    return _lib.library().nt_b200_rotary(args, stream)


rotary_kernel = Kernel(
    name="rotary",
    args=(
        TensorArg("input", 3),
        TensorArg("cos", 2, _F32),
        TensorArg("sin", 2, _F32),
        TensorArg("positions", 1, INDEX_DTYPES),
        TensorArg("output", 3),
    ),
    outputs=("output",),
    launch=_launch_rotary,
    meta=("interleaved", "adjoint"),
    meta_defaults={"interleaved": False, "adjoint": False},
)


def rotary(input, cos, sin, positions, interleaved=False, adjoint=False):
    """`input` [tokens, heads, head_dim] with the first 2 * cos.shape[1] elements
    of every head rotated by row positions[t] of the tables (`rotary_tables`).
    Pairs are (i, i + half) or, interleaved, (2i, 2i + 1).  `adjoint` applies
    the transposed rotation: given the gradient of the output it returns the
    gradient of the input."""
    result = _bound("rotary", input, cos, sin, positions, interleaved, adjoint)
    if result is not None:
        return result
    output = torch.empty_like(input, memory_format=torch.contiguous_format)
    return rotary_kernel(input, cos, sin, positions, output, interleaved=interleaved, adjoint=adjoint)


# --------------------------------------------------------------------- paged cache
_cache_values = itemgetter("key_cache", "value_cache", "key_scale", "value_scale")


def _cache_args(v):
    """The fields of NtB200PagedCache, with the checks that need no device."""
    key, value, ks, vs = _cache_values(v)
    check_same_dtype(v, ("key_cache", "value_cache"))
    pages, heads, page, dim = key.shape
    if value.shape != key.shape or ks.shape != (pages, heads) or vs.shape != (pages, heads):
        raise TypeError(
            f"paged cache shapes {tuple(key.shape)}, {tuple(value.shape)} and scales {tuple(ks.shape)}, "
            f"{tuple(vs.shape)} disagree."
        )
    if page % 16 or dim % 16 or page > 4096:
        raise TypeError(
            f"a paged cache needs page size (at most 4096) and head dimension in multiples of 16; got {page} and {dim}."
        )
    k0, k1, k2, k3 = key.stride()
    v0, v1, v2, v3 = value.stride()
    if k3 != 1 or v3 != 1:
        raise TypeError("Kernel arguments `key_cache`, `value_cache` must have unit stride along their last dimension.")
    return (
        key.data_ptr(), value.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, heads, page, dim,
        dtype_code(key.dtype), k0, k1, k2, v0, v1, v2, *ks.stride(), *vs.stride(),
    )


_CACHE_ARGS = (
    TensorArg("key_cache", 4, CODE_DTYPES),
    TensorArg("value_cache", 4, CODE_DTYPES),
    TensorArg("key_scale", 2, _F32),
    TensorArg("value_scale", 2, _F32),
)


_append_values = itemgetter("key", "value", "query", "offsets", "past", "block_table", "query_out", "key_out", "cos",
                            "sin")


def _launch_paged_append(v, stream):
    key, value, query, offsets, past, table, query_out, key_out, cos, sin = _append_values(v)
    check_same_dtype(v, ("key", "value"))
    check_same_dtype(v, ("offsets", "past", "block_table"))
    cache = _cache_args(v)
    tokens, kv_heads, dim = key.shape
    batch = past.shape[0]
    if value.shape != key.shape or (kv_heads, dim) != (cache[5], cache[7]):
        raise TypeError(
            f"paged_append key {tuple(key.shape)}, value {tuple(value.shape)} and cache "
            f"{tuple(v['key_cache'].shape)} disagree."
        )
    if offsets.shape[0] != batch + 1 or table.shape[0] != batch:
        raise TypeError(f"paged_append needs {batch + 1} offsets and {batch} block table rows.")
    turns = cos is not None
    if turns != (sin is not None):
        raise TypeError("Kernel arguments `cos`, `sin` must be given together.")
    if turns:
        _check_tables(v, dim)
        if tokens and cos.shape[1] and not cos.shape[0]:
            # their address is null, which would mean that nothing is rotated
            raise TypeError("Kernel arguments `cos`, `sin` have no rows: every position is outside them.")
    if query is not None:
        check_same_dtype(v, ("key", "query"))
        if not turns or query_out is None:
            raise TypeError("paged_append rotates `query` into `query_out` and needs `cos` and `sin` for it.")
        check_same_dtype(v, ("query", "query_out"))
        if query.shape[0] != tokens or query.shape[2] != dim or query_out.shape != query.shape:
            raise TypeError(f"paged_append query {tuple(query.shape)} disagrees with key {tuple(key.shape)}.")
    if key_out is not None:
        check_same_dtype(v, ("key", "key_out"))
        if key_out.shape != key.shape:
            raise TypeError("paged_append key_out must have the key's shape.")
    none3 = (0, 0, 0)
    args = _lib.pack_args(
        *cache, key.data_ptr(), value.data_ptr(), query.data_ptr() if query is not None else 0,
        cos.data_ptr() if turns else 0, sin.data_ptr() if turns else 0, offsets.data_ptr(), past.data_ptr(),
        table.data_ptr(), query_out.data_ptr() if query is not None else 0,
        key_out.data_ptr() if key_out is not None else 0, tokens, batch, query.shape[1] if query is not None else 0,
        2 * cos.shape[1] if turns else 0, cos.shape[0] if turns else 0, table.shape[1], *key.stride(),
        *value.stride(), *(query.stride() if query is not None else none3),
        *(query_out.stride() if query is not None else none3), *(key_out.stride() if key_out is not None else none3),
        cos.stride(0) if turns else 0, sin.stride(0) if turns else 0, offsets.stride(0), past.stride(0),
        *table.stride(), bool(v["interleaved"]), dtype_code(key.dtype), dtype_code(offsets.dtype),
    )
    return _lib.library().nt_b200_paged_append(args, stream)


paged_append_kernel = Kernel(
    name="paged_append",
    args=(
        TensorArg("key", 3),
        TensorArg("value", 3),
        TensorArg("offsets", 1, INDEX_DTYPES),
        TensorArg("past", 1, INDEX_DTYPES),
        TensorArg("block_table", 2, INDEX_DTYPES),
        *_CACHE_ARGS,
        TensorArg("query", 3, optional=True),
        TensorArg("cos", 2, _F32, optional=True),
        TensorArg("sin", 2, _F32, optional=True),
        TensorArg("query_out", 3, optional=True),
        TensorArg("key_out", 3, optional=True),
    ),
    outputs=(),  # the cache is updated in place; the kernel returns None
    launch=_launch_paged_append,
    meta=("interleaved",),
    meta_defaults={"interleaved": False, "query": None, "cos": None, "sin": None, "query_out": None, "key_out": None},
)


def paged_append(key, value, offsets, past, block_table, key_cache, value_cache, key_scale, value_scale, query=None,
                 cos=None, sin=None, interleaved=False, return_key=False):
    """Appends packed tokens to a paged 8-bit cache, in place, and returns
    (rotated query, rotated key).

    `key`, `value` [tokens, kv_heads, head_dim]: the new tokens of all sequences
    one after another, sequence s from offsets[s] to offsets[s + 1] (`offsets`:
    batch + 1 entries); past[s] tokens of it are in the cache already.  Token
    position p goes to page block_table[s, p // page], slot p % page, of
    `key_cache` and `value_cache` [pages, kv_heads, page, head_dim]
    (float8_e4m3fn or int8; page and head_dim multiples of 16) as
    round(x / scale), with one fp32 scale a page and head in `key_scale` and
    `value_scale` [pages, kv_heads].  Where a part-filled page's scale has to
    grow, the codes it holds are rounded again.  A page that several sequences
    share must be full.

    With `cos` and `sin` (`rotary_tables`) the key is rotated at its position
    before it is stored, and `query` [tokens, heads, head_dim], if given, is
    rotated too and returned; `return_key` also returns the rotated key in its
    own dtype (a prompt's attention reads it).  What was not asked for is None.
    Tokens that belong to no sequence are written in neither, nor keys that an
    index out of range keeps from the cache.
    """
    result = _bound("paged_append", key, value, offsets, past, block_table, key_cache, value_cache, key_scale,
                    value_scale, query, cos, sin, interleaved, return_key)
    if result is not None:
        return result
    query_out = None if query is None else torch.empty_like(query, memory_format=torch.contiguous_format)
    key_out = torch.empty_like(key, memory_format=torch.contiguous_format) if return_key else None
    paged_append_kernel(key, value, offsets, past, block_table, key_cache, value_cache, key_scale, value_scale,
                        query, cos, sin, query_out, key_out, interleaved=interleaved)
    return query_out, key_out


# --------------------------------------------------------------------- attention over the cache
_attention_values = itemgetter("query", "output", "lse", "lengths", "block_table")


def _launch_paged_attention(v, stream):
    query, out, lse, lengths, table = _attention_values(v)
    check_same_dtype(v, ("query", "output"))
    check_same_dtype(v, ("lengths", "block_table"))
    cache = _cache_args(v)
    batch, queries, heads, dim = query.shape
    kv_heads, cache_dim = cache[5], cache[7]
    if out.shape != query.shape or dim != cache_dim or not kv_heads or heads % kv_heads:
        raise TypeError(
            f"paged_attention query {tuple(query.shape)}, cache {tuple(v['key_cache'].shape)} and output "
            f"{tuple(out.shape)} disagree."
        )
    if dim > 256:
        raise TypeError("Kernel argument `query` has head dimension above the upper bound 256.")
    if lengths.shape[0] != batch or table.shape[0] != batch:
        raise TypeError(f"paged_attention needs {batch} lengths and block table rows.")
    if lse is not None and lse.shape != query.shape[:3]:
        raise TypeError("paged_attention lse must have the query's shape without the head dimension.")
    lib = _lib.library()
    nbytes = lib.nt_b200_paged_attention_workspace_size()
    workspace = query.new_empty(nbytes, dtype=torch.uint8)
    args = _lib.pack_args(
        *cache, query.data_ptr(), lengths.data_ptr(), table.data_ptr(), out.data_ptr(),
        0 if lse is None else lse.data_ptr(), workspace.data_ptr(), nbytes, batch, queries, heads, table.shape[1],
        *query.stride(), *out.stride(), *((0, 0, 0) if lse is None else lse.stride()), lengths.stride(0),
        *table.stride(), dtype_code(query.dtype), dtype_code(lengths.dtype), scale=_scale(v["scale"], dim),
    )
    return lib.nt_b200_paged_attention(args, stream)


def _scale(scale, dim):
    return dim**-0.5 if scale is None else float(scale)


paged_attention_kernel = Kernel(
    name="paged_attention",
    args=(
        TensorArg("query", 4),
        *_CACHE_ARGS,
        TensorArg("block_table", 2, INDEX_DTYPES),
        TensorArg("lengths", 1, INDEX_DTYPES),
        TensorArg("output", 4),
        TensorArg("lse", 3, _F32, optional=True),
    ),
    outputs=("output",),
    launch=_launch_paged_attention,
    meta=("scale",),
    meta_defaults={"scale": None, "lse": None},
)


def paged_attention(query, key_cache, value_cache, key_scale, value_scale, block_table, lengths, scale=None,
                    return_lse=False):
    """Attention of each sequence's newest tokens over the paged 8-bit cache that
    holds them (`paged_append`); tokens of a page outside the pool are not seen.

    `query` [batch, queries, heads, head_dim]: query i of sequence b sees its
    first lengths[b] - queries + 1 + i tokens (one query: all of them; several,
    such as drafted tokens: each up to itself).  Query head h reads key/value
    head h // (heads // kv_heads).  `scale` is 1 / sqrt(head_dim) by default.
    Returns the output, in the query's shape and dtype, or with `return_lse`
    (output, lse): the fp32 natural logarithm of each query's sum of exponentials
    [batch, queries, heads], by which attention over separate keys is joined.  A
    query that sees no token gets 0, and -inf as its lse."""
    result = _bound("paged_attention", query, key_cache, value_cache, key_scale, value_scale, block_table, lengths,
                    scale, return_lse)
    if result is not None:
        return result
    output = torch.empty_like(query, memory_format=torch.contiguous_format)
    lse = query.new_empty(query.shape[:3], dtype=torch.float32) if return_lse else None
    paged_attention_kernel(query, key_cache, value_cache, key_scale, value_scale, block_table, lengths, output, lse,
                           scale=scale)
    return (output, lse) if return_lse else output


# --------------------------------------------------------------------- attention over prompts
def _launch_prompt_attention(v, stream):
    query, key, value, out, lse = v["query"], v["key"], v["value"], v["output"], v["lse"]
    query_offsets, key_offsets = v["query_offsets"], v["key_offsets"]
    check_same_dtype(v, ("query", "key", "value", "output"))
    check_same_dtype(v, ("query_offsets", "key_offsets"))
    tokens, heads, dim = query.shape
    kv_heads = key.shape[1]
    if value.shape != key.shape or key.shape[2] != dim or out.shape != query.shape or not kv_heads or heads % kv_heads:
        raise TypeError(
            f"prompt_attention query {tuple(query.shape)}, key {tuple(key.shape)}, value {tuple(value.shape)} and "
            f"output {tuple(out.shape)} disagree."
        )
    if dim > 256:
        raise TypeError("Kernel argument `query` has head dimension above the upper bound 256.")
    batch = query_offsets.shape[0] - 1
    if batch < 0 or key_offsets.shape != query_offsets.shape:
        raise TypeError("prompt_attention needs as many query offsets as key offsets, one more than sequences.")
    if lse is not None and lse.shape != query.shape[:2]:
        raise TypeError("prompt_attention lse must have the query's shape without the head dimension.")
    lib = _lib.library()
    nbytes = lib.nt_b200_prompt_attention_workspace_size(tokens, batch, heads, kv_heads)
    workspace = query.new_empty(nbytes, dtype=torch.uint8)
    args = _lib.pack_args(
        query.data_ptr(), key.data_ptr(), value.data_ptr(), query_offsets.data_ptr(), key_offsets.data_ptr(),
        out.data_ptr(), 0 if lse is None else lse.data_ptr(), workspace.data_ptr(), nbytes, tokens, key.shape[0], batch,
        heads, kv_heads, dim, *query.stride(), *key.stride(), *value.stride(), *out.stride(),
        *((0, 0) if lse is None else lse.stride()), query_offsets.stride(0), key_offsets.stride(0),
        bool(v["is_causal"]), dtype_code(query.dtype), dtype_code(query_offsets.dtype), scale=_scale(v["scale"], dim),
    )
    return lib.nt_b200_prompt_attention(args, stream)


prompt_attention_kernel = Kernel(
    name="prompt_attention",
    args=(
        TensorArg("query", 3),
        TensorArg("key", 3),
        TensorArg("value", 3),
        TensorArg("query_offsets", 1, INDEX_DTYPES),
        TensorArg("key_offsets", 1, INDEX_DTYPES),
        TensorArg("output", 3),
        TensorArg("lse", 2, _F32, optional=True),
    ),
    outputs=("output",),
    launch=_launch_prompt_attention,
    meta=("is_causal", "scale"),
    meta_defaults={"is_causal": True, "scale": None, "lse": None},
)


def prompt_attention(query, key, value, offsets, key_offsets=None, is_causal=True, scale=None, return_lse=False):
    """Attention over whole prompts packed one after another.

    `query` [tokens, heads, head_dim], `key` and `value` [tokens, kv_heads,
    head_dim]: sequence s from offsets[s] to offsets[s + 1] (`offsets`: batch + 1
    entries), its keys from key_offsets[s] to key_offsets[s + 1] where they
    differ (a prompt's later part against all of its keys: the last query stands
    at the last key).  Causal queries see the keys up to their own; query head h
    reads key/value head h // (heads // kv_heads).  `scale` is
    1 / sqrt(head_dim) by default.  Returns the output, in the query's shape and
    dtype, or with `return_lse` (output, lse): the fp32 natural logarithm of each
    query's sum of exponentials [tokens, heads].  A query that sees no key gets
    0, and -inf as its lse; tokens that belong to no sequence are not written."""
    result = _bound("prompt_attention", query, key, value, offsets, offsets if key_offsets is None else key_offsets,
                    is_causal, scale, return_lse)
    if result is not None:
        return result
    output = torch.empty_like(query, memory_format=torch.contiguous_format)
    lse = query.new_empty(query.shape[:2], dtype=torch.float32) if return_lse else None
    prompt_attention_kernel(query, key, value, offsets, offsets if key_offsets is None else key_offsets, output, lse,
                            is_causal=is_causal, scale=scale)
    return (output, lse) if return_lse else output


# --------------------------------------------------------------------- attention of chunks over the cache
_chunk_values = itemgetter("query", "output", "lse", "offsets", "lengths", "block_table")


def _launch_chunk_attention(v, stream):
    query, out, lse, offsets, lengths, table = _chunk_values(v)
    check_same_dtype(v, ("query", "output"))
    check_same_dtype(v, ("offsets", "lengths", "block_table"))
    cache = _cache_args(v)
    tokens, heads, dim = query.shape
    kv_heads, cache_dim = cache[5], cache[7]
    batch = lengths.shape[0]
    if out.shape != query.shape or dim != cache_dim or not kv_heads or heads % kv_heads:
        raise TypeError(
            f"chunk_attention query {tuple(query.shape)}, cache {tuple(v['key_cache'].shape)} and output "
            f"{tuple(out.shape)} disagree."
        )
    if dim > 256:
        raise TypeError("Kernel argument `query` has head dimension above the upper bound 256.")
    if offsets.shape[0] != batch + 1 or table.shape[0] != batch:
        raise TypeError(f"chunk_attention needs {batch + 1} offsets and {batch} block table rows.")
    if lse is not None and lse.shape != query.shape[:2]:
        raise TypeError("chunk_attention lse must have the query's shape without the head dimension.")
    lib = _lib.library()
    nbytes = lib.nt_b200_chunk_attention_workspace_size()
    workspace = query.new_empty(nbytes, dtype=torch.uint8)
    args = _lib.pack_args(
        *cache, query.data_ptr(), offsets.data_ptr(), lengths.data_ptr(), table.data_ptr(), out.data_ptr(),
        0 if lse is None else lse.data_ptr(), workspace.data_ptr(), nbytes, tokens, batch, heads, table.shape[1],
        *query.stride(), *out.stride(), *((0, 0) if lse is None else lse.stride()), offsets.stride(0),
        lengths.stride(0), *table.stride(), dtype_code(query.dtype), dtype_code(lengths.dtype),
        scale=_scale(v["scale"], dim),
    )
    return lib.nt_b200_chunk_attention(args, stream)


chunk_attention_kernel = Kernel(
    name="chunk_attention",
    args=(
        TensorArg("query", 3),
        *_CACHE_ARGS,
        TensorArg("block_table", 2, INDEX_DTYPES),
        TensorArg("offsets", 1, INDEX_DTYPES),
        TensorArg("lengths", 1, INDEX_DTYPES),
        TensorArg("output", 3),
        TensorArg("lse", 2, _F32, optional=True),
    ),
    outputs=("output",),
    launch=_launch_chunk_attention,
    meta=("scale",),
    meta_defaults={"scale": None, "lse": None},
)


def chunk_attention(query, key_cache, value_cache, key_scale, value_scale, block_table, offsets, lengths, scale=None,
                    return_lse=False):
    """Causal attention of the next pieces of prompts over the paged 8-bit cache that
    holds them (`paged_append`); tokens of a page outside the pool are not seen.

    `query` [tokens, heads, head_dim]: the new tokens of all sequences one after
    another, sequence s from offsets[s] to offsets[s + 1] (`offsets`: batch + 1
    entries); they are the last of its lengths[s] cached tokens, and each sees the
    tokens up to itself.  Query head h reads key/value head h // (heads // kv_heads).
    `scale` is 1 / sqrt(head_dim) by default.  Returns the output, in the query's
    shape and dtype, or with `return_lse` (output, lse): the fp32 natural logarithm
    of each query's sum of exponentials [tokens, heads].  A query that sees no token
    gets 0, and -inf as its lse; tokens that belong to no sequence are not written."""
    result = _bound("chunk_attention", query, key_cache, value_cache, key_scale, value_scale, block_table, offsets,
                    lengths, scale, return_lse)
    if result is not None:
        return result
    output = torch.empty_like(query, memory_format=torch.contiguous_format)
    lse = query.new_empty(query.shape[:2], dtype=torch.float32) if return_lse else None
    chunk_attention_kernel(query, key_cache, value_cache, key_scale, value_scale, block_table, offsets, lengths, output,
                           lse, scale=scale)
    return (output, lse) if return_lse else output


# --------------------------------------------------------------------- norm
_norm_values = itemgetter("input", "residual", "weight", "output", "total", "scale")


def _launch_rms_norm(v, stream):
    x, residual, weight, out, total, scale = _norm_values(v)
    rows, width = x.shape
    codes, group = out.dtype in CODE_DTYPES, v["group"]
    if weight.dtype not in (x.dtype, torch.float32) or not (codes or out.dtype == x.dtype):
        raise TypeError(
            "rms_norm takes a weight of the input's dtype or float32, and an output of the input's dtype, "
            "float8_e4m3fn or int8."
        )
    if weight.shape[0] != width or out.shape != x.shape:
        raise TypeError(f"rms_norm shapes {tuple(x.shape)}, weight {tuple(weight.shape)} -> {tuple(out.shape)} disagree.")
    if width > 131072:
        raise TypeError("Kernel argument `input` has rows above the upper bound 131072.")
    if (residual is None) != (total is None):
        raise TypeError("Kernel arguments `residual`, `total` must be given together.")
    if residual is not None:
        check_same_dtype(v, ("input", "residual", "total"))
        if residual.shape != x.shape or total.shape != x.shape:
            raise TypeError("rms_norm residual and total must have the input's shape.")
    if codes != (scale is not None):
        raise TypeError("rms_norm needs `scale` with an 8-bit output, and with no other.")
    if codes:
        group = _norm_group(width, group)
        if scale.shape != (rows, -(-width // group)):
            raise TypeError(f"rms_norm scale must be {(rows, -(-width // group))}; got {tuple(scale.shape)}.")
    elif group is not None:
        raise TypeError("rms_norm has groups with an 8-bit output only.")
    eps = float(v["eps"])
    if not eps >= 0.0:
        raise TypeError(f"rms_norm needs an eps of 0 or more; got {eps}.")
    none2 = (0, 0)
    args = _lib.pack_args(
        x.data_ptr(), 0 if residual is None else residual.data_ptr(), weight.data_ptr(), out.data_ptr(),
        0 if total is None else total.data_ptr(), 0 if scale is None else scale.data_ptr(), rows, width, group or width,
        *x.stride(), *(none2 if residual is None else residual.stride()), weight.stride(0), *out.stride(),
        *(none2 if total is None else total.stride()), *(none2 if scale is None else scale.stride()),
        dtype_code(x.dtype), dtype_code(weight.dtype), dtype_code(out.dtype), scale=eps,
    )
    return _lib.library().nt_b200_rms_norm(args, stream)


def _norm_group(width, group):
    """Elements of a row that share a scale."""
    if group is None or group >= width:
        return max(width, 1)
    if group <= 0 or group % 16:
        raise TypeError(f"rms_norm needs groups of a multiple of 16 elements; got {group}.")
    return int(group)


rms_norm_kernel = Kernel(
    name="rms_norm",
    args=(
        TensorArg("input", 2),
        TensorArg("weight", 1),
        TensorArg("output", 2, FLOAT_DTYPES + CODE_DTYPES),
        TensorArg("residual", 2, optional=True),
        TensorArg("total", 2, optional=True),
        TensorArg("scale", 2, _F32, optional=True),
    ),
    outputs=("output",),
    launch=_launch_rms_norm,
    meta=("eps", "group"),
    meta_defaults={"eps": 1e-6, "group": None, "residual": None, "total": None, "scale": None},
)


_NOT_GIVEN = object()


def rms_norm(input, weight, residual=None, eps=1e-6, code_dtype=_NOT_GIVEN, group=None):
    """Root-mean-square norm of the rows of `input` [rows, width]: with t = input
    + residual (or input), t / sqrt(mean(t^2) + eps) * weight (`weight`: [width],
    in the input's dtype or float32).

    Returns the output in the input's dtype, or with `code_dtype` (float8_e4m3fn
    or int8) two tensors: codes round(y / scale), and fp32 scales [rows, groups],
    one for each `group` elements of a row (a multiple of 16; the last may be
    shorter; one for the row by default).  E4M3 scales are the least power of two
    that brings a group's largest element to 448 or less, int8 ones that element /
    127.  With a `residual` the last of the outputs is the sum t in the input's
    dtype, the next residual; the norm is that of t as it is stored.

    `code_dtype` None is no code_dtype: a caller that switches the 8-bit output off so
    leaves `group` as it is, where it has no meaning.  A `group` with no word of
    `code_dtype` is refused."""
    if code_dtype is _NOT_GIVEN or code_dtype is None:
        if code_dtype is _NOT_GIVEN and group is not None:
            raise TypeError("rms_norm has groups with an 8-bit output only.")
        code_dtype = group = None
    result = _bound("rms_norm", input, weight, residual, eps, code_dtype, group)
    if result is not None:
        return result
    total = None if residual is None else torch.empty_like(input, memory_format=torch.contiguous_format)
    output = torch.empty_like(input, dtype=code_dtype, memory_format=torch.contiguous_format)
    scale = None
    if code_dtype is not None:
        rows, width = input.shape
        scale = input.new_empty((rows, -(-width // _norm_group(width, group))), dtype=torch.float32)
    rms_norm_kernel(input, weight, output, residual, total, scale, eps=eps, group=group)
    outputs = (output,) + (() if scale is None else (scale,)) + (() if total is None else (total,))
    return outputs if len(outputs) > 1 else output


# --------------------------------------------------------------------- 4-bit weights
def int4_quantize(weight, group=128, symmetric=True):
    """4-bit weights for `int4_matmul` from `weight` [outer, inner]: (codes, scales,
    zeros).  Each `group` elements of a row (a multiple of 32 that divides inner)
    share a scale, in the weight's dtype, and without `symmetric` a zero point:
    element = (code - zero) * scale with codes from 0 to 15; symmetric groups are
    centred at 8 and have no zeros (None)."""
    if weight.dim() != 2 or weight.dtype not in FLOAT_DTYPES:
        raise TypeError(f"int4_quantize needs a matrix of float16, bfloat16 or float32; got {weight.dtype} {tuple(weight.shape)}.")
    outer, inner = weight.shape
    if group <= 0 or group % 32 or inner % group:
        raise ValueError(f"group must be a multiple of 32 that divides {inner}; got {group}.")
    w = weight.detach().float().reshape(outer, inner // group, group)
    if symmetric:
        scales = (w.abs().amax(dim=2) / 7).to(weight.dtype)
        zero = torch.full_like(scales, 8, dtype=torch.float32)
    else:
        low, high = w.amin(dim=2).clamp(max=0), w.amax(dim=2).clamp(min=0)
        scales = ((high - low) / 15).to(weight.dtype)
        step = scales.float()
        zero = torch.where(step > 0, torch.round(-low / step), 8.0).clamp(0, 15)
    step = scales.float()[:, :, None]
    codes = torch.where(step > 0, torch.round(w / step), 0.0).add_(zero[:, :, None]).clamp_(0, 15).to(torch.uint8)
    codes = codes.view(outer, inner)
    return codes[:, 0::2] | codes[:, 1::2] << 4, scales, None if symmetric else zero.to(torch.uint8)


_int4_values = itemgetter("input", "codes", "scales", "output", "zeros", "input_scale")


def _launch_int4_matmul(v, stream):
    x, codes, scales, out, zeros, input_scale = _int4_values(v)
    rows, inner = x.shape
    outer, groups = scales.shape
    if out.dtype != (scales.dtype if x.dtype in CODE_DTYPES else x.dtype):
        raise TypeError("int4_matmul's output has the input's dtype, or the scales' where the input has 8 bits.")
    if codes.shape != (outer, inner // 2) or out.shape != (rows, outer):
        raise TypeError(
            f"int4_matmul input {tuple(x.shape)}, codes {tuple(codes.shape)}, scales {tuple(scales.shape)} and output "
            f"{tuple(out.shape)} disagree."
        )
    group = inner // groups if groups else 0
    if not group or group * groups != inner or group % 32:
        raise TypeError(f"int4_matmul needs groups of a multiple of 32 elements; got {groups} groups of {inner}.")
    if zeros is not None and zeros.shape != scales.shape:
        raise TypeError("int4_matmul zeros must have the scales' shape.")
    if input_scale is not None and input_scale.shape != (rows,):
        raise TypeError(f"int4_matmul needs one input scale for each of {rows} rows; got {tuple(input_scale.shape)}.")
    none2 = (0, 0)
    args = _lib.pack_args(
        x.data_ptr(), codes.data_ptr(), scales.data_ptr(), 0 if zeros is None else zeros.data_ptr(),
        0 if input_scale is None else input_scale.data_ptr(), out.data_ptr(), rows, inner, outer, group, *x.stride(),
        *codes.stride(), *scales.stride(), *(none2 if zeros is None else zeros.stride()),
        0 if input_scale is None else input_scale.stride(0), *out.stride(), dtype_code(x.dtype),
        dtype_code(scales.dtype), dtype_code(out.dtype),
    )
    return _lib.library().nt_b200_int4_matmul(args, stream)


int4_matmul_kernel = Kernel(
    name="int4_matmul",
    args=(
        TensorArg("input", 2, FLOAT_DTYPES + CODE_DTYPES),
        TensorArg("codes", 2, (torch.uint8,)),
        TensorArg("scales", 2),
        TensorArg("output", 2),
        TensorArg("zeros", 2, (torch.uint8,), optional=True),
        TensorArg("input_scale", 1, _F32, optional=True),
    ),
    outputs=("output",),
    launch=_launch_int4_matmul,
    meta_defaults={"zeros": None, "input_scale": None},
)


def int4_matmul(input, codes, scales, zeros=None, input_scale=None):
    """input [rows, inner] times the transpose of a matrix [outer, inner] of 4-bit
    weights (code - zero) * scale: `codes` uint8 [outer, inner / 2], two a byte with
    the even element in the low half; `scales` [outer, groups], each for inner /
    groups neighbouring elements (a multiple of 32); `zeros` uint8 [outer, groups],
    0 to 63, or 8 throughout (`int4_quantize` makes all three); larger zeros are
    an error that `device_status` tells of.  Made for the few rows of a decoding
    step: on tensor cores up to 8, up to 16, or else every 32 rows read the weights
    once.  float32 inputs and strides off the 16-byte grid run on CUDA cores, where
    every 8 do, 8 to 24 times as long; from some 150 rows on `matmul` with weights of
    16 bits is the faster one.

    The input is float16, bfloat16 or float32, and so is the output; or
    float8_e4m3fn or int8 with `input_scale` fp32 [rows] or [rows, 1] (`rms_norm`'s
    codes with one scale a row), with an output in the scales' dtype."""
    result = _bound("int4_matmul", input, codes, scales, zeros, input_scale)
    if result is not None:
        return result
    if isinstance(input_scale, torch.Tensor) and input_scale.dim() == 2 and input_scale.shape[1] == 1:
        input_scale = input_scale[:, 0]
    dtype = scales.dtype if input.dtype in CODE_DTYPES else input.dtype
    output = input.new_empty((input.shape[0], scales.shape[0]), dtype=dtype)
    return int4_matmul_kernel(input, codes, scales, output, zeros, input_scale)


__all__ = [
    "CODE_DTYPES",
    "INDEX_DTYPES",
    "chunk_attention",
    "chunk_attention_kernel",
    "int4_matmul",
    "int4_matmul_kernel",
    "int4_quantize",
    "paged_append",
    "paged_append_kernel",
    "paged_attention",
    "paged_attention_kernel",
    "prompt_attention",
    "prompt_attention_kernel",
    "rms_norm",
    "rms_norm_kernel",
    "rotary",
    "rotary_kernel",
    "rotary_tables",
]
