"""Cases, plain forms and 64-bit values of the serving operators.

Four operators carry a decoder's attention from the fused q/k/v projection to
the attention output:

  rotary    rotary positions: out = R(position) x over the first `rotary`
            elements of every head, or R^T x (the gradient of that rotation)
  append    rotates q and k, and writes k and v in 8 bits into a paged cache
            with one scale for each page and head
  paged     attention of a few new tokens of each sequence over that cache
  prompt    causal attention over whole prompts packed one after another, with
            grouped heads

`run` computes them in plain torch operations in 32 bits, or, where `own` is
true, through `ninetoothed_b200.programs`.  `exact` computes them in 64 bits.
"""

import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of 32 sequences: q and k of the fused projection,
        # 32 + 8 heads; launch latency is all there is
        dict(name="rotary step", op="rotary", tokens=32, heads=40, dim=128, rotary=128, type="bf16",
             interleaved=False, adjoint=False),
        # the gradient through the rotation of a training batch, half of each
        # head rotated in the interleaved layout
        dict(name="rotary gradient", op="rotary", tokens=16384, heads=40, dim=128, rotary=64, type="f16",
             interleaved=True, adjoint=True),
        # one decoding step of 32 sequences into their 16-token pages
        dict(name="append step", op="append", batch=32, new=1, new_lens=0, past=4096, heads=32, kv_heads=8, dim=128,
             rotary=128, page=16, code="e4m3", type="bf16", interleaved=False),
        # four whole prompts into empty pages
        dict(name="append prompts", op="append", batch=4, new=4096, new_lens=0, past=0, heads=32, kv_heads=8, dim=128,
             rotary=128, page=64, code="e4m3", type="bf16", interleaved=False),
        # the next pieces of prompts that were cut up, each going on inside a
        # part-filled page of 8-bit whole numbers
        dict(name="append pieces", op="append", batch=7, new=777, new_lens=1, past=1500, heads=16, kv_heads=16, dim=64,
             rotary=32, page=32, code="int8", type="f16", interleaved=True),
        # one user's decoding step: latency
        dict(name="paged one", op="paged", batch=1, new=1, longest=1023, ragged=False, heads=32, kv_heads=8, dim=128,
             page=16, code="e4m3", type="f16"),
        # a served batch, every sequence at another length
        dict(name="paged batch", op="paged", batch=64, new=1, longest=8192, ragged=True, heads=32, kv_heads=8, dim=128,
             page=64, code="e4m3", type="bf16"),
        # four drafted tokens of each sequence checked at once, one key head
        # to a query head, a cache of 8-bit whole numbers
        dict(name="paged draft", op="paged", batch=16, new=4, longest=2047, ragged=True, heads=16, kv_heads=16, dim=64,
             page=32, code="int8", type="f16"),
        # a few very long contexts
        dict(name="paged long", op="paged", batch=6, new=1, longest=131072, ragged=False, heads=32, kv_heads=8,
             dim=128, page=64, code="e4m3", type="bf16"),
        # a handful of short prompts, some of a few tokens
        dict(name="prompt short", op="prompt", batch=5, longest=100, ragged=True, heads=8, kv_heads=2, dim=64,
             type="f16"),
        # a served batch of prompts of different lengths
        dict(name="prompt packed", op="prompt", batch=8, longest=2048, ragged=True, heads=32, kv_heads=8, dim=128,
             type="bf16"),
        # four prompts of 4096 tokens: the tensor cores' rate
        dict(name="prompt long", op="prompt", batch=4, longest=4096, ragged=False, heads=32, kv_heads=8, dim=128,
             type="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rotary", "append", "paged", "prompt"))
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 8))
    dim = rng.choice((64, 128, 128, 96))
    half = rng.choice(("f16", "bf16"))
    paged = dict(page=rng.choice((16, 32, 64, 128)), code=rng.choice(("e4m3", "int8")))
    if op == "rotary":
        tokens = _spread(rng, 1, 16384)
        return dict(op=op, tokens=tokens, heads=heads + kv_heads, dim=dim, rotary=dim // rng.choice((1, 2)),
                    type=rng.choice(("f16", "bf16", "f32")), interleaved=rng.random() < 0.5, adjoint=rng.random() < 0.5)
    if op == "append":
        batch = _spread(rng, 1, 64)
        new = rng.choice((1, _spread(rng, 2, max(2, 16384 // batch))))
        return dict(op=op, batch=batch, new=new, new_lens=rng.randrange(1, 1000) if new > 1 else 0,
                    past=rng.choice((0, _spread(rng, 1, 2000))), heads=heads, kv_heads=kv_heads, dim=dim,
                    rotary=dim // rng.choice((1, 2)), type=half, interleaved=rng.random() < 0.5, **paged)
    if op == "paged":
        batch = _spread(rng, 1, 64)
        longest = _spread(rng, 1, min(131072, 6 * 131072 // batch))
        return dict(op=op, batch=batch, new=rng.choice((1, 1, 2, 5)), longest=longest, ragged=rng.random() < 0.7,
                    heads=heads, kv_heads=kv_heads, dim=dim, type=half, **paged)
    longest = _spread(rng, 1, 8192)
    batch = _spread(rng, 1, max(1, min(32, (4 * 4096 * 4096) // (longest * longest))))
    return dict(op=op, batch=batch, longest=longest, ragged=rng.random() < 0.7, heads=min(heads, 32),
                kv_heads=kv_heads, dim=dim, type=half)


def _lengths(case, longest, ragged, key):
    """Lengths of the case's sequences: all `longest`, or spread from 1 to it with one that long."""
    if not ragged:
        return [longest] * case["batch"]
    rng = random.Random("%s %s %s" % (key, case["batch"], longest))
    lens = [rng.randint(1, longest) for _ in range(case["batch"])]
    lens[rng.randrange(len(lens))] = longest
    return lens


def _new_lengths(case):
    return _lengths(case, case["new"], bool(case["new_lens"]), "new %d" % case["new_lens"])


def _past_lengths(case):
    return _lengths(case, case["past"], True, "past") if case["past"] else [0] * case["batch"]


def _kv_lengths(case):
    return _lengths(case, case["longest"], case["ragged"], "kept")


def work(case):
    op = case["op"]
    size = 4 if case["type"] == "f32" else 2
    if op == "rotary":
        n = case["tokens"] * case["heads"] * case["dim"]
        turned = case["tokens"] * case["heads"] * case["rotary"]
        return {"bytes": 2 * n * size + case["tokens"] * case["rotary"] * 4, "flops": 3 * turned}
    if op == "append":
        lens, past = _new_lengths(case), _past_lengths(case)
        t, d, h, g = sum(lens), case["dim"], case["heads"], case["kv_heads"]
        pages = sum((p + n - 1) // case["page"] - p // case["page"] + 1 for p, n in zip(past, lens))
        return {"bytes": 2 * t * h * d * size + 2 * t * g * d * (size + 1) + t * case["rotary"] * 4 + 8 * pages * g,
                "flops": 3 * t * (h + g) * case["rotary"] + 4 * t * g * d}
    if op == "paged":
        kept, d = sum(_kv_lengths(case)), case["dim"]
        pages = sum(-(-n // case["page"]) for n in _kv_lengths(case))
        queries = case["batch"] * case["new"] * case["heads"]
        return {"bytes": 2 * kept * case["kv_heads"] * d + 8 * pages * case["kv_heads"] + 2 * queries * d * size,
                "flops": 4 * kept * case["new"] * case["heads"] * d}
    lens, d = _kv_lengths(case), case["dim"]
    return {"bytes": sum(lens) * d * size * (2 * case["heads"] + 2 * case["kv_heads"]),
            "flops": 4 * d * case["heads"] * sum(n * (n + 1) // 2 for n in lens)}


# ---------------------------------------------------------------- inputs
def _offsets(lens, device):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=device)


def _angles(length, rotary, device):
    """cos and sin of position * 10000^(-2i / rotary), in 64 bits."""
    inverse = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * inverse
    return angle.cos(), angle.sin()


def _block_table(lens, page, gen, device):
    """Pages of each sequence in a shuffled pool, and the pool's size."""
    counts = [max(1, -(-n // page)) for n in lens]
    order = torch.randperm(sum(counts), generator=gen, device=device).to(torch.int32)
    table = torch.zeros((len(lens), max(counts)), dtype=torch.int32, device=device)
    for i, pages in enumerate(torch.split(order, counts)):
        table[i, : len(pages)] = pages
    return table, sum(counts)


def _random_cache(pages, kv_heads, page, dim, code, gen, device):
    """Codes and scales of normally distributed values, some heads larger than others."""
    x = torch.randn((pages, kv_heads, page, dim), generator=gen, device=device)
    x *= torch.rand((1, kv_heads, 1, 1), generator=gen, device=device) * 2 + 0.25
    high = x.abs().amax(dim=(2, 3))
    scale = torch.exp2(torch.ceil(torch.log2(high / 448))) if code == "e4m3" else high / 127
    x /= scale[:, :, None, None]
    return (x if code == "e4m3" else x.round_()).to(CODES[code]), scale


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device).manual_seed(seed)
    op, d = case["op"], case["dim"]
    dtype = TYPES[case["type"]]
    state = dict(case=case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device).to(dtype)

    if op == "rotary":
        t = case["tokens"]
        span = max(4096, t)
        cos, sin = _angles(span, case["rotary"], device)
        first = torch.randint(0, span - t + 1, (1,), generator=gen, device=device, dtype=torch.int32)
        positions = (first + torch.arange(t, device=device, dtype=torch.int32) if t > 64 else
                     torch.randint(0, span, (t,), generator=gen, device=device, dtype=torch.int32))
        # the q and k columns of a fused q/k/v projection (v: as many heads
        # again as a quarter of q's)
        qkv = normal(t, case["heads"] + max(1, case["heads"] // 5), d)
        return state | dict(input=qkv[:, : case["heads"]], cos=cos.float(), sin=sin.float(), positions=positions)
    h, g = case["heads"], case["kv_heads"]
    if op == "append":
        lens, past = _new_lengths(case), _past_lengths(case)
        total = [n + p for n, p in zip(lens, past)]
        table, pages = _block_table(total, case["page"], gen, device)
        qkv = normal(sum(lens), h + 2 * g, d)
        qkv[:, h : h + g] *= torch.rand((g, 1), generator=gen, device=device).to(dtype) * 3 + 0.5
        key_cache, key_scale = _random_cache(pages, g, case["page"], d, case["code"], gen, device)
        value_cache, value_scale = _random_cache(pages, g, case["page"], d, case["code"], gen, device)
        cos, sin = _angles(max(total), case["rotary"], device)
        return state | dict(
            query=qkv[:, :h], key=qkv[:, h : h + g], value=qkv[:, h + g :], offsets=_offsets(lens, device),
            past=torch.tensor(past, dtype=torch.int32, device=device), block_table=table, key_cache=key_cache,
            value_cache=value_cache, key_scale=key_scale, value_scale=value_scale, cos=cos.float(), sin=sin.float())
    lens = _kv_lengths(case)
    if op == "paged":
        table, pages = _block_table(lens, case["page"], gen, device)
        key_cache, key_scale = _random_cache(pages, g, case["page"], d, case["code"], gen, device)
        value_cache, value_scale = _random_cache(pages, g, case["page"], d, case["code"], gen, device)
        return state | dict(
            query=normal(case["batch"], case["new"], h, d), key_cache=key_cache, value_cache=value_cache,
            key_scale=key_scale, value_scale=value_scale, block_table=table, scale=d**-0.5,
            lengths=torch.tensor(lens, dtype=torch.int32, device=device))
    qkv = normal(sum(lens), h + 2 * g, d)
    return state | dict(query=qkv[:, :h], key=qkv[:, h : h + g], value=qkv[:, h + g :], offsets=_offsets(lens, device),
                        scale=d**-0.5)


# ---------------------------------------------------------------- the operators
def run(state):
    return (_run_own if own else _run_plain)[state["case"]["op"]](state)


def _own_rotary(s):
    from ninetoothed_b200 import programs

    return programs.rotary(s["input"], s["cos"], s["sin"], s["positions"], interleaved=s["case"]["interleaved"],
                           adjoint=s["case"]["adjoint"])


def _own_append(s):
    from ninetoothed_b200 import programs

    query, key = programs.paged_append(
        s["key"], s["value"], s["offsets"], s["past"], s["block_table"], s["key_cache"], s["value_cache"],
        s["key_scale"], s["value_scale"], query=s["query"], cos=s["cos"], sin=s["sin"],
        interleaved=s["case"]["interleaved"], return_key=False)
    del key
    return dict(query=query, **{name: s[name] for name in ("key_cache", "value_cache", "key_scale", "value_scale")})


def _own_paged(s):
    from ninetoothed_b200 import programs

    output, lse = programs.paged_attention(s["query"], s["key_cache"], s["value_cache"], s["key_scale"],
                                           s["value_scale"], s["block_table"], s["lengths"], scale=s["scale"],
                                           return_lse=True)
    return dict(output=output, lse=lse)


def _own_prompt(s):
    from ninetoothed_b200 import programs

    output, lse = programs.prompt_attention(s["query"], s["key"], s["value"], s["offsets"], scale=s["scale"],
                                            is_causal=True, return_lse=True)
    return dict(output=output, lse=lse)


def _turn(x, cos, sin, interleaved, adjoint=False):
    """x [T, H, D] with the first 2 * cos.shape[-1] elements rotated, in 32 bits."""
    r = cos.shape[-1]
    x = x.float()
    cos, sin = cos[:, None, :], (-sin if adjoint else sin)[:, None, :]
    a, b = (x[..., 0 : 2 * r : 2], x[..., 1 : 2 * r : 2]) if interleaved else (x[..., :r], x[..., r : 2 * r])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)
    return torch.cat((turned, x[..., 2 * r :]), dim=-1)


def _plain_rotary(s):
    positions = s["positions"].long()
    return _turn(s["input"], s["cos"][positions], s["sin"][positions], s["case"]["interleaved"],
                 s["case"]["adjoint"]).to(s["input"].dtype)


def _plain_store(x, cache, scales, page_of, slot_of, first):
    """Writes x [T, H, D] (32 bits) as codes into `cache` and updates `scales` in place.

    A page's scale covers what it held before and the new tokens; what it held
    is rounded again only where the scale grew.  `first` [pages]: the first
    new slot of each page (the page size where there is none).
    """
    pages, heads, page, _ = cache.shape
    high = torch.zeros((pages, heads), device=x.device)
    high.scatter_reduce_(0, page_of[:, None].expand(-1, heads), x.abs().amax(dim=-1), "amax")
    if cache.dtype == torch.int8:
        fresh = torch.clamp(high / 127, min=2.0**-126)
    else:
        # the least power of two that brings the largest value to 448 or less
        fraction, exponent = torch.frexp(high)
        power = torch.clamp(exponent - 9 + (fraction > 0.875), min=-126)
        fresh = torch.ldexp(torch.ones_like(high), power)
    scale = torch.where(first[:, None] > 0, torch.maximum(scales, fresh), fresh)
    touched = first < page
    scale = torch.where(touched[:, None], scale, scales)
    which = torch.nonzero(touched & (first > 0)).flatten()
    ratio = (scales[which] / scale[which])[:, :, None, None]
    held = cache[which]
    moved = held.float() * ratio
    moved = (torch.round(moved) if cache.dtype == torch.int8 else moved).to(cache.dtype)
    old = torch.arange(page, device=x.device)[None, :] < first[which][:, None]
    cache[which] = torch.where(old[:, None, :, None], moved.view(torch.int8), held.view(torch.int8)).view(cache.dtype)
    codes = x * (1.0 / scale)[page_of][:, :, None]
    cache[page_of, :, slot_of] = (torch.round(codes) if cache.dtype == torch.int8 else codes).to(cache.dtype)
    scales.copy_(scale)


def _plain_append(s):
    case, page = s["case"], s["case"]["page"]
    t = torch.arange(s["key"].shape[0], device=s["key"].device)
    of = torch.bucketize(t, s["offsets"][1:].long(), right=True)
    position = s["past"].long()[of] + t - s["offsets"].long()[of]
    page_of = s["block_table"].long()[of, position // page]
    slot_of = position % page
    first = torch.full((s["key_cache"].shape[0],), page, device=t.device)
    first.scatter_reduce_(0, page_of, slot_of, "amin")
    cos, sin = s["cos"][position], s["sin"][position]
    query = _turn(s["query"], cos, sin, case["interleaved"]).to(s["query"].dtype)
    key = _turn(s["key"], cos, sin, case["interleaved"])
    _plain_store(key, s["key_cache"], s["key_scale"], page_of, slot_of, first)
    _plain_store(s["value"].float(), s["value_cache"], s["value_scale"], page_of, slot_of, first)
    return dict(query=query, **{name: s[name] for name in ("key_cache", "value_cache", "key_scale", "value_scale")})


def _softmax_parts(scores):
    """exp(scores - max), its sum and the maximum, over the last dimension."""
    high = scores.amax(dim=-1, keepdim=True)
    weight = torch.exp(scores - high)
    return weight, weight.sum(dim=-1, keepdim=True), high


def _plain_paged(s):
    b, new, h, d = s["query"].shape
    _, g, page, _ = s["key_cache"].shape
    table = s["block_table"].long()

    def gather(cache, scales):
        x = cache.view(torch.int8)[table].view(cache.dtype).float() * scales[table][:, :, :, None, None]
        return x.transpose(1, 2).reshape(b, g, -1, d)

    longest = table.shape[1] * page
    query = s["query"].float().reshape(b, new, g, h // g, d).permute(0, 2, 1, 3, 4).reshape(b, g, -1, d)
    scores = torch.matmul(query, gather(s["key_cache"], s["key_scale"]).transpose(-1, -2)) * s["scale"]
    limit = s["lengths"][:, None] - new + 1 + torch.arange(new, device=table.device)
    seen = torch.arange(longest, device=table.device) < limit[:, :, None]
    seen = seen[:, None, :, None, :].expand(b, g, new, h // g, longest).reshape(b, g, -1, longest)
    some = (limit > 0)[:, None, :, None].expand(b, g, new, h // g).reshape(b, g, -1, 1)
    weight, total, high = _softmax_parts(scores.masked_fill(~seen, -math.inf).masked_fill(~some, 0.0))
    output = (torch.matmul(weight, gather(s["value_cache"], s["value_scale"])) / total).masked_fill(~some, 0.0)
    lse = (high + torch.log(total)).masked_fill(~some, -math.inf)

    def rows(x):
        return x.reshape(b, g, new, h // g, -1).permute(0, 2, 1, 3, 4).reshape(b, new, h, -1)

    return dict(output=rows(output).to(s["query"].dtype), lse=rows(lse)[..., 0].contiguous())


def _plain_prompt(s):
    total, h, d = s["query"].shape
    g = s["key"].shape[1]
    offsets = s["offsets"].long()
    batch, longest = offsets.numel() - 1, s["case"]["longest"]
    t = torch.arange(total, device=offsets.device)
    of = torch.bucketize(t, offsets[1:], right=True)
    at = t - offsets[of]

    def padded(x):
        out = torch.zeros((batch, longest, x.shape[1], d), device=x.device)
        out[of, at] = x.float()
        return out.transpose(1, 2)

    query, key, value = padded(s["query"]), padded(s["key"]), padded(s["value"])
    query = query.reshape(batch, g, (h // g) * longest, d)
    scores = torch.matmul(query, key.transpose(-1, -2)).view(batch, g, h // g, longest, longest)
    scores *= s["scale"]
    row = torch.arange(longest, device=t.device)
    scores.masked_fill_(row[None, :] > row[:, None], -math.inf)
    weight, sums, high = _softmax_parts(scores)
    output = torch.matmul(weight.view(batch, g, -1, longest), value).view(batch, h, longest, d)
    output = output / sums.view(batch, h, longest, 1)
    lse = (high + torch.log(sums)).view(batch, h, longest)
    return dict(output=output.transpose(1, 2)[of, at].to(s["query"].dtype), lse=lse.transpose(1, 2)[of, at])


_run_plain = dict(rotary=_plain_rotary, append=_plain_append, paged=_plain_paged, prompt=_plain_prompt)
_run_own = dict(rotary=_own_rotary, append=_own_append, paged=_own_paged, prompt=_own_prompt)


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    return _exact[case["op"]](prepare(case, seed))


def _spin(x, angle, interleaved):
    """x with pairs taken as complex numbers and multiplied by exp(i angle), in 64 bits."""
    r = angle.shape[-1]
    x = x.double()
    head = x[..., : 2 * r].unflatten(-1, (r, 2) if interleaved else (2, r))
    pair = torch.view_as_complex((head if interleaved else head.transpose(-1, -2)).contiguous())
    pair = torch.view_as_real(pair * torch.exp(1j * angle)[:, None, :])
    head = (pair if interleaved else pair.transpose(-1, -2)).flatten(-2)
    return torch.cat((head, x[..., 2 * r :]), dim=-1)


def _exact_rotary(s):
    # the tables are inputs: the angle is that of the 32-bit pair, and its
    # length, one up to rounding, is kept
    c, n = s["cos"][s["positions"].long()].double(), s["sin"][s["positions"].long()].double()
    angle = torch.complex(torch.atan2(n, c) * (-1 if s["case"]["adjoint"] else 1), -torch.log(torch.hypot(c, n)))
    return _spin(s["input"], angle, s["case"]["interleaved"])


def _exact_append(s):
    case, page = s["case"], s["case"]["page"]
    whole = case["code"] == "int8"
    lens, past = _new_lengths(case), _past_lengths(case)
    position = torch.cat([torch.arange(p, p + n) for p, n in zip(past, lens)]).to(s["cos"].device)
    c, n = s["cos"][position].double(), s["sin"][position].double()
    angle = torch.complex(torch.atan2(n, c), -torch.log(torch.hypot(c, n)))
    out = dict(query=_spin(s["query"], angle, case["interleaved"]))
    key = _spin(s["key"], angle, case["interleaved"])
    for name, x in (("key", key), ("value", s["value"].double())):
        codes, scales = s[name + "_cache"].double(), s[name + "_scale"].double()
        at = 0
        for i, (p, count) in enumerate(zip(past, lens)):
            for j in range(p // page, (p + count - 1) // page + 1):
                low, high = max(p, j * page), min(p + count, (j + 1) * page)
                block = int(s["block_table"][i, j])
                rows = x[at + low - p : at + high - p].transpose(0, 1)
                top = rows.abs().amax(dim=(1, 2))
                scale = top / 127 if whole else torch.exp2(torch.ceil(torch.log2(top / 448)))
                if low > j * page:
                    scale = torch.maximum(scale, scales[block])
                    held = codes[block, :, : low - j * page] * (scales[block] / scale)[:, None, None]
                    codes[block, :, : low - j * page] = held.round() if whole else held.to(CODES["e4m3"]).double()
                rows = rows / scale[:, None, None]
                codes[block, :, low - j * page : high - j * page] = (
                    rows.round() if whole else rows.float().to(CODES["e4m3"]).double())
                scales[block] = scale
            at += count
        out[name + "_cache"] = None if whole else codes
        out[name + "_scale"] = scales
    return out


def _exact_paged(s):
    b, new, h, d = s["query"].shape
    _, g, page, _ = s["key_cache"].shape
    output = torch.zeros((b, new, h, d), dtype=torch.float64, device=s["query"].device)
    lse = torch.full((b, new, h), -math.inf, dtype=torch.float64, device=s["query"].device)
    for i, length in enumerate(_kv_lengths(s["case"])):
        pages = s["block_table"][i, : -(-length // page)].long()
        for j in range(g):
            k, v = ((s[n + "_cache"][pages, j].double() * s[n + "_scale"][pages, j].double()[:, None, None])
                    .reshape(-1, d)[:length] for n in ("key", "value"))
            group = slice(j * (h // g), (j + 1) * (h // g))
            for t in range(max(0, new - length), new):
                limit = length - new + 1 + t
                logits = s["query"][i, t, group].double() @ k[:limit].T * s["scale"]
                lse[i, t, group] = torch.logsumexp(logits, dim=-1)
                output[i, t, group] = torch.exp(logits - lse[i, t, group, None]) @ v[:limit]
    return dict(output=output, lse=lse)


def _exact_prompt(s):
    total, h, d = s["query"].shape
    g = s["key"].shape[1]
    output = torch.zeros((total, h, d), dtype=torch.float64, device=s["query"].device)
    lse = torch.zeros((total, h), dtype=torch.float64, device=s["query"].device)
    bounds = s["offsets"].tolist()
    for low, high in zip(bounds, bounds[1:]):
        future = torch.ones((high - low, high - low), dtype=torch.bool, device=output.device).triu(1)
        for j in range(h):
            k, v = s["key"][low:high, j // (h // g)].double(), s["value"][low:high, j // (h // g)].double()
            logits = (s["query"][low:high, j].double() @ k.T * s["scale"]).masked_fill(future, -math.inf)
            lse[low:high, j] = torch.logsumexp(logits, dim=-1)
            output[low:high, j] = torch.exp(logits - lse[low:high, j, None]) @ v
    return dict(output=output, lse=lse)


_exact = dict(rotary=_exact_rotary, append=_exact_append, paged=_exact_paged, prompt=_exact_prompt)
