"""Cases, plain forms and 64-bit values of the serving operators around the attention of a decoder.

Three operators complete a decoder's layer beside those of `operators.py`:

  norm   root-mean-square norm of a row after the residual's addition, with an
         output in the row's own type or in 8 bits with scales
  int4   product of a few rows with a matrix of 4-bit weights, a scale (and a
         zero point) for each group of weights
  chunk  causal attention of the next pieces of prompts, packed one after
         another, over the paged 8-bit cache that holds them already

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
        # one decoding step of 32 sequences: launch latency is all there is
        dict(name="norm step", op="norm", rows=32, width=4096, type="bf16", residual=True, code="", group=0),
        # a batch of prompts before an 8-bit matrix product, one scale a row
        dict(name="norm codes", op="norm", rows=16384, width=4096, type="bf16", residual=True, code="e4m3", group=0),
        # a first norm (no residual yet) to whole numbers, a scale for each 128
        # elements
        dict(name="norm groups", op="norm", rows=3001, width=5120, type="f16", residual=False, code="int8", group=128),
        # one user's token through a square projection: latency
        dict(name="int4 token", op="int4", rows=1, inner=4096, outer=4096, group=128, zeros=False, type="bf16",
             scale="bf16"),
        # drafted tokens of one user through a layer's inner projection, with
        # zero points
        dict(name="int4 drafts", op="int4", rows=5, inner=10240, outer=4099, group=64, zeros=True, type="f16",
             scale="f16"),
        # one step of 32 sequences
        dict(name="int4 batch", op="int4", rows=32, inner=8192, outer=8192, group=128, zeros=False, type="bf16",
             scale="bf16"),
        # 16 sequences through an output head, from the norm's 8-bit rows
        dict(name="int4 head", op="int4", rows=16, inner=8192, outer=65536, group=32, zeros=True, type="e4m3",
             scale="bf16"),
        # short follow-ups of short talks: latency
        dict(name="chunk short", op="chunk", batch=4, new=16, longest=1000, ragged=True, heads=8, kv_heads=2, dim=64,
             page=16, code="int8", type="f16"),
        # a served batch, each prompt's next piece at another length
        dict(name="chunk pieces", op="chunk", batch=8, new=512, longest=8192, ragged=True, heads=32, kv_heads=8,
             dim=128, page=64, code="e4m3", type="bf16"),
        # one key head to a query head, a cache of 8-bit whole numbers
        dict(name="chunk heads", op="chunk", batch=6, new=300, longest=4000, ragged=True, heads=16, kv_heads=16,
             dim=64, page=32, code="int8", type="f16"),
        # a piece of a long document: few rows over many keys
        dict(name="chunk document", op="chunk", batch=1, new=256, longest=100000, ragged=False, heads=32, kv_heads=8,
             dim=128, page=64, code="e4m3", type="bf16"),
        # large pieces of two prompts: the tensor cores' rate
        dict(name="chunk long", op="chunk", batch=2, new=2048, longest=24576, ragged=False, heads=32, kv_heads=8,
             dim=128, page=64, code="e4m3", type="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "int4", "chunk"))
    half = rng.choice(("f16", "bf16"))
    if op == "norm":
        width = rng.choice((8 * _spread(rng, 8, 2048), _spread(rng, 64, 16384)))
        return dict(op=op, rows=_spread(rng, 1, 16384 * 4096 // max(width, 4096)), width=width,
                    type=rng.choice(("f16", "bf16", "f32")), residual=rng.random() < 0.6,
                    code=rng.choice(("", "e4m3", "int8")), group=rng.choice((0, 32, 128)))
    if op == "int4":
        group = rng.choice((32, 64, 128))
        return dict(op=op, rows=_spread(rng, 1, 64), inner=group * _spread(rng, 2, 10240 // group),
                    outer=_spread(rng, 64, 32768), group=group, zeros=rng.random() < 0.5,
                    type=rng.choice(("f16", "bf16", "bf16", "f16", "e4m3", "int8")), scale=half)
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 8))
    batch = _spread(rng, 1, 32)
    new = _spread(rng, 1, min(2048, 8192 // batch))
    longest = max(new, _spread(rng, 16, min(65536, 2 * 24576 * 2048 // (new * batch))))
    return dict(op=op, batch=batch, new=new, longest=longest, ragged=rng.random() < 0.7, heads=min(heads, 32),
                kv_heads=kv_heads if heads <= 32 else 4, dim=rng.choice((64, 128, 128, 96)),
                page=rng.choice((16, 32, 64, 128)), code=rng.choice(("e4m3", "int8")), type=half)


def _lengths(case):
    """(new tokens, cached tokens) of a case's sequences: all the same, or new
    ones spread from 1 to `new` and cached ones from the new ones to `longest`."""
    batch, new, longest = case["batch"], case["new"], case["longest"]
    if not case["ragged"]:
        return [new] * batch, [longest] * batch
    rng = random.Random("%s %s %s" % (batch, new, longest))
    fresh = [rng.randint(1, new) for _ in range(batch)]
    fresh[rng.randrange(batch)] = new
    kept = [rng.randint(n, longest) for n in fresh]
    kept[rng.randrange(batch)] = longest
    return fresh, kept


def _groups(case):
    return -(-case["width"] // case["group"]) if case["group"] else 1


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "int8": 1}[case["type"]]
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        out = n + 4 * case["rows"] * _groups(case) if case["code"] else n * size
        return {"bytes": n * size * (3 if case["residual"] else 1) + case["width"] * size + out, "flops": 5 * n}
    if case["op"] == "int4":
        m, k, n = case["rows"], case["inner"], case["outer"]
        return {"bytes": n * k // 2 + n * k // case["group"] * (3 if case["zeros"] else 2) + m * k * size + m * n * 2,
                "flops": 2 * m * n * k}
    fresh, kept = _lengths(case)
    d, h, g, page = case["dim"], case["heads"], case["kv_heads"], case["page"]
    return {"bytes": 2 * sum(kept) * g * d + 8 * g * sum(-(-n // page) for n in kept) + 2 * sum(fresh) * h * d * size,
            "flops": 4 * d * h * sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(fresh, kept))}


# ---------------------------------------------------------------- inputs
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
    state = dict(case=case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    if case["op"] == "norm":
        dtype, shape = TYPES[case["type"]], (case["rows"], case["width"])
        # a layer's output, and the sum of all before it with a few large channels
        channels = torch.ones(case["width"], device=device)
        channels[:: max(1, case["width"] // 7)] = 20.0
        return state | dict(input=normal(*shape).to(dtype),
                            residual=(normal(*shape) * 3 * channels).to(dtype) if case["residual"] else None,
                            weight=(1 + 0.2 * normal(case["width"])).to(dtype), eps=1e-6)
    if case["op"] == "int4":
        m, k, n, group = case["rows"], case["inner"], case["outer"], case["group"]
        codes = torch.randint(0, 256, (n, k // 2), generator=gen, device=device, dtype=torch.uint8)
        spread = torch.rand((n, k // group), generator=gen, device=device) * 1.5 + 0.5
        x, scale = normal(m, k), None
        if case["type"] in CODES:
            scale = x.abs().amax(dim=1) / (448 if case["type"] == "e4m3" else 127)
            x = x / scale[:, None]
            x = (x if case["type"] == "e4m3" else x.round()).to(CODES[case["type"]])
        else:
            x = x.to(TYPES[case["type"]])
        zeros = torch.randint(5, 11, (n, k // group), generator=gen, device=device, dtype=torch.uint8)
        return state | dict(input=x, codes=codes, scales=(spread * 0.2 * k**-0.5).to(TYPES[case["scale"]]),
                            zeros=zeros if case["zeros"] else None, input_scale=scale)
    fresh, kept = _lengths(case)
    h, g, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    counts = [-(-n // page) for n in kept]
    order = torch.randperm(sum(counts), generator=gen, device=device).to(torch.int32)
    table = torch.zeros((len(kept), max(counts)), dtype=torch.int32, device=device)
    for i, pages in enumerate(torch.split(order, counts)):
        table[i, : len(pages)] = pages
    key_cache, key_scale = _random_cache(sum(counts), g, page, d, case["code"], gen, device)
    value_cache, value_scale = _random_cache(sum(counts), g, page, d, case["code"], gen, device)
    offsets = [sum(fresh[:i]) for i in range(len(fresh) + 1)]
    return state | dict(
        query=normal(sum(fresh), h, d).to(TYPES[case["type"]]), key_cache=key_cache, value_cache=value_cache,
        key_scale=key_scale, value_scale=value_scale, block_table=table,
        offsets=torch.tensor(offsets, dtype=torch.int32, device=device),
        lengths=torch.tensor(kept, dtype=torch.int32, device=device))


# ---------------------------------------------------------------- the operators
def run(state):
    return (_run_own if own else _run_plain)[state["case"]["op"]](state)


def _named(case, outputs):
    """The norm's outputs by name: what was asked for, in order."""
    names = ["output"] + (["scale"] if case["code"] else []) + (["total"] if case["residual"] else [])
    return dict(zip(names, outputs if isinstance(outputs, tuple) else (outputs,)))


def _own_norm(s):
    from ninetoothed_b200 import programs

    case = s["case"]
    return _named(case, programs.rms_norm(s["input"], s["weight"], residual=s["residual"], eps=s["eps"],
                                          code_dtype=CODES.get(case["code"]), group=case["group"] or None))


def _own_int4(s):
    from ninetoothed_b200 import programs

    return programs.int4_matmul(s["input"], s["codes"], s["scales"], zeros=s["zeros"], input_scale=s["input_scale"])


def _own_chunk(s):
    from ninetoothed_b200 import programs

    output, lse = programs.chunk_attention(s["query"], s["key_cache"], s["value_cache"], s["key_scale"],
                                           s["value_scale"], s["block_table"], s["offsets"], s["lengths"],
                                           return_lse=True)
    return dict(output=output, lse=lse)


def _plain_norm(s):
    case, x = s["case"], s["input"]
    total = x
    if case["residual"]:
        total = (x.float() + s["residual"].float()).to(x.dtype)
    # the sum of squares in 64 bits: what is rounded to 8 bits afterwards then
    # hangs on the formula, not on the order of a sum
    square = total.double().square().mean(dim=1, keepdim=True)
    y = total.float() * (1.0 / torch.sqrt(square + s["eps"])).float() * s["weight"].float()
    outputs = []
    if case["code"]:
        rows, width = y.shape
        groups = _groups(case)
        group = -(-width // groups) if not case["group"] else case["group"]
        y = torch.nn.functional.pad(y, (0, groups * group - width)).view(rows, groups, group)
        high = y.abs().amax(dim=2)
        if case["code"] == "int8":
            scale = torch.clamp(high * torch.tensor(1.0 / 127.0, device=y.device), min=2.0**-126)
            codes = torch.round(y * (1.0 / scale)[:, :, None])
        else:
            # the least power of two that brings the largest value to 448 or less
            fraction, exponent = torch.frexp(high)
            power = torch.clamp(exponent - 9 + (fraction > 0.875), min=-126)
            scale = torch.ldexp(torch.ones_like(high), power)
            codes = y * (1.0 / scale)[:, :, None]
        outputs = [codes.view(rows, -1)[:, :width].contiguous().to(CODES[case["code"]]), scale]
    else:
        outputs = [y.to(x.dtype)]
    return _named(case, tuple(outputs + [total] if case["residual"] else outputs))


def _plain_int4(s):
    n, half = s["codes"].shape
    codes = torch.stack((s["codes"] & 15, s["codes"] >> 4), dim=2).view(n, s["scales"].shape[1], -1).float()
    zeros = s["zeros"].float()[:, :, None] if s["zeros"] is not None else 8.0
    weight = ((codes - zeros) * s["scales"].float()[:, :, None]).view(n, 2 * half)
    out = torch.matmul(s["input"].float(), weight.T)
    if s["input_scale"] is not None:
        out = out * s["input_scale"][:, None]
    return out.to(TYPES[s["case"]["scale"]] if s["case"]["type"] in CODES else s["input"].dtype)


def _gather(s, name, i, j, count):
    """The first `count` keys or values of head j of sequence i, in 32 bits."""
    pages = s["block_table"][i, : -(-count // s["key_cache"].shape[2])].long()
    codes = s[name + "_cache"].view(torch.int8)[pages, j].view(s[name + "_cache"].dtype).float()
    return (codes * s[name + "_scale"][pages, j][:, None, None]).flatten(0, 1)[:count]


def _plain_chunk(s):
    query = s["query"]
    _, h, d = query.shape
    g = s["key_cache"].shape[1]
    group = h // g
    output = torch.empty(query.shape, device=query.device)
    lse = torch.empty(query.shape[:2], device=query.device)
    at = 0
    for i, (new, kept) in enumerate(zip(*_lengths(s["case"]))):
        limit = kept - new + 1 + torch.arange(new, device=query.device)
        unseen = torch.arange(kept, device=query.device) >= limit[:, None]
        for j in range(g):
            rows = query[at : at + new, j * group : (j + 1) * group].float().transpose(0, 1).reshape(-1, d)
            scores = torch.matmul(rows, _gather(s, "key", i, j, kept).T).mul_(d**-0.5).view(group, new, kept)
            scores.masked_fill_(unseen, -math.inf)
            high = scores.amax(dim=2, keepdim=True)
            weight = scores.sub_(high).exp_()
            total = weight.sum(dim=2, keepdim=True)
            part = torch.matmul(weight.view(-1, kept), _gather(s, "value", i, j, kept)).view(group, new, d) / total
            output[at : at + new, j * group : (j + 1) * group] = part.transpose(0, 1)
            lse[at : at + new, j * group : (j + 1) * group] = (high + torch.log(total))[:, :, 0].T
        at += new
    return dict(output=output.to(query.dtype), lse=lse)


_run_plain = dict(norm=_plain_norm, int4=_plain_int4, chunk=_plain_chunk)
_run_own = dict(norm=_own_norm, int4=_own_int4, chunk=_own_chunk)


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    return _exact[case["op"]](prepare(case, seed))


def _exact_norm(s):
    case = s["case"]
    total = s["input"].double()
    if case["residual"]:
        # what the norm takes is the sum as it is stored
        total = (total + s["residual"].double()).to(s["input"].dtype).double()
    length = torch.linalg.vector_norm(total, dim=1, keepdim=True)
    y = total * s["weight"].double() / torch.hypot(length / math.sqrt(case["width"]),
                                                   torch.full_like(length, math.sqrt(s["eps"])))
    out = dict(output=y)
    if case["code"]:
        group = case["group"] or case["width"]
        scales = torch.zeros((case["rows"], _groups(case)), dtype=torch.float64, device=y.device)
        codes = torch.empty_like(y)
        for j in range(scales.shape[1]):
            part = y[:, j * group : (j + 1) * group]
            top = part.abs().amax(dim=1)
            scales[:, j] = top / 127 if case["code"] == "int8" else torch.exp2(torch.ceil(torch.log2(top / 448)))
            codes[:, j * group : (j + 1) * group] = part / scales[:, j, None]
        out = dict(output=None if case["code"] == "int8" else codes, scale=scales)
    if case["residual"]:
        out["total"] = total
    return out


def _exact_int4(s):
    x = s["input"].double()
    if s["input_scale"] is not None:
        x = x * s["input_scale"].double()[:, None]
    n, half = s["codes"].shape
    group = 2 * half // s["scales"].shape[1]
    out = torch.zeros((x.shape[0], n), dtype=torch.float64, device=x.device)
    for j in range(s["scales"].shape[1]):
        bytes_ = s["codes"][:, j * group // 2 : (j + 1) * group // 2].long()
        zero = s["zeros"][:, j].double()[:, None] if s["zeros"] is not None else 8.0
        part = x[:, j * group : (j + 1) * group]
        dot = part[:, 0::2] @ ((bytes_ % 16).double() - zero).T + part[:, 1::2] @ ((bytes_ // 16).double() - zero).T
        out += dot * s["scales"][:, j].double()
    return out


def _exact_chunk(s):
    query = s["query"].double()
    _, h, d = query.shape
    _, g, page, _ = s["key_cache"].shape
    output, lse = torch.zeros_like(query), torch.zeros(query.shape[:2], dtype=torch.float64, device=query.device)
    bounds, kept = s["offsets"].tolist(), s["lengths"].tolist()
    for i, length in enumerate(kept):
        low, high = bounds[i], bounds[i + 1]
        pages = s["block_table"][i, : -(-length // page)].long()
        future = torch.ones((high - low, length), dtype=torch.bool, device=query.device).triu(length - high + low + 1)
        for j in range(g):
            k, v = ((s[n + "_cache"][pages, j].double() * s[n + "_scale"][pages, j].double()[:, None, None])
                    .reshape(-1, d)[:length] for n in ("key", "value"))
            for head in range(j * (h // g), (j + 1) * (h // g)):
                logits = (query[low:high, head] @ k.T / math.sqrt(d)).masked_fill(future, -math.inf)
                lse[low:high, head] = torch.logsumexp(logits, dim=1)
                output[low:high, head] = torch.exp(logits - lse[low:high, head, None]) @ v
    return dict(output=output, lse=lse)


_exact = dict(norm=_exact_norm, int4=_exact_int4, chunk=_exact_chunk)
