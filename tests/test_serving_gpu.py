"""Serving operators on the GPU against plain 64-bit implementations."""

import math

import pytest
import torch

from ninetoothed_b200 import device_status, programs

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}  # half a step, relative
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 0.0, torch.float32: 0.0}  # half a step among the subnormals
INDEX_OUT_OF_RANGE = 10007


def dev(x):
    return x.to("cuda")


def index(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


# --------------------------------------------------------------------- rotary
def turned(x, cos, sin, interleaved, adjoint=False):
    """The rotation in 64 bits, pair by pair; x [T, H, D], cos and sin [T, R/2]."""
    out = x.double().clone()
    r = cos.shape[1]
    for i in range(r):
        i0, i1 = (2 * i, 2 * i + 1) if interleaved else (i, i + r)
        a, b = x[..., i0].double(), x[..., i1].double()
        c, s = cos[:, i, None].double(), sin[:, i, None].double() * (-1 if adjoint else 1)
        out[..., i0], out[..., i1] = a * c - b * s, b * c + a * s
    return out


def rotation_error(x, r):
    """What rounding products and sum to fp32 one by one can add: 2 steps of |a| + |b|."""
    return 4 * 2.0**-24 * x.double().abs().amax() * torch.ones(())


ROTARY_SHAPES = [
    # tokens, heads, head_dim, rotary_dim
    (1, 1, 2, 2),
    (1, 1, 8, 0),
    (3, 5, 64, 64),
    (17, 40, 128, 128),
    (33, 7, 128, 64),
    (5, 3, 96, 32),
    (9, 2, 80, 40),
    (4, 6, 72, 36),
    (7, 3, 30, 18),
    (257, 1, 256, 128),
]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("shape", ROTARY_SHAPES)
def test_rotary(shape, interleaved, dtype):
    t, h, d, r = shape
    x = torch.randn(t, h, d).to(dtype)
    cos, sin = programs.rotary_tables(300, max(r, 2), scaling="ntk" if r > 2 else None, factor=4.0)
    cos, sin = cos[:, : r // 2].contiguous(), sin[:, : r // 2].contiguous()
    positions = torch.randint(0, 300, (t,))
    for adjoint in (False, True):
        got = programs.rotary(dev(x), dev(cos), dev(sin), dev(positions), interleaved=interleaved, adjoint=adjoint)
        want = turned(x, cos[positions], sin[positions], interleaved, adjoint)
        limit = HALF[dtype] * want.abs() + TINY[dtype] + rotation_error(x, r)
        assert got.dtype == dtype and got.shape == x.shape
        assert ((got.cpu().double() - want).abs() <= limit).all()
        assert torch.equal(got.cpu()[..., r:], x[..., r:])
    assert device_status() == 0


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
def test_rotary_strides_and_int64_positions(dtype):
    """Views of a fused projection, a head-major layout, an element stride, in place."""
    qkv = torch.randn(21, 9, 64).to(dtype)
    cos, sin = programs.rotary_tables(64, 64)
    positions = torch.arange(21, dtype=torch.int64) * 3 % 64
    want = turned(qkv, cos[positions], sin[positions], False)
    limit = HALF[dtype] * want.abs() + TINY[dtype] + rotation_error(qkv, 64)
    tables = dev(cos), dev(sin), dev(positions)
    inputs = (
        dev(qkv)[:, 2:7],
        dev(qkv).transpose(0, 1).contiguous().transpose(0, 1)[:, 2:7],
        torch.stack((dev(qkv), dev(qkv)), dim=-1)[:, 2:7, :, 0],
    )
    for x in inputs:
        got = programs.rotary(x, *tables)
        assert ((got.cpu().double() - want[:, 2:7]).abs() <= limit[:, 2:7]).all()
    spread = torch.zeros(21, 5, 130, dtype=dtype, device="cuda")
    programs.rotary_kernel(inputs[0], *tables, spread[:, :, 1:129:2])
    assert torch.equal(spread[:, :, 1:129:2], programs.rotary(inputs[0], *tables))
    assert not spread[:, :, 0::2].any()
    whole = dev(qkv)
    part = whole[:, 2:7]
    programs.rotary_kernel(part, *tables, part)
    assert torch.equal(part, programs.rotary(inputs[0], *tables))
    assert torch.equal(whole[:, :2].cpu(), qkv[:, :2]) and torch.equal(whole[:, 7:].cpu(), qkv[:, 7:])


def test_rotary_leaves_copied_elements_alone_when_not_finite():
    x = torch.randn(2, 2, 64).half()
    x[..., 8:] = math.inf
    x[0, 0, 40] = math.nan
    cos, sin = programs.rotary_tables(8, 8)
    for interleaved in (False, True):
        got = programs.rotary(dev(x), dev(cos), dev(sin), index([1, 2]), interleaved=interleaved).cpu()
        assert torch.equal(got[..., 8:].nan_to_num(7.0), x[..., 8:].nan_to_num(7.0))
        assert got[..., :8].isfinite().all()


def test_rotary_gradient():
    """The adjoint is the gradient: against the formula (the dot products agree)
    and against differences of a linear map."""
    t, h, d, r = 6, 2, 32, 24
    cos, sin = programs.rotary_tables(16, r, scaling="by_parts", factor=8.0, original_length=16)
    positions = torch.arange(t)
    x, g = torch.randn(t, h, d), torch.randn(t, h, d)
    tables = dev(cos), dev(sin), dev(positions)
    for interleaved in (False, True):
        dx = programs.rotary(dev(g), *tables, interleaved=interleaved, adjoint=True).cpu().double()
        y = programs.rotary(dev(x), *tables, interleaved=interleaved).cpu().double()
        left, right = (y * g.double()).sum(), (x.double() * dx).sum()
        # each of the t h d products is off by at most a few steps of its factors
        assert abs(left - right) <= 16 * 2.0**-24 * t * h * d * 16
        for at in ((0, 0, 0), (3, 1, r - 1), (5, 0, d - 1), (2, 1, 7)):
            step = torch.zeros(t, h, d)
            step[at] = 1.0  # the map is linear: any step is exact up to rounding
            up = programs.rotary(dev(x + step), *tables, interleaved=interleaved).cpu().double()
            moved = ((x + step).double()[at] - x.double()[at])
            assert abs(((up - y) * g.double()).sum() / moved - dx[at]) <= 16 * 2.0**-24 * 16 * 16


def test_rotary_position_outside_the_table():
    cos, sin = programs.rotary_tables(4, 16)
    x = torch.randn(3, 2, 32).half()
    got = programs.rotary(dev(x), dev(cos), dev(sin), index([0, 4, -1])).cpu()
    assert device_status() == INDEX_OUT_OF_RANGE and device_status() == 0
    assert torch.equal(got[0], programs.rotary(dev(x[:1]), dev(cos), dev(sin), index([0])).cpu()[0])
    assert got[1:, :, :16].isnan().all() and torch.equal(got[1:, :, 16:], x[1:, :, 16:])


# --------------------------------------------------------------------- append
class Pages:
    """A cache with shuffled pages and stale contents, and what it should hold, in 64 bits."""

    def __init__(self, lens, page, kv_heads, dim, code, layout="heads"):
        self.page, self.code = page, code
        counts = [max(1, -(-n // page)) for n in lens]
        total = sum(counts) + 2
        order = torch.randperm(total)
        self.table = torch.full((len(lens), max(counts) + 1), -1, dtype=torch.int64)
        at = 0
        for i, n in enumerate(counts):
            self.table[i, :n] = order[at : at + n]
            at += n
        shape = (total, kv_heads, page, dim)
        stale = torch.randint(-128, 128, shape, dtype=torch.int8)
        self.caches = {}
        for name in ("key", "value"):
            if layout == "heads":
                store = stale.cuda().clone()
            else:  # token-major pages: [pages, page, heads, dim]
                store = stale.cuda().transpose(1, 2).contiguous().transpose(1, 2)
            self.caches[name] = store.view(code) if code == torch.int8 or layout == "heads" else (
                store.transpose(1, 2).view(code).transpose(1, 2))
        self.scales = {name: torch.full((total, kv_heads), 1e30, device="cuda") for name in ("key", "value")}

    @property
    def args(self):
        return self.caches["key"], self.caches["value"], self.scales["key"], self.scales["value"]

    def tokens(self, name, s, length):
        """(codes, scales) of a sequence's first tokens: [length, H, D] and [length, H], in 64 bits."""
        pages = self.table[s, : -(-length // self.page)]
        codes = self.caches[name].cpu()[pages].double().transpose(1, 2).flatten(0, 1)[:length]
        scales = self.scales[name].cpu()[pages].double().repeat_interleave(self.page, 0)[:length]
        return codes, scales


def least_scale(high, code):
    """The scale of a block, in 64 bits, from its largest magnitude."""
    if code == torch.int8:
        return max(high / 127, 2.0**-126)
    return 2.0 ** max(-126, math.ceil(math.log2(high / 448))) if high > 0 else 2.0**-126


def code_error(x, scale, code):
    """Half a step of a code that stands for x."""
    if code == torch.int8:
        return scale / 2
    return (x.abs() * 2.0**-4).clamp(min=scale * 2.0**-10)


APPENDS = [
    # past, new, page, heads, kv_heads, dim, rotary
    ([0], [1], 16, 4, 1, 64, 64),
    ([15, 16, 17], [1, 1, 1], 16, 8, 2, 128, 128),
    ([0, 5, 31, 32], [70, 0, 1, 33], 32, 6, 3, 64, 32),
    ([63, 0, 100], [130, 64, 1], 64, 4, 4, 128, 64),
    ([3, 0], [200, 129], 128, 2, 1, 96, 96),
    ([1, 2, 3], [40, 3, 17], 48, 5, 5, 80, 20),
    ([0] * 40, [1, 0, 2, 3] * 10, 16, 2, 2, 16, 16),
]


@pytest.mark.parametrize("code", (torch.float8_e4m3fn, torch.int8), ids=("e4m3", "int8"))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("case", APPENDS, ids=range(len(APPENDS)))
def test_paged_append(case, dtype, code):
    past, new, page, heads, kv_heads, dim, rotary = case
    interleaved = heads % 4 == 0
    total = [p + n for p, n in zip(past, new)]
    cache = Pages(total, page, kv_heads, dim, code, layout="heads" if dim != 96 else "tokens")
    cos, sin = programs.rotary_tables(max(total), rotary)
    held = [(torch.randn(p, kv_heads, dim), torch.randn(p, kv_heads, dim)) for p in past]
    wide = torch.int64 if page == 64 else torch.int32
    table = index(cache.table.tolist(), wide)

    def offsets(lens):
        return index([sum(lens[:i]) for i in range(len(lens) + 1)], wide)

    def append(k, v, lens, before, **kwargs):
        return programs.paged_append(dev(k), dev(v), offsets(lens), index(before, wide), table, *cache.args, **kwargs)

    # what the sequences hold goes in unrotated, in a call of its own
    append(torch.cat([k for k, _ in held]).to(dtype), torch.cat([v for _, v in held]).to(dtype), past, [0] * len(past))
    before = {name: [cache.tokens(name, s, p) for s, p in enumerate(past)] for name in ("key", "value")}
    stored = cache.caches["key"].view(torch.int8).cpu().clone() if cache.caches["key"].is_contiguous() else None
    qkv = (torch.randn(sum(new), heads + 2 * kv_heads, dim) * 3).to(dtype)
    query, key, value = qkv.split((heads, kv_heads, kv_heads), dim=1)
    query_out, key_out = append(key, value, new, past, query=dev(qkv)[:, :heads], cos=dev(cos), sin=dev(sin),
                                interleaved=interleaved, return_key=True)
    assert device_status() == 0

    position = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)])
    slack = rotation_error(qkv, rotary)
    for got, x in ((query_out, query), (key_out, key)):
        want = turned(x, cos[position], sin[position], interleaved)
        assert ((got.cpu().double() - want).abs() <= HALF[dtype] * want.abs() + TINY[dtype] + slack).all()
    rows = {"key": turned(key, cos[position], sin[position], interleaved), "value": value.double()}
    touched = set()
    at = 0
    for s, (p, n) in enumerate(zip(past, new)):
        for name in ("key", "value"):
            codes, scales = cache.tokens(name, s, p + n)
            for j in range(p // page, -(-(p + n) // page)):
                low, high = max(p, j * page), min(p + n, (j + 1) * page)
                if low >= high:
                    continue
                touched.add(int(cache.table[s, j]))
                x = rows[name][at + low - p : at + high - p]
                for h in range(kv_heads):
                    scale = least_scale(float(x[:, h].abs().max()), code)
                    first = low > j * page
                    old_codes, old_scales = before[name][s]
                    if first:
                        scale = max(scale, float(old_scales[low - 1, h]))
                    got = float(scales[low, h])
                    # int8: two roundings of the scale, and those of the largest magnitude
                    assert abs(got - scale) <= (4 * 2.0**-24 * scale if code == torch.int8 else 0)
                    off = (codes[low:high, h] * got - x[:, h]).abs()
                    assert (off <= code_error(x[:, h], got, code) * (1 + 2.0**-20) + slack).all()
                    if first:
                        was = old_codes[j * page : low, h] * old_scales[j * page : low, h, None]
                        now = codes[j * page : low, h] * got
                        grew = got > float(old_scales[low - 1, h])
                        limit = code_error(was, got, code) * (1 + 2.0**-20) if grew else 0 * was
                        if code != torch.int8:  # a power of two: exact but for subnormals
                            limit = torch.full_like(was, got * 2.0**-10) if grew else limit
                        assert ((now - was).abs() <= limit).all()
        at += n
    if stored is not None:  # nothing else was written
        rest = [b for b in range(stored.shape[0]) if b not in touched]
        assert torch.equal(cache.caches["key"].view(torch.int8).cpu()[rest], stored[rest])


@pytest.mark.parametrize("code", (torch.float8_e4m3fn, torch.int8), ids=("e4m3", "int8"))
def test_paged_append_not_finite_zero_and_large(code):
    """Infinities saturate and do not set the scale, NaN stays (int8: 0), zeros
    take the least scale, and the largest values keep theirs."""
    cache = Pages([4, 16, 2], 16, 1, 16, code)
    key = torch.ones(22, 1, 16, dtype=torch.bfloat16)
    key[0, 0, 0], key[1, 0, 1], key[2, 0, 2] = math.inf, -math.inf, math.nan
    key[4:20] = 0
    key[20:] = 3e38
    programs.paged_append(dev(key), dev(key), index([0, 4, 20, 22]), index([0, 0, 0]), index(cache.table.tolist()),
                          *cache.args)
    top = 127.0 if code == torch.int8 else 448.0
    for name in ("key", "value"):
        codes, scales = cache.tokens(name, 0, 4)
        assert scales[0, 0] == pytest.approx(least_scale(1.0, code), rel=1e-6)
        assert codes[0, 0, 0] == top and codes[1, 0, 1] == -top
        assert codes[2, 0, 2] == 0 if code == torch.int8 else codes[2, 0, 2].isnan()
        assert ((codes[3] * scales[3, :, None] - 1).abs() <= 2.0**-7).all()
        codes, scales = cache.tokens(name, 1, 16)
        assert not codes.any() and (scales == 2.0**-126).all()
        codes, scales = cache.tokens(name, 2, 2)
        assert ((codes * scales[..., None] / float(key[20, 0, 0]) - 1).abs() <= 2.0**-4).all()
    assert device_status() == 0


def test_paged_append_bad_indices_are_not_followed():
    cache = Pages([16, 16], 16, 1, 16, torch.int8)
    before = cache.caches["key"].clone()
    key = torch.randn(4, 1, 16).half().cuda()
    good = cache.table[:, :1].tolist()
    bad = [
        ([0, 2, 4], [0, 0], [[-1], [99]]),  # pages outside the pool
        ([0, 2, 4], [16, 40], good),  # positions past the block table
        ([0, 2, 9], [0, 0], [[-1], good[1]]),  # tokens that are not there
        ([0, 2, 4], [-3, -1], good),
    ]
    for offsets, past, table in bad:
        table = [row if isinstance(row, list) else [row] for row in table]
        programs.paged_append(key, key, index(offsets), index(past), index(table), *cache.args)
        assert device_status() == INDEX_OUT_OF_RANGE
        assert torch.equal(cache.caches["key"], before)


# --------------------------------------------------------------------- attention over the cache
def softmax_rows(q, k, v, scale, limit):
    """o and lse of one query row over the first `limit` keys, in 64 bits."""
    if limit <= 0:
        return torch.zeros(v.shape[-1], dtype=torch.float64), -math.inf
    s = (k[:limit] @ q) * scale
    lse = torch.logsumexp(s, 0)
    return torch.exp(s - lse) @ v[:limit], float(lse)


def filled_cache(lens, page, kv_heads, dim, code, spread=1.0):
    """A cache of random codes with a scale for each page and head; unused slots and pages stay stale."""
    cache = Pages(lens, page, kv_heads, dim, code, layout="heads" if dim != 96 else "tokens")
    used = sorted({int(cache.table[s, j]) for s, n in enumerate(lens) for j in range(-(-n // page))})
    for name in ("key", "value"):
        top = 127 if code == torch.int8 else 448
        if used:
            codes = (torch.randn(len(used), kv_heads, page, dim) * top / 6).clamp(-top, top)
            codes = codes.round().to(torch.int8) if code == torch.int8 else codes.to(code)
            view = cache.caches[name].view(torch.int8) if cache.caches[name].is_contiguous() else None
            if view is not None:
                view[used] = codes.view(torch.int8).cuda()
            else:
                cache.caches[name].transpose(1, 2).view(torch.int8)[used] = codes.transpose(1, 2).contiguous().view(
                    torch.int8).cuda()
            scales = 6 / top * torch.exp2(spread * (2 * torch.rand(len(used), kv_heads) - 1))
            cache.scales[name][used] = scales.cuda()
    for s, n in enumerate(lens):  # stale NaN codes and scales after the last token
        if n % page and code != torch.int8:
            block = cache.table[s, n // page]
            for name in ("key", "value"):
                if cache.caches[name].is_contiguous():
                    cache.caches[name].view(torch.int8)[block, :, n % page :] = 127
    return cache


def check_paged(query, cache, lens, scale, got, lse, dtype):
    batch, queries, heads, dim = query.shape
    kv_heads = cache.caches["key"].shape[1]
    got, lse = got.cpu().double(), lse.cpu().double()
    for b, n in enumerate(lens):
        k, v = ((codes * scales[..., None]) for codes, scales in (cache.tokens(name, b, n) for name in ("key", "value")))
        for i in range(queries):
            for h in range(heads):
                g = h // (heads // kv_heads)
                want, want_lse = softmax_rows(query[b, i, h].double(), k[:, g], v[:, g], scale, n - queries + 1 + i)
                if want_lse == -math.inf:
                    assert lse[b, i, h] == -math.inf and not got[b, i, h].any()
                    continue
                # scores: fp32 sums of dim products of exact factors, times a factor of a few roundings
                product = float((k[:, g].abs() @ query[b, i, h].double().abs()).max()) * scale
                score = (dim + 8) * 2.0**-24 * product
                assert abs(lse[b, i, h] - want_lse) <= 2 * score + 2.0**-20 * (1 + abs(want_lse))
                # each weight: the score's error, and half a step of fp16 (half precision inputs)
                top = float(v[:, g].abs().max())
                weight = 2 * score + (2.0**-11 if dtype != torch.float32 else 0) + 2.0**-20
                limit = HALF[dtype] * want.abs() + TINY[dtype] + weight * top
                assert ((got[b, i, h] - want).abs() <= limit).all(), (b, i, h)


PAGED = [
    # lens, queries, page, heads, kv_heads, dim
    ([1], 1, 16, 1, 1, 16),
    ([17, 0, 300], 1, 16, 8, 2, 128),
    ([257, 1, 64, 1000], 1, 64, 8, 1, 64),
    ([5, 2, 0, 700], 4, 32, 4, 2, 128),
    ([513, 3], 7, 48, 6, 2, 96),
    ([1300, 12], 5, 128, 20, 4, 80),
    ([40] * 33 + [777, 1200], 1, 16, 3, 3, 112),
    ([31, 33], 40, 16, 2, 1, 48),
]


@pytest.mark.parametrize("code", (torch.float8_e4m3fn, torch.int8), ids=("e4m3", "int8"))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("case", PAGED, ids=range(len(PAGED)))
def test_paged_attention(case, dtype, code):
    lens, queries, page, heads, kv_heads, dim = case
    cache = filled_cache(lens, page, kv_heads, dim, code, spread=4.0)
    query = (torch.randn(len(lens), queries, heads, dim) * 2).to(dtype)
    wide = torch.int64 if page == 64 else torch.int32
    scale = 0.7 * dim**-0.5
    got, lse = programs.paged_attention(dev(query), *cache.args, index(cache.table.tolist(), wide), index(lens, wide),
                                        scale=scale, return_lse=True)
    assert device_status() == 0 and got.dtype == dtype
    check_paged(query, cache, lens, scale, got, lse, dtype)
    again = programs.paged_attention(dev(query), *cache.args, index(cache.table.tolist(), wide), index(lens, wide), scale)
    assert torch.equal(again, got)


def test_paged_attention_strided_queries_and_output():
    lens, page, heads, kv_heads, dim = [100, 700], 32, 6, 3, 64
    cache = filled_cache(lens, page, kv_heads, dim, torch.int8)
    qkv = torch.randn(2, 1, heads + 2 * kv_heads, 2 * dim).half()
    spread = torch.zeros(heads, 2, 1, dim + 5, dtype=torch.float16, device="cuda")
    lse = torch.zeros(heads, 2, 1, device="cuda").permute(1, 2, 0)
    out = spread.permute(1, 2, 0, 3)[..., 5:]
    programs.paged_attention_kernel(dev(qkv)[:, :, :heads, ::2], *cache.args, index(cache.table.tolist()), index(lens),
                                    out, lse)
    check_paged(qkv[:, :, :heads, ::2], cache, lens, dim**-0.5, out, lse, torch.float16)
    assert not spread[..., :5].any()
    part = programs.paged_attention(dev(qkv)[:, :, 2:4, ::2], *(x[:, 1:2] for x in cache.args),
                                    index(cache.table.tolist()), index(lens))
    # the heads of one group over a slice of the cache
    assert torch.allclose(part, out[:, :, 2:4], rtol=2.0**-9, atol=2.0**-9)


def test_paged_attention_scales_far_apart():
    """Weights value_scale * p from blocks of very different scales keep their bits."""
    lens, page, dim = [640], 16, 64
    cache = filled_cache(lens, page, 1, dim, torch.float8_e4m3fn, spread=14.0)
    query = torch.randn(1, 1, 4, dim).bfloat16()
    cache.scales["key"].fill_(0.02)
    got, lse = programs.paged_attention(dev(query), *cache.args, index(cache.table.tolist()), index(lens), return_lse=True)
    check_paged(query, cache, lens, dim**-0.5, got, lse, torch.bfloat16)
    # a block of zeros with the least scale beside the others, and one of scale 0
    block = int(cache.table[0, 3])
    cache.caches["value"].view(torch.int8)[block] = 0
    cache.scales["value"][block] = 2.0**-126
    cache.scales["value"][int(cache.table[0, 5])] = 0
    got, lse = programs.paged_attention(dev(query), *cache.args, index(cache.table.tolist()), index(lens), return_lse=True)
    check_paged(query, cache, lens, dim**-0.5, got, lse, torch.bfloat16)


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
def test_paged_attention_nan_reaches_only_who_sees_it(dtype):
    lens, queries, dim = [70], 4, 128
    for heads in (2, 4):
        cache = filled_cache(lens, 16, 2, dim, torch.float8_e4m3fn)
        query = torch.randn(1, queries, heads, dim).to(dtype)
        args = index(cache.table.tolist()), index(lens)
        clean = programs.paged_attention(dev(query), *cache.args, *args)
        at = int(cache.table[0, 68 // 16])
        cache.caches["value"].view(torch.int8)[at, 0, 68 % 16, 5] = 127
        got = programs.paged_attention(dev(query), *cache.args, *args)
        bad = got.isnan()
        group = slice(0, heads // 2)
        assert bad[:, 2:, group, 5].all() and bad.sum() == 2 * (heads // 2)
        assert torch.equal(got.nan_to_num(0.0), clean.masked_fill(bad, 0.0))


def test_paged_attention_long_and_lengths_out_of_range():
    cache = filled_cache([5000], 32, 1, 64, torch.int8)
    query = torch.randn(1, 1, 8, 64).half()
    table = index(cache.table.tolist())
    got, lse = programs.paged_attention(dev(query), *cache.args, table, index([5000]), return_lse=True)
    check_paged(query, cache, [5000], 64**-0.5, got, lse, torch.float16)
    whole = table[:, :-1]  # 157 pages: 5024 tokens
    programs.paged_attention(dev(query), *cache.args, whole, index([5025]))
    assert device_status() == INDEX_OUT_OF_RANGE
    out = programs.paged_attention(dev(query), *cache.args, whole, index([-1]))
    assert device_status() == INDEX_OUT_OF_RANGE and not out.any()
    programs.paged_attention(dev(query), *cache.args, table, index([5056]))  # the last column is page -1
    assert device_status() == INDEX_OUT_OF_RANGE


def test_paged_attention_offsets_past_32_bits():
    """Pages whose byte offset needs more than 32 bits."""
    pages, page, dim = 34000, 64, 128
    cache = torch.zeros(pages, 16, page, dim, dtype=torch.int8, device="cuda")
    value = torch.zeros(pages, 1, page, dim, dtype=torch.int8, device="cuda")
    assert cache.numel() > 2**32
    scales = torch.ones(pages, 16, device="cuda")
    last = pages - 1
    value[last, 0, :, :] = 3
    cache[last, 15, 0, 0] = 100
    query = torch.zeros(1, 1, 1, dim, dtype=torch.float16, device="cuda")
    query[..., 0] = 1
    got, lse = programs.paged_attention(query, cache[:, 15:], value, scales[:, :1], scales[:, :1], index([[0, last]]),
                                        index([128]), scale=1.0, return_lse=True)
    assert torch.allclose(got.float(), torch.full_like(got.float(), 3.0), rtol=2.0**-10)
    assert abs(float(lse) - 100.0) < 1e-4
    key = torch.full((1, 1, dim), 2.0, dtype=torch.float16, device="cuda")
    programs.paged_append(key, key, index([0, 1]), index([127]), index([[0, last]]), cache[:, 15:], value,
                          scales[:, :1], scales[:, 1:2])
    assert int(cache[last, 15, 63].float().mean()) == 2 and not cache[0].any()


# --------------------------------------------------------------------- attention over prompts
def check_prompt(q, k, v, q_lens, k_lens, scale, causal, got, lse, dtype):
    got, lse = got.cpu().double(), lse.cpu().double()
    q, k, v = q.double(), k.double(), v.double()
    heads, kv_heads, dim = q.shape[1], k.shape[1], q.shape[2]
    q0 = k0 = 0
    for nq, nk in zip(q_lens, k_lens):
        limit = nk - nq + 1 + torch.arange(nq) if causal else torch.full((nq,), nk)
        hidden = torch.arange(nk)[None] >= limit[:, None]
        for h in range(heads):
            g = h // (heads // kv_heads)
            rows, keys, values = q[q0 : q0 + nq, h], k[k0 : k0 + nk, g], v[k0 : k0 + nk, g]
            s = (rows @ keys.T * scale).masked_fill(hidden, -math.inf)
            want_lse = torch.logsumexp(s, 1)
            weights = torch.exp(s - want_lse[:, None]).masked_fill(hidden, 0.0)
            want = weights @ values
            x, y = got[q0 : q0 + nq, h], lse[q0 : q0 + nq, h]
            some = (limit > 0) if nk else torch.zeros(nq, dtype=torch.bool)
            assert not x[~some].any() and (y[~some] == -math.inf).all()
            if not some.any():
                continue
            # scores: fp32 sums of exact products; weights: the scores' error and half a step of the type
            score = (dim + 8) * 2.0**-24 * float((rows.abs() @ keys.abs().T).max()) * abs(scale)
            assert ((y - want_lse)[some].abs() <= 2 * score + 2.0**-20 * (1 + want_lse[some].abs())).all()
            weight = 2 * score + (HALF[dtype] if dtype != torch.float32 else 0) + 2.0**-20
            top = weights[some] @ values.abs()  # what the weights' relative errors can add up to
            bound = HALF[dtype] * want[some].abs() + TINY[dtype] + weight * top
            assert ((x[some] - want[some]).abs() <= bound).all(), (nq, nk, h)
        q0, k0 = q0 + nq, k0 + nk


PROMPTS = [
    # query lengths, key lengths (None: the same), heads, kv_heads, dim
    ([1], None, 1, 1, 64),
    ([1, 0, 17, 100, 3], None, 8, 2, 64),
    ([300, 129, 128], None, 4, 1, 128),
    ([257, 5], None, 3, 1, 96),
    ([64, 200], None, 10, 2, 40),
    ([700], None, 2, 2, 128),
    ([90, 31], None, 7, 1, 24),
    ([5, 60, 0, 33], [300, 60, 7, 40], 6, 3, 80),  # later parts of prompts
    ([40, 9], [10, 0], 4, 2, 64),  # queries before the first key
    ([33], [1000], 130, 1, 16),  # a group over 128: CUDA cores
]


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("case", PROMPTS, ids=range(len(PROMPTS)))
def test_prompt_attention(case, dtype, causal):
    q_lens, k_lens, heads, kv_heads, dim = case
    q = (torch.randn(sum(q_lens), heads, dim) * 2).to(dtype)
    k, v = (torch.randn(sum(k_lens or q_lens), kv_heads, dim).to(dtype) for _ in range(2))
    wide = torch.int64 if dim == 64 else torch.int32

    def offsets(lens):
        return index([sum(lens[:i]) for i in range(len(lens) + 1)], wide)

    scale = 0.6 * dim**-0.5
    got, lse = programs.prompt_attention(dev(q), dev(k), dev(v), offsets(q_lens), offsets(k_lens) if k_lens else None,
                                         is_causal=causal, scale=scale, return_lse=True)
    assert device_status() == 0 and got.dtype == dtype
    check_prompt(q, k, v, q_lens, k_lens or q_lens, scale, causal, got, lse, dtype)
    assert torch.equal(programs.prompt_attention(dev(q), dev(k), dev(v), offsets(q_lens),
                                                 offsets(k_lens) if k_lens else None, causal, scale), got)


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_prompt_attention_many_sequences_and_scores_far_apart(dtype):
    """More items than SMs, lengths of every kind, rows whose maximum moves block by block."""
    lens = [int(n) for n in torch.randint(0, 400, (40,))] + [1500]
    heads, kv_heads, dim = 8, 4, 128
    q = torch.randn(sum(lens), heads, dim).to(dtype)
    k = (torch.randn(sum(lens), kv_heads, dim) * torch.linspace(0.1, 12.0, sum(lens))[:, None, None]).to(dtype)
    v = torch.randn(sum(lens), kv_heads, dim).to(dtype)
    offsets = index([sum(lens[:i]) for i in range(len(lens) + 1)])
    got, lse = programs.prompt_attention(dev(q), dev(k), dev(v), offsets, return_lse=True)
    check_prompt(q, k, v, lens, lens, dim**-0.5, True, got, lse, dtype)


@pytest.mark.parametrize("scale", (0.0, -0.3))
def test_prompt_attention_scale_not_positive(scale):
    q, k, v = torch.randn(3, 70, 2, 32).half()
    got, lse = programs.prompt_attention(dev(q), dev(k), dev(v), index([0, 70]), scale=scale, return_lse=True)
    check_prompt(q, k, v, [70], [70], scale, True, got, lse, torch.float16)


def test_prompt_attention_strides():
    """Views of a fused projection, an output between other heads, an element stride, a base off the 16-byte grid."""
    lens, heads, kv_heads, dim = [50, 150], 4, 2, 64
    qkv = torch.randn(200, heads + 2 * kv_heads, dim).half()
    q, k, v = qkv.split((heads, kv_heads, kv_heads), 1)
    offsets = index([0, 50, 200])
    parts = dev(qkv).split((heads, kv_heads, kv_heads), 1)
    out = torch.zeros(heads + 2, 200, dim, dtype=torch.float16, device="cuda").transpose(0, 1)
    lse = torch.zeros(heads, 200, device="cuda").T
    programs.prompt_attention_kernel(*parts, offsets, offsets, out[:, 1:-1], lse)
    check_prompt(q, k, v, lens, lens, dim**-0.5, True, out[:, 1:-1], lse, torch.float16)
    assert not out[:, 0].any() and not out[:, -1].any()
    spread = torch.stack((dev(qkv), dev(qkv)), dim=-1)[..., 0].split((heads, kv_heads, kv_heads), 1)
    got, lse = programs.prompt_attention(*spread, offsets, return_lse=True)
    check_prompt(q, k, v, lens, lens, dim**-0.5, True, got, lse, torch.float16)
    odd = torch.zeros(qkv.numel() + 1, dtype=torch.float16, device="cuda")[1:].view(qkv.shape).copy_(qkv)
    got, lse = programs.prompt_attention(*odd.split((heads, kv_heads, kv_heads), 1), offsets, return_lse=True)
    check_prompt(q, k, v, lens, lens, dim**-0.5, True, got, lse, torch.float16)


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
def test_prompt_attention_not_finite_where_it_is_not_seen(dtype):
    """NaN and infinities in keys and values of later tokens, of the next sequence
    and of tokens of no sequence reach nobody who does not see them."""
    lens, heads, kv_heads, dim = [200, 70], 4, 2, 128
    q, k, v = (torch.randn(300, n, dim).to(dtype) for n in (heads, kv_heads, kv_heads))
    offsets = index([0, 200, 270])
    clean = programs.prompt_attention(dev(q), dev(k), dev(v), offsets).cpu()
    for bad in (math.nan, math.inf):
        k2, v2 = k.clone(), v.clone()
        k2[270:], v2[270:] = bad, bad
        v2[150, 1, 3] = bad
        v2[190:200, 0] = bad
        k2[195, 0] = bad
        got = programs.prompt_attention(dev(q), dev(k2), dev(v2), offsets).cpu()
        assert not got[150:200, 2:, 3].isfinite().any() and not got[190:200, :2].isfinite().any()
        same = torch.ones(270, heads, dim, dtype=torch.bool)
        same[150:200, 2:, 3] = False
        same[190:200, :2] = False
        # rows whose sums met the bad values were taken again on other units
        near = (got[:270] - clean[:270]).abs() <= 2.0**-8 * (1 + clean[:270].abs())
        assert near[same].all()


def test_prompt_attention_offsets_out_of_range():
    q = torch.randn(64, 2, 64).half().cuda()
    good = programs.prompt_attention(q, q, q, index([0, 64]))
    # the last: overlapping sequences, more of their tiles than tokens have room for
    for bad in ([0, 65], [-1, 64], [0, 40, 30], [0, 64] * 300):
        programs.prompt_attention(q, q, q, index(bad))
        assert device_status() == INDEX_OUT_OF_RANGE
        programs.prompt_attention(q.float(), q.float(), q.float(), index(bad))
        assert device_status() == INDEX_OUT_OF_RANGE
    assert torch.equal(programs.prompt_attention(q, q, q, index([0, 64])), good)


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
def test_prompt_attention_without_keys_or_queries(dtype):
    q = torch.randn(5, 2, 64).to(dtype).cuda()
    none = q[:0, :1]
    got, lse = programs.prompt_attention(q, none, none, index([0, 3, 5]), index([0, 0, 0]), return_lse=True)
    assert not got.any() and (lse == -math.inf).all()
    got, lse = programs.prompt_attention(q[:0], q[:, :1], q[:, :1], index([0, 0]), index([0, 5]), return_lse=True)
    assert got.shape == (0, 2, 64) and lse.shape == (0, 2)
    assert device_status() == 0


@pytest.mark.parametrize("heads, kv_heads", ((4, 4), (6, 2)))
def test_prompt_attention_head_major(heads, kv_heads):
    """[heads, tokens, head_dim] in memory."""
    lens = [200, 60]
    q, k, v = (torch.randn(n, 260, 64).bfloat16().transpose(0, 1) for n in (heads, kv_heads, kv_heads))
    got, lse = programs.prompt_attention(dev(q), dev(k), dev(v), index([0, 200, 260]), return_lse=True)
    assert not dev(q).is_contiguous()
    check_prompt(q, k, v, lens, lens, 64**-0.5, True, got, lse, torch.bfloat16)


def test_joined_by_lse():
    """Attention over a cached beginning and over a prompt's rest, joined by
    their lse, is attention over both."""
    kept, new, heads, kv_heads, dim = 100, 30, 4, 2, 64
    cache = filled_cache([kept], 16, kv_heads, dim, torch.int8)
    q, k, v = (torch.randn(new, n, dim).half() for n in (heads, kv_heads, kv_heads))
    # every new query sees all that is cached: each as a sequence of its own
    table = index(cache.table.tolist()).repeat(new, 1)
    a, la = programs.paged_attention(dev(q)[:, None], *cache.args, table, index([kept] * new), return_lse=True)
    b, lb = programs.prompt_attention(dev(q), dev(k), dev(v), index([0, new]), return_lse=True)
    la, lb = la[:, 0].cpu().double(), lb.cpu().double()
    both = torch.logaddexp(la, lb)
    joined = (a[:, 0].cpu() * torch.exp(la - both)[..., None] + b.cpu() * torch.exp(lb - both)[..., None])
    old = [codes * scales[..., None] for codes, scales in (cache.tokens(name, 0, kept) for name in ("key", "value"))]
    k2, v2 = (torch.cat((x, y.double())) for x, y in zip(old, (k, v)))
    top = float(v2.abs().max())
    for i in range(new):
        for h in range(heads):
            want, want_lse = softmax_rows(q[i, h].double(), k2[:, h // 2], v2[:, h // 2], dim**-0.5, kept + 1 + i)
            assert abs(both[i, h] - want_lse) < 1e-4
            assert ((joined[i, h] - want).abs() <= 2.0**-10 * (top + want.abs())).all()


def test_serving_refusals():
    x = torch.zeros(4, 2, 32, dtype=torch.float16, device="cuda")
    cos = torch.zeros(8, 16, device="cuda")
    at = index([0, 1, 2, 3])
    with pytest.raises(TypeError, match="rotary shapes"):
        programs.rotary(x, cos, cos, at[:3])
    with pytest.raises(TypeError, match="rotary tables"):
        programs.rotary(x, cos, cos[:, :8], at)
    with pytest.raises(TypeError, match="rotary tables"):
        programs.rotary(x[..., :16], cos, cos, at)
    with pytest.raises(TypeError, match="dtype"):
        programs.rotary(x, cos.half(), cos.half(), at)
    with pytest.raises(TypeError, match="dtype"):
        programs.rotary(x, cos, cos, at.float())
    with pytest.raises(TypeError, match="unit stride"):
        programs.rotary(x, cos.repeat(1, 2)[:, ::2], cos.repeat(1, 2)[:, ::2], at)
    with pytest.raises(TypeError, match="CUDA device"):
        programs.rotary(x, cos.cpu(), cos, at)
    codes = torch.zeros(4, 2, 16, 32, dtype=torch.int8, device="cuda")
    scales = torch.zeros(4, 2, device="cuda")
    good = dict(key=x, value=x, offsets=index([0, 4]), past=index([0]), block_table=index([[0]]), key_cache=codes,
                value_cache=codes.clone(), key_scale=scales, value_scale=scales.clone())
    programs.paged_append(**good)
    for change, message in (
        (dict(value=x[:3]), "disagree"),
        (dict(key=x[:, :1], value=x[:, :1]), "disagree"),
        (dict(value=x.float()), "share one dtype"),
        (dict(past=index([0], torch.int64)), "share one dtype"),
        (dict(offsets=index([0, 2, 4])), "offsets"),
        (dict(key_scale=scales[:3]), "disagree"),
        (dict(value_cache=codes[:3]), "disagree"),
        (dict(key_cache=codes[:, :, :8], value_cache=codes[:, :, :8]), "multiples of 16"),
        (dict(key_cache=codes.half(), value_cache=codes.half()), "dtype"),
        (dict(query=x), "needs `cos`"),
        (dict(cos=cos), "together"),
    ):
        with pytest.raises(TypeError, match=message):
            programs.paged_append(**(good | change))
    query = torch.zeros(1, 1, 4, 32, dtype=torch.float16, device="cuda")
    fine = dict(query=query, lengths=index([0]), **{name: good[name] for name in (
        "key_cache", "value_cache", "key_scale", "value_scale", "block_table")})
    assert not programs.paged_attention(**fine).any()
    for change, message in (
        (dict(query=query[..., :16]), "disagree"),
        (dict(query=query[:, :, :3]), "disagree"),
        (dict(lengths=index([0, 0])), "lengths"),
        (dict(lengths=index([0], torch.int64)), "share one dtype"),
        (dict(query=query.double()), "dtype"),
        (dict(key_scale=scales.half()), "dtype"),
    ):
        with pytest.raises(TypeError, match=message):
            programs.paged_attention(**(fine | change))
    ok = dict(query=x, key=x, value=x, offsets=index([0, 4]))
    programs.prompt_attention(**ok)
    for change, message in (
        (dict(key=x[:, :1]), "disagree"),
        (dict(key=x[..., :16], value=x[..., :16]), "disagree"),
        (dict(query=x[:, :1]), "disagree"),
        (dict(value=x.float()), "share one dtype"),
        (dict(offsets=index([])), "offsets"),
        (dict(key_offsets=index([0, 2, 4])), "offsets"),
        (dict(key_offsets=index([0, 4], torch.int64)), "share one dtype"),
        (dict(offsets=index([[0, 4]])), "rank"),
    ):
        with pytest.raises(TypeError, match=message):
            programs.prompt_attention(**(ok | change))
    with pytest.raises(TypeError, match="unit stride"):
        wide = torch.zeros(4, 2, 16, 64, dtype=torch.int8, device="cuda")[..., ::2]
        programs.paged_append(**(good | dict(key_cache=wide, value_cache=wide)))
    with pytest.raises(programs.KernelLaunchError):  # a base off the 16-byte grid
        odd = torch.zeros(4 * 2 * 16 * 32 + 1, dtype=torch.int8, device="cuda")[1:].view(4, 2, 16, 32)
        programs.paged_append(**(good | dict(key_cache=odd)))
