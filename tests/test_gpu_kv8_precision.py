"""What the attention over the paged 8-bit cache keeps of small contributions, against 64-bit arithmetic on the cache's content.

The bounds count what the kernels round. With S = scale * sum |q_i k_i|, p the exact softmax weights and A = sum of p |v|: a score
(products of exact codes and of queries of 22 bits, FP32 sums, the rotation) is off by at most d = 2^-19 (1 + S), so a weight by a
factor within exp(+-2 d); weights keep 22 bits (2^-20 with their factor and their sum), and below FP16's normal numbers (a step is
rounded by half of it) 2^-40 of the row's largest weight in steps of single tokens, else 2^-36 of its largest product of weight
and value scale, per unit of a code; the result is rounded to the cache's type (half a step)."""

import math

import pytest

from mylocal_llm_b200 import _lib
from test_gpu_kv8_attention import query, random_cache, step

pytestmark = pytest.mark.gpu

BLOCK = 64


@pytest.fixture(autouse=True)
def healthy(cuda):
    _lib.clear_device_status()
    yield
    cuda.cuda.synchronize()
    assert _lib.device_status() == 0


def exact(torch, cache, layer, q, sizes, counts, scale):
    """(result, A, largest S, what may be lost below FP16's normal numbers) of every row and head in 64 bits, [rows, heads, dh or 1]."""
    dh, kv_heads = cache.head_dim, cache.kv_heads
    heads, row, out = q.shape[1] // dh, 0, []
    for s, (total, n) in enumerate(zip(sizes, counts)):
        if not n:
            continue
        pages, rest = cache.table[s, :total // BLOCK].long(), total % BLOCK
        codes, sc = cache.codes[pages, layer].double(), cache.scales[pages, layer].double()
        tail = cache.tail[s, layer, :, :, :rest].double()
        k = torch.cat([(codes[:, 0].reshape(-1, kv_heads, BLOCK, dh) * sc[:, 0, :, None, None]).transpose(0, 1).reshape(kv_heads, -1, dh), tail[0]], 1)
        v = torch.cat([(codes[:, 1].reshape(-1, kv_heads, dh, BLOCK) * sc[:, 1, :, None, None]).permute(1, 0, 3, 2).reshape(kv_heads, -1, dh), tail[1]], 1)
        step_of = torch.cat([sc[:, 1].T.repeat_interleave(BLOCK, 1), cache.peak[s, layer, 1].double()[:, None].expand(-1, rest)], 1)
        x = q[row:row + n].double().reshape(n, kv_heads, heads // kv_heads, dh).permute(1, 2, 0, 3)
        hidden = torch.arange(total, device="cuda") > (torch.arange(n, device="cuda") + total - n)[:, None]
        k, v = k[:, None], v[:, None]
        p = torch.softmax((x @ k.transpose(-1, -2) * scale).masked_fill(hidden, -math.inf), -1)
        big = (x.abs() @ k.abs().transpose(-1, -2) * abs(scale)).masked_fill(hidden, 0).amax(-1, keepdim=True)
        seen, step_of = (~hidden).double(), step_of[:, None, :]
        if max(counts) == 1:
            lost = 2.0 ** -39 * p.amax(-1, keepdim=True) * (seen @ v.abs())
        else:
            lost = 2.0 ** -35 * (p * step_of[:, :, None]).amax(-1, keepdim=True) * (seen @ (v.abs() / step_of[..., None].clamp_min(1e-300)))
        parts = p @ v, p @ v.abs(), big, lost
        out.append([t.permute(2, 0, 1, 3).reshape(n, heads, -1) for t in parts])
        row += n
    return [torch.cat(t) for t in zip(*out)]


def check(torch, cache, layer, q, out, sizes, counts, scale):
    want, a, big, lost = exact(torch, cache, layer, q, sizes, counts, scale)
    kind = torch.finfo(out.dtype)
    d = 2.0 ** -19 * (1 + big)
    bound = (torch.exp(2 * d) - 1 + 2.0 ** -20) * a + lost + kind.eps / 2 * 1.01 * want.abs() + kind.tiny * kind.eps
    got = out.double().reshape(want.shape)
    assert torch.isfinite(got).all()
    off = ((got - want).abs() / bound).max()
    assert off <= 1, f"{float(off)} of the bound"


def levelled_cache(torch, sizes, kv_heads, dh, dtype, levels, value_scales, seed):
    """Every block's keys score about ``levels[b % len]`` (in natural units, for queries of ones and scale 1 / dh) and its values
    have the scale ``value_scales[b % len]``."""
    cache = random_cache(torch, sizes, 1, kv_heads, dh, dtype, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for s, n in enumerate(sizes):
        for b in range(n // BLOCK):
            page, level = int(cache.table[s, b]), levels[b % len(levels)]
            keys = torch.randint(60, 69, (kv_heads, BLOCK * dh), device="cuda", generator=gen)
            cache.codes[page, 0, 0] = (keys if level > 0 else -keys).to(torch.int8)
            cache.scales[page, 0, 0] = abs(level) / 64
            cache.scales[page, 0, 1] = value_scales[b % len(value_scales)]
        rest = n % BLOCK
        if rest:
            cache.tail[s, 0, 0, :, :rest] = levels[n // BLOCK % len(levels)]
            cache.peak[s, 0, 0] = cache.tail[s, 0, 0, :, :rest].float().abs().amax((-1, -2))
            values = torch.randn(kv_heads, rest, dh, device="cuda", generator=gen) * 60 * value_scales[n // BLOCK % len(value_scales)]
            cache.tail[s, 0, 1, :, :rest] = values.to(cache.dtype)
            cache.peak[s, 0, 1] = cache.tail[s, 0, 1, :, :rest].float().abs().amax((-1, -2))
    return cache


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("heads,kv_heads,dh", [(4, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("levels,value_scales", [
    ([-20, 5], [0.25, 2.0 ** -30]),              # large values under weights of e^-25: what counts is 2^-28 of them in scale
    ([5, -20], [2.0 ** -30, 0.25]),
    ([-30, -10, 10], [0.25, 2.0 ** -20, 2.0 ** -42]),
    ([10, -10, -30], [2.0 ** -42, 2.0 ** -20, 0.25]),
    ([3, 3, 3, 3, 3, 3, -40], [2.0 ** -40] * 6 + [0.25])])
@pytest.mark.parametrize("sizes,counts", [([700, 260], [700, 260]), ([3000, 900], [400, 300]), ([3000, 900], [1, 1])])
def test_large_value_scales_under_small_weights(cuda, dtype, heads, kv_heads, dh, levels, value_scales, sizes, counts):
    """Blocks count by weight times value, whatever the scales of blocks that hardly count or that a row does not see."""
    torch = cuda
    if dtype == "float16":                       # results in its range
        value_scales = [v * 2.0 ** 12 if v < 0.2 else v for v in value_scales]
    cache = levelled_cache(torch, sizes, kv_heads, dh, dtype, levels, value_scales, 1)
    q = torch.ones(sum(counts), heads * dh, device="cuda", dtype=getattr(torch, dtype))
    out = cache.attention(0, q, step(cache, sizes, counts), scale=1 / dh)
    check(torch, cache, 0, q, out, sizes, counts, 1 / dh)


@pytest.mark.parametrize("scale", [0.0, 2.0 ** -126, 2.0 ** -60, 2.0 ** -30, 2.0 ** 60, 2.0 ** 100])
@pytest.mark.parametrize("counts", [[200], [500], [1]])
def test_value_scales_of_any_size(cuda, scale, counts):
    """All values zero, tiny or huge, and blocks of ordinary ones among them."""
    torch = cuda
    for mixed in (False, True):
        cache = random_cache(torch, [500], 1, 2, 64, "bfloat16", 3)
        pages = cache.table[0, :7].long()
        cache.scales[pages[::2] if mixed else pages, 0, 1] = max(scale, 2.0 ** -126)
        if scale == 0:
            cache.codes[pages[::2] if mixed else pages, 0, 1] = 0
        if not mixed:
            cache.tail[0, 0, 1, :, :52] *= 0.0 if scale == 0 else scale
            cache.peak[0, 0, 1] = cache.tail[0, 0, 1, :, :52].float().abs().amax((-1, -2))
        q = query(torch, counts[0], 32 * 64, "bfloat16", 3)
        out = cache.attention(0, q, step(cache, [500], counts))
        if scale == 0 and not mixed:
            assert not out.any()
        check(torch, cache, 0, q, out, [500], counts, 0.125)


@pytest.mark.parametrize("dtype,q_dtype", [("bfloat16", "float32"), ("float16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("heads,kv_heads,dh", [(96, 6, 64), (96, 6, 128)])
@pytest.mark.parametrize("pairs,count", [(1, 1), (20, 1), (200, 1), (1, 9), (1, 63), (4, 50), (10, 33), (16, 63), (40, 60)])
def test_weights_and_queries_keep_22_bits(cuda, dtype, q_dtype, heads, kv_heads, dh, pairs, count):
    """Pairs of blocks whose contributions cancel, so that neither the result's rounding nor an average hides what is lost: the
    queries lie between two FP16 numbers, the weights anywhere. (The tokens behind them have values of zero.)"""
    torch = cuda
    size = 128 * pairs + count
    cache = random_cache(torch, [size], 1, kv_heads, dh, dtype, pairs + count)
    gen = torch.Generator().manual_seed(pairs)
    cache.codes[:, :, 0] = 64
    cache.codes[:, :, 1] = 100
    cache.tail[0, 0, 1, :, :count] = 0
    cache.peak[0, 0, 1] = 0
    cache.tail[0, 0, 0, :, :count] = 0.125
    cache.peak[0, 0, 0] = 0.125
    level = 1.0 + 2.0 ** -12 if q_dtype == "float32" else 1.0
    q = torch.full((count, heads * dh), level, device="cuda", dtype=getattr(torch, q_dtype))
    keys = torch.rand(2 * pairs, kv_heads, generator=gen).float() * 0.5 / 64              # a block's keys score 64 times that
    values = torch.rand(2 * pairs, kv_heads, generator=gen).float() * 0.5 + 0.5
    scores = keys.double() * 64 * level
    values[1::2] = (values[::2].double() * torch.exp(scores[::2] - scores[1::2]) * 100 / 64).float()
    pages = cache.table[0, :2 * pairs].long()
    cache.scales[pages, 0, 0] = keys.cuda()
    cache.scales[pages, 0, 1] = values.cuda()
    cache.codes[pages[1::2], 0, 1] = -64                                        # (as large a product as 100, by another weight)
    out = cache.attention(0, q, step(cache, [size], [count]), scale=1 / dh)
    want = exact(torch, cache, 0, q, [size], [count], 1 / dh)
    assert (want[0].abs() <= 2.0 ** -20 * want[1]).all()                        # they do cancel
    check(torch, cache, 0, q, out, [size], [count], 1 / dh)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,dh,count", [(2, 2, 64, 1), (4, 1, 128, 1), (16, 1, 64, 1), (4, 1, 64, 3), (32, 1, 64, 40)])
@pytest.mark.parametrize("bits", [18.3, 23.7, 24.4, 25.1])
def test_many_small_weights_behind_a_dominant_one(cuda, dtype, heads, kv_heads, dh, count, bits):
    """One key of weight 1 with values of zero, then tens of thousands of keys of nearly equal weights 2^-bits whose values do not
    average out: they are the result."""
    torch = cuda
    size = 64 * 1100 + count
    cache = random_cache(torch, [size], 1, kv_heads, dh, dtype, 2)
    pages = cache.table[0, :1100].long()
    gap = bits * math.log(2)
    keys = torch.zeros(kv_heads, BLOCK, dh, device="cuda", dtype=torch.int8)
    keys[:, 0] = 127
    cache.codes[:, 0, 0] = 0
    cache.codes[pages[0], 0, 0] = keys.reshape(kv_heads, -1)
    cache.scales[:, :, 0] = gap / 127
    values = torch.randint(40, 128, (1100, kv_heads, dh, BLOCK), device="cuda", dtype=torch.int8, generator=torch.Generator("cuda").manual_seed(3))
    values[0] = 0
    cache.codes[pages, 0, 1] = values.reshape(1100, kv_heads, -1)
    cache.scales[:, :, 1] = 2.0 ** 7
    cache.tail[0, :, :, :, :count] = 0
    cache.peak[0] = 0
    q = torch.ones(count, heads * dh, device="cuda", dtype=getattr(torch, dtype))
    out = cache.attention(0, q, step(cache, [size], [count]), scale=1 / dh)
    check(torch, cache, 0, q, out, [size], [count], 1 / dh)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,dh", [(4, 2, 64), (32, 2, 128)])
@pytest.mark.parametrize("count", [1, 4, 50])
def test_small_values_next_to_large_ones_in_the_tail(cuda, dtype, heads, kv_heads, dh, count):
    """Every dimension has its own order of magnitude: values of one token, seen alone, come back as they are, and keys that only
    score by their small dimensions decide the weights."""
    torch = cuda
    cache = random_cache(torch, [count], 1, kv_heads, dh, dtype, count)
    size = 2.0 ** torch.linspace(0, -16, dh, device="cuda")                     # (FP16: normal numbers of eleven bits)
    cache.tail[0, 0, :, :, :count] = ((1 + torch.rand(2, kv_heads, count, dh, device="cuda", generator=torch.Generator("cuda").manual_seed(5))) * size * 8).to(cache.dtype)
    cache.peak[0, 0] = cache.tail[0, 0, :, :, :count].float().abs().amax((-1, -2))
    q = torch.zeros(count, heads, dh, device="cuda")
    q[..., dh // 2:] = 1 / (8 * size[dh // 2:])
    q = q.reshape(count, -1)
    out = cache.attention(0, q, step(cache, [count], [count]))
    first = cache.tail[0, 0, 1, :, 0].repeat_interleave(heads // kv_heads, 0).reshape(-1)
    assert torch.equal(out[0], first)
    check(torch, cache, 0, q, out, [count], [count], dh ** -0.5)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,dh", [(4, 2, 64), (32, 2, 128)])
@pytest.mark.parametrize("count,few", [(5, 1), (60, 1), (4, 4), (50, 50), (300, 300)])
def test_small_values_next_to_large_ones_in_a_row_of_queries(cuda, dtype, heads, kv_heads, dh, count, few):
    """One dimension of the queries is 2^15 times the others that score; those decide the weights."""
    torch = cuda
    gen = torch.Generator("cuda").manual_seed(count)
    rest = count % BLOCK
    cache = random_cache(torch, [count], 1, kv_heads, dh, dtype, count)
    signs = lambda *shape: torch.randint(0, 2, shape, device="cuda", generator=gen) * 2 - 1  # noqa: E731
    cache.codes[:, 0] = 0
    for b in range(count // BLOCK):
        page = int(cache.table[0, b])
        keys = torch.zeros(kv_heads, BLOCK, dh, device="cuda")
        keys[..., -8:] = signs(kv_heads, BLOCK, 8) * 64
        cache.codes[page, 0, 0] = keys.reshape(kv_heads, -1).to(torch.int8)
        cache.codes[page, 0, 1] = (signs(kv_heads, dh, BLOCK) * 64).reshape(kv_heads, -1).to(torch.int8)
        cache.scales[page, 0, 0], cache.scales[page, 0, 1] = 1 / 16, 1 / 64
    cache.tail[0, 0, :, :, :rest] = 0
    cache.tail[0, 0, 0, :, :rest, -8:] = signs(kv_heads, rest, 8).to(cache.dtype) * 4
    cache.tail[0, 0, 1, :, :rest] = signs(kv_heads, rest, dh).to(cache.dtype)
    cache.peak[0, 0, 0], cache.peak[0, 0, 1] = 4, 1
    q = torch.zeros(few, heads, dh, device="cuda")
    q[..., 0] = 2.0 ** 10
    q[..., -8:] = (1 + torch.rand(few, heads, 8, device="cuda", generator=gen)) * 2.0 ** -5
    q = q.reshape(few, -1)
    out = cache.attention(0, q, step(cache, [count], [few]), scale=1.0)
    check(torch, cache, 0, q, out, [count], [few], 1.0)


@pytest.mark.parametrize("count", [11, 31, 43, 54, 85, 86, 97, 171])
@pytest.mark.parametrize("context", [0, 6000])
def test_rows_that_fill_no_warp(cuda, count, context):
    """Three rows per token: lanes without a row next to lanes with one, in one part of the keys and in many."""
    torch = cuda
    sizes, counts = [context + count, context // 2 + 200], [count, 190]
    for dh in (64, 128):
        cache = random_cache(torch, sizes, 1, 2, dh, "float16", count)
        q = query(torch, sum(counts), 6 * dh, "float16", count)
        out = cache.attention(0, q, step(cache, sizes, counts))
        check(torch, cache, 0, q, out, sizes, counts, dh ** -0.5)
