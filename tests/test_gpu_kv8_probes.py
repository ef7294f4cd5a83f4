"""Whether every page and every key of a context reaches its rows, exactly once, at any length: probes whose answer is one page's or
one key's contribution, where a bound on sums of random values would let lost pages pass.

A page probe has queries of zero, so all weights are equal, and values of zero but for one page, whose values are 100: a row that
sees n keys, m of them in the page, answers 100 m / n up to the rounding of the result and of FP32 sums (2^-18). A key probe has one
key whose score lies 60 above all others: the answer is that key's values, to e^-60 and the same roundings."""

import pytest

from mylocal_llm_b200 import _lib
from test_gpu_kv8_attention import random_cache, step

pytestmark = pytest.mark.gpu

BLOCK = 64


@pytest.fixture(autouse=True)
def healthy(cuda):
    _lib.clear_device_status()
    yield
    cuda.cuda.synchronize()
    assert _lib.device_status() == 0


CASES = [                                            # heads, kv_heads, head_dim, type, tokens held, new tokens, bound on the keys
    (8, 1, 128, "bfloat16", [70001], [1], None),     # one sequence in many parts
    (4, 4, 64, "float16", [4097], [1], None),
    (8, 2, 128, "float16", [11771, 127, 64, 5000, 63], [1] * 5, None),
    (8, 2, 64, "bfloat16", [11771, 127, 64, 5000, 63], [5, 5, 5, 0, 5], None),
    (32, 2, 64, "float16", [777, 100, 1300], [1] * 3, None),         # whole sequences per CTA
    (32, 2, 64, "float16", [777, 100, 1300], [1] * 3, 1300),
    (8, 8, 64, "bfloat16", [60 + 7 * i for i in range(40)], [1] * 40, 340),
    (8, 8, 64, "bfloat16", [60 + i * 37 % 70 for i in range(300)], [1] * 300, None),         # sequences of a warp each
    (4, 1, 128, "float16", [60000, 40], [20, 3], None),
    (16, 1, 64, "float16", [9000], [63], None),      # chunks whose keys are divided
    (4, 1, 128, "bfloat16", [4001, 900], [300, 64], None),
    (6, 2, 64, "bfloat16", [1000, 640, 129], [1000, 640, 129], None)]            # whole prompts


def ids(case):
    heads, kv_heads, dh, dtype, sizes, counts, _ = case
    return f"{heads}-{kv_heads}-{dh}-{dtype}-{len(sizes)}x{max(sizes)}-{max(counts)}"


def chosen(pages):
    """All pages of a short context; of a long one the first and last and every few, in steps that meet every remainder."""
    return list(range(pages)) if pages <= 64 else sorted({0, 1, 2, 3, pages - 3, pages - 2, pages - 1, *range(0, pages, max(1, pages // 97) | 1)})


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_every_page_counts_once(cuda, case):
    torch = cuda
    heads, kv_heads, dh, dtype, sizes, counts, max_keys = case
    cache = random_cache(torch, sizes, 1, kv_heads, dh, dtype, 1)
    cache.codes[:, :, 1] = 0
    cache.tail[:, :, 1] = torch.where(torch.isnan(cache.tail[:, :, 1]), cache.tail[:, :, 1], torch.zeros_like(cache.tail[:, :, 1]))
    held = cache.table[cache.table >= 0].long()
    cache.scales[held, 0, 1] = 1.0
    q = torch.zeros(sum(counts), heads * dh, device="cuda")
    batch = step(cache, sizes, counts, max_keys=max_keys)
    eps = torch.finfo(cache.dtype).eps
    row = 0
    worst = torch.zeros((), device="cuda", dtype=torch.float64)
    for s, (total, n) in enumerate(zip(sizes, counts)):
        seen = torch.arange(total - n + 1, total + 1, device="cuda", dtype=torch.float64)          # keys that the rows see
        full = total // BLOCK
        for b in chosen(full) + ([full] if total % BLOCK else []):
            if b < full:
                cache.codes[int(cache.table[s, b]), 0, 1] = 100
            else:
                cache.tail[s, 0, 1, :, :total % BLOCK] = 100
                cache.peak[s, 0, 1] = 100
            out = cache.attention(0, q, batch).double()
            if b < full:
                cache.codes[int(cache.table[s, b]), 0, 1] = 0
            else:
                cache.tail[s, 0, 1, :, :total % BLOCK] = 0
            want = torch.zeros(sum(counts), device="cuda", dtype=torch.float64)
            want[row:row + n] = 100 * (seen - b * BLOCK).clamp(0, BLOCK) / seen
            bound = (eps / 2 * 1.01 + 2.0 ** -18) * want + torch.finfo(cache.dtype).tiny * eps
            worst = torch.maximum(worst, ((out - want[:, None]).abs() / bound[:, None]).max())
        row += n
    assert float(worst) <= 1, f"{float(worst)} of the bound"


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_the_key_that_dominates_is_the_answer(cuda, case):
    torch = cuda
    heads, kv_heads, dh, dtype, sizes, counts, max_keys = case
    cache = random_cache(torch, sizes, 1, kv_heads, dh, dtype, 2)
    cache.codes[:, :, 0] = 0
    cache.tail[:, :, 0] = torch.where(torch.isnan(cache.tail[:, :, 0]), cache.tail[:, :, 0], torch.zeros_like(cache.tail[:, :, 0]))
    held = cache.table[cache.table >= 0].long()
    cache.scales[held, 0, 0] = 60 / 100
    q = torch.zeros(sum(counts), heads, dh, device="cuda")
    q[..., dh - 3] = 1.0
    q = q.reshape(sum(counts), -1)
    batch = step(cache, sizes, counts, max_keys=max_keys)
    eps = torch.finfo(cache.dtype).eps
    gen = torch.Generator().manual_seed(3)
    row = 0
    worst = torch.zeros((), device="cuda", dtype=torch.float64)
    for s, (total, n) in enumerate(zip(sizes, counts)):
        full, first = total // BLOCK, total - n                                   # every new token sees the keys up to `first`
        if not n:
            continue
        blocks = [b for b in chosen(full) if b * BLOCK <= first] + ([full] if full * BLOCK <= first and total % BLOCK else [])
        for b in blocks:
            key = int(torch.randint(0, min(BLOCK, first + 1 - b * BLOCK), (1,), generator=gen))
            if b < full:
                page = int(cache.table[s, b])
                cache.codes[page, 0, 0].reshape(kv_heads, BLOCK, dh)[:, key, dh - 3] = 100
                want = cache.codes[page, 0, 1].reshape(kv_heads, dh, BLOCK)[..., key].double() * cache.scales[page, 0, 1].double()[:, None]
            else:
                cache.tail[s, 0, 0, :, key, dh - 3] = 60
                cache.peak[s, 0, 0] = 60
                want = cache.tail[s, 0, 1, :, key].double()
            out = cache.attention(0, q, batch, scale=1.0)[row:row + n].double().reshape(n, kv_heads, heads // kv_heads, dh)
            if b < full:
                cache.codes[page, 0, 0] = 0
            else:
                cache.tail[s, 0, 0, :, :total % BLOCK] = 0
            want = want[None, :, None]
            bound = (eps / 2 * 1.01 + 2.0 ** -18) * want.abs() + torch.finfo(cache.dtype).tiny * eps + 1e-20
            worst = torch.maximum(worst, ((out - want).abs() / bound).max())
        row += n
    assert float(worst) <= 1, f"{float(worst)} of the bound"
