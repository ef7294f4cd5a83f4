"""Attention over the paged 8-bit cache against 64-bit arithmetic on the cache's own content.

Bound of an output element, with S the sum of |q_i k_i| * scale over a key's dimensions, p the exact softmax weights and A = sum
of p |v|: a query is rounded to FP16 (relative 2^-11, or 2^-24 of the row's largest magnitude below FP16's normal numbers), so
a score is off by at most d = 2^-11 max S + 2^-24 max|q| scale max sum |k| + 2^-20 (1 + max S) for the FP32 sums, rotation and
exponentials; a weight by a factor within exp(+-2 d); weights pass the tensor cores as FP16 (2^-11, or 2^-24 of the largest one,
over at most `keys` of them); the result is rounded to the cache's type (half a step). Tails pass as FP16 relative to their
power-of-two scale: 2^-24 of the largest magnitude of the block, already counted for K in the second term, and added for V."""

import math

import pytest

from mylocal_llm_b200 import PagedKV8Cache, _lib

pytestmark = pytest.mark.gpu

BLOCK = 64


@pytest.fixture(autouse=True)
def healthy(cuda):
    _lib.clear_device_status()
    yield
    cuda.cuda.synchronize()
    assert _lib.device_status() == 0


def rope_tables(torch, rows, dh):
    inv = 10000.0 ** (-torch.arange(dh // 2, dtype=torch.float64, device="cuda") * 2.0 / dh)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def random_cache(torch, sizes, layers, kv_heads, dh, dtype, seed, max_length=None, spare=3):
    """A cache that holds ``sizes`` tokens, pages in random order, everything that must not be read poisoned with NaN."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pages = sum(n // BLOCK for n in sizes) + spare
    blocks = max(1, -(-(max_length or max(max(sizes), 1)) // BLOCK))
    codes = torch.randint(-127, 128, (pages, layers, 2, kv_heads, BLOCK * dh), dtype=torch.int8, device="cuda", generator=gen)
    scales = torch.rand((pages, layers, 2, kv_heads), device="cuda", generator=gen) * 0.02 + 0.001
    tail = torch.randn((len(sizes), layers, 2, kv_heads, BLOCK, dh), device="cuda", generator=gen).to(getattr(torch, dtype))
    peak = torch.zeros((len(sizes), layers, 2, kv_heads), device="cuda")
    table = torch.full((len(sizes), blocks), -1, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int(), 0
    refs = torch.zeros(pages, dtype=torch.int32)
    for s, n in enumerate(sizes):
        table[s, :n // BLOCK] = order[at:at + n // BLOCK]
        refs[order[at:at + n // BLOCK].long()] = 1
        at += n // BLOCK
        tail[s, :, :, :, n % BLOCK:] = math.nan
        if n % BLOCK:
            peak[s] = tail[s, :, :, :, :n % BLOCK].float().abs().amax((-1, -2))
        else:
            peak[s] = math.nan
    scales[order[at:].long().cuda()] = math.nan
    lengths = torch.tensor(sizes, dtype=torch.int32)
    return PagedKV8Cache.from_tensors(codes, scales, tail, peak, table.cuda(), lengths.cuda(), refs.cuda(), max_length)


def step(cache, sizes, counts, max_keys=None, slots=None):
    """A batch whose new tokens are the last of each sequence, all of them in the cache already."""
    slots = list(range(len(sizes))) if slots is None else slots
    batch = cache.batch(slots, counts, max_keys=max_keys)
    batch.starts.copy_(type(cache.lengths).new_tensor(cache.lengths, [sizes[s] - n for s, n in zip(slots, counts)]))
    return batch


def check(torch, cache, layer, q, out, sizes, counts, rope=None, scale=None, slots=None):
    dh, kv_heads = cache.head_dim, cache.kv_heads
    heads = q.shape[1] // dh
    scale = dh ** -0.5 if scale is None else scale
    eps = torch.finfo(out.dtype).eps
    row = 0
    for s, n in zip(range(len(sizes)) if slots is None else slots, counts):
        if not n:
            continue
        total = sizes[s]
        pages, rest = cache.table[s, :total // BLOCK].long(), total % BLOCK
        codes, sc = cache.codes[pages, layer].double(), cache.scales[pages, layer].double()
        tail = cache.tail[s, layer, :, :, :rest].double()
        k = torch.cat([(codes[:, 0].reshape(-1, kv_heads, BLOCK, dh) * sc[:, 0, :, None, None]).transpose(0, 1).reshape(kv_heads, -1, dh), tail[0]], 1)
        v = torch.cat([(codes[:, 1].reshape(-1, kv_heads, dh, BLOCK) * sc[:, 1, :, None, None]).permute(1, 0, 3, 2).reshape(kv_heads, -1, dh), tail[1]], 1)
        x = q[row:row + n].double().reshape(n, heads, dh)
        if rope is not None:
            c, si = (t[total - n:total, None].double() for t in rope)
            x = torch.cat([x[..., :dh // 2] * c - x[..., dh // 2:] * si, x[..., :dh // 2] * si + x[..., dh // 2:] * c], -1)
        x = x.reshape(n, kv_heads, heads // kv_heads, dh).permute(1, 2, 0, 3)                       # [kv, group, n, dh]
        hidden = torch.arange(total, device="cuda") > (torch.arange(n, device="cuda") + total - n)[:, None]
        k, v = k[:, None], v[:, None]
        p = torch.softmax((x @ k.transpose(-1, -2) * scale).masked_fill(hidden, -math.inf), -1)
        want = p @ v
        biggest = (x.abs() @ k.abs().transpose(-1, -2) * abs(scale)).amax(-1, keepdim=True)
        d = 2.0 ** -11 * biggest + 2.0 ** -24 * x.abs().amax(-1, keepdim=True) * abs(scale) * k.abs().sum(-1).amax() + 2.0 ** -20 * (1 + biggest)
        a = p @ v.abs()
        bound = (torch.exp(2 * d) - 1 + 2.0 ** -11 + 2.0 ** -18) * a + (2.0 ** -24 * total + 2.0 ** -23) * v.abs().amax() + eps / 2 * want.abs() * 1.01
        got = out[row:row + n].double().reshape(n, kv_heads, heads // kv_heads, dh).permute(1, 2, 0, 3)
        off = (got - want).abs()
        assert torch.isfinite(got).all()
        assert (off <= bound).all(), f"sequence {s}: {float((off / bound).max())} of the bound"
        row += n
    assert row == out.shape[0]


def query(torch, rows, width, dtype, seed, extra=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((rows, width + extra), device="cuda", generator=gen).to(getattr(torch, dtype))[:, :width]


@pytest.mark.parametrize("heads,kv_heads,dh", [(32, 32, 64), (8, 2, 128), (5, 1, 64), (40, 2, 128), (16, 1, 64), (17, 1, 128), (6, 3, 64)])
@pytest.mark.parametrize("dtype,q_dtype", [("bfloat16", "float32"), ("float16", "float16")])
def test_single_tokens_over_ragged_contexts(cuda, heads, kv_heads, dh, dtype, q_dtype):
    torch = cuda
    sizes = [1, 2, 63, 64, 65, 127, 128, 129, 1000, 640, 3333]
    cache = random_cache(torch, sizes, 2, kv_heads, dh, dtype, heads + dh)
    q = query(torch, len(sizes), heads * dh, q_dtype, 1, extra=8)
    batch = step(cache, sizes, [1] * len(sizes))
    rope = rope_tables(torch, cache.max_length, dh)
    check(torch, cache, 1, q, cache.attention(1, q, batch, rope=rope), sizes, [1] * len(sizes), rope)
    check(torch, cache, 0, q, cache.attention(0, q, batch, scale=0.2), sizes, [1] * len(sizes), None, 0.2)


@pytest.mark.parametrize("size", [1, 31, 64, 4096, 4097, 70001])
@pytest.mark.parametrize("heads,kv_heads,dh", [(4, 4, 64), (8, 1, 128)])
def test_one_long_sequence(cuda, size, heads, kv_heads, dh):
    torch = cuda
    cache = random_cache(torch, [size], 1, kv_heads, dh, "bfloat16", size)
    q = query(torch, 1, heads * dh, "bfloat16", size)
    check(torch, cache, 0, q, cache.attention(0, q, step(cache, [size], [1])), [size], [1])


def test_many_short_sequences(cuda):
    torch = cuda
    sizes = [1 + (i * 37) % 300 for i in range(700)]
    cache = random_cache(torch, sizes, 1, 2, 64, "bfloat16", 9)
    q = query(torch, 700, 4 * 64, "float32", 9)
    out = cache.attention(0, q, step(cache, sizes, [1] * 700))
    check(torch, cache, 0, q, out, sizes, [1] * 700)
    # the same sequences in another order, a few of them, with a tighter bound on their lengths
    slots = [699, 3, 250, 17]
    some = step(cache, sizes, [1] * 4, max_keys=300, slots=slots)
    alone = cache.attention(0, q[slots].contiguous(), some)
    check(torch, cache, 0, q[slots], alone, sizes, [1] * 4, slots=slots)


@pytest.mark.parametrize("heads,kv_heads,dh", [(4, 4, 64), (8, 2, 128), (3, 1, 64), (7, 1, 128), (24, 1, 64)])
@pytest.mark.parametrize("dtype,q_dtype", [("bfloat16", "float32"), ("float16", "bfloat16")])
@pytest.mark.parametrize("sizes,counts", [
    ([1, 2, 64, 65, 300, 129], [1, 2, 64, 65, 300, 129]),                # whole prompts
    ([200, 513, 70, 1000, 640], [7, 0, 70, 129, 64]),                    # chunks behind a context, one idle, one from the start
    ([1999, 5], [2, 3])])                                                # a few tokens (verification of a draft)
def test_several_tokens_per_sequence(cuda, heads, kv_heads, dh, dtype, q_dtype, sizes, counts):
    torch = cuda
    cache = random_cache(torch, sizes, 2, kv_heads, dh, dtype, heads)
    q = query(torch, sum(counts), heads * dh, q_dtype, 2, extra=4)
    rope = rope_tables(torch, cache.max_length, dh)
    batch = step(cache, sizes, counts)
    check(torch, cache, 1, q, cache.attention(1, q, batch, rope=rope), sizes, counts, rope)


def test_a_long_prompt(cuda):
    torch = cuda
    sizes, counts = [2500, 3100], [2500, 700]
    cache = random_cache(torch, sizes, 1, 2, 128, "bfloat16", 4)
    q = query(torch, 3200, 8 * 128, "bfloat16", 4)
    check(torch, cache, 0, q, cache.attention(0, q, step(cache, sizes, counts)), sizes, counts)


@pytest.mark.parametrize("counts", [[1, 1], [40, 70]])
def test_rows_at_odd_addresses(cuda, counts):
    """Rows of queries that start at any element, and an odd stride between them."""
    torch = cuda
    sizes = [200, 70]
    cache = random_cache(torch, sizes, 1, 2, 64, "bfloat16", 6)
    for dtype in ("float32", "bfloat16"):
        wide = query(torch, sum(counts), 4 * 64 + 3, dtype, 6)
        q = wide[:, 1:257]
        rope = rope_tables(torch, cache.max_length, 64)
        check(torch, cache, 0, q, cache.attention(0, q, step(cache, sizes, counts), rope=rope), sizes, counts, rope)


@pytest.mark.parametrize("factor", [1e-30, 3e4, 1e15])
@pytest.mark.parametrize("counts", [[1, 1], [64, 100]])
def test_queries_and_values_far_from_one(cuda, factor, counts):
    """Queries beyond FP16's range (their row is scaled by a power of two) and values whose scales differ by orders of magnitude
    between the blocks."""
    torch = cuda
    sizes = [300, 140]
    cache = random_cache(torch, sizes, 1, 2, 64, "bfloat16", 8)
    cache.scales[:, :, 0] /= factor                                   # keys so that the scores stay moderate
    cache.tail[:, :, 0] /= factor
    cache.peak[:, :, 0] /= factor
    cache.scales[::2, :, 1] *= 1e-12
    q = query(torch, sum(counts), 4 * 64, "float32", 8) * factor
    check(torch, cache, 0, q, cache.attention(0, q, step(cache, sizes, counts)), sizes, counts)


@pytest.mark.parametrize("counts", [[1, 1, 1], [130, 3, 64]])
def test_scores_of_large_magnitude(cuda, counts):
    """Softmax weights of exactly one key: the running maximum moves through blocks of scores in the thousands."""
    torch = cuda
    sizes = [400, 100, 64]
    cache = random_cache(torch, sizes, 1, 1, 64, "float16", 10)
    q = torch.ones(sum(counts), 2 * 64, device="cuda")
    cache.codes[:, :, 0] = 1
    cache.scales[:, :, 0] = torch.arange(cache.pages, device="cuda")[:, None, None].float() * 10 + 1
    cache.tail[:, :, 0] = torch.where(torch.isnan(cache.tail[:, :, 0]), cache.tail[:, :, 0], torch.ones_like(cache.tail[:, :, 0]))
    cache.peak[:, :, 0] = 1
    check(torch, cache, 0, q, cache.attention(0, q, step(cache, sizes, counts)), sizes, counts)


@pytest.mark.parametrize("counts", [[1, 1], [100, 30]])
def test_what_is_not_finite_shows_where_it_is_seen(cuda, counts):
    torch = cuda
    sizes = [200, 90]
    cache = random_cache(torch, sizes, 1, 2, 64, "bfloat16", 11)
    q = query(torch, sum(counts), 4 * 64, "float32", 11)
    clean = cache.attention(0, q, step(cache, sizes, counts)).clone()
    page = int(cache.table[0, 1])                                     # tokens 64..127 of the first sequence, head 1, values
    cache.scales[page, 0, 1, 1] = math.nan
    out = cache.attention(0, q, step(cache, sizes, counts)).reshape(sum(counts), 4, 64)
    sees = torch.zeros(sum(counts), dtype=torch.bool, device="cuda")
    sees[:counts[0]] = torch.arange(200 - counts[0], 200, device="cuda") >= 64
    assert torch.isnan(out[sees][:, 2:]).all() and torch.isfinite(out[:, :2]).all() and torch.isfinite(out[~sees]).all()
    cache.scales[page, 0, 1, 1] = 0.01
    cache.scales[int(cache.table[0, 1]), 0, 1, 1] = 0.01
    q[0, 70] = math.inf                                               # head 1 of the first row
    out = cache.attention(0, q, step(cache, sizes, counts)).reshape(sum(counts), 4, 64)
    assert torch.isnan(out[0, 1]).all() and torch.isfinite(out[1:]).all() and torch.isfinite(out[0, [0, 2, 3]]).all()
    assert torch.equal(out[1:, :2], clean.reshape(sum(counts), 4, 64)[1:, :2])


@pytest.mark.parametrize("part", [0, 1])
@pytest.mark.parametrize("where", ["page", "tail"])
@pytest.mark.parametrize("count", [4, 60])
def test_a_block_that_is_not_finite_leaves_the_rows_before_it_alone(cuda, part, where, count):
    """New tokens on both sides of a block's border: only those behind it see the block."""
    torch = cuda
    size = 130 if where == "tail" else 200
    border = 128
    cache = random_cache(torch, [size], 1, 1, 64, "bfloat16", 13)
    counts = [size - border + count // 2]
    q = query(torch, counts[0], 3 * 64, "float32", 13)
    clean = cache.attention(0, q, step(cache, [size], counts)).clone()
    if where == "tail":
        cache.tail[0, 0, part, 0, 1, 7] = math.inf
        cache.peak[0, 0, part, 0] = math.inf
    else:
        cache.scales[int(cache.table[0, 2]), 0, part, 0] = math.nan
    out = cache.attention(0, q, step(cache, [size], counts))
    assert torch.equal(out[:count // 2], clean[:count // 2]) and torch.isnan(out[count // 2:]).all()


@pytest.mark.parametrize("counts", [[1], [90]])
@pytest.mark.parametrize("entry", [-1, 10 ** 6])
def test_a_page_that_the_table_lacks_shows(cuda, counts, entry):
    """A table entry outside the pool: nothing is read beyond it, and the rows that would see the block are NaN."""
    torch = cuda
    cache = random_cache(torch, [200], 1, 2, 64, "bfloat16", 14)
    q = query(torch, counts[0], 4 * 64, "float32", 14)
    clean = cache.attention(0, q, step(cache, [200], counts)).clone()
    cache.table[0, 2] = entry                                         # tokens 128..191
    out = cache.attention(0, q, step(cache, [200], counts))
    sees = torch.arange(200 - counts[0], 200, device="cuda") >= 128
    assert torch.isnan(out[sees]).all() and torch.equal(out[~sees], clean[~sees])


def test_a_few_tokens_over_a_very_long_context(cuda):
    """Few rows and many keys: the keys are divided among many CTAs."""
    torch = cuda
    sizes, counts = [60000, 40], [20, 3]
    cache = random_cache(torch, sizes, 1, 1, 128, "float16", 15)
    q = query(torch, 23, 4 * 128, "float16", 15)
    check(torch, cache, 0, q, cache.attention(0, q, step(cache, sizes, counts)), sizes, counts)


def test_more_sequences_than_one_launch_takes(cuda):
    torch = cuda
    sizes = [1 + (i * 53) % 200 + (4000 if i % 700 == 5 else 0) for i in range(1500)]
    cache = random_cache(torch, sizes, 1, 1, 64, "bfloat16", 16)
    q = query(torch, 1500, 2 * 64, "bfloat16", 16)
    counts = [0 if i % 11 == 3 else 1 for i in range(1500)]
    q = q[:sum(counts)]
    check(torch, cache, 0, q, cache.attention(0, q, step(cache, sizes, counts)), sizes, counts)


def test_offsets_beyond_32_bits(cuda):
    """A pool of more than 2^32 bytes whose last pages are the ones in use."""
    torch = cuda
    layers, kv_heads, dh = 16, 32, 128
    pages = 2 ** 32 // (layers * 2 * kv_heads * 64 * dh) + 24
    sizes = [64 * 16 + 5, 64 * 3]
    cache = PagedKV8Cache(layers, kv_heads, dh, pages=pages, sequences=2, max_length=2048)
    gen = torch.Generator(device="cuda").manual_seed(0)
    used = list(range(pages - 19, pages))
    for p in used:
        cache.codes[p] = torch.randint(-127, 128, cache.codes[p].shape, dtype=torch.int8, device="cuda", generator=gen)
        cache.scales[p] = 0.01
    cache.table[0, :16] = torch.tensor(used[:16], dtype=torch.int32)
    cache.table[1, :3] = torch.tensor(used[16:], dtype=torch.int32)
    cache.lengths.copy_(torch.tensor(sizes))
    cache.tail[0, :, :, :, :5] = 0.5
    cache.peak[0] = 0.5
    for counts in ([1, 1], [30, 64]):
        q = query(torch, sum(counts), kv_heads * dh, "bfloat16", 12)
        check(torch, cache, 15, q, cache.attention(15, q, step(cache, sizes, counts)), sizes, counts)


def test_a_step_captured_and_replayed_and_on_another_stream(cuda):
    """Decode steps replayed from one graph equal the same steps called directly on another stream, bit for bit."""
    torch = cuda
    heads, kv_heads, dh, layers = 8, 2, 64, 2
    sizes = [60, 127, 3]

    def steps(use_graph):
        cache = random_cache(torch, sizes, layers, kv_heads, dh, "bfloat16", 21, max_length=300, spare=9)
        cache.tail.nan_to_num_(0.0)
        cache.peak.nan_to_num_(0.0)
        rope = rope_tables(torch, 300, dh)
        batch = cache.batch([0, 1, 2], [1, 1, 1])
        gen = torch.Generator(device="cuda").manual_seed(22)
        inputs = torch.randn(10, 3, (heads + 2 * kv_heads) * dh, device="cuda", generator=gen)
        x = inputs[0].clone()
        qd, kd = heads * dh, kv_heads * dh

        def one():
            cache.extend(batch)
            outs = []
            for layer in range(layers):
                cache.append(layer, x[:, qd:qd + kd], x[:, qd + kd:], batch, rope=rope)
                outs.append(cache.attention(layer, x[:, :qd], batch, rope=rope))
            return outs

        got = []
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got.append([o.clone() for o in one()])
            if use_graph:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    outs = one()
            for i in range(1, 10):
                x.copy_(inputs[i])
                if use_graph:
                    graph.replay()
                else:
                    outs = one()
                got.append([o.clone() for o in outs])
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        assert cache.read_lengths() == [70, 137, 13]
        return got, cache

    direct, first = steps(False)
    replayed, second = steps(True)
    assert all(torch.equal(a, b) for u, w in zip(direct, replayed) for a, b in zip(u, w))
    assert torch.equal(first.codes, second.codes) and torch.equal(first.tail, second.tail) and torch.equal(first.table, second.table)


def test_two_steps_at_once_on_two_caches(cuda):
    """Calls on two streams share nothing."""
    torch = cuda
    sizes = [5000, 77]
    caches = [random_cache(torch, sizes, 1, 2, 128, "bfloat16", 30 + i) for i in range(2)]
    q = query(torch, 2, 8 * 128, "bfloat16", 30)
    want = [c.attention(0, q, step(c, sizes, [1, 1])).clone() for c in caches]
    batches = [step(c, sizes, [1, 1]) for c in caches]
    streams = [torch.cuda.Stream() for _ in caches]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for c, b, s in zip(caches, batches, streams):
            with torch.cuda.stream(s):
                got.append(c.attention(0, q, b))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("heads,kv_heads,dh", [(8, 2, 128), (8, 2, 64), (3, 3, 128), (15, 1, 64)])
@pytest.mark.parametrize("sizes,counts", [
    ([8000, 8000, 5003, 7999], [8, 8, 3, 1]),                            # a few tokens each behind long contexts
    ([4001], [64]), ([4001], [300]), ([700], [17]),                      # chunks of one sequence, tails of 33 and 60 tokens
    ([11771, 127, 64, 5000, 63], [5, 5, 5, 0, 5]),                       # cut into many parts, some of them empty
    ([215], [3]), ([60] * 40, [7] * 40), ([1500] * 3, [33] * 3)])
def test_chunks_between_single_tokens_and_prompts(cuda, dtype, heads, kv_heads, dh, sizes, counts):
    """Sizes at which the kernels for few and for many rows meet, each with its ways to divide the work."""
    torch = cuda
    cache = random_cache(torch, sizes, 1, kv_heads, dh, dtype, heads + sum(counts))
    q = query(torch, sum(counts), heads * dh, dtype, 3)
    rope = rope_tables(torch, cache.max_length, dh)
    for max_keys in (None, max(sizes)):
        out = cache.attention(0, q, step(cache, sizes, counts, max_keys=max_keys), rope=rope)
        check(torch, cache, 0, q, out, sizes, counts, rope)
        assert torch.equal(out, cache.attention(0, q, step(cache, sizes, counts, max_keys=max_keys), rope=rope))


@pytest.mark.parametrize("rest", [1, 2, 15, 16, 17, 33, 63])
@pytest.mark.parametrize("heads,kv_heads,dh", [(2, 2, 64), (4, 1, 128), (16, 1, 64), (12, 1, 128)])
def test_tails_of_every_kind(cuda, rest, heads, kv_heads, dh):
    """Single tokens and a few, whose own keys are in the tail, over contexts of a tail alone and of pages and a tail."""
    torch = cuda
    sizes = [rest, 64 + rest, 640 + rest, 6400 + rest]
    for n in (1, min(rest, 6)):
        cache = random_cache(torch, sizes, 1, kv_heads, dh, "float16", rest)
        q = query(torch, n * len(sizes), heads * dh, "float32", rest)
        out = cache.attention(0, q, step(cache, sizes, [n] * len(sizes)))
        check(torch, cache, 0, q, out, sizes, [n] * len(sizes))


def test_a_batch_belongs_to_its_cache(cuda):
    torch = cuda
    cache = random_cache(torch, [100, 70], 1, 1, 64, "bfloat16", 0)
    other = random_cache(torch, [100], 1, 1, 64, "bfloat16", 0)
    q = query(torch, 1, 64, "bfloat16", 0)
    with pytest.raises(ValueError):
        other.attention(0, q, step(cache, [100, 70], [1], slots=[1]))
    out = torch.empty(65, dtype=torch.bfloat16, device="cuda")[1:].view(1, 64)
    with pytest.raises(ValueError):
        cache.attention(0, q, step(cache, [100, 70], [1], slots=[0]), out=out)              # not 16-byte aligned
