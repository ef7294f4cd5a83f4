"""Paged 8-bit key/value cache: what appending leaves in it and the page operations, against plain 64-bit computations.

Codes are whole numbers and have to be equal: keys and values are rounded to the cache's type first (the rotation in 64 bits,
rounded to FP32 and then to that type), scale = max |x| / 127 as an FP32 number, code = x / scale to the nearest integer."""

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
    _lib.clear_device_status()


def rope_tables(torch, rows, dh):
    inv = 10000.0 ** (-torch.arange(dh // 2, dtype=torch.float64, device="cuda") * 2.0 / dh)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def rotated(torch, x, cos, sin):
    """[tokens, heads, dh] by the tables' rows, in 64 bits."""
    half = x.shape[-1] // 2
    x0, x1, c, s = x[..., :half].double(), x[..., half:].double(), cos[:, None].double(), sin[:, None].double()
    return torch.cat([x0 * c - x1 * s, x0 * s + x1 * c], -1).float()


def content(torch, cache, slot):
    """(codes [blocks, layers, 2, heads, 64, dh] in token order, scales, tail rows) of a sequence, from table and lengths."""
    length = int(cache.lengths[slot])
    full, rest = length // BLOCK, length % BLOCK
    pages = cache.table[slot, :full].long()
    assert (pages >= 0).all() and (cache.table[slot, full:] == -1).all()
    raw = cache.codes[pages]
    shape = raw.shape[:2]
    keys = raw[:, :, 0].reshape(*shape, cache.kv_heads, BLOCK, cache.head_dim)
    values = raw[:, :, 1].reshape(*shape, cache.kv_heads, cache.head_dim, BLOCK).transpose(-1, -2)
    return torch.stack([keys, values], 2), cache.scales[pages], cache.tail[slot, :, :, :, :rest]


def quantised(torch, x):
    """x [..., 64, dh] -> codes, scales [...] from the definition, in 64 bits."""
    scale = (x.double().abs().amax((-1, -2)) / 127).float().clamp_min(2.0 ** -126)
    return (x.double() / scale.double()[..., None, None]).round().to(torch.int8), scale


def bookkeeping(torch, cache):
    """Reference counts and free bits follow from the table; no page is in a row twice."""
    held = cache.table[cache.table >= 0].long()
    refs = torch.bincount(held, minlength=cache.pages).int()
    assert torch.equal(refs, cache.refs)
    bits = (cache.free_bits.long()[:, None] >> torch.arange(32, device="cuda") & 1).reshape(-1)[:cache.pages]
    assert torch.equal(bits == 1, refs == 0)
    assert torch.equal((cache.table >= 0).sum(1), (cache.lengths // BLOCK).long())


def fill(torch, cache, slots, counts, gen, history, rope, q_dtype, strided):
    batch = cache.batch(slots, counts)
    cache.extend(batch)
    width = cache.kv_heads * cache.head_dim
    for layer in range(cache.layers):
        fused = torch.randn((batch.rows, 2 * width + (3 if strided == "odd" else 8)), device="cuda", generator=gen).to(q_dtype)
        k, v = fused[:, :width], fused[:, width:2 * width]
        if strided == "odd":
            k, v = fused[:, 1:width + 1], fused[:, width + 2:2 * width + 2]
        cache.append(layer, k, v, batch, rope=rope)
        row = 0
        for slot, n in zip(slots, counts):
            history[slot][layer].append(tuple(x[row:row + n].reshape(n, cache.kv_heads, cache.head_dim) for x in (k, v)))
            row += n
    return batch


@pytest.mark.parametrize("dh,kv_heads,dtype,q_dtype,rope,strided", [
    (64, 3, "bfloat16", "float32", True, "even"), (128, 2, "float16", "float16", True, "odd"), (128, 1, "bfloat16", "bfloat16", False, "odd"),
    (64, 8, "float16", "float32", False, "even"), (64, 2, "float16", "bfloat16", True, "even")])
def test_appending_equals_the_formula_whatever_the_chunks(cuda, dh, kv_heads, dtype, q_dtype, rope, strided):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(dh + kv_heads)
    cache = PagedKV8Cache(2, kv_heads, dh, pages=40, sequences=7, max_length=500, dtype=dtype)
    tables = rope_tables(torch, 500, dh) if rope else None
    history = [[[], []] for _ in range(7)]
    steps = [([0, 1, 2, 3, 4, 5], [1, 63, 64, 65, 200, 0]), ([2, 0, 4], [1, 1, 1])] + [([1, 3, 5, 6], [1, 1, 1, 2])] * 3
    steps += [([4, 0, 6], [100, 126, 130]), ([5, 1], [189, 0]), ([6], [60])] + [([0, 1, 2, 3], [1, 1, 1, 1])] * 2
    for slots, counts in steps:
        fill(torch, cache, slots, counts, gen, history, tables, getattr(torch, q_dtype), strided)
    assert _lib.device_status() == 0
    bookkeeping(torch, cache)
    kind = getattr(torch, dtype)
    for slot in range(7):
        length = int(cache.lengths[slot])
        codes, scales, tail = content(torch, cache, slot)
        for layer in range(2):
            k = torch.cat([p[0] for p in history[slot][layer]])
            v = torch.cat([p[1] for p in history[slot][layer]])
            assert k.shape[0] == length
            if rope:
                k = rotated(torch, k, tables[0][:length], tables[1][:length])
            kv = torch.stack([k.to(kind), v.to(kind)]).permute(0, 2, 1, 3)                    # [2, heads, tokens, dh]
            full = length // BLOCK * BLOCK
            want, scale = quantised(torch, kv[:, :, :full].reshape(2, kv_heads, -1, BLOCK, dh).permute(2, 0, 1, 3, 4))
            assert torch.equal(codes[:, layer], want)
            assert torch.equal(scales[:, layer], scale)
            assert torch.equal(tail[layer], kv[:, :, full:])
            if length > full:
                assert torch.equal(cache.peak[slot, layer], kv[:, :, full:].float().abs().amax((-1, -2)))


def test_rows_behind_a_tail_stay(cuda):
    torch = cuda
    cache = PagedKV8Cache(1, 2, 64, pages=4, sequences=2, max_length=128)
    cache.tail.fill_(7.0)
    batch = cache.batch([1], [10])
    cache.extend(batch)
    x = torch.randn(10, 128, device="cuda")
    cache.append(0, x, x, batch)
    assert (cache.tail[0] == 7).all() and (cache.tail[1, :, :, :, 10:] == 7).all() and not (cache.tail[1, :, :, :, :10] == 7).any()


@pytest.mark.parametrize("value,expected", [("zero", 0.0), ("tiny", 1.0), ("nan", math.nan), ("inf", math.nan)])
def test_edge_values_of_a_block(cuda, value, expected):
    """All zero: codes 0. Numbers below the smallest scale: rounded to multiples of it. A value that is not finite: scale NaN for
    its head only."""
    torch = cuda
    cache = PagedKV8Cache(1, 2, 64, pages=4, sequences=1, max_length=128)
    x = torch.zeros(64, 128, device="cuda")
    if value == "tiny":
        x[3, 5] = 2.0 ** -126
    elif value != "zero":
        x[:, 64:] = 1.0
        x[3, 5] = math.nan if value == "nan" else -math.inf
    batch = cache.extend(cache.batch([0], [64]))
    cache.append(0, x, x, batch)
    page = int(cache.table[0, 0])
    scale = cache.scales[page, 0]
    codes = cache.codes[page, 0].reshape(2, 2, 64, 64)
    if math.isnan(expected):
        assert torch.isnan(scale[:, 0]).all()
        assert torch.equal(scale[:, 1], torch.full((2,), 1.0 / 127, device="cuda")) and (codes[:, 1] == 127).all()
    else:
        assert (scale == 2.0 ** -126).all()
        assert codes.abs().sum() == (2 if expected else 0)
        assert codes[0, 0, 3, 5] == expected and codes[1, 0, 5, 3] == expected


def test_codes_next_to_every_border(cuda):
    """Quotients a rounding error away from k + 1/2, for every k: ties go to the even code, neighbours of a tie to their side."""
    torch = cuda
    cache = PagedKV8Cache(1, 1, 128, pages=9, sequences=1, max_length=512, dtype="float16")
    top = 1.75 * 127 / 64                        # scale 1.75 / 64: k + 1/2 codes are exact FP16 numbers up to 11 bits
    half = (torch.arange(127, device="cuda", dtype=torch.float64) + 0.5) * (1.75 / 64)
    near = half.to(torch.float16)
    bits = near.view(torch.int16)
    values = torch.cat([near, (bits + 1).view(torch.float16), (bits - 1).view(torch.float16), -near])
    x = torch.zeros(64 * 128, dtype=torch.float16, device="cuda")
    x[:values.numel()] = values
    x[-1] = top
    x = x.reshape(64, 128)
    batch = cache.extend(cache.batch([0], [64]))
    cache.append(0, x, x, batch)
    want, scale = quantised(torch, x)
    page = int(cache.table[0, 0])
    assert torch.equal(cache.codes[page, 0, 0, 0].reshape(64, 128), want) and float(cache.scales[page, 0, 0, 0]) == float(scale)


def test_extend_is_all_or_nothing(cuda):
    torch = cuda
    cache = PagedKV8Cache(1, 1, 64, pages=5, sequences=3, max_length=300)
    cache.extend(cache.batch([0, 1], [130, 70]))                # three pages
    state = [t.clone() for t in (cache.table, cache.lengths, cache.refs, cache.free_bits)]
    batch = cache.batch([2, 1, 0], [128, 60, 1])                # needs three, two are free
    cache.extend(batch)
    assert _lib.device_status() == 501 and (batch.starts == -1).all()
    assert all(torch.equal(a, b) for a, b in zip(state, (cache.table, cache.lengths, cache.refs, cache.free_bits)))
    x = torch.randn(189, 64, device="cuda")
    before = cache.codes.clone(), cache.tail.clone()
    cache.append(0, x, x, batch)                                # a refused step writes nothing and answers NaN
    assert torch.equal(cache.codes, before[0]) and torch.equal(cache.tail, before[1])
    assert torch.isnan(cache.attention(0, x, batch)).all()
    _lib.clear_device_status()
    batch = cache.batch([2, 0], [10, 171])                      # 130 + 171 > 300
    cache.extend(batch)
    assert _lib.device_status() == 502 and (batch.starts == -1).all()
    assert all(torch.equal(a, b) for a, b in zip(state, (cache.table, cache.lengths, cache.refs, cache.free_bits)))
    _lib.clear_device_status()
    cache.extend(cache.batch([2, 0], [10, 126]))                # exactly what is left
    assert cache.read_lengths() == [256, 70, 10] and _lib.device_status() == 0
    bookkeeping(torch, cache)


@pytest.mark.parametrize("pages,sequences", [(37, 5), (5000, 1500), (70000, 40)])
def test_pages_come_lowest_first_and_return(cuda, pages, sequences):
    torch = cuda
    cache = PagedKV8Cache(1, 1, 64, pages=pages, sequences=sequences, max_length=64 * 2000)
    rng = torch.Generator().manual_seed(pages)
    free, rows, lengths = list(range(pages)), [[] for _ in range(sequences)], [0] * sequences
    for step in range(6):
        slots = torch.randperm(sequences, generator=rng).tolist()[:max(1, sequences * 2 // 3)]
        most = max(1, 64 * len(free) // max(1, 2 * len(slots)))
        counts = [int(torch.randint(0, min(most, 64 * 2000 - lengths[s]) + 1, (1,), generator=rng)) for s in slots]
        batch = cache.extend(cache.batch(slots, counts))
        assert batch.starts.tolist() == [lengths[s] for s in slots]
        for s, n in zip(slots, counts):
            need = (lengths[s] + n) // 64 - lengths[s] // 64
            rows[s] += free[:need]
            free, lengths[s] = free[need:], lengths[s] + n
        drop = torch.randperm(sequences, generator=rng).tolist()[:max(1, sequences // 3)]
        cache.free(drop)
        for s in drop:
            free, rows[s], lengths[s] = sorted(free + rows[s]), [], 0
        assert cache.read_lengths() == lengths
        table = cache.table.tolist()
        assert all(t[:len(r)] == r for t, r in zip(table, rows))
        bookkeeping(torch, cache)
    assert _lib.device_status() == 0


def test_fork_shares_pages_and_parts_ways(cuda):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(3)
    cache = PagedKV8Cache(2, 2, 64, pages=30, sequences=8, max_length=400)
    history = [[[], []] for _ in range(8)]
    fill(torch, cache, [0, 1, 2], [150, 64, 5], gen, history, None, torch.float32, "even")
    cache.tail[4:] = 9.0
    cache.fork([0, 0, 1, 2], [4, 5, 6, 7])
    bookkeeping(torch, cache)
    assert cache.read_lengths() == [150, 64, 5, 0, 150, 150, 64, 5] and cache.read_live_pages() == 3
    for a, b in ((0, 4), (0, 5), (1, 6), (2, 7)):
        assert all(torch.equal(x, y) for x, y in zip(content(torch, cache, a), content(torch, cache, b)))
        rest = int(cache.lengths[a]) % 64
        assert (cache.tail[b, :, :, :, rest:] == 9).all()
    kept = [t.clone() for t in content(torch, cache, 0)]
    fill(torch, cache, [4, 5], [50, 120], gen, history, None, torch.float32, "even")       # each copy goes on by itself
    assert all(torch.equal(x, y) for x, y in zip(kept, content(torch, cache, 0)))
    first, second = content(torch, cache, 4), content(torch, cache, 5)
    assert torch.equal(first[0][:2], second[0][:2]) and not torch.equal(first[0][2], second[0][2])
    bookkeeping(torch, cache)
    cache.free([0, 5])
    assert all(torch.equal(x, y) for x, y in zip(first, content(torch, cache, 4)))          # shared pages outlive a holder
    bookkeeping(torch, cache)
    cache.free([1, 2, 3, 4, 6, 7])
    assert cache.read_live_pages() == 0 and (cache.table == -1).all()
    bookkeeping(torch, cache)
    assert _lib.device_status() == 0


def test_fork_and_free_refusals(cuda):
    torch = cuda
    cache = PagedKV8Cache(1, 1, 64, pages=8, sequences=4, max_length=200)
    cache.extend(cache.batch([0, 1], [130, 3]))
    state = [t.clone() for t in (cache.table, cache.lengths, cache.refs, cache.free_bits)]
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for src, dst in ((ints(0, 0), ints(2, 2)), (ints(0), ints(1)), (ints(0, 2), ints(2, 3)), (ints(0), ints(4)), (ints(-1), ints(2)), (ints(2), ints(2))):
        cache.fork(src, dst)                                     # twice the same target, not empty, also a source, out of range
        assert _lib.device_status() == 503
        _lib.clear_device_status()
        assert all(torch.equal(a, b) for a, b in zip(state, (cache.table, cache.lengths, cache.refs, cache.free_bits)))
    for src, dst in (([0], [0]), ([0, 1], [2, 2]), ([4], [2]), ([0], [4]), ([0, 1], [2])):
        with pytest.raises(ValueError):
            cache.fork(src, dst)
    with pytest.raises(ValueError):
        cache.free([1, 1])
    cache.free(ints(0, 0, 0))                                    # the same slot in a tensor: freed once
    assert _lib.device_status() == 0
    bookkeeping(torch, cache)
    assert cache.read_lengths() == [0, 3, 0, 0]
    cache.free(ints(9, 1))
    assert _lib.device_status() == 503 and cache.read_lengths() == [0, 0, 0, 0]


def test_compact_keeps_everything_in_fewer_pages(cuda):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(5)
    cache = PagedKV8Cache(3, 2, 128, pages=70, sequences=6, max_length=700, dtype="float16")
    history = [[[], [], []] for _ in range(6)]
    fill(torch, cache, [0, 1, 2, 3], [300, 200, 640, 65], gen, history, None, torch.float32, "even")
    cache.fork([2], [5])
    cache.free([1, 2])
    before = [[t.clone() for t in content(torch, cache, s)] for s in range(6)]
    old = [t.clone() for t in (cache.codes, cache.table, cache.refs)]
    for pages in (None, 15, 33):
        small = cache.compact(pages)
        assert small.pages == (pages or 15) and small.read_live_pages() == 15
        bookkeeping(torch, small)
        for s in range(6):
            assert all(torch.equal(a, b) for a, b in zip(before[s], content(torch, small, s)))
        assert torch.equal(small.tail, cache.tail) and torch.equal(small.peak, cache.peak) and small.read_lengths() == cache.read_lengths()
        assert sorted(small.table[small.table >= 0].tolist()) == list(range(15))
    assert all(torch.equal(a, b) for a, b in zip(old, (cache.codes, cache.table, cache.refs)))
    with pytest.raises(ValueError):
        cache.compact(14)
    fill(torch, small, [1], [130], gen, history, None, torch.float32, "even")               # the copy is a cache of its own
    bookkeeping(torch, small)
    assert torch.equal(old[1], cache.table)
    assert _lib.device_status() == 0


def test_refusals_of_the_python_layer(cuda):
    torch = cuda
    cache = PagedKV8Cache(2, 2, 64, pages=4, sequences=2, max_length=128)
    for slots, counts in (([0, 0], [1, 1]), ([2], [1]), ([-1], [1]), ([0], [-1]), ([0], [129]), ([], []), ([0, 1], [1])):
        with pytest.raises(ValueError):
            cache.batch(slots, counts)
    with pytest.raises(ValueError):
        cache.batch([0], [5], max_keys=4)
    batch = cache.extend(cache.batch([0], [5]))
    good = torch.randn(5, 128, device="cuda")
    with pytest.raises(ValueError):
        cache.append(2, good, good, batch)                       # no such layer
    with pytest.raises(ValueError):
        cache.append(0, good[:4], good, batch)
    with pytest.raises(ValueError):
        cache.append(0, good.t().contiguous().t(), good, batch)  # columns are not consecutive
    with pytest.raises(TypeError):
        cache.append(0, good, good.half(), batch)
    with pytest.raises(TypeError):
        cache.append(0, good.double(), good.double(), batch)
    with pytest.raises(ValueError):
        cache.append(0, good, good, batch, rope=rope_tables(torch, 127, 64))
    with pytest.raises(ValueError):
        cache.append(0, good, good, batch, rope=rope_tables(torch, 128, 128))
    with pytest.raises(ValueError):
        cache.attention(0, torch.randn(5, 192, device="cuda"), batch)      # three heads over two
    with pytest.raises(ValueError):
        cache.attention(0, good, batch, out=torch.empty(5, 128, device="cuda"))
    with pytest.raises(NotImplementedError):
        PagedKV8Cache(1, 1, 96, pages=1, sequences=1, max_length=64)
    with pytest.raises(NotImplementedError):
        PagedKV8Cache(1, 1, 64, pages=1, sequences=1, max_length=64, dtype="float32")
    with pytest.raises(ValueError):
        PagedKV8Cache.from_tensors(cache.codes, cache.scales, cache.tail, cache.peak, cache.table.long(), cache.lengths, cache.refs)
    with pytest.raises(ValueError):
        PagedKV8Cache.from_tensors(cache.codes, cache.scales, cache.tail, cache.peak, cache.table, cache.lengths, cache.refs, max_length=200)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("pages", [30000, 40000])
def test_steps_of_more_sequences_than_a_cta_has_threads(cuda, pages):
    torch = cuda
    sequences = 2300
    cache = PagedKV8Cache(1, 1, 64, pages=pages, sequences=sequences, max_length=64 * 40)
    free, rows, lengths = list(range(pages)), [[] for _ in range(sequences)], [0] * sequences
    for counts in ([(i * 89) % 800 for i in range(sequences)], [64] * sequences, [i % 2 for i in range(sequences)]):
        slots = [(7 * i + 3) % sequences for i in range(sequences)]
        batch = cache.extend(cache.batch(slots, counts))
        assert batch.starts.tolist() == [lengths[s] for s in slots]
        for s, n in zip(slots, counts):
            need = (lengths[s] + n) // 64 - lengths[s] // 64
            rows[s] += free[:need]
            free, lengths[s] = free[need:], lengths[s] + n
        assert cache.read_lengths() == lengths
        assert all(t[:len(r)] == r for t, r in zip(cache.table.tolist(), rows))
    bookkeeping(torch, cache)
    assert _lib.device_status() == 0
    refused = cache.extend(cache.batch(range(sequences), [1500] * sequences))           # more pages than there are
    assert set(refused.starts.tolist()) == {-1} and cache.read_lengths() == lengths and _lib.device_status() in (501, 502)
