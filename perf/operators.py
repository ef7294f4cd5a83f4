"""Operators of 8-bit serving, as cases that can be timed and compared: a paged key/value cache held in 8 bits with the
attention that reads it and the page operations of a scheduler, and the matrix product in 8-bit integers.

``listed()`` names the standing cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` builds what a
serving program holds before the call, ``run(state)`` is one pass and ``work(case)`` the bytes and operations it cannot do
without. With ``own`` false a pass computes the plain form in elementary torch operations; with ``own`` true it makes the
calls of the package. Four operators:

``append``     new keys (rotated to their positions) and values of a ragged batch enter the cache: blocks of 64 tokens that
               become full are quantised to int8 with one scale per block and head and written to their page (the values
               transposed), the tokens behind the last full block wait in a 16-bit tail.
``attention``  causal attention of a ragged batch of new tokens over that cache: one token per sequence (decode), whole
               prompts, or chunks of prompts behind a cached context.
``branch``     scheduler work on the page table: sequences are forked (full pages shared, tails copied), the copies grow
               by some tokens (pages are taken from the pool) and are dropped again (pages return to the pool).
``compact``    a new, independent cache with a smaller pool: all live pages move to its front and the page table follows.
``int8``       ``y = x @ W.T`` with int8 weights (one scale per output channel) and activations quantised per token.

Layout of a cache: ``codes`` int8 [pages, layers, 2, kv_heads, 64 * head_dim] (keys [64][head_dim], values
[head_dim][64]), ``scales`` FP32 [pages, layers, 2, kv_heads], ``tail`` [sequences, layers, 2, kv_heads, 64, head_dim] in
the model's type, ``peak`` FP32 [sequences, layers, 2, kv_heads] (largest magnitude in the tail), ``table`` int32
[sequences, blocks], ``lengths`` int32 [sequences], ``refs`` int32 [pages].
"""

import math

import torch

own = False

BLOCK = 64
FLOOR = 2.0 ** -126                              # smallest scale: the smallest normal FP32 number
ESIZE = {"float32": 4, "float16": 2, "bfloat16": 2}


# ------------------------------------------------------------------------------------------------ cases
def _attention(batch, context, new, heads, kv_heads, dh, dtype="bfloat16", q_dtype="float32", ragged=False, layers=2):
    return {"op": "attention", "batch": batch, "context": context, "new": new, "heads": heads, "kv_heads": kv_heads, "dh": dh,
            "dtype": dtype, "q_dtype": q_dtype, "ragged": ragged, "layers": layers}


def _append(batch, context, new, kv_heads, dh, dtype="bfloat16", q_dtype="float32", ragged=False, layers=2):
    return {"op": "append", "batch": batch, "context": context, "new": new, "kv_heads": kv_heads, "dh": dh, "dtype": dtype,
            "q_dtype": q_dtype, "ragged": ragged, "layers": layers}


def _branch(batch, context, new, kv_heads, dh, layers, dtype="bfloat16"):
    return {"op": "branch", "batch": batch, "context": context, "new": new, "kv_heads": kv_heads, "dh": dh, "layers": layers,
            "dtype": dtype}


def _int8(m, n, k, dtype="bfloat16", out="bfloat16"):
    return {"op": "int8", "m": m, "n": n, "k": k, "dtype": dtype, "out": out}


def listed():
    cases = {
        # one sequence of a 1.7B decoder (32 heads of 64, not grouped) in the middle of an answer: latency counts
        "attention_decode_b1_c777": _attention(1, 777, 1, 32, 32, 64),
        # a serving batch of ragged contexts, grouped heads of 128
        "attention_decode_b48_c8192": _attention(48, 8192, 1, 32, 8, 128, q_dtype="bfloat16", ragged=True),
        # few sequences with very long contexts: the work of a head has to be split
        "attention_decode_b4_c131072": _attention(4, 131072, 1, 32, 8, 128, "float16", layers=1),
        # a batch of whole prompts
        "attention_prompt_b4_t2048": _attention(4, 2048, 2048, 32, 32, 64),
        # chunks of long prompts behind what is cached already, ragged, one sequence of the batch idle
        "attention_chunk_b3_t512_c16000": _attention(3, 16000, 512, 32, 8, 128, "float16", "float16", ragged=True),
        # a decode step of a serving batch, and long prompts, entering the cache
        "append_b64_t1": _append(64, 4096, 1, 8, 128, ragged=True),
        "append_b3_t8192": _append(3, 8192, 8192, 8, 128, q_dtype="bfloat16", ragged=True),
        # one sequence tries two continuations; a beam over a whole batch
        "branch_b2": _branch(2, 1500, 40, 8, 128, 16),
        "branch_b64": _branch(64, 3000, 200, 8, 64, 24),
        # a pool whose sequences came and went, packed into as many pages as are alive
        "compact_b40_c4096": {"op": "compact", "batch": 40, "context": 4096, "kv_heads": 8, "dh": 64, "layers": 24, "dtype": "bfloat16"},
        # the projections of a step: a decode token, a ragged batch on sizes that fill no tile, a prompt
        "int8_m1_8192x2048": _int8(1, 8192, 2048),
        "int8_m4096_8192x8192": _int8(4096, 8192, 8192),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "append", "append", "branch", "compact", "int8", "int8", "int8"))
    kv_heads, dh = rng.choice((1, 2, 4, 5, 8, 16, 32)), rng.choice((64, 128))
    dtype = rng.choice(("bfloat16", "float16"))
    if op == "int8":
        # activations and outputs of any floating type; a decode batch to a long prompt
        n, k = _log_int(rng, 250, 16384), _log_int(rng, 250, 16384)
        m = min(_log_int(rng, 1, 8192), 4096 * 8192 * 8192 // (n * k))
        return _int8(max(1, m), n, k, rng.choice(("float32", "float16", "bfloat16")), rng.choice(("float32", "float16", "bfloat16")))
    if op == "attention":
        heads = kv_heads * rng.choice((1, 2, 3, 4, 6, 8) if kv_heads <= 8 else (1, 2))
        q_dtype = rng.choice(("float32", dtype))
        if rng.random() < 0.5:
            batch = _log_int(rng, 1, 128)
            context = min(_log_int(rng, 1, 131072), max(1, 4 * 131072 * 8 * 128 // (batch * kv_heads * dh)))
            new = 1
        else:
            batch = rng.choice((1, 2, 3, 5, 8))
            context = _log_int(rng, 2, 16384)
            new = min(context, _log_int(rng, 2, 4096), max(2, 2 ** 29 // (batch * context * heads)))
        return _attention(batch, context, new, heads, kv_heads, dh, dtype, q_dtype, rng.random() < 0.6, rng.choice((1, 2, 3)))
    if op == "append":
        batch = _log_int(rng, 1, 128)
        new = rng.choice((1, _log_int(rng, 2, 8192)))
        new = max(1, min(new, 3 * 8192 * 8 * 128 // (batch * kv_heads * dh)))
        context = min(16384, max(new, _log_int(rng, 1, 8192)))
        return _append(batch, context, new, kv_heads, dh, dtype, rng.choice(("float32", dtype)), rng.random() < 0.6, rng.choice((1, 2, 3)))
    layers = rng.choice((2, 5, 12, 24))
    kv_heads = min(kv_heads, 8)
    if op == "branch":
        return _branch(_log_int(rng, 1, 64), _log_int(rng, 1, 3000), _log_int(rng, 1, 300), kv_heads, dh // 2 if layers == 24 and dh == 128 else dh,
                       layers, dtype)
    return {"op": "compact", "batch": rng.choice((3, 10, 24, 40)), "context": _log_int(rng, 100, 4096), "kv_heads": kv_heads, "dh": 64,
            "layers": layers, "dtype": dtype}


# ------------------------------------------------------------------------------------------------ sizes of a case
def _spread(i, high, ragged):
    """Size of entry ``i`` of a batch: ``high``, or sizes spread over 1..high with ``high`` itself first."""
    return high if not ragged or i == 0 else max(1, round(high * ((i * 0.6180339887498949) % 1.0)))


def _lengths(case):
    """(tokens in the cache after the step, new tokens among them) of every sequence."""
    out = []
    for i in range(case["batch"]):
        total = _spread(i, case["context"], case.get("ragged", False))
        new = 1 if case["new"] == 1 else min(total, _spread(i + 1 if i else 0, case["new"], case.get("ragged", False)))
        if case["new"] > 1 and case.get("ragged") and i == 1 and case["batch"] > 2:
            new = 0                                                  # idle in this step
        if case["op"] == "append" and case["new"] > 1:
            total = (total - new) // BLOCK * BLOCK + new             # chunks of a prompt begin at a block
        out.append((total, new))
    return out


def _branch_sizes(case):
    """(parents' lengths, tokens their copies grow by, pages in the pool)."""
    parents = [_spread(i, case["context"], True) for i in range(case["batch"])]
    grow = [_spread(i, case["new"], True) for i in range(case["batch"])]
    held = sum(n // BLOCK for n in parents)
    taken = sum((n + g) // BLOCK - n // BLOCK for n, g in zip(parents, grow))
    return parents, grow, held + taken + 17


def _compact_sizes(case):
    return [_spread(i, case["context"], True) for i in range(case["batch"])]


def work(case):
    op = case["op"]
    if op == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * ESIZE[case["dtype"]] + n * k + 4 * n + m * n * ESIZE[case["out"]], "flops": 2 * m * n * k}
    kvh, dh, e = case["kv_heads"], case["dh"], ESIZE[case["dtype"]]
    token = 2 * kvh * dh                                             # elements of a token's keys and values in one layer
    if op == "compact":
        sizes = _compact_sizes(case)
        pages = sum(n // BLOCK for n in sizes)
        return {"bytes": 2 * case["layers"] * (pages * (BLOCK * token + 8 * kvh) + case["batch"] * BLOCK * token * e), "flops": 0}
    if op == "branch":
        parents, _, _ = _branch_sizes(case)
        tails = sum(n % BLOCK for n in parents) * token * e * case["layers"]
        return {"bytes": 2 * tails + 4 * 3 * sum(n // BLOCK + 1 for n in parents), "flops": 0}
    sizes = _lengths(case)
    rows = sum(n for _, n in sizes)
    if op == "append":
        full = sum(t // BLOCK - (t - n) // BLOCK for t, n in sizes)
        old = sum((t - n) % BLOCK for t, n in sizes if t // BLOCK > (t - n) // BLOCK)
        fresh = sum(min(n, t % BLOCK) for t, n in sizes)
        return {"bytes": rows * token * ESIZE[case["q_dtype"]] + old * token * e + full * (BLOCK * token + 8 * kvh) + fresh * token * e
                + rows * dh * 4, "flops": 0}
    cached = sum((t // BLOCK * BLOCK) * token + t // BLOCK * 8 * kvh + t % BLOCK * token * e for t, n in sizes if n)
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for t, n in sizes)
    heads = case["heads"]
    return {"bytes": cached + rows * heads * dh * (ESIZE[case["q_dtype"]] + e), "flops": 4 * heads * dh * pairs}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 11)
    return gen


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", dtype=dtype, generator=gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(case, sizes, sequences, pages, gen):
    """A cache that holds ``sizes[s]`` tokens of sequence ``s``, in pages scattered over the pool, and the host's copy of the
    page table."""
    layers, kvh, dh = case["layers"], case["kv_heads"], case["dh"]
    dtype = getattr(torch, case["dtype"])
    codes = torch.empty((pages, layers, 2, kvh, BLOCK * dh), dtype=torch.int8, device="cuda")
    for part in codes.split(max(1, 2 ** 27 // codes[0].numel())):     # codes of normally distributed blocks: peak near 4 sigma
        part.copy_((_normal(gen, *part.shape, dtype=torch.float16) * 32.0).round_().clamp_(-127, 127))
    scales = torch.rand((pages, layers, 2, kvh), device="cuda", generator=gen) * 0.02 + 0.02
    tail = torch.empty((sequences, layers, 2, kvh, BLOCK, dh), dtype=dtype, device="cuda")
    for part in tail.split(max(1, 2 ** 27 // tail[0].numel())):
        part.copy_(_normal(gen, *part.shape, dtype=dtype))
    held = [n // BLOCK for n in sizes]
    width = -(-max(_longest(case), 1) // BLOCK)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(pages)).tolist()
    table, at = [], 0
    for n in held:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    table += [[-1] * width] * (sequences - len(held))
    refs = [0] * pages
    for p in order[:at]:
        refs[p] = 1
    lengths = list(sizes) + [0] * (sequences - len(sizes))
    inside = torch.arange(BLOCK, device="cuda")[None, :] < (_ints(lengths) % BLOCK)[:, None]
    peak = torch.where(inside[:, None, None, None, :, None], tail.abs(), torch.zeros((), dtype=dtype, device="cuda")).amax((-1, -2)).float()
    return {"codes": codes, "scales": scales, "tail": tail, "peak": peak, "table": _ints(table).reshape(sequences, width),
            "lengths": _ints(lengths), "refs": _ints(refs)}


def _longest(case):
    return max(_lengths_after(case))


def _lengths_after(case):
    if case["op"] == "branch":
        parents, grow, _ = _branch_sizes(case)
        return [n + g for n, g in zip(parents, grow)]
    return _compact_sizes(case) if case["op"] == "compact" else [t for t, _ in _lengths(case)]


def _rope_tables(rows, dh):
    inv = 10000.0 ** (-torch.arange(dh // 2, dtype=torch.float64, device="cuda") * 2.0 / dh)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    gen = _generator(seed)
    state = {"case": case}
    if case["op"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        x = _normal(gen, m, k) * torch.exp(0.5 * _normal(gen, m, 1))
        x[:, torch.randint(0, k, (max(1, k // 500),), device="cuda", generator=gen)] *= 12.0     # channels that stand out
        state["x"] = x.to(getattr(torch, case["dtype"]))
        state["codes"] = (_normal(gen, n, k, dtype=torch.float16) * 32.0).round_().clamp_(-127, 127).to(torch.int8)
        state["scales"] = torch.rand(n, device="cuda", generator=gen) * 4e-4 + 4e-4
        if own:
            from mylocal_llm_b200 import Int8Weight
            state["weight"] = Int8Weight(state["codes"], state["scales"])
        return state
    if case["op"] in ("branch", "compact"):
        if case["op"] == "branch":
            sizes, grow, pages = _branch_sizes(case)
            state |= _cache(case, sizes, 2 * case["batch"], pages, gen)
            b = case["batch"]
            state |= {"src": _ints(list(range(b))), "dst": _ints(list(range(b, 2 * b))), "grow": _ints(grow),
                      "most": max(-(-g // BLOCK) for g in grow) + 1}
        else:
            sizes = _compact_sizes(case)
            held = sum(n // BLOCK for n in sizes)
            state |= _cache(case, sizes, case["batch"], 2 * held + 5, gen)
            state["held"] = held
        if own:
            from mylocal_llm_b200 import PagedKV8Cache
            state["cache"] = PagedKV8Cache.from_tensors(**{n: state[n] for n in ("codes", "scales", "tail", "peak", "table", "lengths", "refs")},
                                                        max_length=_longest(case))
            if case["op"] == "branch":
                state["batch"] = state["cache"].batch(list(range(b, 2 * b)), grow)
        return state
    # a step of a ragged batch: the cache as it is before the attention (all tokens in it), or before the new tokens enter
    sizes = _lengths(case)
    b, dh, kvh = case["batch"], case["dh"], case["kv_heads"]
    blocks = sum(t // BLOCK for t, _ in sizes)
    state |= _cache(case, [t for t, _ in sizes], b, blocks + max(3, blocks // 16), gen)
    starts, counts = [t - n for t, n in sizes], [n for _, n in sizes]
    offsets = [sum(counts[:i]) for i in range(b + 1)]
    rows = offsets[-1]
    cos, sin = _rope_tables(max(t for t, _ in sizes), dh)
    q_heads = case.get("heads", kvh)
    # column slices of one projection output, as the stacked q|k|v projection leaves them
    width = (q_heads + 2 * kvh) * dh
    fused = _normal(gen, rows, width, dtype=getattr(torch, case["q_dtype"]))
    state |= {"q": fused[:, :q_heads * dh], "k": fused[:, q_heads * dh:(q_heads + kvh) * dh], "v": fused[:, (q_heads + kvh) * dh:],
              "cos": cos, "sin": sin, "layer": case["layers"] - 1, "starts": _ints(starts), "counts": _ints(counts),
              "offsets": _ints(offsets), "sizes": sizes}
    seq = torch.repeat_interleave(torch.arange(b, device="cuda"), state["counts"], output_size=rows)
    pos = torch.arange(rows, device="cuda") - (state["offsets"][:-1] - state["starts"])[seq]
    state |= {"seq": seq, "pos": pos}                                                    # sequence and position of every row
    if case["op"] == "append":
        # the blocks that the new tokens touch: their sequence and number, where each begins in the list, which become full
        touched = [(i, blk) for i, (t, n) in enumerate(sizes) if n for blk in range((t - n) // BLOCK, (t - 1) // BLOCK + 1)]
        first = [0] * b
        for at, (i, blk) in reversed(list(enumerate(touched))):
            first[i] = at - blk
        idx = lambda v: torch.tensor(v, dtype=torch.int64, device="cuda")  # noqa: E731
        opened = [at for at, (i, blk) in enumerate(touched) if starts[i] > blk * BLOCK]
        full = [at for at, (i, blk) in enumerate(touched) if (blk + 1) * BLOCK <= sizes[i][0]]
        part = [at for at, (i, blk) in enumerate(touched) if (blk + 1) * BLOCK > sizes[i][0]]
        state |= {"touched": len(touched), "block_seq": idx([i for i, _ in touched]), "block_no": idx([blk for _, blk in touched]),
                  "row_block": idx(first)[seq] + pos // BLOCK, "opened": idx(opened), "full": idx(full), "part": idx(part),
                  "rows_part": torch.nonzero(pos >= (_ints([t for t, _ in sizes]) // BLOCK * BLOCK)[seq])[:, 0]}
    if own:
        from mylocal_llm_b200 import PagedKV8Cache
        state["cache"] = PagedKV8Cache.from_tensors(**{n: state[n] for n in ("codes", "scales", "tail", "peak", "table", "lengths", "refs")},
                                                    max_length=_longest(case))
        state["batch"] = state["cache"].batch(list(range(b)), counts)
        state["batch"].starts.copy_(state["starts"])
        if case["op"] == "append":
            # the peaks that the new tokens of a tail meet are those of the tokens before the step
            of, layer = state["block_seq"][state["part"]], state["layer"]
            before = torch.arange(BLOCK, device="cuda") < (state["starts"][of] - state["block_no"][state["part"]] * BLOCK)[:, None]
            magnitude = state["tail"][of, layer].float().abs()
            state["peak"][of, layer] = (magnitude * before[:, None, None, :, None]).amax((-1, -2))
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"int8": _run_int8, "attention": _run_attention, "append": _run_append, "branch": _run_branch,
            "compact": _run_compact}[state["case"]["op"]](state)


def _quantised(x, dims):
    """(codes, scales) of ``x`` with one scale over ``dims``: scale = max |x| / 127, code = x / scale rounded to the nearest,
    ties to even. The quotient is formed in 64 bits, where it lies on the right side of every border."""
    scale = (x.abs().amax(dims, keepdim=True).double() / 127.0).float().clamp_min(FLOOR)
    return (x.double() / scale.double()).round().to(torch.int8), scale


def _run_int8(state):
    case = state["case"]
    out = getattr(torch, case["out"])
    if own:
        from mylocal_llm_b200 import int8_linear
        return int8_linear(state["x"], state["weight"], out_dtype=out)
    codes, scale = _quantised(state["x"].float(), (-1,))
    return (torch.matmul(codes.float(), state["codes"].float().t()) * scale * state["scales"]).to(out)


def _rotated(x, cos, sin):
    half = x.shape[-1] // 2
    x0, x1 = x[..., :half], x[..., half:]
    return torch.cat([x0 * cos - x1 * sin, x0 * sin + x1 * cos], dim=-1)


def _run_append(state):
    if own:
        cache, batch, layer = state["cache"], state["batch"], state["layer"]
        cache.append(layer, state["k"], state["v"], batch, rope=(state["cos"], state["sin"]))
        return {"codes": cache.codes, "scales": cache.scales, "tail": cache.tail, "peak": cache.peak}
    case, layer = state["case"], state["layer"]
    kvh, dh, dtype = case["kv_heads"], case["dh"], getattr(torch, case["dtype"])
    pos, seq = state["pos"], state["seq"]
    rows = pos.shape[0]
    # far positions and borders of the rounding: the rotation in 64 bits
    cos, sin = state["cos"][pos][:, None].double(), state["sin"][pos][:, None].double()
    k = _rotated(state["k"].reshape(rows, kvh, dh).double(), cos, sin).float().to(dtype)
    kv = torch.stack([k, state["v"].reshape(rows, kvh, dh).to(dtype)], dim=1)            # [rows, 2, kvh, dh]
    blocks = torch.zeros((state["touched"], 2, kvh, BLOCK, dh), dtype=torch.float32, device=kv.device)
    opened = state["opened"]                                                             # blocks that hold older tokens
    of = state["block_seq"][opened]
    older = torch.arange(BLOCK, device=kv.device) < (state["starts"][of] % BLOCK)[:, None]
    blocks[opened] = torch.where(older[:, None, None, :, None], state["tail"][of, layer].float(), blocks[opened])
    blocks[state["row_block"], :, :, pos % BLOCK] = kv.float()
    full, part = state["full"], state["part"]
    codes, scale = _quantised(blocks[full], (-1, -2))
    page = state["table"][state["block_seq"][full], state["block_no"][full]].long()
    state["codes"][page, layer, 0] = codes[:, 0].reshape(-1, kvh, BLOCK * dh)
    state["codes"][page, layer, 1] = codes[:, 1].transpose(-1, -2).reshape(-1, kvh, BLOCK * dh)
    state["scales"][page, layer] = scale[..., 0, 0]
    keep = state["rows_part"]
    state["tail"][seq[keep], layer, :, :, pos[keep] % BLOCK] = kv[keep]
    state["peak"][state["block_seq"][part], layer] = blocks[part].abs().amax((-1, -2))
    return {"codes": state["codes"], "scales": state["scales"], "tail": state["tail"], "peak": state["peak"]}


def _run_attention(state):
    case, layer = state["case"], state["layer"]
    b, heads, kvh, dh = case["batch"], case["heads"], case["kv_heads"], case["dh"]
    if own:
        return state["cache"].attention(layer, state["q"], state["batch"], rope=(state["cos"], state["sin"]))
    group, device, most = heads // kvh, state["q"].device, max(1, max(n for _, n in state["sizes"]))
    seq, pos = state["seq"], state["pos"]
    q = state["q"].reshape(-1, heads, dh).float()
    q = _rotated(q, state["cos"][pos][:, None], state["sin"][pos][:, None]) * (dh ** -0.5)
    # keys and values in order: the full pages of each sequence and, behind them, its tail
    table = state["table"].clamp_min(0).long()
    width = table.shape[1]
    total = state["starts"] + state["counts"]
    blocks = state["codes"][table, layer].float() * state["scales"][table, layer][..., None]      # [b, width, 2, kvh, 64 * dh]
    keys = torch.zeros((b, kvh, width + 1, BLOCK, dh), device=device)
    values = torch.zeros((b, kvh, width + 1, BLOCK, dh), device=device)
    keys[:, :, :width] = blocks[:, :, 0].reshape(b, width, kvh, BLOCK, dh).transpose(1, 2)
    values[:, :, :width] = blocks[:, :, 1].reshape(b, width, kvh, dh, BLOCK).permute(0, 2, 1, 4, 3)
    every, last = torch.arange(b, device=device), (total // BLOCK).long()
    keys[every, :, last] = state["tail"][:, layer, 0].float()
    values[every, :, last] = state["tail"][:, layer, 1].float()
    keys, values = keys.reshape(b, kvh, -1, dh), values.reshape(b, kvh, -1, dh)
    # rows as [sequence, key/value head, group x new token]
    at = pos - state["starts"][seq]
    padded = torch.zeros((b, most, heads, dh), device=device)
    padded[seq, at] = q
    grouped = padded.reshape(b, most, kvh, group, dh).permute(0, 2, 3, 1, 4).reshape(b, kvh, group * most, dh)
    scores = torch.matmul(grouped, keys.transpose(-1, -2)).reshape(b, kvh, group, most, -1)
    limit = state["starts"][:, None] + torch.arange(most, device=device)                  # last key that a row sees
    seen = torch.arange(keys.shape[2], device=device) <= limit[..., None]
    scores = scores.masked_fill_(~seen[:, None, None], float("-inf"))
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    norm = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.reshape(b, kvh, group * most, -1), values).reshape(b, kvh, group, most, dh) / norm
    out = out.permute(0, 3, 1, 2, 4).reshape(b, most, heads * dh)
    return out[seq, at].to(getattr(torch, case["dtype"]))


def _run_branch(state):
    if own:
        cache, batch = state["cache"], state["batch"]
        cache.fork(state["src"], state["dst"])
        cache.extend(batch)
        out = {"table": cache.table.clone(), "refs": cache.refs.clone(), "lengths": cache.lengths.clone(), "starts": batch.starts,
               "tail": cache.tail, "peak": cache.peak}
        cache.free(state["dst"])
        return out
    src, dst, grow = state["src"].long(), state["dst"].long(), state["grow"]
    table, refs, lengths, tail, peak = (state[n] for n in ("table", "refs", "lengths", "tail", "peak"))
    width, pages = table.shape[1], refs.shape[0]
    # fork: the full pages are shared, the tokens of the tail are copied
    have = lengths[src]
    columns = torch.arange(width, device=table.device)
    shared = columns < (have // BLOCK)[:, None]
    table[dst] = torch.where(shared, table[src], torch.full_like(table[src], -1))
    refs.index_add_(0, table[dst].clamp_min(0).reshape(-1).long(), shared.reshape(-1).int())
    lengths[dst] = have
    inside = (torch.arange(BLOCK, device=table.device) < (have % BLOCK)[:, None])[:, None, None, None, :, None]
    tail[dst] = torch.where(inside, tail[src], tail[dst])
    peak[dst] = peak[src]
    # grow: the lowest free pages, in the order of the requests
    need = (have + grow) // BLOCK - have // BLOCK
    before = need.cumsum(0) - need
    free = refs == 0
    rank = torch.where(free, free.cumsum(0) - 1, pages)
    page_of = torch.full((pages + 1,), -1, dtype=torch.int32, device=table.device)
    page_of[rank] = torch.arange(pages, dtype=torch.int32, device=table.device)
    request = torch.arange(state["most"], device=table.device)
    asked = request < need[:, None]
    page = page_of[torch.where(asked, before[:, None] + request, pages).long()]
    column = torch.where(asked, (have // BLOCK)[:, None] + request, width).long()
    wide = torch.cat([table[dst], table.new_zeros((dst.shape[0], 1))], dim=1)            # a column for what was not asked
    table[dst] = wide.scatter(1, column, page)[:, :width]
    refs.index_add_(0, torch.where(asked, page, 0).reshape(-1).long(), asked.reshape(-1).int())
    lengths[dst] = have + grow
    out = {"table": table.clone(), "refs": refs.clone(), "lengths": lengths.clone(), "starts": have, "tail": tail, "peak": peak}
    # free: what no sequence refers to any more returns to the pool
    held = table[dst] >= 0
    refs.index_add_(0, table[dst].clamp_min(0).reshape(-1).long(), -held.reshape(-1).int())
    table[dst] = -1
    lengths[dst] = 0
    return out


def _run_compact(state):
    if own:
        small = state["cache"].compact(state["held"])
        return {n: getattr(small, n) for n in ("codes", "scales", "tail", "peak", "table", "lengths", "refs")}
    refs, table = state["refs"], state["table"]
    live = refs > 0
    place = live.cumsum(0) - 1                                                           # of every live page in the new pool
    source = torch.zeros(state["held"] + 1, dtype=torch.int64, device=refs.device)
    source[torch.where(live, place, state["held"])] = torch.arange(refs.shape[0], device=refs.device)
    source = source[:-1]
    moved = torch.where(table >= 0, place[table.clamp_min(0).long()].int(), -1)
    return {"codes": state["codes"][source], "scales": state["scales"][source], "tail": state["tail"].clone(),
            "peak": state["peak"].clone(), "table": moved, "lengths": state["lengths"].clone(), "refs": refs[source]}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """What ``run`` returns, from the definitions, in 64 bits; ``None`` for what is moved and not computed."""
    if case["op"] in ("branch", "compact"):
        return None
    state = prepare(case, seed)
    if case["op"] == "int8":
        x = state["x"].double()
        scale = torch.clamp(x.abs().max(dim=1).values / 127, min=FLOOR).float().double()
        codes = torch.round(x / scale[:, None])
        out = torch.empty((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for at in range(0, case["n"], 2048):
            part = state["codes"][at:at + 2048].double()
            out[:, at:at + 2048] = (codes @ part.T) * scale[:, None] * state["scales"][at:at + 2048].double()
        return out
    layer, kvh, dh = state["layer"], case["kv_heads"], case["dh"]

    def turned(x, first):
        """[tokens, heads, dh] in 64 bits, turned by the angles of the positions from ``first`` on (as complex numbers)."""
        n = x.shape[0]
        z = torch.complex(x[..., :dh // 2], x[..., dh // 2:])
        z = z * torch.complex(state["cos"][first:first + n].double(), state["sin"][first:first + n].double())[:, None]
        return torch.cat([z.real, z.imag], -1)

    row = 0
    if case["op"] == "append":
        scales, peak = state["scales"].double(), state["peak"].double()
        for s, (total, new) in enumerate(state["sizes"]):
            if not new:
                continue
            start = total - new
            low = start // BLOCK * BLOCK
            dtype = state["tail"].dtype
            k = turned(state["k"][row:row + new].double().reshape(new, kvh, dh), start).to(dtype)
            v = state["v"][row:row + new].reshape(new, kvh, dh).to(dtype)
            for part, x in enumerate((k, v)):
                old = state["tail"][s, layer, part, :, :start - low].transpose(0, 1)
                x = torch.cat([old, x]).double().abs()                                   # tokens low .. total - 1
                for blk in range(low // BLOCK, (total - 1) // BLOCK + 1):
                    top = x[blk * BLOCK - low:(blk + 1) * BLOCK - low].amax((0, 2))
                    if (blk + 1) * BLOCK <= total:
                        scales[int(state["table"][s, blk]), layer, part] = torch.clamp(top / 127, min=FLOOR)
                    else:
                        peak[s, layer, part] = top
            row += new
        return {"codes": None, "scales": scales, "tail": None, "peak": peak}
    heads = case["heads"]
    outs = []
    for s, (total, new) in enumerate(state["sizes"]):
        if not new:
            continue
        pages = state["table"][s, :total // BLOCK].long()
        codes, scales = state["codes"][pages, layer].double(), state["scales"][pages, layer].double()
        rest = total % BLOCK
        q = turned(state["q"][row:row + new].double().reshape(new, heads, dh), total - new)
        mask = torch.arange(total, device="cuda") > (torch.arange(new, device="cuda") + total - new)[:, None]
        result = torch.empty((new, heads, dh), dtype=torch.float64, device="cuda")
        for h in range(heads):
            g = h // (heads // kvh)
            tail = state["tail"][s, layer, :, g, :rest].double()
            k = torch.cat([(codes[:, 0, g] * scales[:, 0, g, None]).reshape(-1, dh), tail[0]])
            v = torch.cat([(codes[:, 1, g] * scales[:, 1, g, None]).reshape(-1, dh, BLOCK).transpose(1, 2).reshape(-1, dh), tail[1]])
            weights = torch.softmax((q[:, h] @ k.T / math.sqrt(dh)).masked_fill(mask, -math.inf), dim=-1)
            result[:, h] = weights @ v
        outs.append(result.reshape(new, heads * dh))
        row += new
    return torch.cat(outs)
