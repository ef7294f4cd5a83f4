"""The 8-bit cache and the int8 product as a serving program uses them together, and in the Llama model.

Every attention call is compared with 64-bit arithmetic on the cache's content (the bound of test_gpu_kv8_attention), every
sequence's content with what was appended to it (the definition of test_gpu_kv8_cache)."""

import numpy as np
import pytest

from mylocal_llm_b200 import Int8Weight, PagedKV8Cache, _lib, int8_linear
from mylocal_llm_b200.llama_model import ExternalLlamaConfig, ExternalLlamaModel, PagedGenerationState
from oracle import llama_oracle as lo
from test_gpu_kv8_attention import check, rope_tables
from test_gpu_kv8_cache import bookkeeping, content, quantised, rotated
from test_gpu_llama_model import CFG, make_weights

pytestmark = pytest.mark.gpu

BLOCK = 64


@pytest.fixture(autouse=True)
def healthy(cuda):
    _lib.clear_device_status()
    yield
    cuda.cuda.synchronize()
    assert _lib.device_status() == 0


def test_a_schedule_of_prompts_steps_forks_and_ends(cuda):
    """Projections in 8 bits, prompts in chunks, decode steps, forks that go on by themselves, ends, a smaller pool: whatever
    happened before, each sequence's content and each row's context are those of its own tokens."""
    torch = cuda
    heads, kv_heads, dh, d, layers, horizon = 8, 2, 64, 256, 2, 700
    qd, kd = heads * dh, kv_heads * dh
    gen = torch.Generator(device="cuda").manual_seed(0)
    rng = np.random.default_rng(0)
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    qkv = [Int8Weight.quantize(randn(qd + 2 * kd, d) / 16) for _ in range(layers)]
    back = [Int8Weight.quantize(randn(d, qd) / 24) for _ in range(layers)]
    rope = rope_tables(torch, horizon, dh)
    cache = PagedKV8Cache(layers, kv_heads, dh, pages=70, sequences=9, max_length=horizon)
    history = [[[] for _ in range(layers)] for _ in range(9)]                   # keys and values before rotation
    lengths = [0] * 9

    def step(slots, counts):
        batch = cache.extend(cache.batch(slots, counts, max_keys=max(max(lengths[s] + n for s, n in zip(slots, counts)), 1)))
        for s, n in zip(slots, counts):
            lengths[s] += n
        x = randn(batch.rows, d).to(torch.bfloat16)
        for layer in range(layers):
            fused = int8_linear(x, qkv[layer], out_dtype=torch.float32)
            q, k, v = fused[:, :qd], fused[:, qd:qd + kd], fused[:, qd + kd:]
            cache.append(layer, k, v, batch, rope=rope)
            row = 0
            for s, n in zip(slots, counts):
                history[s][layer].append((k[row:row + n].reshape(n, kv_heads, dh), v[row:row + n].reshape(n, kv_heads, dh)))
                row += n
            context = cache.attention(layer, q, batch, rope=rope)
            check(torch, cache, layer, q, context, lengths, counts, rope, slots=slots)
            x = x + int8_linear(context, back[layer])
        assert torch.isfinite(x).all()

    def verify():
        bookkeeping(torch, cache)
        assert cache.read_lengths() == lengths
        for s in range(9):
            codes, scales, tail = content(torch, cache, s)
            for layer in range(layers):
                if not lengths[s]:
                    continue
                k, v = (torch.cat([p[i] for p in history[s][layer]]) for i in range(2))
                k = rotated(torch, k, rope[0][:lengths[s]], rope[1][:lengths[s]])
                kv = torch.stack([k.to(torch.bfloat16), v.to(torch.bfloat16)]).permute(0, 2, 1, 3)
                full = lengths[s] // BLOCK * BLOCK
                want, scale = quantised(torch, kv[:, :, :full].reshape(2, kv_heads, -1, BLOCK, dh).permute(2, 0, 1, 3, 4))
                assert torch.equal(codes[:, layer], want) and torch.equal(scales[:, layer], scale) and torch.equal(tail[layer], kv[:, :, full:])

    step([0, 3], [200, 64])
    step([0, 3, 1], [1, 1, 130])
    for _ in range(3):
        step([3, 0, 1], [1, 1, 1])
    cache.fork([0, 0, 1], [4, 5, 8])
    for src, dst in ((0, 4), (0, 5), (1, 8)):
        history[dst] = [list(parts) for parts in history[src]]
        lengths[dst] = lengths[src]
    verify()
    for i in range(6):
        slots = [int(s) for s in rng.permutation([0, 1, 3, 4, 5, 8])[:4]]
        step(slots, [int(n) for n in rng.integers(0, 70 if i % 2 else 3, 4)] if i else [60, 1, 64, 3])
    cache.free([0, 3])
    for s in (0, 3):
        lengths[s], history[s] = 0, [[] for _ in range(layers)]
    verify()
    cache = cache.compact(60)
    verify()
    step([0, 4, 2], [300, 1, 7])
    cache.free([4, 5])
    for s in (4, 5):
        lengths[s], history[s] = 0, [[] for _ in range(layers)]
    step([8, 0, 1], [33, 2, 1])
    verify()


@pytest.mark.parametrize("uniform", [False, True])
def test_llama_on_an_8_bit_cache_matches_the_oracle(cuda, uniform):
    """Up to 63 tokens lie in the 16-bit tail: the same tolerance as with the dense cache."""
    torch = cuda
    model = ExternalLlamaModel(ExternalLlamaConfig(**CFG), dtype="bfloat16")
    packed, oracle = make_weights(model, uniform=uniform)
    model.set_weights(packed)
    tokens = np.random.default_rng(1).integers(0, CFG["vocab_size"], 12)
    state = model.create_generation_state(1, 32, "int8")
    assert isinstance(state, PagedGenerationState)
    ref = lo.llama_logits(oracle, CFG, tokens)
    scale = np.abs(ref).max()
    for _ in range(2):                                                          # a second prompt replaces the first
        logits = model.prefill(torch.from_numpy(tokens[:9][None]).cuda(), state)
        np.testing.assert_allclose(logits[0].cpu().numpy(), ref[8], rtol=6e-2, atol=6e-2 * scale)
        for i in range(9, 12):
            logits = model.decode_one(torch.from_numpy(tokens[i:i + 1]).cuda(), state)
            np.testing.assert_allclose(logits[0].cpu().numpy(), ref[i], rtol=6e-2, atol=6e-2 * scale)
        assert state.length == 12 and state.cache.read_lengths() == [12]


@pytest.mark.parametrize("fused", [True, False])
def test_llama_calls_the_cache_with_its_own_keys_and_positions(cuda, monkeypatch, fused):
    """Prompts over several blocks and decode steps across a block's border: each layer's attention is that of its cache, and the
    first layer's cache holds what the dense one holds (keys of both are roundings of values that differ by FP32 roundings of the
    rotation, at most 2^-22 of the two products: one step of BF16 at most)."""
    torch = cuda
    cfg = dict(CFG, max_position_embeddings=256)
    model = ExternalLlamaModel(ExternalLlamaConfig(**cfg), dtype="bfloat16")
    packed, _ = make_weights(model, seed=3, uniform=True)
    model.set_weights(packed)
    model.fused_decode = fused
    tokens = torch.from_numpy(np.random.default_rng(2).integers(0, CFG["vocab_size"], (2, 135))).cuda()
    state, dense = model.create_generation_state(2, 200, "int8"), model.create_generation_state(2, 200)
    calls = []
    real = PagedKV8Cache.attention

    def checked(self, layer, q, batch, **kw):
        out = real(self, layer, q, batch, **kw)
        counts = (batch.offsets[1:] - batch.offsets[:-1]).tolist()
        check(torch, self, layer, q, out, self.read_lengths(), counts, kw["rope"])
        calls.append((layer, q.shape[0]))
        return out

    monkeypatch.setattr(PagedKV8Cache, "attention", checked)
    model.prefill(tokens[:, :125].contiguous(), state)
    model.prefill(tokens[:, :125].contiguous(), dense)
    for i in range(125, 135):
        model.decode_one(tokens[:, i].contiguous(), state)
        model.decode_one(tokens[:, i].contiguous(), dense)
    assert calls == [(0, 250), (1, 250)] + [(0, 2), (1, 2)] * 10
    for s in range(2):
        codes, scales, tail = content(torch, state.cache, s)
        for part, cache in ((0, dense.k), (1, dense.v)):
            want = cache[0, s, :, :135].double()
            held = codes[:, 0, part].double() * scales[:, 0, part, :, None, None].double()
            held = held.permute(1, 0, 2, 3).reshape(2, 128, 64)
            step = 2.0 ** -7 * want.abs() + 1e-5
            assert ((held - want[:, :128]).abs() <= step[:, :128] + 0.51 * scales[:, 0, part].double().T.repeat_interleave(64, 1)[..., None]).all()
            assert ((tail[0, part].double() - want[:, 128:]).abs() <= step[:, 128:]).all()


def test_llama_decode_on_an_8_bit_cache_is_capturable(cuda):
    torch = cuda
    cfg = dict(CFG, max_position_embeddings=256)
    model = ExternalLlamaModel(ExternalLlamaConfig(**cfg), dtype="bfloat16")
    packed, _ = make_weights(model, seed=5, uniform=True)
    model.set_weights(packed)
    tokens = torch.from_numpy(np.random.default_rng(6).integers(0, CFG["vocab_size"], (3, 90))).cuda()

    def run(graphed):
        state = model.create_generation_state(3, 128, "int8")
        model.prefill(tokens[:, :60].contiguous(), state)
        ids = tokens[:, 60].clone()
        outs = [model.decode_one(ids, state).clone()]
        torch.cuda.synchronize()
        if graphed:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                logits = model.decode_one(ids, state)
        for i in range(61, 70):
            ids.copy_(tokens[:, i])
            if graphed:
                graph.replay()
            else:
                logits = model.decode_one(ids, state)
            outs.append(logits.clone())
        torch.cuda.synchronize()
        assert state.cache.read_lengths() == [70] * 3
        return outs

    assert all(torch.equal(a, b) for a, b in zip(run(False), run(True)))


def test_llama_states_share_a_pool_by_forking(cuda):
    """Two continuations of one prompt: the fork's first step gives the logits of its source's."""
    torch = cuda
    cfg = dict(CFG, max_position_embeddings=256)
    model = ExternalLlamaModel(ExternalLlamaConfig(**cfg), dtype="bfloat16")
    packed, _ = make_weights(model, seed=9, uniform=True)
    model.set_weights(packed)
    tokens = torch.from_numpy(np.random.default_rng(7).integers(0, CFG["vocab_size"], (2, 100))).cuda()
    tokens[1] = tokens[0]
    state = model.create_generation_state(1, 200, "int8", sequences=2, pages=6)
    model.prefill(tokens[:1, :80].contiguous(), state)
    state.cache.fork([0], [1])
    pair = model.create_generation_state(1, 200, "int8", sequences=2, pages=6)
    pair.cache, pair.slots, pair.batch, pair.length = state.cache, [0, 1], 2, state.length
    pair.step = pair.cache.batch([0, 1], [1, 1])
    for i in range(80, 100):
        logits = model.decode_one(tokens[:, i].contiguous(), pair)
        assert torch.equal(logits[0], logits[1])
    assert state.cache.read_lengths() == [100, 100] and state.cache.read_live_pages() == 1


def test_llama_refuses_what_an_8_bit_cache_cannot_hold(cuda):
    model = ExternalLlamaModel(ExternalLlamaConfig(**CFG), dtype="float32")
    packed, _ = make_weights(model, uniform=True)
    model.set_weights(packed)
    with pytest.raises(NotImplementedError):
        model.create_generation_state(1, 32, "int8")
    with pytest.raises(ValueError):
        model.create_generation_state(1, 32, "int4")
    with pytest.raises(ValueError):
        model.create_generation_state(1, 32, pages=4)
    half = ExternalLlamaModel(ExternalLlamaConfig(**CFG), dtype="float16")
    half.set_weights(packed)
    with pytest.raises(ValueError):
        half.create_generation_state(2, 32, "int8", sequences=1)
    state = half.create_generation_state(1, 8, "int8")
    with pytest.raises(ValueError):
        half.prefill(cuda.zeros((1, 9), dtype=cuda.int64, device="cuda"), state)
    half.prefill(cuda.zeros((1, 8), dtype=cuda.int64, device="cuda"), state)
    with pytest.raises(ValueError):
        half.decode_one(cuda.zeros(1, dtype=cuda.int64, device="cuda"), state)
