"""What a refused step of the 8-bit cache leaves behind it, in the cache and in the Llama model."""

import numpy as np
import pytest

from mylocal_llm_b200 import Int8Weight, PagedKV8Cache, _lib, int8_linear, quantize_int8_rows
from mylocal_llm_b200.llama_model import ExternalLlamaConfig, ExternalLlamaModel
from test_gpu_kv8_cache import bookkeeping
from test_gpu_llama_model import CFG, make_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def healthy(cuda):
    _lib.clear_device_status()
    yield
    cuda.cuda.synchronize()
    _lib.clear_device_status()


def llama(torch, **changes):
    model = ExternalLlamaModel(ExternalLlamaConfig(**dict(CFG, max_position_embeddings=256, **changes)), dtype="bfloat16")
    packed, _ = make_weights(model, seed=4, uniform=True)
    model.set_weights(packed)
    tokens = torch.from_numpy(np.random.default_rng(8).integers(0, CFG["vocab_size"], (2, 200))).cuda()
    return model, tokens


@pytest.mark.parametrize("fused", [True, False])
def test_no_step_goes_on_from_a_refused_prompt(cuda, fused):
    torch = cuda
    model, tokens = llama(torch)
    model.fused_decode = fused
    state = model.create_generation_state(2, 200, "int8", pages=2)
    assert torch.isnan(model.prefill(tokens[:, :130].contiguous(), state)).all()          # four pages, two are there
    assert _lib.device_status() == 501
    for i in range(3):
        assert torch.isnan(model.decode_one(tokens[:, 130 + i].contiguous(), state)).all()
    assert _lib.device_status() == 501 and state.cache.read_lengths() == [0, 0]
    _lib.clear_device_status()
    assert torch.isnan(model.decode_one(tokens[:, 133].contiguous(), state)).all() and _lib.device_status() == 504
    _lib.clear_device_status()
    good = model.create_generation_state(2, 200, "int8")
    for s in (state, good):                                                               # a prompt that fits starts anew
        s.logits = [model.prefill(tokens[:, :100].contiguous(), s), model.decode_one(tokens[:, 100].contiguous(), s)]
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(state.logits, good.logits))
    assert _lib.device_status() == 0 and state.cache.read_lengths() == [101, 101]
    bookkeeping(torch, state.cache)


@pytest.mark.parametrize("graphed", [False, True])
def test_no_step_goes_on_from_a_refused_token(cuda, graphed):
    """A token that found no page for its block is missing from the sequence, also when there are pages again."""
    torch = cuda
    model, tokens = llama(torch)
    state = model.create_generation_state(1, 200, "int8", sequences=2, pages=2)
    other = state.cache.extend(state.cache.batch([1], [64]))                              # one of the two pages
    x = torch.zeros(64, CFG["num_key_value_heads"] * state.cache.head_dim, device="cuda")
    for layer in range(state.cache.layers):
        state.cache.append(layer, x, x, other)
    model.prefill(tokens[:1, :126].contiguous(), state)
    ids = tokens[:1, 126].clone()
    assert torch.isfinite(model.decode_one(ids, state)).all()
    torch.cuda.synchronize()
    if graphed:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = model.decode_one(ids, state)

    def step():
        if graphed:
            graph.replay()
            return logits
        return model.decode_one(ids, state)

    assert torch.isnan(step()).all() and _lib.device_status() == 501                      # token 128 of 128
    state.cache.free([1])
    for _ in range(2):
        assert torch.isnan(step()).all()
    assert state.cache.read_lengths() == [127, 0]
    model.prefill(tokens[:1, :127].contiguous(), state)
    assert torch.isfinite(step()).all() and state.cache.read_lengths() == [128, 0]


@pytest.mark.parametrize("sequences", [3, 1100])
def test_extending_after_a_refusal(cuda, sequences):
    torch = cuda
    cache = PagedKV8Cache(1, 1, 64, pages=2, sequences=sequences, max_length=256)
    batch = cache.batch(list(range(sequences)), [100] + [1] * (sequences - 1))
    assert (batch.starts == -2).all()
    assert (cache.extend(batch, after=True).starts == 0).all() and _lib.device_status() == 0
    assert (cache.extend(batch, after=True).starts == -1).all() and _lib.device_status() == 501     # 200 tokens: two pages more
    cache.free(list(range(1, sequences)))
    cache.free([0])
    assert (cache.extend(batch, after=True).starts == -1).all() and _lib.device_status() == 501
    _lib.clear_device_status()
    assert (cache.extend(batch, after=True).starts == -1).all() and _lib.device_status() == 504
    _lib.clear_device_status()
    assert cache.read_lengths() == [0] * sequences
    assert (cache.extend(batch).starts == 0).all() and _lib.device_status() == 0                    # the caller knows
    bookkeeping(torch, cache)


@pytest.mark.parametrize("length", [-1, -64, -200, -2 ** 31, 257, 2 ** 31 - 1])
@pytest.mark.parametrize("sequences", [3, 1100])
def test_lengths_that_no_sequence_has(cuda, length, sequences):
    """A cache over existing tensors with a length outside 0 .. max_length: the step is refused, nothing is written."""
    torch = cuda
    first = PagedKV8Cache(1, 1, 64, pages=40, sequences=sequences, max_length=256)
    first.lengths[1] = length
    parts = [getattr(first, n) for n in ("codes", "scales", "tail", "peak", "table", "lengths", "refs")]
    before = [t.clone() for t in parts]
    cache = PagedKV8Cache.from_tensors(*parts, max_length=256)
    batch = cache.extend(cache.batch(list(range(sequences)), [70, 200] + [1] * (sequences - 2)))
    assert _lib.device_status() == 502 and (batch.starts == -1).all()
    assert all(torch.equal(a, b) for a, b in zip(before, parts))


@pytest.mark.parametrize("layer", [2 ** 32, 2 ** 32 + 1, -2 ** 32, 2 ** 31, 2, -1])
@pytest.mark.parametrize("native", ["0", "1"])
def test_layers_that_the_cache_lacks(cuda, monkeypatch, layer, native):
    """Also those whose low 32 bits name one."""
    torch = cuda
    monkeypatch.setenv("B200Q_HOST", native)
    cache = PagedKV8Cache(2, 1, 64, pages=2, sequences=1, max_length=64)
    batch = cache.extend(cache.batch([0], [3]))
    x = torch.ones(3, 64, device="cuda")
    with pytest.raises(ValueError):
        cache.append(layer, x, x, batch)
    with pytest.raises(ValueError):
        cache.attention(layer, x, batch)
    assert not cache.tail.any()


def test_more_rows_than_32_bits_count(cuda):
    """Not the rows that the low 32 bits count."""
    torch = cuda
    weight = Int8Weight(torch.ones(4, 1, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda"))
    x = torch.empty(2 ** 32 + 1, 1, dtype=torch.float16, device="cuda")
    for call in (lambda: quantize_int8_rows(x), lambda: int8_linear(x, weight), lambda: int8_linear(x[None], weight),
                 lambda: quantize_int8_rows(x.reshape(1, -1))):
        with pytest.raises(NotImplementedError):
            call()
