"""The kernels of the 8-bit cache start while their predecessor drains and wait for it before they touch memory: the same bits
with and without chained launches (``B200Q_CHAIN``), eagerly and replayed back to back from a graph."""

import numpy as np
import pytest

from mylocal_llm_b200 import Int8Weight, PagedKV8Cache, _lib, int8_linear
from mylocal_llm_b200.llama_model import ExternalLlamaConfig, ExternalLlamaModel
from test_gpu_chained_launch import LLAMA
from test_gpu_kv8_attention import rope_tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 40, 1], [150, 0, 70]])
@pytest.mark.parametrize("graphed", [False, True])
def test_a_step_of_the_cache(cuda, monkeypatch, counts, graphed):
    """Projection, growth, append, attention, projection back, a fork and its end, over and over on the same buffers."""
    torch = cuda
    layers, kv_heads, dh, heads, d = 3, 2, 64, 8, 256
    width, horizon = (heads + 2 * kv_heads) * dh, 1600
    gen = torch.Generator(device="cuda").manual_seed(1)
    into = [Int8Weight.quantize(torch.randn(width, d, device="cuda", generator=gen) / 16) for _ in range(layers)]
    back = [Int8Weight.quantize(torch.randn(d, heads * dh, device="cuda", generator=gen) / 24) for _ in range(layers)]
    inputs = torch.randn(8, sum(counts), d, device="cuda", generator=gen)
    rope = rope_tables(torch, horizon, dh)

    def run(chain):
        monkeypatch.setenv("B200Q_CHAIN", chain)
        cache = PagedKV8Cache(layers, kv_heads, dh, pages=60, sequences=4, max_length=horizon)
        batch = cache.batch([0, 1, 2], counts)
        src, dst = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (0, 3))
        x = inputs[0].clone()

        def step():
            cache.extend(batch)
            y = x
            for layer in range(layers):
                fused = int8_linear(y, into[layer])
                q, k, v = fused[:, :heads * dh], fused[:, heads * dh:(heads + kv_heads) * dh], fused[:, (heads + kv_heads) * dh:]
                cache.append(layer, k, v, batch, rope=rope)
                y = y + int8_linear(cache.attention(layer, q, batch, rope=rope), back[layer], out_dtype=torch.float32)
            cache.fork(src, dst)
            cache.free(dst)
            return y

        seen = [step().clone()]
        torch.cuda.synchronize()
        if graphed:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = step()
        for row in inputs[1:]:
            x.copy_(row)
            if graphed:
                graph.replay()
            else:
                y = step()
            seen.append(y.clone())
        torch.cuda.synchronize()
        assert cache.read_lengths()[:3] == [8 * n for n in counts] and _lib.device_status() == 0
        return seen + [cache.tail, cache.table, cache.refs, cache.free_bits]

    plain, chained = run("0"), run("1")
    assert all(torch.equal(a, b) for a, b in zip(plain, chained)) and all(torch.isfinite(t).all() for t in plain[:8])


def test_the_llama_model_on_the_8_bit_cache(cuda, monkeypatch):
    torch = cuda
    model = ExternalLlamaModel.synthetic(ExternalLlamaConfig(**LLAMA), seed=1)
    prompt = torch.from_numpy(np.random.default_rng(2).integers(0, LLAMA["vocab_size"], (2, 61))).cuda()

    def generate(chain, graphed):
        monkeypatch.setenv("B200Q_CHAIN", chain)
        state = model.create_generation_state(2, 100, "int8")
        token = model.prefill(prompt, state).argmax(dim=-1)
        seen = [model.decode_one(token, state).clone()]
        token.copy_(seen[0].argmax(dim=-1))
        torch.cuda.synchronize()
        if graphed:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                logits = model.decode_one(token, state)
                token.copy_(logits.argmax(dim=-1))
        for _ in range(10):
            if graphed:
                graph.replay()
            else:
                logits = model.decode_one(token, state)
                token.copy_(logits.argmax(dim=-1))
            seen.append(logits.clone())
        torch.cuda.synchronize()
        return seen

    reference = generate("0", False)
    for chain, graphed in (("1", False), ("1", True), ("0", True)):
        assert all(torch.equal(a, b) for a, b in zip(reference, generate(chain, graphed)))
