"""What a serving program's host does between steps waits for nothing on the device: batches, forks and ends given as Python
integers, and a whole prompt of the Llama model."""

import pytest

from mylocal_llm_b200 import PagedKV8Cache, _lib
from mylocal_llm_b200.llama_model import ExternalLlamaConfig, ExternalLlamaModel
from test_gpu_kv8_cache import bookkeeping
from test_gpu_llama_model import CFG, make_weights

pytestmark = pytest.mark.gpu


def busy(torch):
    """The current stream gets a kernel of about a tenth of a second (it ends by itself); an event behind it."""
    torch.cuda._sleep(200_000_000)
    event = torch.cuda.Event()
    event.record()
    return event


def test_batches_forks_and_ends_do_not_wait(cuda):
    torch = cuda
    cache = PagedKV8Cache(1, 1, 64, pages=8, sequences=6, max_length=200)

    def work():
        cache.extend(cache.batch([0, 1], [130, 5]))
        cache.fork([0, 1], [2, 3])
        cache.free([0])
        cache.extend(cache.batch([2, 3, 0], [1, 1, 3]))
        cache.free([0, 1, 2, 3])

    work()                                       # (pinned memory and kernels are there)
    torch.cuda.synchronize()
    event = busy(torch)
    work()
    assert not event.query()
    torch.cuda.synchronize()
    assert _lib.device_status() == 0 and cache.read_lengths() == [0] * 6
    bookkeeping(torch, cache)


def test_many_batches_under_way_keep_their_own_numbers(cuda):
    """Their host memory is not used again before it has been copied."""
    torch = cuda
    cache = PagedKV8Cache(1, 1, 64, pages=8, sequences=50, max_length=64)
    cache.batch([0], [1])
    torch.cuda.synchronize()
    event = busy(torch)
    batches = [cache.batch([i % 50, (i + 1) % 50], [i % 7, i % 5]) for i in range(300)]
    assert not event.query()
    torch.cuda.synchronize()
    for i, b in enumerate(batches):
        assert b.slots.tolist() == [i % 50, (i + 1) % 50] and b.offsets.tolist() == [0, i % 7, i % 7 + i % 5] and b.starts.tolist() == [-2, -2]


def test_a_prompt_of_the_model_does_not_wait(cuda):
    torch = cuda
    model = ExternalLlamaModel(ExternalLlamaConfig(**dict(CFG, max_position_embeddings=256)), dtype="bfloat16")
    packed, _ = make_weights(model, seed=4, uniform=True)
    model.set_weights(packed)
    tokens = torch.randint(0, CFG["vocab_size"], (2, 70), device="cuda")
    state = model.create_generation_state(2, 200, "int8")
    want = [model.prefill(tokens, state).clone(), model.decode_one(tokens[:, 0].contiguous(), state).clone()]
    torch.cuda.synchronize()
    event = busy(torch)
    got = [model.prefill(tokens, state), model.decode_one(tokens[:, 0].contiguous(), state)]
    assert not event.query()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_python_integers_are_not_captured(cuda):
    """A graph would copy them from host memory that is used for something else by then; tensors on the device it may hold."""
    torch = cuda
    cache = PagedKV8Cache(1, 1, 64, pages=8, sequences=6, max_length=200)
    batch = cache.extend(cache.batch([0], [70]))
    src, dst = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (0, 1))
    cache.fork(src, dst)
    cache.free(dst)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: cache.batch([1], [1]), lambda: cache.fork([0], [1]), lambda: cache.fork(src, [1]), lambda: cache.free([0])):
            with pytest.raises(RuntimeError):
                call()
        cache.fork(src, dst)
        cache.extend(batch)
        cache.free(dst)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert _lib.device_status() == 502                       # 70 + 70 + 70 > 200
    _lib.clear_device_status()
    assert cache.read_lengths() == [140, 0, 0, 0, 0, 0]
    bookkeeping(torch, cache)
