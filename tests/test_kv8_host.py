"""Refusals of the 8-bit cache's and the int8 product's entry points: decided on the host before any launch (no GPU here)."""

import ctypes

import pytest

from mylocal_llm_b200 import Int8Weight, PagedKV8Cache, _lib, int8_linear, quantize_int8_rows

ONE = 16                                   # an aligned address that nothing dereferences


def cache(**changes):
    fields = dict(codes=ONE, scales=ONE, tail=ONE, peak=ONE, table=ONE, lengths=ONE, refs=ONE, free_bits=ONE, layers=2, kv_heads=4,
                  head_dim=64, pages=10, sequences=3, blocks=4, max_length=256, dtype=2)
    fields.update(changes)
    return _lib.KV8CacheStruct(**fields)


def rc(name, *args):
    return getattr(_lib.load(), name)(*args)


@pytest.mark.parametrize("field", ["codes", "scales", "tail", "peak", "table", "lengths", "refs", "free_bits"])
def test_every_part_of_a_cache_is_needed(field):
    assert rc("b200q_kv8_free", ctypes.byref(cache(**{field: None})), ONE, 1, None) == 1


@pytest.mark.parametrize("change,code", [
    (dict(layers=0), 1), (dict(kv_heads=0), 1), (dict(pages=0), 1), (dict(sequences=0), 1), (dict(blocks=0), 1), (dict(max_length=0), 1),
    (dict(head_dim=80), 3), (dict(dtype=0), 3), (dict(sequences=65537), 3), (dict(pages=(1 << 20) + 1), 3),
    (dict(max_length=320), 1),                              # five full blocks in a table of four
    (dict(codes=8), 1), (dict(tail=24), 1)])                # not 16-byte aligned
def test_sizes_of_a_cache(change, code):
    bad = ctypes.byref(cache(**change))
    assert rc("b200q_kv8_extend", bad, ONE, ONE, 1, ONE, None) == code
    assert rc("b200q_kv8_append", bad, 0, ONE, ONE, 0, 256, 256, ONE, ONE, ONE, 1, 1, None, None, 0, None) == code
    assert rc("b200q_kv8_attention", bad, 0, ONE, 0, 256, 4, ONE, ONE, ONE, 1, 1, 1, 1, None, None, 0, 0.1, ONE, ONE, 1 << 20, None) == code
    assert rc("b200q_kv8_fork", bad, ONE, ONE, 1, ONE, None) == code
    assert b"kv8_fork" in _lib.load().b200q_last_error()


def test_none_null_cache():
    assert rc("b200q_kv8_extend", None, ONE, ONE, 1, ONE, None) == 1


@pytest.mark.parametrize("change", [
    dict(layer=2), dict(layer=-1), dict(k=None), dict(starts=None), dict(dtype=5), dict(k_row=255), dict(v_row=0), dict(batch=4),
    dict(max_new=257), dict(cos=None), dict(rows=255), dict(cos=ONE + 4)])
def test_append_refuses(change):
    a = dict(layer=1, k=ONE, v=ONE, dtype=0, k_row=256, v_row=256, slots=ONE, offsets=ONE, starts=ONE, batch=2, max_new=3, cos=ONE,
             sin=ONE, rows=256)
    a.update(change)
    assert rc("b200q_kv8_append", ctypes.byref(cache()), *a.values(), None) == 1


@pytest.mark.parametrize("change", [
    dict(layer=2), dict(q=None), dict(dtype=3), dict(q_row=511), dict(heads=6), dict(heads=0), dict(batch=4), dict(rows=-1),
    dict(max_new=0), dict(max_new=6), dict(max_new=257, rows=300), dict(keys=0), dict(keys=257), dict(sin=None), dict(positions=10), dict(out=None)])
def test_attention_refuses(change):
    a = dict(layer=0, q=ONE, dtype=0, q_row=512, heads=8, slots=ONE, offsets=ONE, starts=ONE, batch=2, rows=5, max_new=4, keys=100,
             cos=ONE, sin=ONE, positions=256, scale=0.1, out=ONE, workspace=ONE, bytes=1 << 30)
    a.update(change)
    assert rc("b200q_kv8_attention", ctypes.byref(cache()), *a.values(), None) == 1


def test_page_operations_refuse():
    good = ctypes.byref(cache())
    assert rc("b200q_kv8_extend", good, ONE, ONE, 4, ONE, None) == 1            # more entries than sequences
    assert rc("b200q_kv8_extend", good, ONE, None, 1, ONE, None) == 1
    assert rc("b200q_kv8_fork", good, ONE, ONE, 4, ONE, None) == 1
    assert rc("b200q_kv8_fork", good, ONE, ONE, 1, None, None) == 1
    assert rc("b200q_kv8_free", good, None, 1, None) == 1
    assert rc("b200q_kv8_free", good, ONE, -1, None) == 1
    other = cache(codes=32, tail=32, table=32, pages=5)
    need = rc("b200q_kv8_compact_workspace", good, ctypes.byref(other))
    assert need == 4 * 16
    for name in ("b200q_kv8_compact_plan", "b200q_kv8_compact_move"):
        assert rc(name, good, ctypes.byref(other), ONE, need - 1, None) == 1
        assert rc(name, good, ctypes.byref(cache(codes=32, tail=32, table=32, layers=3)), ONE, 1 << 20, None) == 1
        assert rc(name, good, ctypes.byref(cache(codes=32, table=32)), ONE, 1 << 20, None) == 1     # shares the tails
    for name, args in (("b200q_kv8_extend", (ONE, ONE, 0, ONE)), ("b200q_kv8_fork", (ONE, ONE, 0, ONE)), ("b200q_kv8_free", (ONE, 0))):
        assert rc(name, good, *args, None) == 0                                  # nothing to do: no launch


@pytest.mark.parametrize("change,code", [
    (dict(x=None), 1), (dict(dtype=4), 1), (dict(k=0), 1), (dict(x_row=99), 1), (dict(codes_row=104), 1), (dict(codes_row=96), 1),
    (dict(codes=ONE + 4), 1), (dict(rows=-1), 1)])
def test_int8_quantize_refuses(change, code):
    a = dict(x=ONE, dtype=0, rows=3, k=100, x_row=100, codes=ONE, codes_row=112, scales=ONE, early=0)
    a.update(change)
    assert rc("b200q_int8_quantize", *a.values(), None) == code


@pytest.mark.parametrize("change,code", [
    (dict(w=None), 1), (dict(xs=None), 1), (dict(dtype=4), 1), (dict(n=0), 1), (dict(m=-1), 1), (dict(k=131072, w_row=131072, x_row=131072), 3),
    (dict(w_row=104), 1), (dict(x_row=96), 1), (dict(x=ONE + 8), 1)])
def test_int8_gemm_refuses(change, code):
    a = dict(w=ONE, w_row=112, ws=ONE, n=5, k=100, x=ONE, x_row=112, xs=ONE, m=3, y=ONE, dtype=0)
    a.update(change)
    assert rc("b200q_int8_gemm", *a.values(), None) == code


def test_python_layers_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    with pytest.raises(TypeError):
        quantize_int8_rows(torch.zeros(2, 32))
    with pytest.raises(TypeError):
        Int8Weight(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2))
    with pytest.raises(TypeError):
        int8_linear(torch.zeros(2, 32), torch.zeros(2, 32))
    with pytest.raises(TypeError):
        PagedKV8Cache(1, 1, 64, pages=1, sequences=1, max_length=64, device="cpu")
    with pytest.raises(ValueError):
        PagedKV8Cache(1, 1, 64, pages=0, sequences=1, max_length=64)


@pytest.mark.parametrize("max_new,rows", [(1, 2), (4, 5), (200, 300)])
def test_attention_refuses_outputs_that_are_not_aligned(max_new, rows):
    assert rc("b200q_kv8_attention", ctypes.byref(cache()), 0, ONE, 0, 512, 8, ONE, ONE, ONE, 2, rows, max_new, 100, None, None, 0, 0.1, ONE + 8,
              ONE, 1 << 20, None) == 1


def test_a_step_that_append_could_not_take_is_not_begun():
    """The lengths would have grown by tokens that no call can store."""
    whole = ctypes.byref(cache(sequences=65536))
    for name in ("b200q_kv8_extend", "b200q_kv8_extend_after"):
        assert rc(name, whole, ONE, ONE, 65536, ONE, None) == 3
    assert rc("b200q_kv8_append", whole, 0, ONE, ONE, 0, 256, 256, ONE, ONE, ONE, 65536, 1, None, None, 0, None) == 3


@pytest.mark.parametrize("size", [2 ** 30 + 1, 2 ** 31 - 1])
def test_int8_sizes_whose_indexes_do_not_fit_32_bits(size):
    wide = -(-size // 16) * 16
    assert rc("b200q_int8_quantize", ONE, 0, size, 100, 100, ONE, 112, ONE, 0, None) == 3
    assert rc("b200q_int8_quantize", ONE, 0, 3, size, wide, ONE, wide, ONE, 0, None) == 3
    for name in ("b200q_int8_gemm", "b200q_int8_gemm_behind_quantize"):
        assert rc(name, ONE, 112, ONE, size, 100, ONE, 112, ONE, 3, ONE, 0, None) == 3
        assert rc(name, ONE, 112, ONE, 5, 100, ONE, 112, ONE, size, ONE, 0, None) == 3
