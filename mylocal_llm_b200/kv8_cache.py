"""Paged key/value cache in 8 bits and the attention that reads it.

The dense caches of ``llama_model.GenerationState`` (and of the reference, ``mini_llm/ops/attention_inference.py:255-277``)
reserve a full horizon per sequence in the model's type. Here a block of 64 tokens that has become full is held as int8 codes
with one FP32 scale per block, key/value head and part (keys, values) in a page of a shared pool; the up to 63 tokens behind
it wait in the model's 16-bit type. A token costs about half the memory and half the memory traffic of every later step. A
page is written once, so sequences share pages by reference: a fork copies only the tail.

    cache = PagedKV8Cache(layers, kv_heads, head_dim, pages=2048, sequences=16, max_length=8192)
    batch = cache.batch([0, 1, 5], [512, 1, 1])        # slots and their new tokens: one prompt, two single tokens
    cache.extend(batch)                                # lengths grow, pages are taken from the pool
    for layer in range(layers):
        cache.append(layer, k, v, batch, rope=(cos, sin))          # k, v [514, kv_heads * head_dim]
        context = cache.attention(layer, q, batch, rope=(cos, sin))  # q [514, heads * head_dim] -> same shape
    cache.fork([0], [7]); cache.free([1, 5]); cache = cache.compact()

All bookkeeping (lengths, page table, reference counts, the pool's free pages) lives on the device, nothing but ``compact``
and the ``read_*`` helpers waits for it, and a step whose ``batch`` is kept can be captured into a CUDA graph and replayed:
``extend`` reads the lengths anew each time (``fork`` and ``free`` are captured with slots in device tensors). What the device
refuses - too few free pages, a sequence that would pass ``max_length``, a fork onto a slot that is not empty - changes nothing
and sets the device status word (``_lib.device_status``: 501, 502, 503); the rows of a refused step are NaN, and so are those of
the steps behind it where a batch is extended with ``after=True``. Calls on one cache have to be ordered by their streams.

A key or value that is not finite (in the cache's type) makes its block (its 64 tokens, of its head and layer) NaN, and with it
every row that sees the block. Scores, softmax statistics and sums are FP32, and the codes enter the products exactly. Queries and
softmax weights enter them with 22 bits (an FP16 number and its remainder), whichever of two kernels a step takes, which follows
from an estimate of their times. Below FP16's normal numbers
2^-36 of a row's largest product of weight and value scale is kept in steps of many tokens, 2^-40 of its largest weight in steps
of few; values of the tail are held to 2^-31 of the largest magnitude among them.
"""

import ctypes

from . import _lib

BLOCK_TOKENS = 64


def _torch():
    import torch
    return torch


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _launch(device, name, *args):
    """The entry point on the current stream of ``device`` (appended as the last argument), whatever device is current."""
    torch = _torch()
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        _lib.call(name, *args, stream)
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, stream)


def _dtype_id(t, what):
    ident = _lib.DTYPE_ID.get(str(t.dtype)[6:])
    if ident is None:
        raise TypeError(f"{what} must be FP32, FP16 or BF16")
    return ident


def _ints(values, device):
    """Python integers as an int32 tensor on ``device``, on its current stream: from pinned memory, so that nothing waits for what
    the stream still has to do. Not while the stream is captured: a replay would read host memory that others have by then."""
    torch = _torch()
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("make batches before the capture, and give fork and free tensors on the device")
    return torch.tensor(values, dtype=torch.int32, pin_memory=True).to(device, non_blocking=True)


class KV8Batch:
    """One step's sequences: ``slots`` [B], ``offsets`` [B + 1] (row of each sequence's first new token) and ``starts`` [B]
    (tokens before the step, written by ``PagedKV8Cache.extend``; -1: it was refused, -2: there was none yet), int32 on the device; on the host the number of rows, the most
    new tokens of a sequence and a bound on the tokens a sequence holds after the step."""

    def __init__(self, slots, offsets, starts, rows, max_new, max_keys, limits):
        self.limits = limits                             # sequences and max_length of the cache that it was made for
        self.slots, self.offsets, self.starts = slots, offsets, starts
        self.rows, self.max_new, self.max_keys = rows, max_new, max_keys
        self.size = slots.shape[0]
        self._pointers = (slots.data_ptr(), offsets.data_ptr(), starts.data_ptr())


class PagedKV8Cache:
    def __init__(self, layers, kv_heads, head_dim, *, pages, sequences, max_length, dtype="bfloat16", device="cuda"):
        torch = _torch()
        if min(layers, kv_heads, pages, sequences, max_length) < 1:
            raise ValueError("layers, kv_heads, pages, sequences and max_length must be positive")
        dtype = getattr(torch, dtype) if isinstance(dtype, str) else dtype
        blocks = max(1, -(-max_length // BLOCK_TOKENS))
        zeros = lambda shape, kind: torch.zeros(shape, dtype=kind, device=device)  # noqa: E731
        self._bind(zeros((pages, layers, 2, kv_heads, BLOCK_TOKENS * head_dim), torch.int8),
                   zeros((pages, layers, 2, kv_heads), torch.float32),
                   zeros((sequences, layers, 2, kv_heads, BLOCK_TOKENS, head_dim), dtype),
                   zeros((sequences, layers, 2, kv_heads), torch.float32),
                   zeros((sequences, blocks), torch.int32) - 1, zeros(sequences, torch.int32), zeros(pages, torch.int32),
                   None, max_length)

    @classmethod
    def from_tensors(cls, codes, scales, tail, peak, table, lengths, refs, max_length=None):
        """A cache over existing tensors (a snapshot that was saved, another program's pool), which it uses in place: shapes and
        meaning as in include/b200q.h. ``max_length`` defaults to what the table has room for."""
        cache = cls.__new__(cls)
        cache._bind(codes, scales, tail, peak, table, lengths, refs, None, max_length)
        return cache

    def _bind(self, codes, scales, tail, peak, table, lengths, refs, free_bits, max_length):
        torch = _torch()
        parts = (codes, scales, tail, peak, table, lengths, refs)
        if not all(isinstance(t, torch.Tensor) and t.is_cuda for t in parts):
            raise TypeError("a cache is made of torch CUDA tensors")
        if tail.ndim != 6 or table.ndim != 2 or codes.ndim != 5:
            raise ValueError("codes, tail and table have 5, 6 and 2 dimensions")
        pages, layers, _, kv_heads, _ = codes.shape
        sequences, head_dim, blocks = tail.shape[0], tail.shape[5], table.shape[1]
        if head_dim not in (64, 128):
            raise NotImplementedError("head_dim must be 64 or 128")
        if tail.dtype not in (torch.float16, torch.bfloat16):
            raise NotImplementedError("the tail is FP16 or BF16 (softmax weights pass the tensor cores in 16 bits)")
        expected = {"codes": (codes, (pages, layers, 2, kv_heads, BLOCK_TOKENS * head_dim), torch.int8),
                    "scales": (scales, (pages, layers, 2, kv_heads), torch.float32),
                    "tail": (tail, (sequences, layers, 2, kv_heads, BLOCK_TOKENS, head_dim), tail.dtype),
                    "peak": (peak, (sequences, layers, 2, kv_heads), torch.float32),
                    "table": (table, (sequences, blocks), torch.int32), "lengths": (lengths, (sequences,), torch.int32),
                    "refs": (refs, (pages,), torch.int32)}
        for name, (t, shape, dtype) in expected.items():
            if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous() or t.device != codes.device:
                raise ValueError(f"{name}: expected a contiguous {dtype} tensor {shape} on {codes.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
        room = blocks * BLOCK_TOKENS + BLOCK_TOKENS - 1
        max_length = blocks * BLOCK_TOKENS if max_length is None else int(max_length)
        if not 1 <= max_length <= room:
            raise ValueError(f"max_length must be 1..{room} for a table of {blocks} blocks")
        if free_bits is None:
            free = torch.zeros(-(-pages // 32) * 32, dtype=torch.int64, device=codes.device)
            free[:pages] = refs == 0
            words = (free.reshape(-1, 32) << torch.arange(32, device=codes.device)).sum(1)
            free_bits = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
        self.codes, self.scales, self.tail, self.peak = codes, scales, tail, peak
        self.table, self.lengths, self.refs, self.free_bits = table, lengths, refs, free_bits
        self.layers, self.kv_heads, self.head_dim, self.pages = layers, kv_heads, head_dim, pages
        self.sequences, self.max_length, self.dtype, self.device = sequences, max_length, tail.dtype, codes.device
        self._struct = _lib.KV8CacheStruct(*[_ptr(t) for t in (codes, scales, tail, peak, table, lengths, refs, free_bits)],
                                           layers, kv_heads, head_dim, pages, sequences, blocks, max_length,
                                           _lib.DTYPE_ID[str(tail.dtype)[6:]])
        self._c, self._index = ctypes.addressof(self._struct), codes.device.index

    # ------------------------------------------------------------------------------------------------ sequences and pages
    def batch(self, slots, counts, *, max_keys=None):
        """The sequences of a step (distinct slots, Python integers) and how many new tokens each brings (0: it takes part
        without any). ``max_keys`` bounds the tokens a sequence holds after the step; the default ``max_length`` is always right,
        a smaller one lets ``attention`` divide short contexts better."""
        slots, counts = [int(s) for s in slots], [int(n) for n in counts]
        if not slots or len(slots) != len(counts):
            raise ValueError("slots and counts must be of the same length, at least one")
        if len(set(slots)) != len(slots) or min(slots) < 0 or max(slots) >= self.sequences:
            raise ValueError(f"slots must be distinct and within 0..{self.sequences - 1}")
        if min(counts) < 0 or max(counts) > self.max_length:
            raise ValueError(f"new tokens must be within 0..{self.max_length}")
        max_keys = self.max_length if max_keys is None else int(max_keys)
        if not max(1, max(counts)) <= max_keys <= self.max_length:
            raise ValueError(f"max_keys must be within {max(1, max(counts))}..{self.max_length}")
        offsets = [0]
        for n in counts:
            offsets.append(offsets[-1] + n)
        if offsets[-1] >= 2 ** 31:
            raise ValueError("too many tokens in one step")
        ints = _ints(slots + offsets + [-2] * len(slots), self.device)
        b = len(slots)
        return KV8Batch(ints[:b], ints[b:2 * b + 1], ints[2 * b + 1:], offsets[-1], max(counts), max_keys,
                        (self.sequences, self.max_length))

    def _check_batch(self, batch):
        if not isinstance(batch, KV8Batch) or batch.slots.device != self.device:
            raise TypeError("batch must come from this cache's batch()")
        if batch.limits != (self.sequences, self.max_length):
            raise ValueError("batch was made for a cache of other sizes")
        return batch

    def extend(self, batch, *, after=False):
        """The sequences of ``batch`` grow by their new tokens: ``batch.starts`` gets their lengths before, pages are taken for the
        blocks that become full. All sequences or none (status 501 / 502, ``starts`` -1). ``after``: a batch whose step before was
        refused (its ``starts`` are -1) is refused again (status 504), for programs that do not look at every step."""
        self._check_batch(batch)
        slots, offsets, starts = batch._pointers
        host = _lib.host()
        if host is None or not host.kv8_extend(self._c, self._index, slots, offsets, batch.size, starts, bool(after)):
            _launch(self.device, "b200q_kv8_extend_after" if after else "b200q_kv8_extend", self._c, slots, offsets, batch.size, starts)
        return batch

    def _slots(self, slots):
        torch = _torch()
        if isinstance(slots, torch.Tensor):
            if slots.dtype != torch.int32 or slots.ndim != 1 or not slots.is_contiguous() or slots.device != self.device:
                raise ValueError(f"slots must be a contiguous int32 tensor on {self.device}")
            if slots.shape[0] > self.sequences:
                raise ValueError("more slots than sequences")
            return slots
        slots = [int(s) for s in slots]
        if len(set(slots)) != len(slots) or (slots and (min(slots) < 0 or max(slots) >= self.sequences)):
            raise ValueError(f"slots must be distinct and within 0..{self.sequences - 1}")
        return _ints(slots, self.device)

    def fork(self, src, dst):
        """Every empty sequence ``dst[i]`` becomes a copy of ``src[i]`` (sources may repeat): full pages are shared, the tail is
        copied. Python integers or int32 device tensors; all pairs or none (status 503)."""
        torch = _torch()
        if not isinstance(src, torch.Tensor):
            src = [int(s) for s in src]
            if src and (min(src) < 0 or max(src) >= self.sequences):
                raise ValueError(f"slots must be within 0..{self.sequences - 1}")
            if not isinstance(dst, torch.Tensor) and set(src) & {int(d) for d in dst}:
                raise ValueError("a target of a fork cannot be a source too")
            src = _ints(src, self.device)
        src, dst = self._slots(src), self._slots(dst)
        if src.shape != dst.shape:
            raise ValueError("src and dst must be of the same length")
        if src.shape[0]:
            host = _lib.host()
            if host is None or not host.kv8_fork(self._c, self._index, src.data_ptr(), dst.data_ptr(), src.shape[0]):
                scratch = torch.empty(1, dtype=torch.int32, device=self.device)
                _launch(self.device, "b200q_kv8_fork", self._c, src.data_ptr(), dst.data_ptr(), src.shape[0], scratch.data_ptr())

    def free(self, slots):
        """The sequences become empty; pages that no sequence refers to any more return to the pool."""
        slots = self._slots(slots)
        if slots.shape[0]:
            host = _lib.host()
            if host is None or not host.kv8_free(self._c, self._index, slots.data_ptr(), slots.shape[0]):
                _launch(self.device, "b200q_kv8_free", self._c, slots.data_ptr(), slots.shape[0])

    def compact(self, pages=None):
        """A new cache, independent of this one, with the same sequences and a pool of ``pages`` pages (default: the live ones)
        that begins with the live pages in their order. Waits for the device to count them (not for the copies)."""
        torch = _torch()
        if pages is None:
            pages = max(1, self.read_live_pages())
        pages = int(pages)
        if pages < 1:
            raise ValueError("pages must be positive")
        like = lambda t, n=None: torch.empty((n or t.shape[0],) + t.shape[1:], dtype=t.dtype, device=self.device)  # noqa: E731
        new = type(self).__new__(type(self))
        new._bind(like(self.codes, pages), like(self.scales, pages), like(self.tail), like(self.peak), like(self.table),
                  like(self.lengths), like(self.refs, pages), torch.empty(-(-pages // 32), dtype=torch.int32, device=self.device),
                  self.max_length)
        size = _lib.load().b200q_kv8_compact_workspace(self._c, new._c)
        space = torch.empty(size // 4, dtype=torch.int32, device=self.device)
        with torch.cuda.device(self.device):
            _launch(self.device, "b200q_kv8_compact_plan", self._c, new._c, space.data_ptr(), size)
            live = torch.empty(1, dtype=torch.int32, pin_memory=True)
            live.copy_(space[:1], non_blocking=True)
            counted = torch.cuda.Event()
            counted.record()
            _launch(self.device, "b200q_kv8_compact_move", self._c, new._c, space.data_ptr(), size)
            counted.synchronize()
        if int(live) > pages:
            raise ValueError(f"{int(live)} live pages do not fit a pool of {pages}")
        return new

    def read_live_pages(self):
        """Pages that some sequence refers to (waits for the device)."""
        return int(_torch().count_nonzero(self.refs))

    def read_lengths(self):
        """Tokens held by every sequence, as a list (waits for the device)."""
        return self.lengths.tolist()

    # ------------------------------------------------------------------------------------------------ tokens
    def _rope(self, rope):
        if rope is None:
            return None, None, 0
        cos, sin = rope
        torch = _torch()
        for t in (cos, sin):
            if (t.dtype != torch.float32 or t.ndim != 2 or t.shape[1] * 2 != self.head_dim or not t.is_contiguous()
                    or t.device != self.device):
                raise ValueError(f"RoPE tables must be contiguous FP32 [positions, {self.head_dim // 2}] on {self.device}")
        if cos.shape != sin.shape or cos.shape[0] < self.max_length:
            raise ValueError(f"RoPE tables of {cos.shape[0]} positions for sequences of up to {self.max_length} tokens")
        return cos.data_ptr(), sin.data_ptr(), cos.shape[0]

    def _layer(self, layer):
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} out of range 0..{self.layers - 1}")
        return layer

    def _rows(self, x, batch, width, what):
        if x.ndim != 2 or x.shape[0] != batch.rows or x.shape[1] != width or x.device != self.device:
            raise ValueError(f"{what} must be [{batch.rows}, {width}] on {self.device}, got {tuple(x.shape)} on {x.device}")
        if x.shape[0] and (x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < width)):
            raise ValueError(f"{what} must have rows of consecutive elements that do not overlap")
        return x.stride(0) if x.shape[0] > 1 else width

    def append(self, layer, k, v, batch, *, rope=None):
        """Keys and values ``[rows, kv_heads * head_dim]`` (FP32, FP16 or BF16; column slices of a projection output will do) of
        the new tokens of one layer, after ``extend(batch)``. ``rope`` = (cos, sin) tables ``[positions, head_dim / 2]``: the keys
        are rotated to their positions (rotate-half) first."""
        self._check_batch(batch)
        host = _lib.host()
        if host is not None and type(layer) is int:
            cos, sin = rope or (None, None)
            if host.kv8_append(self._c, self._index, layer, k, v, *batch._pointers, batch.size, batch.rows, batch.max_new, cos, sin):
                return
        width = self.kv_heads * self.head_dim
        k_row, v_row = self._rows(k, batch, width, "k"), self._rows(v, batch, width, "v")
        if k.dtype != v.dtype:
            raise TypeError("k and v must have the same type")
        cos, sin, positions = self._rope(rope)
        if batch.rows:
            _launch(self.device, "b200q_kv8_append", self._c, self._layer(layer), k.data_ptr(), v.data_ptr(), _dtype_id(k, "k"), k_row, v_row,
                    *batch._pointers, batch.size, batch.max_new, cos, sin, positions)

    def attention(self, layer, q, batch, *, rope=None, scale=None, out=None):
        """Causal attention of the new tokens over the cache they are in (after ``append``): ``q`` ``[rows, heads * head_dim]``
        (FP32, FP16 or BF16; rotated here when ``rope`` is given) -> ``[rows, heads * head_dim]`` in the cache's type. ``heads`` is a
        multiple of ``kv_heads``; ``scale`` defaults to ``head_dim ** -0.5``."""
        self._check_batch(batch)
        host = _lib.host()
        if host is not None and type(layer) is int:
            cos, sin = rope or (None, None)
            result = host.kv8_attention(self._c, self._index, layer, q, *batch._pointers, batch.size, batch.rows, batch.max_new, batch.max_keys,
                                        cos, sin, self.head_dim ** -0.5 if scale is None else scale, out)
            if result is not None:
                return result
        torch = _torch()
        heads = q.shape[1] // self.head_dim if q.ndim == 2 else 0
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"q must be [rows, heads * {self.head_dim}] with heads a multiple of {self.kv_heads}")
        q_row = self._rows(q, batch, heads * self.head_dim, "q")
        cos, sin, positions = self._rope(rope)
        if out is None:
            out = torch.empty(q.shape, dtype=self.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != self.dtype or not out.is_contiguous() or out.device != self.device:
            raise ValueError(f"out must be a contiguous {self.dtype} tensor {tuple(q.shape)} on {self.device}")
        if batch.rows:
            size = _lib.load().b200q_kv8_attention_workspace(self._c, heads, batch.size, batch.rows, batch.max_new, batch.max_keys)
            space = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
            _launch(self.device, "b200q_kv8_attention", self._c, self._layer(layer), q.data_ptr(), _dtype_id(q, "q"), q_row, heads,
                    *batch._pointers, batch.size, batch.rows, batch.max_new, batch.max_keys, cos, sin, positions,
                    float(self.head_dim ** -0.5 if scale is None else scale), out.data_ptr(), _ptr(space), size)
        return out
