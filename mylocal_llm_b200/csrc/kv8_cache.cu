// Paged 8-bit key/value cache (layout: kv8_cache.cuh): taking pages, appending tokens, sharing, dropping and packing pages.
#include "kv8_cache.cuh"

namespace b200q {

constexpr int EXTEND_THREADS = 1024;

// Exclusive prefix sum over the CTA (1024 threads); *total gets the sum.
__device__ __forceinline__ int block_prefix(int v, int *total) {
    __shared__ int warp_sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    __syncthreads();                                     // (the sums of a previous call have been read)
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        const int s = lane < blockDim.x / 32 ? warp_sums[lane] : 0;
        int t = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += up;
        }
        warp_sums[lane] = t;
    }
    __syncthreads();
    *total = warp_sums[31];
    return incl - v + (warp ? warp_sums[warp - 1] : 0);
}

// Every sequence slots[b] grows by offsets[b + 1] - offsets[b] tokens: it gets a page for each block that becomes full
// (the lowest free pages, in the order of the requests), starts[b] its length before. All or nothing: without enough pages,
// or where a sequence would pass max_length, nothing changes, every start is -1 (which the other kernels skip) and the
// status word tells. `after`: the batch's starts are those of the step before, and where that was refused this one is too: a
// program that has not looked must not go on with a sequence that lacks those tokens. One CTA: the work is a prefix sum over the
// batch and, only when a block becomes full, a pass over the free bits (32 pages per word), so a decode step costs little more
// than its launch.
__global__ void __launch_bounds__(EXTEND_THREADS) kv8_extend_kernel(const b200q_kv8_cache c, const int32_t *slots,
                                                                    const int32_t *offsets, int batch, int32_t *starts, int after,
                                                                    int *status) {
    chain_trigger();
    chain_wait();
    // A batch that fits is held by the threads, entry by entry; shared memory has what every page taken looks up: its entry's
    // first request, slot and length.
    __shared__ int first_s[EXTEND_THREADS], slot_s[EXTEND_THREADS], have_s[EXTEND_THREADS];
    const int tid = threadIdx.x, words = (c.pages + 31) / 32;
    const bool small = batch <= EXTEND_THREADS;
    const uint32_t early = tid < words ? c.free_bits[tid] : 0u;          // the first words are on their way meanwhile
    int carry = 0, bad = 0, my_slot = 0, my_have = 0, my_add = 0;        // bad: the status word
    for (int b0 = 0; b0 < batch; b0 += EXTEND_THREADS) {
        const int b = b0 + tid;
        int need = 0;
        if (b < batch) {
            my_slot = slots[b];
            my_add = offsets[b + 1] - offsets[b];
            if (after && starts[b] == KV8_REFUSED) {
                bad = STATUS_KV8_FOLLOWS;
            } else if (my_slot < 0 || my_slot >= c.sequences || my_add < 0) {
                bad = STATUS_KV8_LENGTH;
            } else {
                my_have = c.lengths[my_slot];
                if (my_have < 0 || my_add > c.max_length - my_have) bad = STATUS_KV8_LENGTH;
                else need = (my_have + my_add) / KV8_BLOCK - my_have / KV8_BLOCK;
            }
        }
        int sum;
        const int before = block_prefix(need, &sum);
        if (b < batch) {                                 // first page request of the entry, until the pages are assigned
            if (small) {
                first_s[b] = before;
                slot_s[b] = my_slot;
                have_s[b] = my_have;
            } else {
                starts[b] = carry + before;
            }
        }
        carry += sum;
    }
    if (bad == STATUS_KV8_FOLLOWS) atomicCAS(status, 0, bad);            // (the first refusal's word says why)
    else if (bad) atomicExch(status, bad);
    bad = __syncthreads_or(bad);
    const int *request = small ? first_s : starts;
    const int total = carry;
    if (total > 0 && !bad) {
        int all, first_rank = 0;
        if (words <= EXTEND_THREADS) {                   // one pass over the words
            first_rank = block_prefix(__popc(early), &all);
        } else {
            int have = 0;
            for (int w = tid; w < words; w += EXTEND_THREADS) have += __popc(c.free_bits[w]);
            block_prefix(have, &all);
        }
        if (all < total) {
            if (tid == 0) atomicExch(status, STATUS_KV8_POOL);
            for (int b = tid; b < batch; b += EXTEND_THREADS) starts[b] = KV8_REFUSED;
            return;
        }
        int rank = 0;
        for (int w0 = 0; w0 < words && rank < total; w0 += EXTEND_THREADS) {
            const int w = w0 + tid;
            const uint32_t bits = w0 == 0 ? early : w < words ? c.free_bits[w] : 0u;
            int sum = all, r = first_rank;
            if (words > EXTEND_THREADS) r = rank + block_prefix(__popc(bits), &sum);
            rank += sum;
            if (bits == 0u || r >= total) continue;
            uint32_t left = bits;
            int e = 0;                                   // entry of request r: the last with starts[e] <= r that needs any
            for (int lo = 0, hi = batch - 1; lo <= hi;) {
                const int mid = (lo + hi) >> 1;
                if (request[mid] <= r) { e = mid; lo = mid + 1; } else { hi = mid - 1; }
            }
            while (left && r < total) {
                const int bit = __ffs(left) - 1;
                left &= left - 1;
                while (e + 1 < batch && request[e + 1] <= r) ++e;
                const int page = w * 32 + bit, slot = small ? slot_s[e] : slots[e], have = small ? have_s[e] : c.lengths[slot];
                c.table[static_cast<size_t>(slot) * c.blocks + have / KV8_BLOCK + (r - request[e])] = page;
                c.refs[page] = 1;
                ++r;
            }
            c.free_bits[w] = left;
        }
        __syncthreads();
    }
    for (int b = tid; b < batch; b += EXTEND_THREADS) {
        if (bad) {
            starts[b] = KV8_REFUSED;
        } else {
            if (!small) {
                my_slot = slots[b];
                my_have = c.lengths[my_slot];
                my_add = offsets[b + 1] - offsets[b];
            }
            starts[b] = my_have;
            c.lengths[my_slot] = my_have + my_add;
        }
    }
}

// ------------------------------------------------------------------------------------------------------------- append
struct Kv8Append {
    const void *k, *v;
    long long k_row, v_row;
    int layer;
    const int32_t *slots, *offsets, *starts;
    const float *cos_t, *sin_t;           // [rope_rows][head_dim / 2], or NULL: keys are stored as they come
};

// Four consecutive values of type IN as they are loaded (held in few registers until they are used). VEC: base and strides are
// such that one 8- or 16-byte load fetches them.
template <int IN> struct RawQuad { uint2 w; };
template <> struct RawQuad<B200Q_F32> { float4 w; };
template <int IN, bool VEC>
__device__ __forceinline__ RawQuad<IN> load_quad(const void *p, size_t i) {
    RawQuad<IN> r;
    if constexpr (IN == B200Q_F32) {
        const float *q = static_cast<const float *>(p) + i;
        if (VEC) r.w = *reinterpret_cast<const float4 *>(q);
        else r.w = make_float4(q[0], q[1], q[2], q[3]);
    } else {
        const uint16_t *q = static_cast<const uint16_t *>(p) + i;
        if (VEC) r.w = *reinterpret_cast<const uint2 *>(q);
        else r.w = make_uint2(q[0] | (static_cast<uint32_t>(q[1]) << 16), q[2] | (static_cast<uint32_t>(q[3]) << 16));
    }
    return r;
}
template <bool BF16> __device__ __forceinline__ float2 unpack16(uint32_t w);
template <int IN>
__device__ __forceinline__ void quad_values(const RawQuad<IN> &r, float (&f)[4]) {
    if constexpr (IN == B200Q_F32) {
        f[0] = r.w.x; f[1] = r.w.y; f[2] = r.w.z; f[3] = r.w.w;
    } else {
        const float2 a = unpack16<IN == B200Q_BF16>(r.w.x), b = unpack16<IN == B200Q_BF16>(r.w.y);
        f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&p);
    }
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&p);
}
template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
    return BF16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

// Rotated pairs of four consecutive dimensions, rounded to FP32 and then to the cache's type as if both products and their sum
// were exact up to 64 bits (both products are): what a cache holds then follows from the inputs alone, whatever order another
// program computes in. FP32 first: with the error's bound added and taken off, both ends round to the same 16-bit number
// unless a border lies between them, which about one in 2^11 (BF16) values meets; then the quad goes through 64 bits.
template <bool BF16>
static __device__ __noinline__ uint4 rotate_exact(float4 x0, float4 x1, float4 c, float4 s) {
    auto lo = [](float a, float b, float cc, float ss) {
        return __double2float_rn(__fma_rn(static_cast<double>(a), static_cast<double>(cc), -__dmul_rn(static_cast<double>(b), static_cast<double>(ss))));
    };
    auto hi = [](float a, float b, float cc, float ss) {
        return __double2float_rn(__fma_rn(static_cast<double>(a), static_cast<double>(ss), __dmul_rn(static_cast<double>(b), static_cast<double>(cc))));
    };
    return make_uint4(pack16<BF16>(lo(x0.x, x1.x, c.x, s.x), lo(x0.y, x1.y, c.y, s.y)), pack16<BF16>(lo(x0.z, x1.z, c.z, s.z), lo(x0.w, x1.w, c.w, s.w)),
                      pack16<BF16>(hi(x0.x, x1.x, c.x, s.x), hi(x0.y, x1.y, c.y, s.y)), pack16<BF16>(hi(x0.z, x1.z, c.z, s.z), hi(x0.w, x1.w, c.w, s.w)));
}
// out: the quad at i as two words, then its partner's.
template <bool BF16>
__device__ __forceinline__ void rotate_quad(const float (&x0)[4], const float (&x1)[4], const float (&c)[4], const float (&s)[4], uint32_t (&out)[4]) {
    constexpr float BOUND = 1.1920929e-7f;               // 2^-23: product, sum and the reference's own FP32 rounding, 2^-24 each
    uint32_t differ = 0u;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            float v[2], w[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int i = 2 * p + e;
                const float product = h ? __fmul_rn(x1[i], c[i]) : -__fmul_rn(x1[i], s[i]);
                v[e] = __fmaf_rn(x0[i], h ? s[i] : c[i], product);
                w[e] = __fmul_rn(fabsf(product) + fabsf(v[e]), BOUND);
            }
            out[2 * h + p] = pack16<BF16>(v[0] + w[0], v[1] + w[1]);
            differ |= out[2 * h + p] ^ pack16<BF16>(v[0] - w[0], v[1] - w[1]);
        }
    if (differ) {                                        // (by value: arrays that a call gets by address live in memory)
        const uint4 r = rotate_exact<BF16>(make_float4(x0[0], x0[1], x0[2], x0[3]), make_float4(x1[0], x1[1], x1[2], x1[3]),
                                           make_float4(c[0], c[1], c[2], c[3]), make_float4(s[0], s[1], s[2], s[3]));
        out[0] = r.x;
        out[1] = r.y;
        out[2] = r.z;
        out[3] = r.w;
    }
}

// One CTA of 2 DH threads = the keys or the values of one block of 64 tokens of one sequence and head; the CTAs of a row's heads
// follow one another, so that rows are read whole. A thread holds four consecutive tokens x (a quad of dimensions at i and its
// partner at i + DH / 2, which the rotation needs), as 16-bit pairs. A block that becomes full takes its older tokens from the tail and finds the largest
// magnitude (16-bit integers order 16-bit floats, NaN and infinities on top); keys go out as words of four codes, values as words
// of four tokens of a dimension (a transposition of bytes in registers) that pass through shared memory. One that does not become
// full goes to the tail. Bound by memory - every new token is read once, as projection output, and written once - and, next to
// it, by the instructions per element: with 64-bit rotations, exact codes one by one and byte stores 3 x 8192 tokens took 83 us, now 26
// (10 at the measured bandwidth; 0.65 of the issue slots).
// All loads of inputs are issued before the first is used (rows past the ends repeat the first or last one); registers are held to
// what lets half of an SM's threads be resident.
template <int DH, bool BF16, int IN, bool VEC>
__global__ void __launch_bounds__(2 * DH, 1024 / (2 * DH)) kv8_append_kernel(const b200q_kv8_cache c, const Kv8Append a) {
    constexpr int HALF = DH / 2, QUADS = HALF / 4, WARPS = DH / 16, LD = KV8_BLOCK / 4 + 1;      // warps per part; words of a row
    __shared__ uint32_t v_s[DH * LD];
    __shared__ uint32_t peaks[WARPS];
    chain_trigger();
    chain_wait();
    const int at = threadIdx.x, part = blockIdx.x & 1, b = blockIdx.z, head = blockIdx.x >> 1;
    const int start = a.starts[b], row0 = a.offsets[b], n = a.offsets[b + 1] - row0;
    if (start < 0 || n <= 0) return;
    const int total = start + n, first = start / KV8_BLOCK, last = (total - 1) / KV8_BLOCK;
    int block = first + blockIdx.y;
    if (block > last) return;
    const bool opened = start % KV8_BLOCK != 0;          // the first block holds older tokens
    // The tail is read for the first block and written for the last: where these are two blocks, one CTA does both, in that
    // order.
    const bool both = opened && last > first && total % KV8_BLOCK != 0;
    if (both && block == last) return;
    const int slot = a.slots[b];
    const size_t unit = kv8_unit(slot, c.layers, a.layer, part, c.kv_heads, head);
    uint16_t *tail = static_cast<uint16_t *>(c.tail) + unit * (KV8_BLOCK * DH);
    const int i = (at % QUADS) * 4, t0 = at / QUADS * 4;
    const void *in = part ? a.v : a.k;
    const long long in_row = part ? a.v_row : a.k_row;

    for (;; block = last) {
        const int base = block * KV8_BLOCK;
        const bool full = base + KV8_BLOCK <= total;
        uint32_t x[4][4];                                // [token][quad as two words, partner]
        uint32_t top = 0u;
        const bool turn = part == 0 && a.cos_t;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0u;
        const int page = full ? c.table[static_cast<size_t>(slot) * c.blocks + block] : 0;
        if (full || (base + t0 + 3 >= start && base + t0 < total)) {         // (few threads have a token of a decode step)
            RawQuad<IN> lo[4], hi[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int pos = min(max(base + t0 + j, start), total - 1);
                const size_t from = (row0 + (pos - start)) * static_cast<size_t>(in_row) + static_cast<size_t>(head) * DH + i;
                lo[j] = load_quad<IN, VEC>(in, from);
                hi[j] = load_quad<IN, VEC>(in, from + HALF);
            }
#pragma unroll
            for (int jj = 0; jj < 4; jj += 2) {
                float4 cq[2], sq[2];
                if (turn)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const size_t from = static_cast<size_t>(min(max(base + t0 + jj + j, start), total - 1)) * HALF + i;
                        cq[j] = *reinterpret_cast<const float4 *>(a.cos_t + from);
                        sq[j] = *reinterpret_cast<const float4 *>(a.sin_t + from);
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float l4[4], h4[4];
                    quad_values<IN>(lo[jj + j], l4);
                    quad_values<IN>(hi[jj + j], h4);
                    if (turn) {
                        const float cv[4] = {cq[j].x, cq[j].y, cq[j].z, cq[j].w}, sv[4] = {sq[j].x, sq[j].y, sq[j].z, sq[j].w};
                        rotate_quad<BF16>(l4, h4, cv, sv, x[jj + j]);
                    } else {
                        x[jj + j][0] = pack16<BF16>(l4[0], l4[1]);
                        x[jj + j][1] = pack16<BF16>(l4[2], l4[3]);
                        x[jj + j][2] = pack16<BF16>(h4[0], h4[1]);
                        x[jj + j][3] = pack16<BF16>(h4[2], h4[3]);
                    }
                }
            }
            if (base < start || !full)                       // (only the first block has older tokens, only the last empty places)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int pos = base + t0 + j;
                    if (pos >= start && pos < total) continue;
                    uint2 u = make_uint2(0u, 0u), w = u;
                    if (full) {
                        u = *reinterpret_cast<const uint2 *>(tail + (t0 + j) * DH + i);
                        w = *reinterpret_cast<const uint2 *>(tail + (t0 + j) * DH + i + HALF);
                    }
                    x[j][0] = u.x;
                    x[j][1] = u.y;
                    x[j][2] = w.x;
                    x[j][3] = w.y;
                }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = __vmaxu2(top, x[j][e] & 0x7fff7fffu);
        }
        top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
        if ((at & 31) == 0) peaks[at >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = max(top, peaks[w]);
        const uint32_t peak = abs_bits(unpack16<BF16>(top).x);
        if (full) {
            const float s = int8_scale(peak), inv = __fdiv_rn(1.f, s);
            const bool held = page >= 0 && page < c.pages;       // (a table that lacks the page loses the block, not memory)
            const size_t u = kv8_unit(held ? page : 0, c.layers, a.layer, part, c.kv_heads, head);
            int8_t *to = c.codes + u * (KV8_BLOCK * DH);
            uint32_t code[2][4];                         // [half][token]: four dimensions
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 p = unpack16<BF16>(x[j][2 * h]), q = unpack16<BF16>(x[j][2 * h + 1]);
                    const float v[4] = {p.x, p.y, q.x, q.y};
                    code[h][j] = int8_codes(v, s, inv);
                }
            if (part == 0) {
                if (held)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int h = 0; h < 2; ++h) *reinterpret_cast<uint32_t *>(to + (t0 + j) * DH + i + h * HALF) = code[h][j];
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {            // four tokens x four dimensions of bytes, transposed
                    const uint32_t a01 = __byte_perm(code[h][0], code[h][1], 0x5140), b01 = __byte_perm(code[h][0], code[h][1], 0x7362);
                    const uint32_t a23 = __byte_perm(code[h][2], code[h][3], 0x5140), b23 = __byte_perm(code[h][2], code[h][3], 0x7362);
                    uint32_t *row = v_s + (i + h * HALF) * LD + t0 / 4;
                    row[0] = __byte_perm(a01, a23, 0x5410);
                    row[LD] = __byte_perm(a01, a23, 0x7632);
                    row[2 * LD] = __byte_perm(b01, b23, 0x5410);
                    row[3 * LD] = __byte_perm(b01, b23, 0x7632);
                }
                __syncthreads();
                if (held)
#pragma unroll
                    for (int j = at; j < DH * 4; j += 2 * DH) {
                        const uint32_t *row = v_s + (j >> 2) * LD + 4 * (j & 3);
                        reinterpret_cast<uint4 *>(to)[j] = make_uint4(row[0], row[1], row[2], row[3]);
                    }
            }
            if (at == 0 && held) c.scales[u] = s;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int pos = base + t0 + j;
                if (pos < start || pos >= total) continue;
                *reinterpret_cast<uint2 *>(tail + (t0 + j) * DH + i) = make_uint2(x[j][0], x[j][1]);
                *reinterpret_cast<uint2 *>(tail + (t0 + j) * DH + i + HALF) = make_uint2(x[j][2], x[j][3]);
            }
            if (at == 0) {
                const uint32_t older = block == first && opened ? abs_bits(c.peak[unit]) : 0u;
                c.peak[unit] = __uint_as_float(max(peak, older));
            }
        }
        if (!both || block != first) break;
        __syncthreads();                                 // every thread has read the tail and the shared peaks
    }
}

// --------------------------------------------------------------------------------------------------------- fork, free
// fork, first kernel (one CTA): the pairs are looked over as a whole. A slot out of range, a target named twice, one that is
// not empty or that is a source too: nothing happens but status 503. *ok tells the copying kernel.
__global__ void __launch_bounds__(1024) kv8_fork_check_kernel(const b200q_kv8_cache c, const int32_t *src, const int32_t *dst,
                                                              int count, int32_t *ok, int *status) {
    __shared__ uint32_t named[KV8_MAX_SEQUENCES / 32];
    chain_trigger();
    chain_wait();
    const int tid = threadIdx.x;
    for (int w = tid; w < KV8_MAX_SEQUENCES / 32; w += 1024) named[w] = 0u;
    __syncthreads();
    int bad = 0;
    for (int i = tid; i < count; i += 1024) {
        const int s = src[i], d = dst[i];
        if (s < 0 || s >= c.sequences || d < 0 || d >= c.sequences) {
            bad = 1;
            continue;
        }
        if (atomicOr(&named[d >> 5], 1u << (d & 31)) & (1u << (d & 31))) bad = 1;
        if (c.lengths[d] != 0) bad = 1;
    }
    __syncthreads();
    if (!bad)
        for (int i = tid; i < count; i += 1024)
            if (src[i] >= 0 && src[i] < c.sequences && (named[src[i] >> 5] >> (src[i] & 31) & 1u)) bad = 1;
    bad = __syncthreads_or(bad);
    if (tid == 0) {
        *ok = !bad;
        if (bad) atomicExch(status, STATUS_KV8_SLOTS);
    }
    if (bad) return;
    for (int i = tid; i < count; i += 1024) c.lengths[dst[i]] = c.lengths[src[i]];
}

constexpr int COPY_PIECES = 8;               // 16-byte pieces in flight per thread of the copying kernels

// fork, second kernel: CTA (0, i) copies the table row of pair i and counts its pages, CTA (1 + layer, i) the tokens of the
// tail of one layer - rows below length % 64 only, as 16-byte pieces.
__global__ void __launch_bounds__(256) kv8_fork_copy_kernel(const b200q_kv8_cache c, const int32_t *src, const int32_t *dst,
                                                            const int32_t *ok) {
    chain_trigger();
    chain_wait();
    if (!*ok) return;
    const int tid = threadIdx.x, s = src[blockIdx.y], d = dst[blockIdx.y], length = c.lengths[s];
    if (blockIdx.x == 0) {
        const int held = min(length / KV8_BLOCK, c.blocks);
        for (int j = tid; j < held; j += 256) {
            const int page = c.table[static_cast<size_t>(s) * c.blocks + j];
            c.table[static_cast<size_t>(d) * c.blocks + j] = page;
            if (page >= 0 && page < c.pages) atomicAdd(c.refs + page, 1);
        }
        return;
    }
    const int layer = blockIdx.x - 1, units = 2 * c.kv_heads;
    const size_t from = kv8_unit(s, c.layers, layer, 0, c.kv_heads, 0), to = kv8_unit(d, c.layers, layer, 0, c.kv_heads, 0);
    const int pieces = (length % KV8_BLOCK) * c.head_dim / 8, unit_pieces = KV8_BLOCK * c.head_dim / 8, all = units * pieces;
    const uint4 *tail_from = static_cast<const uint4 *>(c.tail) + from * unit_pieces;
    uint4 *tail_to = static_cast<uint4 *>(c.tail) + to * unit_pieces;
    for (int j0 = tid; j0 < all; j0 += 256 * COPY_PIECES) {
        uint4 v[COPY_PIECES];
        size_t at[COPY_PIECES];
#pragma unroll
        for (int q = 0; q < COPY_PIECES; ++q) {
            const int j = min(j0 + 256 * q, all - 1), u = j / pieces;        // (the last piece again, past the end)
            at[q] = static_cast<size_t>(u) * unit_pieces + (j - u * pieces);
            v[q] = __ldcs(tail_from + at[q]);
        }
#pragma unroll
        for (int q = 0; q < COPY_PIECES; ++q) __stcs(tail_to + at[q], v[q]);
    }
    for (int u = tid; u < units; u += 256) c.peak[to + u] = c.peak[from + u];
}

// One CTA per slot: the sequence becomes empty, and a page that no sequence refers to any more becomes free. Counts and
// free bits are the same whatever the order; a slot named twice is freed once.
__global__ void __launch_bounds__(256) kv8_free_kernel(const b200q_kv8_cache c, const int32_t *slots, int *status) {
    __shared__ int length;
    chain_trigger();
    chain_wait();
    const int slot = slots[blockIdx.x];
    if (slot < 0 || slot >= c.sequences) {
        if (threadIdx.x == 0) atomicExch(status, STATUS_KV8_SLOTS);
        return;
    }
    if (threadIdx.x == 0) length = atomicExch(c.lengths + slot, 0);
    __syncthreads();
    const int held = min(length / KV8_BLOCK, c.blocks);
    for (int j = threadIdx.x; j < held; j += 256) {
        int32_t *entry = c.table + static_cast<size_t>(slot) * c.blocks + j;
        const int page = *entry;
        *entry = -1;
        if (page >= 0 && page < c.pages && atomicSub(c.refs + page, 1) == 1)
            atomicOr(c.free_bits + (page >> 5), 1u << (page & 31));
    }
}

// ------------------------------------------------------------------------------------------------------------ compact
// First kernel (one CTA): place[page] = the live page's number in the new pool (live pages keep their order), source[] the
// reverse, and the new pool's counts and free bits.
__global__ void __launch_bounds__(1024) kv8_compact_plan_kernel(const b200q_kv8_cache c, const b200q_kv8_cache to,
                                                                int32_t *count, int32_t *place, int32_t *source) {
    chain_trigger();
    chain_wait();
    const int tid = threadIdx.x;
    int live = 0;
    for (int p0 = 0; p0 < c.pages; p0 += 1024) {
        const int p = p0 + tid;
        const int refs = p < c.pages ? c.refs[p] : 0;
        int sum;
        const int at = live + block_prefix(refs > 0, &sum);
        if (p < c.pages) place[p] = refs > 0 && at < to.pages ? at : -1;
        if (refs > 0 && at < to.pages) {
            source[at] = p;
            to.refs[at] = refs;
        }
        live += sum;
    }
    if (tid == 0) *count = live;
    for (int p = min(live, to.pages) + tid; p < to.pages; p += 1024) {
        source[p] = -1;
        to.refs[p] = 0;
    }
    for (int w = tid; w < (to.pages + 31) / 32; w += 1024) {
        const int lo = max(live - 32 * w, 0), hi = min(to.pages - 32 * w, 32);        // bits lo .. hi - 1 are free
        uint32_t bits = lo >= 32 ? 0u : 0xffffffffu << lo;
        if (hi < 32) bits &= (1u << hi) - 1u;
        to.free_bits[w] = bits;
    }
}

// Second kernel: a grid over equal pieces of everything that moves - codes and scales of the live pages, the tails and
// peaks of all sequences, table and lengths. Pure copying, bound by memory.
__global__ void __launch_bounds__(256) kv8_compact_copy_kernel(const b200q_kv8_cache c, const b200q_kv8_cache to,
                                                               const int32_t *place, const int32_t *source,
                                                               int chunks_per_page, int page_ctas, int tail_ctas) {
    chain_trigger();
    chain_wait();
    const int tid = threadIdx.x;
    const size_t page_pieces = static_cast<size_t>(c.layers) * 2 * c.kv_heads * KV8_BLOCK * c.head_dim / 16;
    const int page_scales = c.layers * 2 * c.kv_heads;
    if (static_cast<int>(blockIdx.x) < page_ctas) {
        const int page = blockIdx.x / chunks_per_page, chunk = blockIdx.x - page * chunks_per_page, from = source[page];
        if (from < 0) return;
        const uint4 *in = reinterpret_cast<const uint4 *>(c.codes) + from * page_pieces;
        uint4 *out = reinterpret_cast<uint4 *>(to.codes) + page * page_pieces;
        const size_t at = static_cast<size_t>(chunk) * 256 * COPY_PIECES + tid;
        uint4 v[COPY_PIECES];
#pragma unroll
        for (int j = 0; j < COPY_PIECES; ++j)
            if (at + 256 * j < page_pieces) v[j] = __ldcs(in + at + 256 * j);
#pragma unroll
        for (int j = 0; j < COPY_PIECES; ++j)
            if (at + 256 * j < page_pieces) __stcs(out + at + 256 * j, v[j]);
        if (chunk == 0)
            for (int j = tid; j < page_scales; j += 256)
                to.scales[static_cast<size_t>(page) * page_scales + j] = c.scales[static_cast<size_t>(from) * page_scales + j];
        return;
    }
    int cta = blockIdx.x - page_ctas;
    if (cta < tail_ctas) {
        const size_t pieces = static_cast<size_t>(c.sequences) * page_scales * KV8_BLOCK * c.head_dim / 8;
        const size_t at = static_cast<size_t>(cta) * 256 * COPY_PIECES + tid;
        uint4 v[COPY_PIECES];
#pragma unroll
        for (int j = 0; j < COPY_PIECES; ++j)
            if (at + 256 * j < pieces) v[j] = static_cast<const uint4 *>(c.tail)[at + 256 * j];
#pragma unroll
        for (int j = 0; j < COPY_PIECES; ++j)
            if (at + 256 * j < pieces) static_cast<uint4 *>(to.tail)[at + 256 * j] = v[j];
        return;
    }
    cta -= tail_ctas;                                    // the last CTAs: one per sequence
    for (int j = tid; j < c.blocks; j += 256) {
        const int page = c.table[static_cast<size_t>(cta) * c.blocks + j];
        to.table[static_cast<size_t>(cta) * c.blocks + j] = page >= 0 && page < c.pages ? place[page] : -1;
    }
    for (int j = tid; j < page_scales; j += 256)
        to.peak[static_cast<size_t>(cta) * page_scales + j] = c.peak[static_cast<size_t>(cta) * page_scales + j];
    if (tid == 0) to.lengths[cta] = c.lengths[cta];
}

// ----------------------------------------------------------------------------------------------------------- host side
using AppendFn = void (*)(const b200q_kv8_cache, const Kv8Append);
template <int DH, bool BF16, int IN>
static AppendFn append_kernel_of(bool vec) { return vec ? kv8_append_kernel<DH, BF16, IN, true> : kv8_append_kernel<DH, BF16, IN, false>; }
template <int DH>
static AppendFn append_kernel(int dtype, int in, bool vec) {
    if (dtype == B200Q_BF16)
        return in == B200Q_F32 ? append_kernel_of<DH, true, B200Q_F32>(vec) : in == B200Q_F16 ? append_kernel_of<DH, true, B200Q_F16>(vec)
                                                                                           : append_kernel_of<DH, true, B200Q_BF16>(vec);
    return in == B200Q_F32 ? append_kernel_of<DH, false, B200Q_F32>(vec) : in == B200Q_F16 ? append_kernel_of<DH, false, B200Q_F16>(vec)
                                                                                        : append_kernel_of<DH, false, B200Q_BF16>(vec);
}

int kv8_check(const char *what, const b200q_kv8_cache *c) {
    if (!c || !c->codes || !c->scales || !c->tail || !c->peak || !c->table || !c->lengths || !c->refs || !c->free_bits)
        return fail(B200Q_EINVAL, "%s: NULL pointer", what);
    if (c->layers < 1 || c->kv_heads < 1 || c->pages < 1 || c->sequences < 1 || c->blocks < 1 || c->max_length < 1)
        return fail(B200Q_EINVAL, "%s: layers, heads, pages, sequences, blocks and max_length must be positive", what);
    if (c->head_dim != 64 && c->head_dim != 128) return fail(B200Q_EUNSUPPORTED, "%s: head_dim must be 64 or 128", what);
    if (c->dtype != B200Q_F16 && c->dtype != B200Q_BF16)
        return fail(B200Q_EUNSUPPORTED, "%s: the tail is FP16 or BF16", what);
    if (c->sequences > KV8_MAX_SEQUENCES || c->pages > KV8_MAX_PAGES || c->kv_heads > 1024 || c->layers > 4096)
        return fail(B200Q_EUNSUPPORTED, "%s: at most %d sequences, %d pages, 1024 heads and 4096 layers", what,
                    KV8_MAX_SEQUENCES, KV8_MAX_PAGES);
    if (c->max_length / KV8_BLOCK > c->blocks)
        return fail(B200Q_EINVAL, "%s: max_length %d needs %d blocks, the table has %d", what, c->max_length,
                    c->max_length / KV8_BLOCK, c->blocks);
    if ((reinterpret_cast<uintptr_t>(c->codes) | reinterpret_cast<uintptr_t>(c->tail)) & 15)
        return fail(B200Q_EINVAL, "%s: codes and tail must be 16-byte aligned", what);
    return B200Q_OK;
}

}  // namespace b200q

using namespace b200q;

static int extend(const b200q_kv8_cache *cache, const int32_t *slots, const int32_t *offsets, int batch, int32_t *starts, int after,
                  void *stream) {
    if (int rc = kv8_check("kv8_extend", cache)) return rc;
    if (batch == 0) return B200Q_OK;
    if (!slots || !offsets || !starts) return fail(B200Q_EINVAL, "kv8_extend: NULL pointer");
    if (batch < 0 || batch > cache->sequences) return fail(B200Q_EINVAL, "kv8_extend: batch %d out of range", batch);
    if (batch > KV8_MAX_STEP) return fail(B200Q_EUNSUPPORTED, "kv8_extend: at most %d sequences per step", KV8_MAX_STEP);
    int *status = device_status_word();
    if (!status) return fail(B200Q_ECUDA, "kv8_extend: no CUDA device");
    launch_chained(kv8_extend_kernel, dim3(1), dim3(EXTEND_THREADS), 0, static_cast<cudaStream_t>(stream), *cache, slots,
                   offsets, batch, starts, after, status);
    return check_launch("kv8_extend");
}

extern "C" int b200q_kv8_extend(const b200q_kv8_cache *cache, const int32_t *slots, const int32_t *offsets, int batch,
                                int32_t *starts, void *stream) {
    return extend(cache, slots, offsets, batch, starts, 0, stream);
}

extern "C" int b200q_kv8_extend_after(const b200q_kv8_cache *cache, const int32_t *slots, const int32_t *offsets, int batch,
                                      int32_t *starts, void *stream) {
    return extend(cache, slots, offsets, batch, starts, 1, stream);
}

extern "C" int b200q_kv8_append(const b200q_kv8_cache *cache, int layer, const void *k, const void *v, int in_dtype,
                                int64_t k_row, int64_t v_row, const int32_t *slots, const int32_t *offsets,
                                const int32_t *starts, int batch, int max_new, const float *cos_table,
                                const float *sin_table, int rope_rows, void *stream) {
    if (int rc = kv8_check("kv8_append", cache)) return rc;
    if (batch == 0 || max_new == 0) return B200Q_OK;
    if (!k || !v || !slots || !offsets || !starts) return fail(B200Q_EINVAL, "kv8_append: NULL pointer");
    if (layer < 0 || layer >= cache->layers) return fail(B200Q_EINVAL, "kv8_append: layer %d out of range", layer);
    if (!dtype_valid(in_dtype)) return fail(B200Q_EINVAL, "kv8_append: bad dtype");
    if (batch < 0 || batch > cache->sequences || max_new < 0 || max_new > cache->max_length)
        return fail(B200Q_EINVAL, "kv8_append: batch %d, new tokens %d out of range", batch, max_new);
    const int64_t width = static_cast<int64_t>(cache->kv_heads) * cache->head_dim;
    if (k_row < width || v_row < width) return fail(B200Q_EINVAL, "kv8_append: row stride below kv_heads * head_dim");
    if (!cos_table != !sin_table) return fail(B200Q_EINVAL, "kv8_append: one of the two RoPE tables is NULL");
    if (cos_table && rope_rows < cache->max_length)
        return fail(B200Q_EINVAL, "kv8_append: RoPE tables of %d rows for sequences of up to %d tokens", rope_rows,
                    cache->max_length);
    if ((reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) & 15)
        return fail(B200Q_EINVAL, "kv8_append: RoPE tables must be 16-byte aligned");
    if (batch > KV8_MAX_STEP) return fail(B200Q_EUNSUPPORTED, "kv8_append: at most %d sequences per step", KV8_MAX_STEP);
    Kv8Append a{};
    a.k = k; a.v = v; a.k_row = k_row; a.v_row = v_row; a.layer = layer;
    a.slots = slots; a.offsets = offsets; a.starts = starts;
    a.cos_t = cos_table; a.sin_t = sin_table;
    const size_t quad = 4 * dtype_size(in_dtype);
    const bool vec = (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % quad == 0 && k_row % 4 == 0 && v_row % 4 == 0;
    const dim3 grid(2 * cache->kv_heads, (max_new + 2 * KV8_BLOCK - 2) / KV8_BLOCK, batch);
    if (grid.y > 65535) return fail(B200Q_EUNSUPPORTED, "kv8_append: too many new tokens");
    auto kernel = cache->head_dim == 64 ? append_kernel<64>(cache->dtype, in_dtype, vec) : append_kernel<128>(cache->dtype, in_dtype, vec);
    launch_chained(kernel, grid, dim3(2 * cache->head_dim), 0, static_cast<cudaStream_t>(stream), *cache, a);
    return check_launch("kv8_append");
}

extern "C" int b200q_kv8_fork(const b200q_kv8_cache *cache, const int32_t *src, const int32_t *dst, int count,
                              int32_t *scratch, void *stream) {
    if (int rc = kv8_check("kv8_fork", cache)) return rc;
    if (count == 0) return B200Q_OK;
    if (!src || !dst || !scratch) return fail(B200Q_EINVAL, "kv8_fork: NULL pointer");
    if (count < 0 || count > cache->sequences || count > 65535) return fail(B200Q_EINVAL, "kv8_fork: count %d out of range", count);
    int *status = device_status_word();
    if (!status) return fail(B200Q_ECUDA, "kv8_fork: no CUDA device");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    launch_chained(kv8_fork_check_kernel, dim3(1), dim3(1024), 0, s, *cache, src, dst, count, scratch, status);
    if (int rc = check_launch("kv8_fork")) return rc;
    launch_chained(kv8_fork_copy_kernel, dim3(1 + cache->layers, count), dim3(256), 0, s, *cache, src, dst,
                   static_cast<const int32_t *>(scratch));
    return check_launch("kv8_fork");
}

extern "C" int b200q_kv8_free(const b200q_kv8_cache *cache, const int32_t *slots, int count, void *stream) {
    if (int rc = kv8_check("kv8_free", cache)) return rc;
    if (count == 0) return B200Q_OK;
    if (!slots) return fail(B200Q_EINVAL, "kv8_free: NULL pointer");
    if (count < 0 || count > cache->sequences) return fail(B200Q_EINVAL, "kv8_free: count %d out of range", count);
    int *status = device_status_word();
    if (!status) return fail(B200Q_ECUDA, "kv8_free: no CUDA device");
    launch_chained(kv8_free_kernel, dim3(count), dim3(256), 0, static_cast<cudaStream_t>(stream), *cache, slots, status);
    return check_launch("kv8_free");
}

extern "C" long long b200q_kv8_compact_workspace(const b200q_kv8_cache *from, const b200q_kv8_cache *to) {
    if (!from || !to || from->pages < 1 || to->pages < 1) return 0;
    return 4ll * (1 + static_cast<long long>(from->pages) + to->pages);
}

static int compact_check(const char *what, const b200q_kv8_cache *from, const b200q_kv8_cache *to, const void *workspace,
                         long long workspace_bytes) {
    if (int rc = kv8_check(what, from)) return rc;
    if (int rc = kv8_check(what, to)) return rc;
    if (from->layers != to->layers || from->kv_heads != to->kv_heads || from->head_dim != to->head_dim ||
        from->sequences != to->sequences || from->blocks != to->blocks || from->dtype != to->dtype)
        return fail(B200Q_EINVAL, "%s: the caches differ in more than their pages", what);
    if (from->codes == to->codes || from->tail == to->tail || from->table == to->table)
        return fail(B200Q_EINVAL, "%s: the new cache must have memory of its own", what);
    if (!workspace || workspace_bytes < b200q_kv8_compact_workspace(from, to))
        return fail(B200Q_EINVAL, "%s: workspace too small", what);
    return B200Q_OK;
}

extern "C" int b200q_kv8_compact_plan(const b200q_kv8_cache *from, const b200q_kv8_cache *to, void *workspace,
                                      long long workspace_bytes, void *stream) {
    if (int rc = compact_check("kv8_compact_plan", from, to, workspace, workspace_bytes)) return rc;
    int32_t *count = static_cast<int32_t *>(workspace), *place = count + 1;
    launch_chained(kv8_compact_plan_kernel, dim3(1), dim3(1024), 0, static_cast<cudaStream_t>(stream), *from, *to, count, place,
                   place + from->pages);
    return check_launch("kv8_compact_plan");
}

extern "C" int b200q_kv8_compact_move(const b200q_kv8_cache *from, const b200q_kv8_cache *to, const void *workspace,
                                      long long workspace_bytes, void *stream) {
    if (int rc = compact_check("kv8_compact_move", from, to, workspace, workspace_bytes)) return rc;
    const int32_t *place = static_cast<const int32_t *>(workspace) + 1, *source = place + from->pages;
    const long long units = static_cast<long long>(from->layers) * 2 * from->kv_heads;
    const long long chunk = 256 * COPY_PIECES, page_pieces = units * KV8_BLOCK * from->head_dim / 16;
    const long long chunks = (page_pieces + chunk - 1) / chunk;
    const long long tail_ctas = (from->sequences * units * KV8_BLOCK * from->head_dim / 8 + chunk - 1) / chunk;
    const long long ctas = chunks * to->pages + tail_ctas + from->sequences;
    if (ctas > 0x7fffffffll) return fail(B200Q_EUNSUPPORTED, "kv8_compact_move: pool too large");
    launch_chained(kv8_compact_copy_kernel, dim3(static_cast<unsigned>(ctas)), dim3(256), 0, static_cast<cudaStream_t>(stream), *from,
                   *to, place, source, static_cast<int>(chunks), static_cast<int>(chunks * to->pages), static_cast<int>(tail_ctas));
    return check_launch("kv8_compact_move");
}
