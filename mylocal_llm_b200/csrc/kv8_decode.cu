// Attention of single tokens (and of a few per sequence) over the paged 8-bit cache.
//
// Bound by memory: every byte of a context is read once per key/value head, for the `group` query heads that share it (one or
// two tiles of eight rows, kv8_attention.cuh). The work of a call is a list of
// units - blocks of 64 keys of (key/value head, tile of rows, sequence) - cut into equal parts, one per CTA and two CTAs per SM,
// wherever the borders of the sequences lie; a sequence cut in two leaves FP32 partial results (maximum, sum, values) that a
// second kernel joins. Short sequences are not cut, and very short ones (SOLO) belong to one warp each, which needs no other. Inside a CTA the units of a part go to the warps in turn. A warp keeps its next pages on their way with
// one bulk copy each for keys and values (contiguous in a page) into its own stages in shared memory, so 100 to 200 KB per SM
// are in flight without a register, and its warps meet only at the end of a sequence.
#include <algorithm>

#include "kv8_attention.cuh"

namespace b200q {

constexpr int STATUS_KV8_WAIT = 511;        // gave up waiting for a page
constexpr int KV8_MAX_BATCH = 1024;         // sequences of one launch
constexpr int KV8_MAX_PARTS = 1024;         // parts that a joining kernel looks through

// Warps of a CTA and pages that a warp has in shared memory. The work of a page is a long chain of dependent instructions
// (1400 for a head dimension of 128): warps hide it, so there are as many as their registers allow.
// What parts consist of: any units, with two CTAs per SM so that one's work goes on while the other's warps meet; whole
// sequences; whole sequences for each warp by itself.
enum DecodeMode { CUT = 0, WHOLE = 1, SOLO = 2 };
template <int DH, int RT, int MODE> struct DecodeShape {
    static constexpr int CTAS = MODE == CUT ? 2 : 1, WARPS = (RT == 1 ? 12 : 8) / CTAS, STAGES = DH == 64 ? 2 : 1;
};

// Weights pass the tensor cores times 2^15, so that the largest one is at the top of FP16's range: a number and its remainder then
// keep 22 bits down to 2^-29 of it and 2^-40 of it below. (At 1 the many small weights behind a dominant key lost theirs, up to all:
// 131071 keys at 2^-25 of it are 0.4 % of the result.) The factor is taken off with the block's value scale and in the sum.
constexpr float KV8_WEIGHT_RANGE = 15.f, KV8_WEIGHT_UNIT = 1.f / 32768.f;

struct Kv8Decode {
    Kv8Attention a;
    int group, tiles;             // query heads per key/value head; lists of 8 RT rows (tokens x heads of the group) per head
    float *partial;               // [CTA][2][8 RT][DH + 4]: values, maximum, sum
    int4 *cuts;                   // [CTA], for the joining kernel: slot of the sequence that begins in the part and goes on behind
                                  // it (-1: none), its list, its number; list * batch + number of the one that goes on from
                                  // the part before (-1: none)
    int *status;
};

// Blocks that a sequence's step reads; 0 without new tokens or where the step was refused.
__device__ __forceinline__ int units_of(const Kv8Attention &a, int b) {
    const int start = a.starts[b], n = a.offsets[b + 1] - a.offsets[b];
    return start < 0 || n <= 0 ? 0 : (start + n + KV8_BLOCK - 1) / KV8_BLOCK;
}

template <int DH, bool BF16, int RT, int MODE>
__global__ void __launch_bounds__(DecodeShape<DH, RT, MODE>::WARPS * 32, DecodeShape<DH, RT, MODE>::CTAS) kv8_decode_kernel(const b200q_kv8_cache c, const Kv8Decode p) {
    constexpr int W = DecodeShape<DH, RT, MODE>::WARPS, ST = DecodeShape<DH, RT, MODE>::STAGES, HALF_PAGE = KV8_BLOCK * DH, DT = DH / 8, LD = DH + 4;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem;                                                            // [W][ST][2][HALF_PAGE]
    float *merged = reinterpret_cast<float *>(smem + W * ST * 2 * HALF_PAGE);        // [W][4][LD]: values of 4 rows, maximum, sum
    uint64_t *bars = reinterpret_cast<uint64_t *>(merged + W * 4 * LD);              // [W][2][ST]: keys, values
    int32_t *prefix = reinterpret_cast<int32_t *>(bars + 2 * W * ST);                    // [batch + 1]
    __shared__ int warp_sums[W];
    const Kv8Attention &a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    if (tid < 2 * W * ST) mbar_init(&bars[tid], 1);
    fence_barrier_init();
    chain_trigger();
    chain_wait();

    // ---- units before each sequence
    if (tid == 0) prefix[0] = 0;
    int total_units = 0;
    for (int b0 = 0; b0 < a.batch; b0 += W * 32) {
        const int b = b0 + tid;
        const int n = b < a.batch ? units_of(a, b) : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        __syncthreads();
        if (lane == 31) warp_sums[warp] = incl;
        __syncthreads();
        int before = total_units;
        for (int w = 0; w < W; ++w) {
            if (w < warp) before += warp_sums[w];
            total_units += warp_sums[w];
        }
        if (b < a.batch) prefix[b + 1] = before + incl;
    }
    __syncthreads();
    // rows of refused sequences
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
        if (a.starts[b] < 0)
            for (long long i = static_cast<long long>(a.offsets[b]) * a.heads * DH + tid;
                 i < static_cast<long long>(a.offsets[b + 1]) * a.heads * DH; i += W * 32)
                store_from_float(a.out, c.dtype, i, kv8_nan());

    const int lists = c.kv_heads * p.tiles;                  // a list of all sequences per head and tile
    const long long all = static_cast<long long>(lists) * total_units;
    long long lo, hi;
    if constexpr (MODE != CUT) {
        const long long segments = static_cast<long long>(lists) * a.batch;
        const int parts = MODE == SOLO ? gridDim.x * W : gridDim.x, part = MODE == SOLO ? blockIdx.x * W + warp : blockIdx.x;
        const long long s0 = segments * part / parts, s1 = segments * (part + 1) / parts;
        lo = s0 / a.batch * total_units + prefix[s0 % a.batch];
        hi = s1 / a.batch * total_units + prefix[s1 % a.batch];
    } else {
        // (contexts may be far shorter than the bound that the grid was made for: with a round of units per sequence on average, a
        // part each, 256 of four units 15 us instead of 21 by cutting)
        const long long segments = static_cast<long long>(lists) * a.batch;
        const long long parts = segments < gridDim.x && all <= segments * W ? segments : gridDim.x;
        lo = all * min(static_cast<long long>(blockIdx.x), parts) / parts;
        hi = all * min(blockIdx.x + 1ll, parts) / parts;
    }
    if (lo >= hi) {                                          // (SOLO: the warp; nothing below is for the whole CTA then)
        if (MODE == CUT && tid == 0) p.cuts[blockIdx.x] = make_int4(-1, 0, 0, -1);
        return;
    }

    // ---- this warp's units of the part, numbered from its beginning: every W-th, or all of them
    constexpr int STEP = MODE == SOLO ? 1 : W;
    const int first = MODE == SOLO ? 0 : warp;
    const int count = static_cast<int>(hi - lo);
    uint8_t *my_ring = ring + warp * ST * 2 * HALF_PAGE;
    uint64_t *my_bars = bars + warp * 2 * ST;
    int list = static_cast<int>(lo / total_units), s = 0, at = 0;
    int begin;                                               // first unit of sequence s of the list (may lie before the part)
    {
        const int r = static_cast<int>(lo - static_cast<long long>(list) * total_units);
        int right = a.batch - 1;                             // the last sequence that begins at or before r (with units)
        while (s < right) {
            const int mid = (s + right + 1) >> 1;
            if (prefix[mid] <= r) s = mid; else right = mid - 1;
        }
        begin = prefix[s] - r;
    }

    // The next unit to be looked up: its page is read from the table one unit before its copies are requested.
    constexpr int PAGE = 0, TAIL = 1, NONE = 2;
    int pu = first, plist = list, pseq = s, pbegin = begin, pend = begin, pfull = 0;
    const int32_t *prow = nullptr;
    struct Unit { int kind, page, list, seq; };
    auto open = [&] {                                        // sequence pseq of plist
        pbegin = pend;
        pend += prefix[pseq + 1] - prefix[pseq];
        if (pend > pu) {
            pfull = (a.starts[pseq] + a.offsets[pseq + 1] - a.offsets[pseq]) / KV8_BLOCK;
            prow = c.table + static_cast<size_t>(a.slots[pseq]) * c.blocks;
        }
    };
    open();
    auto look_up = [&]() -> Unit {
        if (pu >= count) return {NONE, 0, plist, pseq};
        while (pend <= pu) {
            if (++pseq == a.batch) {
                pseq = 0;
                ++plist;
            }
            open();
        }
        const int unit = pu - pbegin;
        pu += STEP;
        return unit < pfull ? Unit{PAGE, prow[unit], plist, pseq} : Unit{TAIL, 0, plist, pseq};
    };
    // (a table that lacks the page: another one is read, not beyond the pool, and its scale is NaN)
    auto page_of = [&](const Unit &x) { return x.page >= 0 && x.page < c.pages ? x.page : 0; };
    auto tail_of = [&](const Unit &x, int part) {
        return static_cast<const uint16_t *>(c.tail) +
               kv8_unit(a.slots[x.seq], c.layers, a.layer, part, c.kv_heads, x.list / p.tiles) * HALF_PAGE;
    };
    // part 0: the keys, 1: the values. A stage's keys are replaced as soon as the scores are formed, its values after the value
    // product: each half has the time of the other's work to arrive. A tail's values are 16 bits, so its keys take both halves
    // and its values follow them when the scores are formed (asked into L2 with the keys).
    bool gave_up = false;                                    // the whole warp: a copy did not arrive, nothing more is requested
    auto arrived = [&](int part, int st, uint32_t &phases) {
        if (!gave_up)
            gave_up = !__all_sync(0xffffffffu, mbar_wait_bounded(&my_bars[part * ST + st], (phases >> st) & 1u, p.status, STATUS_KV8_WAIT));
        phases ^= 1u << st;
    };
    auto request = [&](int part, const Unit &x, int st) {
        if (gave_up || x.kind == NONE) return;
        uint64_t *bar = &my_bars[part * ST + st];
        uint8_t *to = my_ring + st * 2 * HALF_PAGE;
        if (x.kind == PAGE) {
            if (lane == 0) {
                const size_t u = kv8_unit(page_of(x), c.layers, a.layer, part, c.kv_heads, x.list / p.tiles);
                mbar_arrive_expect_tx(bar, HALF_PAGE);
                bulk_copy_g2s(to + part * HALF_PAGE, c.codes + u * HALF_PAGE, HALF_PAGE, bar);
            }
        } else {
            const int bytes = (a.starts[x.seq] + a.offsets[x.seq + 1] - a.offsets[x.seq]) % KV8_BLOCK * DH * 2;
            if (lane == 0) {
                mbar_arrive_expect_tx(bar, bytes);
                bulk_copy_g2s(to, tail_of(x, part), bytes, bar);
            }
            if (part == 0) {
                const char *v = reinterpret_cast<const char *>(tail_of(x, 1));
                for (int o = lane * 128; o < bytes; o += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(v + o));
            }
        }
    };
    // the unit's scales: lane 0 the keys', lane 1 the values' (of a tail: the largest magnitudes)
    auto scale_of = [&](const Unit &x) -> float {
        if (lane >= 2 || x.kind == NONE) return 0.f;
        if (x.kind == PAGE) {
            const float scale = c.scales[kv8_unit(page_of(x), c.layers, a.layer, lane, c.kv_heads, x.list / p.tiles)];
            return page_of(x) == x.page ? scale : kv8_nan();
        }
        return c.peak[kv8_unit(a.slots[x.seq], c.layers, a.layer, lane, c.kv_heads, x.list / p.tiles)];
    };
    int kind_at[ST], st = 0;                                 // units in the stages, oldest first
    float scale_at[ST];
    uint32_t k_phases = 0u, v_phases = 0u;                   // of the stages' barriers
#pragma unroll
    for (int i = 0; i < ST; ++i) {
        const Unit x = look_up();
        kind_at[i] = x.kind;
        request(0, x, i);
        if (x.kind == PAGE) request(1, x, i);
        scale_at[i] = scale_of(x);
    }
    Unit next = look_up();
    auto advance = [&] {
#pragma unroll
        for (int i = 0; i + 1 < ST; ++i) {
            kind_at[i] = kind_at[i + 1];
            scale_at[i] = scale_at[i + 1];
        }
        kind_at[ST - 1] = next.kind;
        scale_at[ST - 1] = scale_of(next);
        next = look_up();
        if (++st == ST) st = 0;
    };

    int u = first, from_before = -1;
    for (;;) {
        // ---- one segment: the units [at, end) of sequence s
        const int seq_end = begin + prefix[s + 1] - prefix[s], end = min(seq_end, count);
        const int head = list / p.tiles, row0 = (list - head * p.tiles) * 8 * RT;
        const int start = a.starts[s], row_of = a.offsets[s], n = a.offsets[s + 1] - row_of, total = start + n;
        const int rows = min(n * p.group - row0, 8 * RT);    // rows of this list (row = token * group + head of the group)
        float m[RT], l[RT], o[RT][DT][2];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int i = 0; i < DT; ++i) o[r][i][0] = o[r][i][1] = 0.f;
        }
        if (u < end && rows > 0) {
            uint32_t qf[RT][DH / 16][4];
            float factor[RT];
            int pos[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int row = row0 + g + 8 * r, token = row / p.group;
                const bool valid = g + 8 * r < rows;
                pos[r] = valid ? start + token : start;
                factor[r] = query_split<DH>(
                    a, valid ? (row_of + token) * a.q_row + static_cast<long long>(head * p.group + row - token * p.group) * DH : -1,
                    pos[r], t, qf[r]);
            }
            for (; u < end; u += STEP) {
                const int unit = u - begin;
                const bool tail = kind_at[0] == TAIL;
                const uint8_t *stage = my_ring + st * 2 * HALF_PAGE;
                float acc[RT][8][4];
                float kscale = __shfl_sync(0xffffffffu, scale_at[0], 0), vscale = __shfl_sync(0xffffffffu, scale_at[0], 1), vinv = 0.f;
                const int rest = total - unit * KV8_BLOCK;   // keys of the block (64 or more: all)
                arrived(0, st, k_phases);
                if (!tail) {
                    score_codes<DH, RT>(stage, qf, g, t, acc);
                    __syncwarp();
                    if (next.kind == PAGE) request(0, next, st);
                } else {
                    kscale = tail_scale(abs_bits(kscale));
                    vscale = tail_scale(abs_bits(vscale));
                    vinv = power_inverse(vscale);
                    score_tail<DH, BF16, RT>(stage, power_inverse(kscale), rest, qf, g, t, acc);
                    __syncwarp();
                    request(1, {TAIL, 0, list, s}, st);
                }
                // ---- softmax weights; a row sees the keys up to its own position
                uint32_t pf[RT][4][4];
                float alpha[RT];
                bool moved = false;
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    // (not below the smallest normal number, where a hidden key's -inf would meet a zero)
                    float f = factor[r] * kscale, x[8][2], top = -INFINITY;
                    if (f < KV8_MIN_SCALE || pos[r] < unit * KV8_BLOCK) f = KV8_MIN_SCALE;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) x[j][e] = acc[r][j][e] + acc[r][j][2 + e];
                    if ((unit + 1) * KV8_BLOCK > start + 1) {                // (the same for the whole warp)
                        const int limit = pos[r] - unit * KV8_BLOCK - 16 * t;
#pragma unroll
                        for (int j = 0; j < 8; ++j)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if (2 * j + e > limit) x[j][e] = -INFINITY;
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = fmaxf(top, fmaxf(x[j][0], x[j][1]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    top = fmaxf(m[r], top * f);              // (f >= 0)
                    const float shift = top == -INFINITY ? 0.f : top;        // (no key seen yet: weights are 0)
                    const float move = KV8_WEIGHT_RANGE - shift;
                    alpha[r] = exp2_approx(m[r] - shift);
                    moved |= alpha[r] != 1.f;
                    m[r] = top;
                    float sum = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float p0 = exp2_approx(fmaf(x[j][0], f, move)), p1 = exp2_approx(fmaf(x[j][1], f, move));
                        sum += p0 + p1;
                        split_half(p0, p1, pf[r][j >> 1][2 * (j & 1)], pf[r][j >> 1][2 * (j & 1) + 1]);
                    }
                    l[r] = fmaf(sum, KV8_WEIGHT_UNIT, l[r] * alpha[r]);
                }
                if (__any_sync(0xffffffffu, moved)) {        // a maximum moved: rarely, after the first pages
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int i = 0; i < DT; ++i)
#pragma unroll
                            for (int e = 0; e < 2; ++e) o[r][i][e] *= alpha[r];
                }
                // ---- values, four tiles at a time (a block that a row does not see leaves it alone, even where its values are
                // not finite)
                arrived(1, st, v_phases);
                vscale = gave_up ? kv8_nan() : vscale * KV8_WEIGHT_UNIT;
                auto add = [&](int i, const float (&v)[RT][4][4]) {
#pragma unroll
                    for (int r = 0; r < RT; ++r)
                        if (pos[r] >= unit * KV8_BLOCK)
#pragma unroll
                            for (int b = 0; b < 4; ++b)
#pragma unroll
                                for (int e = 0; e < 2; ++e)
                                    o[r][i + b][e] = fmaf(vscale, v[r][b][e], fmaf(vscale, v[r][b][2 + e], o[r][i + b][e]));
                };
                if (!tail) {
#pragma unroll
                    for (int i = 0; i < DT; i += 4) {
                        float v[RT][4][4];
                        uint32_t word[4][4];
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const uint4 w = *reinterpret_cast<const uint4 *>(stage + HALF_PAGE + (8 * (i + b) + g) * KV8_BLOCK + 16 * t);
                            word[b][0] = w.x; word[b][1] = w.y; word[b][2] = w.z; word[b][3] = w.w;
                        }
#pragma unroll
                        for (int q = 0; q < 4; ++q)
#pragma unroll
                            for (int b = 0; b < 4; ++b) {
                                uint32_t b0, b1;
                                codes_to_half(word[b][q], b0, b1);
#pragma unroll
                                for (int r = 0; r < RT; ++r) {
                                    if (q == 0) mma_f16_first(v[r][b], pf[r][q], b0, b1);
                                    else mma_f16(v[r][b], pf[r][q], b0, b1);
                                }
                            }
                        add(i, v);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < DT; i += 4) {
                        float v[RT][4][4];
#pragma unroll
                        for (int b = 0; b < 4; ++b)
#pragma unroll
                            for (int q = 0; q < 4; q += 2) {
                                uint32_t w[4];
                                tail_values<DH, BF16>(smem_u32(stage), vinv, rest, i + b, q, lane, w);
#pragma unroll
                                for (int r = 0; r < RT; ++r) {
                                    if (q == 0) mma_f16_first(v[r][b], pf[r][q], w[0], w[1]);
                                    else mma_f16(v[r][b], pf[r][q], w[0], w[1]);
                                    mma_f16(v[r][b], pf[r][q + 1], w[2], w[3]);
                                }
                            }
                        add(i, v);
                    }
                }
                __syncwarp();
                if (tail || next.kind == TAIL) request(0, next, st);
                if (next.kind == PAGE) request(1, next, st);
                advance();
            }
        } else {
            for (; u < end; u += STEP) {                     // rows that do not exist: the units pass by
                arrived(0, st, k_phases);
                if (kind_at[0] == PAGE) arrived(1, st, v_phases);
                request(0, next, st);
                if (next.kind == PAGE) request(1, next, st);
                advance();
            }
        }
        // ---- a warp by itself has its rows' results
        if constexpr (MODE == SOLO) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                float sum = l[r];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (g + 8 * r >= rows) continue;
                const int row = row0 + g + 8 * r, token = row / p.group;
                const size_t to = (static_cast<size_t>(row_of + token) * a.heads + head * p.group + row - token * p.group) * DH + 2 * t;
#pragma unroll
                for (int i = 0; i < DT; ++i) {
                    store_from_float(a.out, c.dtype, to + 8 * i, o[r][i][0] / sum);
                    store_from_float(a.out, c.dtype, to + 8 * i + 1, o[r][i][1] / sum);
                }
            }
        } else {
        // ---- join the warps, four rows at a time
        const bool complete = at == begin && end == seq_end;
#pragma unroll
        for (int r4 = 0; r4 < 2 * RT; ++r4) {
            if (4 * r4 >= rows) break;
            const int r = r4 >> 1;
            float sum = l[r];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (g >> 2 == (r4 & 1)) {
                float *mine = merged + (warp * 4 + (g & 3)) * LD;
#pragma unroll
                for (int i = 0; i < DT; ++i) *reinterpret_cast<float2 *>(mine + 8 * i + 2 * t) = make_float2(o[r][i][0], o[r][i][1]);
                if (t == 0) *reinterpret_cast<float2 *>(mine + DH) = make_float2(m[r], sum);
            }
            __syncthreads();
            const int here = min(rows - 4 * r4, 4);
            for (int i = tid; i < here * DH; i += W * 32) {
                const int row = i / DH, d = i - row * DH;
                const float *from = merged + row * LD;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < W; ++w) top = fmaxf(top, from[w * 4 * LD + DH]);
                const float shift = top == -INFINITY ? 0.f : top;
                float value = 0.f, weight = 0.f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float f = exp2_approx(from[w * 4 * LD + DH] - shift);
                    value += f * from[w * 4 * LD + d];
                    weight += f * from[w * 4 * LD + DH + 1];
                }
                if (complete) {
                    const int rr = row0 + 4 * r4 + row, token = rr / p.group;
                    store_from_float(a.out, c.dtype, (static_cast<size_t>(row_of + token) * a.heads + head * p.group + rr - token * p.group) * DH + d,
                                     value / weight);
                } else {
                    float *to = p.partial + ((static_cast<size_t>(blockIdx.x) * 2 + (at == 0 ? 0 : 1)) * 8 * RT + 4 * r4 + row) * (DH + 4);
                    to[d] = value;
                    if (d == 0) {
                        to[DH] = top;
                        to[DH + 1] = weight;
                    }
                }
            }
            __syncthreads();
        }
        }
        if (MODE == CUT && begin < 0) from_before = list * a.batch + s;
        if (end == count) {
            if (MODE == CUT && tid == 0)
                p.cuts[blockIdx.x] = make_int4(begin >= 0 && seq_end > count ? (at == 0 ? 0 : 1) : -1, list, s, from_before);
            break;
        }
        at = end;
        begin = seq_end;
        do {
            if (++s == a.batch) {
                s = 0;
                ++list;
            }
        } while (prefix[s + 1] == prefix[s]);
    }
    if (gave_up) {
        // copies already requested still write shared memory: they complete on their own within microseconds
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 100000) {
        }
    }
}

// Joins the partial results of a sequence that was cut, one row of it per CTA (grid: sequences x rows). Which sequence: that of
// number blockIdx.x, or, where there are fewer parts than sequences, the one that begins in part blockIdx.x and goes on behind it.
// A part's results are a row of DH values away from the next one's, so the parts are read by 8 or 16 groups of threads at once
// (one thread after the other's 72 parts took 110 us for five sequences of up to 11771 keys).
template <int DH>
__global__ void __launch_bounds__(256) kv8_decode_join_kernel(const b200q_kv8_cache c, const Kv8Decode p, int ctas, int tile, int by_part) {
    constexpr int LANES = DH / 4, GROUPS = 256 / LANES;
    __shared__ float factors[KV8_MAX_PARTS];                 // of the parts' results; -1: the part holds none of the sequence
    __shared__ float4 sums[GROUPS][LANES];
    __shared__ float warp_top[8], warp_weight[8];
    __shared__ int first_s, last_s, slot_s;
    chain_trigger();
    chain_wait();
    const Kv8Attention &a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int segment = blockIdx.x;
    if (by_part) {
        const int4 cut = p.cuts[blockIdx.x];
        if (cut.x < 0) return;
        segment = cut.y * a.batch + cut.z;
    }
    const int list = segment / a.batch, s = segment - list * a.batch, head = list / p.tiles, row0 = (list - head * p.tiles) * tile;
    const int row = blockIdx.y, row_of = a.offsets[s];
    if (row >= min((a.offsets[s + 1] - row_of) * p.group - row0, tile)) return;
    if (tid == 0) first_s = last_s = -1;
    __syncthreads();
    for (int q = tid; q < ctas; q += 256) {
        const int4 cut = p.cuts[q];
        const bool begins = cut.x >= 0 && cut.y * a.batch + cut.z == segment;
        if (begins) {
            first_s = q;
            slot_s = cut.x;
        }
        factors[q] = begins || cut.w == segment ? 0.f : -1.f;
        if (cut.w == segment) atomicMax(&last_s, q);
    }
    __syncthreads();
    const int first = first_s, last = last_s, slot0 = slot_s;
    if (first < 0) return;                                   // not cut
    auto part = [&](int q) { return p.partial + ((static_cast<size_t>(q) * 2 + (q == first ? slot0 : 0)) * tile + row) * (DH + 4); };
    constexpr int MINE = KV8_MAX_PARTS / 256;
    float2 stat[MINE];                                       // maximum and sum of weights
    float top = -INFINITY, weight = 0.f;
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        const int q = first + tid + 256 * j;
        stat[j] = make_float2(-INFINITY, 0.f);
        if (q <= last && factors[q] >= 0.f) stat[j] = *reinterpret_cast<const float2 *>(part(q) + DH);
        top = fmaxf(top, stat[j].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) warp_top[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, warp_top[w]);
    const float shift = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        const int q = first + tid + 256 * j;
        const float f = exp2_approx(stat[j].x - shift);
        weight += f * stat[j].y;
        if (q <= last && factors[q] >= 0.f) factors[q] = f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) weight += __shfl_xor_sync(0xffffffffu, weight, o);
    if (lane == 0) warp_weight[warp] = weight;
    __syncthreads();
    const int group = tid / LANES, at = tid - group * LANES;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int q = first + group; q <= last; q += GROUPS) {
        const float f = factors[q];
        if (!(f < 0.f)) {                                    // (NaN belongs to the result)
            const float4 v = reinterpret_cast<const float4 *>(part(q))[at];
            sum.x += f * v.x; sum.y += f * v.y; sum.z += f * v.z; sum.w += f * v.w;
        }
    }
    sums[group][at] = sum;
    __syncthreads();
    if (tid >= DH) return;
    float value = 0.f;
    weight = 0.f;
    for (int g = 0; g < GROUPS; ++g) value += reinterpret_cast<const float *>(sums[g])[tid];
    for (int w = 0; w < 8; ++w) weight += warp_weight[w];
    const int rr = row0 + row, token = rr / p.group;
    store_from_float(a.out, c.dtype, (static_cast<size_t>(row_of + token) * a.heads + head * p.group + rr - token * p.group) * DH + tid, value / weight);
}

// ----------------------------------------------------------------------------------------------------------- host side
// How a call is divided: CTAs, and what their parts consist of.
struct DecodePlan {
    int tile, tiles, rows, ctas, mode;  // rows per list (8 or 16), lists per head, rows that a list has at most
    long long bytes;
    double time;                        // estimate, us
};

// What a mode costs, in us, as measured with 8 to 4096 sequences x heads of 1 to 94 units, all of the same length (caches in L2): a
// CTA per sequence (its queries and the warps' meeting) and round of its warps; a warp by itself per sequence and unit; parts per
// sequence and unit of the whole device. For such batches the best mode's estimate is within a third of its measured time; of ragged
// ones the longest sequence alone is known, so they are overestimated (48 of up to 8192 keys: 167 for 93). Measured (head
// dimension 128, four rows): 8 sequences x heads of 1500 keys 13.7 cut, 16.1 whole, 87 by single warps; 256 of 777 keys 30 / 30 /
// 66; 4096 of 60 keys 133 / 253 / 58.
struct DecodeTimes {
    double whole, whole_round, solo, solo_unit, cut, cut_unit;
};
static constexpr DecodeTimes DECODE_TIMES[2][2] = {          // [head dimension 128][16 rows]
    {{3.0, 2.9, 8.0, 2.7, 0.02, 0.0018}, {5.5, 3.3, 9.5, 3.2, 0.04, 0.0031}},
    {{4.0, 4.2, 11.0, 3.6, 0.03, 0.0029}, {9.0, 4.9, 15.0, 5.2, 0.06, 0.0046}},
};

static DecodePlan decode_plan(const b200q_kv8_cache *c, int heads, int batch, int max_new, int max_keys) {
    DecodePlan d{};
    const int group = heads / c->kv_heads;
    const int b = std::min(batch, KV8_MAX_BATCH);
    d.tile = max_new * static_cast<long long>(group) <= 8 ? 8 : 16;
    d.tiles = static_cast<int>((max_new * static_cast<long long>(group) + d.tile - 1) / d.tile);
    d.rows = static_cast<int>(std::min<long long>(max_new * static_cast<long long>(group), d.tile));
    const int warps = d.tile == 8 ? DecodeShape<64, 1, WHOLE>::WARPS : DecodeShape<64, 2, WHOLE>::WARPS;
    const long long units = (max_keys + KV8_BLOCK - 1) / KV8_BLOCK, segments = static_cast<long long>(c->kv_heads) * d.tiles * b;
    const int sms = sm_count();
    const DecodeTimes &t = DECODE_TIMES[c->head_dim == 128][d.tile == 16];
    const double whole = 2.5 + (segments + sms - 1) / sms * (t.whole + t.whole_round * ((units + warps - 1) / warps));
    const double solo = 3. + (segments + sms * warps - 1) / (sms * warps) * (t.solo + t.solo_unit * units);
    const double cut = 13. + segments * (t.cut + t.cut_unit * units) * (148. / sms);
    // Long sequences are always cut, which also evens out lengths that differ (the estimates know the longest only).
    d.time = units > 4 * warps ? cut : std::min(std::min(whole, solo), cut);
    d.mode = d.time == cut ? CUT : d.time == whole ? WHOLE : SOLO;
    const long long work = d.mode == SOLO ? (segments + warps - 1) / warps : d.mode == WHOLE ? segments : std::max<long long>(1, segments * units / (warps / 2));
    d.ctas = static_cast<int>(std::min<long long>({d.mode == CUT ? 2 * sms : sms, work, KV8_MAX_PARTS}));
    d.bytes = d.mode != CUT ? 0 : static_cast<long long>(d.ctas) * (16 + 2 * d.tile * (c->head_dim + 4) * 4);
    return d;
}

// Sizes whose units a CTA can number.
static bool decode_supported(const b200q_kv8_cache *c, const DecodePlan &d) {
    return static_cast<long long>(c->kv_heads) * d.tiles <= 65535 &&
           static_cast<long long>(KV8_MAX_BATCH) * ((c->max_length + KV8_BLOCK - 1) / KV8_BLOCK) <= 0x7fffffffll / std::max(1, c->kv_heads * d.tiles / d.ctas + 1);
}

double kv8_decode_time(const b200q_kv8_cache *c, int heads, int batch, int max_new, int max_keys) {
    const DecodePlan d = decode_plan(c, heads, batch, max_new, max_keys);
    return decode_supported(c, d) ? d.time : 1e30;
}

long long kv8_decode_workspace(const b200q_kv8_cache *c, int heads, int batch, int max_new, int max_keys) {
    return decode_plan(c, heads, batch, max_new, max_keys).bytes;
}

template <int DH, bool BF16, int RT, int MODE>
static int launch_decode(const b200q_kv8_cache &c, Kv8Decode p, const DecodePlan &d, cudaStream_t stream) {
    constexpr int W = DecodeShape<DH, RT, MODE>::WARPS, ST = DecodeShape<DH, RT, MODE>::STAGES;
    constexpr size_t fixed = static_cast<size_t>(W) * ST * 2 * KV8_BLOCK * DH + W * 4 * (DH + 4) * 4 + W * ST * 16;
    const size_t smem = fixed + (KV8_MAX_BATCH + 1) * 4;
    static_assert((fixed + (KV8_MAX_BATCH + 1) * 4 + 128 + 1024) * DecodeShape<DH, RT, MODE>::CTAS <= 228 * 1024, "shared memory of the decode kernel");
    if (int rc = allow_large_shared_memory(reinterpret_cast<const void *>(kv8_decode_kernel<DH, BF16, RT, MODE>))) return rc;
    const Kv8Attention whole = p.a;
    for (int b0 = 0; b0 < whole.batch; b0 += KV8_MAX_BATCH) {
        p.a.batch = std::min(KV8_MAX_BATCH, whole.batch - b0);
        p.a.slots = whole.slots + b0;
        p.a.offsets = whole.offsets + b0;
        p.a.starts = whole.starts + b0;
        launch_chained(kv8_decode_kernel<DH, BF16, RT, MODE>, dim3(d.ctas), dim3(W * 32), smem, stream, c, p);
        if (int rc = check_launch("kv8_attention")) return rc;
        if (MODE != CUT) continue;
        const long long segments = static_cast<long long>(c.kv_heads) * p.tiles * p.a.batch;
        const int by_part = segments >= d.ctas;
        if (d.ctas > 1)
            launch_chained(kv8_decode_join_kernel<DH>, dim3(by_part ? d.ctas - 1 : static_cast<int>(segments), d.rows), dim3(256), 0, stream, c, p,
                           d.ctas, d.tile, by_part);
        if (int rc = check_launch("kv8_attention (join)")) return rc;
    }
    return B200Q_OK;
}

using DecodeLaunch = int (*)(const b200q_kv8_cache &, Kv8Decode, const DecodePlan &, cudaStream_t);
template <int DH, bool BF16, int RT>
static DecodeLaunch decode_launch_of(int mode) {
    return mode == CUT ? launch_decode<DH, BF16, RT, CUT> : mode == WHOLE ? launch_decode<DH, BF16, RT, WHOLE> : launch_decode<DH, BF16, RT, SOLO>;
}
template <int DH>
static DecodeLaunch decode_launch(bool bf16, bool wide, int mode) {
    return bf16 ? (wide ? decode_launch_of<DH, true, 2>(mode) : decode_launch_of<DH, true, 1>(mode))
                : (wide ? decode_launch_of<DH, false, 2>(mode) : decode_launch_of<DH, false, 1>(mode));
}

int kv8_decode(const b200q_kv8_cache *c, const Kv8Attention &a, int max_new, int max_keys, void *workspace,
               long long workspace_bytes, cudaStream_t stream) {
    const DecodePlan d = decode_plan(c, a.heads, a.batch, max_new, max_keys);
    if (d.bytes > workspace_bytes || (d.bytes && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15))))
        return fail(B200Q_EINVAL, "kv8_attention: workspace of %lld bytes, 16-byte aligned, needed", d.bytes);
    if (!decode_supported(c, d))
        return fail(B200Q_EUNSUPPORTED, "kv8_attention: too many heads or keys");
    Kv8Decode p{};
    p.a = a;
    p.group = a.heads / c->kv_heads;
    p.tiles = d.tiles;
    p.cuts = static_cast<int4 *>(workspace);
    p.partial = reinterpret_cast<float *>(p.cuts + (d.mode == CUT ? d.ctas : 0));
    p.status = device_status_word();
    if (!p.status) return fail(B200Q_ECUDA, "kv8_attention: no CUDA device");
    const bool bf16 = c->dtype == B200Q_BF16;
    auto launch = c->head_dim == 64 ? decode_launch<64>(bf16, d.tile == 16, d.mode) : decode_launch<128>(bf16, d.tile == 16, d.mode);
    return launch(*c, p, d, stream);
}

}  // namespace b200q
