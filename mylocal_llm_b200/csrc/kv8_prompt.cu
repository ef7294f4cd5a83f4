// Attention of many tokens per sequence (whole prompts, chunks of prompts) over the paged 8-bit cache, on the 5th-generation
// tensor cores.
//
// One CTA owns 256 rows of one key/value head of one sequence (row = token * group + head of the group: the heads that share keys
// are neighbours) as two tiles of 128, and walks the blocks of 64 keys that its last row sees, or a part of them. Warps have
// roles that meet at mbarriers:
//   loader      one bulk copy each for the keys and the values of a page (int8, contiguous) into a ring
//   converters  (4 warps) codes -> FP16, exact, into the 128-byte-swizzled K-major operands: the keys as [64][head_dim], the
//               values, which a page holds transposed, as [head_dim][64]; the 16-bit tail of a sequence goes the same way
//   MMA         scores S = Q K^T (FP32, tensor memory) of one tile while the other tile's softmax runs, then O += P V with the
//               softmax weights P read from tensor memory
//   softmax     (2 x 4 warps) a thread per row: maximum, weights, sum; the weights go back to tensor memory as FP16, times the
//               block's value scale relative to a power of two U that follows the largest scale seen. A row's reference maximum
//               moves only when it is passed by 2^8, so O is rescaled rarely (FP16 has the room for weights up to 2^8).
// With a head dimension of 128 the tensor cores and the 16 exponentials per clock of an SM take about the same time, with 64
// the exponentials take twice as long. Queries are rounded to FP16 (a power of two per row keeps them in range); where the
// result is FP16 too the rounding would show next to the result's own, and a second product with the remainders (SPLIT) removes
// it. Weights are rounded to FP16. Block scales below 2^-14 of the largest lose bits of their share accordingly.
//
// Every wait is bounded: on expiry the status word tells, all roles leave, and the CTA ends.
#include <algorithm>

#include "kv8_attention.cuh"
#include "umma.cuh"

namespace b200q {

constexpr int STATUS_KV8_PROMPT = 512;       // gave up waiting at a barrier of the prompt kernel
constexpr int KP_ROWS = 128, KP_CTA_ROWS = 256;
constexpr int KP_SOFTMAX_WARPS = 8, KP_CONVERT_WARPS = 4;
constexpr int KP_THREADS = (KP_SOFTMAX_WARPS + KP_CONVERT_WARPS + 2) * 32;

template <int DH, bool SPLIT> struct PromptShape {
    static constexpr int STAGES = DH == 64 ? 4 : SPLIT ? 2 : 3;          // operand stages, and as many pages of codes
    static constexpr int Q = 2 * KP_ROWS * DH * 2, K = KV8_BLOCK * DH * 2, RAW = 2 * KV8_BLOCK * DH;
    static constexpr int BYTES = (SPLIT ? 2 : 1) * Q + STAGES * (2 * K + RAW);
};

struct Kv8Prompt {
    Kv8Attention a;
    int group, splits;            // query heads per key/value head; parts of the keys
    float *partial;               // [splits][rows][heads][DH + 2] when splits > 1
    int *status;
};

// D[tmem] (+)= A[tmem] * B[smem desc]
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Instruction descriptor of kind::f16 with FP16 operands (bits [7,10), [10,13) = 0) and an FP32 accumulator.
__host__ __device__ constexpr uint32_t umma_idesc_f16(int m, int n) {
    return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
        "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
        "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Byte offset of 16-byte chunk c (eight FP16 values) of a row in a swizzled operand of 128-byte rows.
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// Sixteen codes -> two chunks (2q, 2q + 1) of an operand row.
__device__ __forceinline__ void convert16(const uint4 &w, uint8_t *operand, int row, int q) {
    uint4 a, b;
    codes_to_half(w.x, a.x, a.y);
    codes_to_half(w.y, a.z, a.w);
    codes_to_half(w.z, b.x, b.y);
    codes_to_half(w.w, b.z, b.w);
    *reinterpret_cast<uint4 *>(operand + swizzled(row, 2 * q)) = a;
    *reinterpret_cast<uint4 *>(operand + swizzled(row, 2 * q + 1)) = b;
}

template <int DH, bool BF16, bool SPLIT>
__global__ void __launch_bounds__(KP_THREADS, 1) kv8_prompt_kernel(const b200q_kv8_cache c, const Kv8Prompt p) {
    using Shape = PromptShape<DH, SPLIT>;
    constexpr int ST = Shape::STAGES, SLABS = DH / 64, HALF_PAGE = KV8_BLOCK * DH;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t raw_full[ST], raw_free[ST], k_full[ST], k_free[ST], v_full[ST], v_free[ST], s_full[2], p_full[2],
        o_done[2], q_full;
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile int abort_flag;
    const Kv8Attention &a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    chain_trigger();
    chain_wait();
    // blocks of rows are numbered from the last (which sees most keys) to the first
    const int kvh = blockIdx.x % c.kv_heads, part = (blockIdx.x / c.kv_heads) % p.splits, b = blockIdx.x / (c.kv_heads * p.splits);
    const int start = a.starts[b], first = a.offsets[b], n = a.offsets[b + 1] - first, slot = a.slots[b], total = start + n;
    const int rows = n * p.group, row0 = (gridDim.y - 1 - blockIdx.y) * KP_CTA_ROWS;
    if (n <= 0 || row0 >= rows) return;
    if (start < 0) {                             // a refused step
        if (part == 0)
            for (int i = tid; i < min(KP_CTA_ROWS, rows - row0) * DH; i += KP_THREADS) {
                const int row = row0 + i / DH, token = row / p.group;
                store_from_float(a.out, c.dtype, (static_cast<size_t>(first + token) * a.heads + kvh * p.group + row - token * p.group) * DH + i % DH, kv8_nan());
            }
        return;
    }
    // units (blocks of keys) of both tiles: all that the tile's last row sees; this CTA's part of the longer one
    auto units_to = [&](int end_row) { return (start + (min(end_row, rows) - 1) / p.group) / KV8_BLOCK + 1; };
    const int all = units_to(row0 + KP_CTA_ROWS), u0 = static_cast<int>(static_cast<long long>(all) * part / p.splits);
    const int u1 = static_cast<int>(static_cast<long long>(all) * (part + 1) / p.splits);
    if (u0 >= u1) return;                        // (the joining kernel knows)
    const int count1 = row0 + KP_ROWS < rows ? u1 - u0 : 0;
    const int count0 = max(0, min(units_to(row0 + KP_ROWS), u1) - u0), count = max(count0, count1);
    const int full_units = total / KV8_BLOCK;    // units from here on are the tail

    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *q_s = smem, *k_s = smem + (SPLIT ? 2 : 1) * Shape::Q, *v_s = k_s + ST * Shape::K, *raw_s = v_s + ST * Shape::K;
    if (tid == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(&raw_full[s], 1);
            mbar_init(&raw_free[s], KP_CONVERT_WARPS);
            mbar_init(&k_full[s], KP_CONVERT_WARPS);
            mbar_init(&k_free[s], 1);
            mbar_init(&v_full[s], KP_CONVERT_WARPS);
            mbar_init(&v_free[s], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t], 4);
            mbar_init(&o_done[t], 1);
        }
        mbar_init(&q_full, KP_SOFTMAX_WARPS);
        abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0) {
        tmem_alloc<false>(&tmem_base_slot, 512);
        tmem_relinquish<false>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_slot;
    const uint32_t S_COL = 0, P_COL = 128, O_COL = 192;
    // the whole warp: false once anybody has given up
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        bool ok = mbar_try_wait(bar, parity);
        if (!__all_sync(0xffffffffu, ok)) {
            if (abort_flag) ok = false;
            else ok = mbar_wait_bounded(bar, parity, p.status, STATUS_KV8_PROMPT);
            if (!__all_sync(0xffffffffu, ok)) {
                abort_flag = 1;
                return false;
            }
        }
        return true;
    };

    if (warp == KP_SOFTMAX_WARPS + KP_CONVERT_WARPS) {
        // ---- loader
        int pages = 0;
        bool loading = false;
        for (int i = 0; i < count; ++i) {
            const int unit = u0 + i, s = i % ST;
            if ((i & 31) == 0) pages = unit + lane < full_units ? c.table[static_cast<size_t>(slot) * c.blocks + unit + lane] : 0;
            int page = __shfl_sync(0xffffffffu, pages, i & 31);
            page = page >= 0 && page < c.pages ? page : 0;       // (a table that lacks the page: not beyond the pool)
            if (i >= ST && !wait(&raw_free[s], (i / ST - 1) & 1)) break;
            if (lane == 0) {
                if (unit < full_units) {
                    const size_t u = kv8_unit(page, c.layers, a.layer, 0, c.kv_heads, kvh);
                    mbar_arrive_expect_tx(&raw_full[s], 2 * HALF_PAGE);
                    bulk_copy_g2s(raw_s + s * Shape::RAW, c.codes + u * HALF_PAGE, HALF_PAGE, &raw_full[s]);
                    bulk_copy_g2s(raw_s + s * Shape::RAW + HALF_PAGE, c.codes + (u + c.kv_heads) * HALF_PAGE, HALF_PAGE, &raw_full[s]);
                } else {
                    mbar_arrive(&raw_full[s]);                   // the converters read the tail themselves
                }
            }
            __syncwarp();
            loading = true;
        }
        if (abort_flag && loading) {
            // copies already requested still write shared memory; they complete on their own within microseconds
            const uint64_t t0 = global_timer_ns();
            while (global_timer_ns() - t0 < 100000) {
            }
        }
        __syncwarp();
    } else if (warp == KP_SOFTMAX_WARPS + KP_CONVERT_WARPS + 1) {
        // ---- MMAs (the whole warp walks the loop, one elected lane issues)
        constexpr uint32_t s_idesc = umma_idesc_f16(KP_ROWS, KV8_BLOCK), o_idesc = umma_idesc_f16(KP_ROWS, DH);
        const uint64_t q_desc = smem_desc_sw128(q_s), k_desc = smem_desc_sw128(k_s), v_desc = smem_desc_sw128(v_s);
        auto scores = [&](int t, int i) {        // S of tile t for unit i
            const uint64_t kd = k_desc + static_cast<uint32_t>((i % ST) * Shape::K >> 4);
            const uint64_t qd = q_desc + static_cast<uint32_t>(t * (Shape::Q / 2) >> 4);
            if (elect_one()) {
#pragma unroll
                for (int part_q = 0; part_q < (SPLIT ? 2 : 1); ++part_q)
#pragma unroll
                    for (int k = 0; k < DH / 16; ++k)
                        umma_bf16<false>(tmem + S_COL + 64 * t, qd + static_cast<uint32_t>((part_q * Shape::Q + (k / 4) * (KP_ROWS * 128)) >> 4) + 2 * (k % 4),
                                         kd + static_cast<uint32_t>(((k / 4) * (KV8_BLOCK * 128)) >> 4) + 2 * (k % 4), s_idesc, part_q + k > 0);
                umma_commit<false>(smem_u32(&s_full[t]));
            }
            __syncwarp();
        };
        auto values = [&](int t, int i, bool last) {
            const uint64_t vd = v_desc + static_cast<uint32_t>((i % ST) * Shape::K >> 4);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_f16_ts(tmem + O_COL + DH * t, tmem + P_COL + 32 * t + 8 * k, vd + 2 * k, o_idesc, i + k > 0);
                if (last) umma_commit<false>(smem_u32(&o_done[t]));
            }
            __syncwarp();
        };
        auto release = [&](uint64_t *bar) {
            if (elect_one()) umma_commit<false>(smem_u32(bar));
            __syncwarp();
        };
        bool fine = wait(&q_full, 0) && wait(&k_full[0], 0);
        if (fine) {
            tc_fence_after();
            if (count0) scores(0, 0);
            if (count1) scores(1, 0);
            release(&k_free[0]);
        }
        for (int i = 0; fine && i < count; ++i) {
            const int s = i % ST, s_next = (i + 1) % ST;
            if (!wait(&v_full[s], (i / ST) & 1)) break;
            if (i < count0) {
                if (!wait(&p_full[0], i & 1)) break;
                tc_fence_after();
                values(0, i, i + 1 == count0);
            }
            if (i + 1 < count && !wait(&k_full[s_next], ((i + 1) / ST) & 1)) break;
            tc_fence_after();
            if (i + 1 < count0) scores(0, i + 1);
            if (i < count1) {
                if (!wait(&p_full[1], i & 1)) break;
                tc_fence_after();
                values(1, i, i + 1 == count1);
            }
            release(&v_free[s]);
            if (i + 1 < count1) scores(1, i + 1);
            if (i + 1 < count) release(&k_free[s_next]);
        }
    } else if (warp >= KP_SOFTMAX_WARPS) {
        // ---- converters
        const int ct = tid - KP_SOFTMAX_WARPS * 32;
        for (int i = 0; i < count; ++i) {
            const int s = i % ST, unit = u0 + i;
            uint8_t *k_to = k_s + s * Shape::K, *v_to = v_s + s * Shape::K;
            const uint8_t *raw = raw_s + s * Shape::RAW;
            const size_t tail = kv8_unit(slot, c.layers, a.layer, 0, c.kv_heads, kvh);
            const uint16_t *tail_k = static_cast<const uint16_t *>(c.tail) + tail * HALF_PAGE, *tail_v = tail_k + static_cast<size_t>(c.kv_heads) * HALF_PAGE;
            const int rest = total - unit * KV8_BLOCK;
            // Tail values pass relative to a power of two; where the largest is not finite the scale is NaN and they are zeros
            // (a NaN here would reach rows that do not see the block).
            auto tail_inverse = [&](int values_part) {
                const uint32_t top = abs_bits(c.peak[tail + (values_part ? c.kv_heads : 0)]);
                return top < 0x7f800000u ? power_inverse(power_of(top)) : 0.f;
            };
            auto half_of = [&](uint32_t w, float inv) { return inv == 0.f ? 0u : tail_to_half<BF16>(w, inv); };
            if (!wait(&raw_full[s], (i / ST) & 1)) break;
            if (i >= ST && !wait(&k_free[s], (i / ST - 1) & 1)) break;
            if (unit < full_units) {
#pragma unroll
                for (int j = 0; j < SLABS * 2; ++j) {
                    const int id = ct + 128 * j, key = (id >> 2) & 63, q = id & 3, slab = id >> 8;
                    convert16(*reinterpret_cast<const uint4 *>(raw + key * DH + slab * 64 + q * 16), k_to + slab * (KV8_BLOCK * 128), key, q);
                }
            } else {
                const float inv = tail_inverse(0);
                for (int id = ct; id < KV8_BLOCK * DH / 8; id += 128) {
                    const int key = id / (DH / 8), chunk = id % (DH / 8);
                    uint4 w = make_uint4(0u, 0u, 0u, 0u);
                    if (key < rest) w = *reinterpret_cast<const uint4 *>(tail_k + key * DH + 8 * chunk);
                    *reinterpret_cast<uint4 *>(k_to + (chunk >> 3) * (KV8_BLOCK * 128) + swizzled(key, chunk & 7)) =
                        make_uint4(half_of(w.x, inv), half_of(w.y, inv), half_of(w.z, inv), half_of(w.w, inv));
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_full[s]);
            if (i >= ST && !wait(&v_free[s], (i / ST - 1) & 1)) break;
            if (unit < full_units) {
#pragma unroll
                for (int j = 0; j < SLABS * 2; ++j) {
                    const int id = ct + 128 * j;
                    convert16(*reinterpret_cast<const uint4 *>(raw + HALF_PAGE + id * 16), v_to, id >> 2, id & 3);
                }
            } else {
                const float inv = tail_inverse(1);
                for (int id = ct; id < KV8_BLOCK * DH / 2; id += 128) {
                    const int key = id / (DH / 2), d = id % (DH / 2) * 2;
                    const uint32_t w = key < rest ? half_of(*reinterpret_cast<const uint32_t *>(tail_v + key * DH + d), inv) : 0u;
                    *reinterpret_cast<uint16_t *>(v_to + swizzled(d, key >> 3) + (key & 7) * 2) = static_cast<uint16_t>(w);
                    *reinterpret_cast<uint16_t *>(v_to + swizzled(d + 1, key >> 3) + (key & 7) * 2) = static_cast<uint16_t>(w >> 16);
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&v_full[s]);
                mbar_arrive(&raw_free[s]);
            }
        }
    } else {
        // ---- softmax: a thread per row
        const int t = warp >> 2, local = 32 * (warp & 3) + lane, row = row0 + t * KP_ROWS + local, mine = t ? count1 : count0;
        const bool valid = row < rows;
        const int token = valid ? row / p.group : 0, pos = start + token;
        const size_t out_row = static_cast<size_t>(first + token) * a.heads + kvh * p.group + (valid ? row - token * p.group : 0);
        float factor = 0.f;
        {
            // the row's query: the largest magnitude, then FP16 (and remainders) into the operand; dimensions i and i + DH / 2 a
            // sixteen at a time
            constexpr int HALF = DH / 2;
            const size_t base = (first + token) * static_cast<size_t>(a.q_row) + static_cast<size_t>(kvh * p.group + (valid ? row - token * p.group : 0)) * DH;
            auto rotated = [&](int i, float (&x0)[16], float (&x1)[16]) {
                load16f(a.q, a.q_dtype, base + i, a.vec, x0);
                load16f(a.q, a.q_dtype, base + i + HALF, a.vec, x1);
                if (a.cos_t) {
                    float cv[16], sv[16];
                    load16f(a.cos_t, B200Q_F32, static_cast<size_t>(pos) * HALF + i, true, cv);
                    load16f(a.sin_t, B200Q_F32, static_cast<size_t>(pos) * HALF + i, true, sv);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float lo = x0[e] * cv[e] - x1[e] * sv[e], hi = x0[e] * sv[e] + x1[e] * cv[e];
                        x0[e] = lo;
                        x1[e] = hi;
                    }
                }
            };
            uint32_t top = 0u;
            if (valid && mine)
#pragma unroll 1
                for (int i = 0; i < HALF; i += 16) {
                    float x0[16], x1[16];
                    rotated(i, x0, x1);
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = max(top, max(abs_bits(x0[e]), abs_bits(x1[e])));
                }
            const float power = power_of(top), inv = a.scale < 0.f ? -power_inverse(power) : power_inverse(power);
            factor = power * (fabsf(a.scale) * 1.4426950408889634f);
            uint8_t *q_to = q_s + t * (Shape::Q / 2);
            if (mine)
#pragma unroll 1
                for (int i = 0; i < HALF; i += 16) {
                    float x[2][16];
                    if (valid) {
                        rotated(i, x[0], x[1]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[0][e] = x[1][e] = 0.f;
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int d = i + h * HALF;
                        uint8_t *to = q_to + (d / 64) * (KP_ROWS * 128);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int w = 0; w < 4; ++w) split_half(x[h][8 * e + 2 * w] * inv, x[h][8 * e + 2 * w + 1] * inv, hi[w], lo[w]);
                            const uint32_t at = swizzled(local, (d % 64) / 8 + e);
                            *reinterpret_cast<uint4 *>(to + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                            if (SPLIT) *reinterpret_cast<uint4 *>(to + Shape::Q + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        }
                    }
                }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full);
        }
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        float m = -INFINITY, l = 0.f, reference = 0.f;       // reference: U
        bool fine = true;
        // scales of the next unit, read a unit ahead (their page two units ahead)
        auto page_at = [&](int unit) { return unit < full_units ? c.table[static_cast<size_t>(slot) * c.blocks + unit] : 0; };
        auto scales_at = [&](int unit, int page, float &ks, float &vs) {
            if (unit < full_units) {
                const size_t u = kv8_unit(page >= 0 && page < c.pages ? page : 0, c.layers, a.layer, 0, c.kv_heads, kvh);
                ks = c.scales[u];
                vs = c.scales[u + c.kv_heads];
            } else {
                const size_t u = kv8_unit(slot, c.layers, a.layer, 0, c.kv_heads, kvh);
                ks = power_of(abs_bits(c.peak[u]));
                vs = power_of(abs_bits(c.peak[u + c.kv_heads]));
            }
        };
        float ks_next = 0.f, vs_next = 0.f;
        int page_next = 0;
        if (mine) {
            scales_at(u0, page_at(u0), ks_next, vs_next);
            if (mine > 1) page_next = page_at(u0 + 1);
        }
        for (int i = 0; i < mine; ++i) {
            const int unit = u0 + i;
            const float ks = ks_next, vs = vs_next;
            if (i + 1 < mine) scales_at(unit + 1, page_next, ks_next, vs_next);
            if (i + 2 < mine) page_next = page_at(unit + 2);
            const bool sees = pos >= unit * KV8_BLOCK;
            // (not below the smallest normal number, where a hidden key's -inf would meet a zero)
            float f = factor * ks;
            if (f < KV8_MIN_SCALE || !sees) f = KV8_MIN_SCALE;
            // U follows the largest scale: the same in every thread
            float beta = 1.f;
            const float power = power_of(abs_bits(vs));
            if (power > 8.f * reference) {
                beta = __fdiv_rn(reference, power);
                reference = power;
            }
            const float relative = sees ? __fdiv_rn(vs, reference) : 0.f;
            if (!wait(&s_full[t], i & 1)) {
                fine = false;
                break;
            }
            tc_fence_after();
            uint32_t s0[32], s1[32];
            tmem_ld32(tmem + lanes + S_COL + 64 * t, s0);
            tmem_ld32(tmem + lanes + S_COL + 64 * t + 32, s1);
            tmem_ld_wait();
            if (__any_sync(0xffffffffu, pos < unit * KV8_BLOCK + KV8_BLOCK - 1)) {
                const int limit = pos - unit * KV8_BLOCK;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    if (e > limit) s0[e] = 0xff800000u;
                    if (e + 32 > limit) s1[e] = 0xff800000u;
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 32; ++e) top = fmaxf(top, fmaxf(__uint_as_float(s0[e]), __uint_as_float(s1[e])));
            top *= f;
            float alpha = beta;
            if (top > m + 8.f) {
                const float keep = exp2_approx(m - top);
                alpha *= keep;
                l *= keep;
                m = top;
            }
            if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
                for (int d = 0; d < DH; d += 32) {
                    uint32_t o[32];
                    tmem_ld32(tmem + lanes + O_COL + DH * t + d, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                    tmem_st32(tmem + lanes + O_COL + DH * t + d, o);
                }
            }
            const float shift = m == -INFINITY ? 0.f : m;
            float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                const float x = exp2_approx(fmaf(__uint_as_float(s0[e]), f, -shift)), y = exp2_approx(fmaf(__uint_as_float(s1[e]), f, -shift));
                sum0 += x;
                sum1 += y;
                s0[e] = __float_as_uint(x * relative);
                s1[e] = __float_as_uint(y * relative);
            }
            l += sum0 + sum1;
            uint32_t w[32];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                w[e] = pack_half(__uint_as_float(s0[2 * e]), __uint_as_float(s0[2 * e + 1]));
                w[16 + e] = pack_half(__uint_as_float(s1[2 * e]), __uint_as_float(s1[2 * e + 1]));
            }
            tmem_st32(tmem + lanes + P_COL + 32 * t, w);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t]);
        }
        // ---- results
        if (mine && fine && wait(&o_done[t], 0)) {
            tc_fence_after();
            const float gain = p.splits == 1 ? __fdiv_rn(reference, l) : reference;
            float *to = p.splits == 1 ? nullptr : p.partial + ((static_cast<size_t>(part) * a.rows) * a.heads + out_row) * (DH + 2);
#pragma unroll 1
            for (int d = 0; d < DH; d += 32) {
                uint32_t o[32];
                tmem_ld32(tmem + lanes + O_COL + DH * t + d, o);
                tmem_ld_wait();
                if (!valid) continue;
                float v[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(o[e]) * gain;
                if (p.splits == 1) {
                    uint4 *out = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + out_row * DH + d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t w[4];
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            if (BF16) {
                                const __nv_bfloat162 x = __floats2bfloat162_rn(v[8 * e + 2 * h], v[8 * e + 2 * h + 1]);
                                w[h] = *reinterpret_cast<const uint32_t *>(&x);
                            } else {
                                w[h] = pack_half(v[8 * e + 2 * h], v[8 * e + 2 * h + 1]);
                            }
                        }
                        out[e] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 2) *reinterpret_cast<float2 *>(to + d + e) = make_float2(v[e], v[e + 1]);
                }
            }
            if (valid && p.splits > 1) *reinterpret_cast<float2 *>(to + DH) = make_float2(m, l);
        } else if (!mine && valid && p.splits > 1) {         // no key of this part: an empty share
            float *to = p.partial + ((static_cast<size_t>(part) * a.rows) * a.heads + out_row) * (DH + 2);
            for (int d = 0; d < DH; ++d) to[d] = 0.f;
            to[DH] = -INFINITY;
            to[DH + 1] = 0.f;
        }
    }
    if (abort_flag) {                            // (MMAs in flight end by themselves before the tensor memory is freed)
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 100000) {
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc<false>(tmem, 512);
}

// Joins the parts of a row: one warp per row and head, DH / 32 dimensions per lane.
template <int DH>
__global__ void __launch_bounds__(256) kv8_prompt_join_kernel(const b200q_kv8_cache c, const Kv8Prompt p) {
    chain_trigger();
    chain_wait();
    const Kv8Attention &a = p.a;
    const long long at = blockIdx.x * 8ll + (threadIdx.x >> 5);
    if (at >= static_cast<long long>(a.rows) * a.heads) return;
    const int lane = threadIdx.x & 31, token_row = static_cast<int>(at / a.heads), head = static_cast<int>(at % a.heads);
    int b = 0;
    for (int lo = 0, hi = a.batch - 1; lo <= hi;) {          // the sequence of the row
        const int mid = (lo + hi) >> 1;
        if (a.offsets[mid] <= token_row) { b = mid; lo = mid + 1; } else { hi = mid - 1; }
    }
    const int start = a.starts[b], n = a.offsets[b + 1] - a.offsets[b], rows = n * p.group;
    if (start < 0) return;
    const int row = (token_row - a.offsets[b]) * p.group + head % p.group;
    const int end = min(row / KP_CTA_ROWS * KP_CTA_ROWS + KP_CTA_ROWS, rows);
    const int all = (start + (end - 1) / p.group) / KV8_BLOCK + 1;       // units of the row's CTA
    float top = -INFINITY, weight = 0.f, value[DH / 32];
#pragma unroll
    for (int e = 0; e < DH / 32; ++e) value[e] = 0.f;
    auto share = [&](int q) { return p.partial + (static_cast<size_t>(q) * a.rows * a.heads + at) * (DH + 2); };
    auto empty = [&](int q) { return static_cast<long long>(all) * q / p.splits == static_cast<long long>(all) * (q + 1) / p.splits; };
    for (int q = 0; q < p.splits; ++q)
        if (!empty(q)) top = fmaxf(top, share(q)[DH]);
    const float shift = top == -INFINITY ? 0.f : top;
    for (int q = 0; q < p.splits; ++q) {
        if (empty(q)) continue;
        const float *from = share(q), f = exp2_approx(from[DH] - shift);
        weight += f * from[DH + 1];
#pragma unroll
        for (int e = 0; e < DH / 32; ++e) value[e] += f * from[lane + 32 * e];
    }
#pragma unroll
    for (int e = 0; e < DH / 32; ++e) store_from_float(a.out, c.dtype, at * DH + lane + 32 * e, value[e] / weight);
}

// ----------------------------------------------------------------------------------------------------------- host side
int kv8_shared_memory(const void *kernel, int bytes);        // kv8_decode.cu

// Parts of the keys: as many as give every SM two CTAs, of eight blocks at least.
static int prompt_splits(const b200q_kv8_cache *c, int heads, int batch, int max_new, int max_keys) {
    const long long rows = static_cast<long long>(max_new) * (heads / c->kv_heads), units = (max_keys + KV8_BLOCK - 1) / KV8_BLOCK;
    const long long ctas = (rows + KP_CTA_ROWS - 1) / KP_CTA_ROWS * c->kv_heads * batch;
    return static_cast<int>(std::max(1ll, std::min({(2ll * sm_count() + ctas - 1) / ctas, units / 8, 16ll})));
}

long long kv8_prompt_workspace(const b200q_kv8_cache *c, int heads, int batch, int rows, int max_new, int max_keys) {
    const int splits = prompt_splits(c, heads, batch, max_new, max_keys);
    return splits == 1 ? 0 : static_cast<long long>(splits) * rows * heads * (c->head_dim + 2) * 4;
}

int kv8_prompt(const b200q_kv8_cache *c, const Kv8Attention &a, int max_new, int max_keys, void *workspace, long long workspace_bytes,
               cudaStream_t stream) {
    Kv8Prompt p{};
    p.a = a;
    p.group = a.heads / c->kv_heads;
    p.splits = prompt_splits(c, a.heads, a.batch, max_new, max_keys);
    const long long bytes = kv8_prompt_workspace(c, a.heads, a.batch, a.rows, max_new, max_keys);
    if (bytes > workspace_bytes || (bytes && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15))))
        return fail(B200Q_EINVAL, "kv8_attention: workspace of %lld bytes, 16-byte aligned, needed", bytes);
    if (reinterpret_cast<uintptr_t>(a.out) & 15) return fail(B200Q_EINVAL, "kv8_attention: out must be 16-byte aligned");
    p.partial = static_cast<float *>(workspace);
    p.status = device_status_word();
    if (!p.status) return fail(B200Q_ECUDA, "kv8_attention: no CUDA device");
    const long long blocks = (static_cast<long long>(max_new) * p.group + KP_CTA_ROWS - 1) / KP_CTA_ROWS;
    const long long across = static_cast<long long>(c->kv_heads) * p.splits * a.batch;
    const long long joins = (static_cast<long long>(a.rows) * a.heads + 7) / 8;
    if (blocks > 65535 || across > 0x7fffffffll || joins > 0x7fffffffll || static_cast<long long>(max_new) * p.group > 0x40000000ll)
        return fail(B200Q_EUNSUPPORTED, "kv8_attention: too many rows");
    const bool bf16 = c->dtype == B200Q_BF16;
    auto kernel = c->head_dim == 64 ? (bf16 ? kv8_prompt_kernel<64, true, false> : kv8_prompt_kernel<64, false, true>)
                                    : (bf16 ? kv8_prompt_kernel<128, true, false> : kv8_prompt_kernel<128, false, true>);
    const int smem = 1024 + (c->head_dim == 64 ? (bf16 ? PromptShape<64, false>::BYTES : PromptShape<64, true>::BYTES)
                                               : (bf16 ? PromptShape<128, false>::BYTES : PromptShape<128, true>::BYTES));
    if (int rc = kv8_shared_memory(reinterpret_cast<const void *>(kernel), smem)) return rc;
    launch_chained(kernel, dim3(static_cast<unsigned>(across), static_cast<unsigned>(blocks)), dim3(KP_THREADS), smem, stream, *c, p);
    if (int rc = check_launch("kv8_attention")) return rc;
    if (p.splits == 1) return B200Q_OK;
    launch_chained(c->head_dim == 64 ? kv8_prompt_join_kernel<64> : kv8_prompt_join_kernel<128>, dim3(static_cast<unsigned>(joins)), dim3(256), 0,
                   stream, *c, p);
    return check_launch("kv8_attention (join)");
}

}  // namespace b200q
