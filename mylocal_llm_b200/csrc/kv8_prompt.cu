// Attention of many tokens per sequence (whole prompts, chunks of prompts) over the paged 8-bit cache, on the 5th-generation
// tensor cores.
//
// One CTA owns 256 rows of one key/value head of one sequence (row = token * group + head of the group: the heads that share keys
// are neighbours) as two tiles of 128, and walks the units of 128 keys (two pages) that its last row sees, or a part of them.
// Warps have roles that meet at mbarriers:
//   converters  (4 warps) codes -> registers, a half page ahead (and asked into L2 four units ahead) -> FP16, exact, into the 128-byte-swizzled K-major operands: the
//               keys as [128][head_dim], the values, which a page holds transposed, as [head_dim][64] twice; the 16-bit tail of a
//               sequence goes the same way. (A ring of codes in shared memory took 64 KB of its traffic per unit, which the
//               operands of the MMAs need: at head dimension 128 they read 256 to 320 KB per unit at 128 bytes a clock.)
//   MMA         (a warp per tile) scores S = Q K^T (FP32, tensor memory), then, when the tile's softmax is done, O += P V with
//               the softmax weights P read from tensor memory, where they and their remainders replace their scores; one tile's
//               products run while the other's softmax does. (One warp for both tiles needed more time to issue the
//               instructions, among three other busy warps of its scheduler, than the tensor cores to execute them.)
//   softmax     (2 x 4 warps) a thread per row: maximum, weights, sum; the weights go back to tensor memory as FP16, times the
//               block's value scale (its logarithm is an addend of the exponent, which costs nothing; the sum is divided by it).
//               A row's reference M is the largest such product that it has seen, so a block counts by what it adds to the
//               row and not by its scale: a large scale under a small weight does not push the others out of FP16's range.
//               M moves only when it is passed by 2^4, so O is rescaled rarely; products are held as 2^11 times what they are
//               next to M, FP16's whole range. The sum and the largest weight have a reference of their own, since M may lie
//               2^126 above or below it. A unit's first page is handed over before the second's weights are worked out (chunks
//               of head dimension 128 397 -> 363 us).
// 128 keys per step because an MMA of 128 rows x 64 keys reads 6 KB of operands for 32 clocks of work, more than shared memory
// gives: with units of 64 keys the MMAs took 3200 of 3900 clocks per 64 keys (head dimension 128). Queries (a power of two per row
// keeps them in range) and products of weight and scale are an FP16 number and what is left of it as another, each with an MMA of
// its own, so both keep 22 bits as in kv8_decode.cu, whichever kernel a step gets. As FP16 numbers alone the weights cost 1.4 times
// the result's own rounding in FP16 results (2.9e-4 for 2.1e-4 against 64 bits); prompts of head dimension 64 took 207 us instead of
// 243, chunks of dimension 128 and FP16 (queries in two parts) 321 instead of 358. Below FP16's normal numbers 2^-36 of the row's M
// is kept.
//
// Every wait is bounded: on expiry the status word tells, all roles leave, and the CTA ends.
#include <algorithm>

#include "kv8_attention.cuh"
#include "umma.cuh"

namespace b200q {

constexpr int STATUS_KV8_PROMPT = 512;       // gave up waiting at a barrier of the prompt kernel
constexpr int KP_ROWS = 128, KP_CTA_ROWS = 256;
constexpr int KP_SOFTMAX_WARPS = 8, KP_CONVERT_WARPS = 4;
constexpr int KP_THREADS = 512;              // and two MMA warps and two that only help with the queries
// Registers per thread: a softmax thread holds its row's 128 scores, a converter DH / 8 words of codes (4 x 2048 tokens of head
// dimension 64: 253 us with 176 and 80, 241 so; three chunks of dimension 128 with 184 and 72 the same time, with 192 and 64 16 us more).
// Together 512 x 128, what the launch has.
template <int DH> constexpr int KP_SOFTMAX_REGS = DH == 64 ? 192 : 176;
template <int DH> constexpr int KP_OTHER_REGS = 256 - KP_SOFTMAX_REGS<DH>;

constexpr int KP_KEYS = 2 * KV8_BLOCK;       // keys of a unit

// Operand stages of keys and values (of a unit each), by what shared memory holds next to the queries and their remainders.
template <int DH> struct PromptShape {
    static constexpr int KS = 2, VS = DH == 128 ? 1 : 2;
    static constexpr int Q = 2 * KP_ROWS * DH * 2, K = KP_KEYS * DH * 2;
    static constexpr int BYTES = 2 * Q + (KS + VS) * K;
};
constexpr int KP_AHEAD = 4;                  // units between a page's request to L2 and its use
// Exponents of two: products of weight and value scale are held times 2^KP_RANGE / M and pass M by 2^KP_SLACK at most, which uses
// FP16's range up to 2^15; those below 2^-KP_NOTHING M only enter the sum. (Ranges of 7, 11 and 13: 235, 235 and 240 us for 4 x 2048 tokens of
// head dimension 64, 358, 363 and 370 for three chunks of dimension 128: more room below, O rescaled more often.)
constexpr float KP_RANGE = 11.f, KP_SLACK = 15.f - KP_RANGE, KP_NOTHING = 100.f;

struct Kv8Prompt {
    Kv8Attention a;
    int group, splits;            // query heads per key/value head; parts of the keys
    float *partial;               // [splits][rows][heads][DH + 2] when splits > 1
    int *status;
};

// D[tmem] (+)= A * B, A described in shared memory or read from tensor memory. Descriptors as their low words (the address is in
// them) and one high word, so that an operand costs one addition.
__device__ __forceinline__ void umma_f16_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
        "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
// A pair as FP16 numbers, cut off.
__device__ __forceinline__ uint32_t cut_half(float lo, float hi) {
    uint32_t r;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float log2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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

template <int DH, bool BF16>
__global__ void __launch_bounds__(KP_THREADS, 1) kv8_prompt_kernel(const b200q_kv8_cache c, const Kv8Prompt p) {
    using Shape = PromptShape<DH>;
    constexpr int KS = Shape::KS, VS = Shape::VS, SLABS = DH / 64, HALF_PAGE = KV8_BLOCK * DH;
    constexpr int K_SLAB = KP_KEYS * 128, V_PAGE = DH * 128;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t k_full[KS], k_free[KS], v_full[VS], v_free[VS], s_full[2], p_full[2][2], o_done[2], q_full;
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile int abort_flag;
    __shared__ float factor_s[KP_CTA_ROWS];
    const Kv8Attention &a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    chain_wait();
    // CTAs start in the order of their numbers, so the last to start should be short. Blocks of rows go from the last (which sees
    // most keys) to the first: over all sequences where these are alike, else (up to 32) one sequence after the other, the longest
    // first (chunks of 512 behind 16000 and 3800 tokens: 381 us in the first order, 336 us in the second; four prompts of 2048
    // tokens: 198 and 208 us).
    const int blocks = gridDim.z;
    int kvh = blockIdx.x, part = 0, b = blockIdx.y, row_block = blockIdx.z;
    if (p.splits > 1) {
        part = blockIdx.x / c.kv_heads;
        kvh = blockIdx.x - part * c.kv_heads;
    }
    int start = a.starts[b], first = a.offsets[b], next = a.offsets[b + 1], slot = a.slots[b];
    if (a.batch > 1 && a.batch <= 32) {
        const int size = lane < a.batch ? a.starts[lane] + a.offsets[lane + 1] - a.offsets[lane] : 0;
        const int first_size = __shfl_sync(0xffffffffu, size, 0);
        if (__any_sync(0xffffffffu, lane < a.batch && size != first_size)) {
            const int number = b + a.batch * row_block;
            int rank = 0;
            for (int q = 0; q < a.batch; ++q) {
                const int other = __shfl_sync(0xffffffffu, size, q);
                rank += other > size || (other == size && q < lane);
            }
            row_block = number % blocks;
            b = __ffs(__ballot_sync(0xffffffffu, lane < a.batch && rank == number / blocks)) - 1;
            start = a.starts[b];
            first = a.offsets[b];
            next = a.offsets[b + 1];
            slot = a.slots[b];
        }
    }
    const int n = next - first, total = start + n;
    const int rows = n * p.group, row0 = (blocks - 1 - row_block) * KP_CTA_ROWS;
    if (n <= 0 || row0 >= rows) return;
    if (start < 0) {                             // a refused step
        if (part == 0)
            for (int i = tid; i < min(KP_CTA_ROWS, rows - row0) * DH; i += KP_THREADS) {
                const int row = row0 + i / DH, token = row / p.group;
                store_from_float(a.out, c.dtype, (static_cast<size_t>(first + token) * a.heads + kvh * p.group + row - token * p.group) * DH + i % DH, kv8_nan());
            }
        return;
    }
    // units of both tiles: all that the tile's last row sees; this CTA's part of the longer one
    auto units_to = [&](int end_row) { return (start + (min(end_row, rows) - 1) / p.group) / KP_KEYS + 1; };
    const int all = units_to(row0 + KP_CTA_ROWS), u0 = static_cast<int>(static_cast<long long>(all) * part / p.splits);
    const int u1 = static_cast<int>(static_cast<long long>(all) * (part + 1) / p.splits);
    if (u0 >= u1) return;                        // (the joining kernel knows)
    const int count1 = row0 + KP_ROWS < rows ? u1 - u0 : 0;
    const int count0 = max(0, min(units_to(row0 + KP_ROWS), u1) - u0), count = max(count0, count1);
    const int full_pages = total / KV8_BLOCK;    // the block after them is the tail, what follows does not exist

    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *q_s = smem, *k_s = smem + 2 * Shape::Q, *v_s = k_s + KS * Shape::K;
    if (tid == 0) {
        for (int s = 0; s < KS; ++s) {
            mbar_init(&k_full[s], KP_CONVERT_WARPS);
            mbar_init(&k_free[s], 2);            // both tiles
        }
        for (int s = 0; s < VS; ++s) {
            mbar_init(&v_full[s], KP_CONVERT_WARPS);
            mbar_init(&v_free[s], 2);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t][0], 4);
            mbar_init(&p_full[t][1], 4);
            mbar_init(&o_done[t], 1);
        }
        mbar_init(&q_full, KP_THREADS / 32);
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
    // Only now may the next kernel come: one that allocates tensor memory before it waits for this one must not find it free while
    // a CTA here still needs it.
    chain_trigger();
    const uint32_t tmem = tmem_base_slot;                    // (all 512 columns: 0)
    const uint32_t S_COL = 0, P_COL = 64, O_COL = 256;       // per tile: S 128 columns (then the remainders of P, and P from column 64), O DH columns
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

    constexpr int MMA = KP_SOFTMAX_WARPS + KP_CONVERT_WARPS;
    {
        // ---- queries, by all warps: DH / 8 lanes hold four dimensions of a row and their partners; the largest
        // magnitude, then FP16 numbers and remainders relative to its power of two
        constexpr int HALF = DH / 2, LANES = DH / 8, AT_ONCE = 32 / LANES, WARPS = KP_THREADS / 32, STEPS = (KP_CTA_ROWS / AT_ONCE + WARPS - 1) / WARPS;
        const int i = lane % LANES * 4;
#pragma unroll 3
        for (int step = 0; step < STEPS; ++step) {
            const int local = (warp + WARPS * step) * AT_ONCE + lane / LANES, row = row0 + local, token = row / p.group;
            float x[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[h][e] = 0.f;
            if (local < KP_CTA_ROWS && row < rows) {
                const size_t base = (first + token) * static_cast<size_t>(a.q_row) + static_cast<size_t>(kvh * p.group + row - token * p.group) * DH + i;
                load4f(a.q, a.q_dtype, base, a.vec, x[0]);
                load4f(a.q, a.q_dtype, base + HALF, a.vec, x[1]);
                if (a.cos_t) {
                    const float4 c4 = *reinterpret_cast<const float4 *>(a.cos_t + static_cast<size_t>(start + token) * HALF + i);
                    const float4 s4 = *reinterpret_cast<const float4 *>(a.sin_t + static_cast<size_t>(start + token) * HALF + i);
                    const float cv[4] = {c4.x, c4.y, c4.z, c4.w}, sv[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float lo = x[0][e] * cv[e] - x[1][e] * sv[e], hi = x[0][e] * sv[e] + x[1][e] * cv[e];
                        x[0][e] = lo;
                        x[1][e] = hi;
                    }
                }
            }
            uint32_t top = 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max(abs_bits(x[0][e]), abs_bits(x[1][e])));
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float power = query_scale(top), inv = a.scale < 0.f ? -power_inverse(power) : power_inverse(power);
            if (local < KP_CTA_ROWS) {
                if (i == 0) factor_s[local] = power * (fabsf(a.scale) * 1.4426950408889634f);
                uint8_t *q_to = q_s + (local / KP_ROWS) * (Shape::Q / 2);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = i + h * HALF;
                    uint32_t hi[2], lo[2];
                    split_half(x[h][0] * inv, x[h][1] * inv, hi[0], lo[0]);
                    split_half(x[h][2] * inv, x[h][3] * inv, hi[1], lo[1]);
                    uint8_t *to = q_to + (d / 64) * (KP_ROWS * 128) + swizzled(local % KP_ROWS, d % 64 / 8) + d % 8 * 2;
                    *reinterpret_cast<uint2 *>(to) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2 *>(to + Shape::Q) = make_uint2(lo[0], lo[1]);
                }
            }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full);
        __syncwarp();                            // (the roles begin with an instruction of the whole warp)
    }

    if (warp >= MMA) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KP_OTHER_REGS<DH>));
        if (warp < MMA + 2) {
        // ---- MMAs of tile t (the whole warp walks the loop, one elected lane issues). Units that the tile does not need are
        // released as they come.
        constexpr uint32_t s_idesc = umma_idesc_f16(KP_ROWS, KP_KEYS), o_idesc = umma_idesc_f16(KP_ROWS, DH);
        const int t = warp - MMA, mine = t ? count1 : count0;
        const uint64_t any_desc = smem_desc_sw128(smem);
        const uint32_t hi = static_cast<uint32_t>(any_desc >> 32), lo = static_cast<uint32_t>(any_desc);
        const uint32_t q_lo = lo + t * (Shape::Q / 2 >> 4), k_lo = lo + (2 * Shape::Q >> 4), v_lo = k_lo + (KS * Shape::K >> 4);
        const uint32_t s_at = tmem + S_COL + 128 * t, o_at = tmem + O_COL + DH * t;
        auto scores = [&](int i) {
            const int s = i % KS;
            const uint32_t kd = k_lo + s * (Shape::K >> 4);
            if (elect_one()) {
                if (i < mine) {
#pragma unroll
                    for (int part_q = 0; part_q < 2; ++part_q)
#pragma unroll
                        for (int k = 0; k < DH / 16; ++k)
                            umma_f16_ss(s_at, q_lo + ((part_q * Shape::Q + (k / 4) * (KP_ROWS * 128)) >> 4) + 2 * (k % 4),
                                        kd + (((k / 4) * K_SLAB) >> 4) + 2 * (k % 4), hi, s_idesc, part_q + k > 0);
                    umma_commit<false>(smem_u32(&s_full[t]));
                    umma_commit<false>(smem_u32(&k_free[s]));
                } else {
                    mbar_arrive(&k_free[s]);
                }
            }
            __syncwarp();
        };
        // (the products of the first page's keys run while the second page's weights are worked out)
        auto values = [&](int i, int page) {
            const int s = i % VS;
            const uint32_t vd = v_lo + s * (Shape::K >> 4) + page * (V_PAGE >> 4);
            if (elect_one()) {
                if (i < mine) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        umma_f16_ts(o_at, s_at + P_COL + 32 * page + 8 * k, vd + 2 * k, hi, o_idesc, i + page + k > 0);
                        umma_f16_ts(o_at, s_at + 32 * page + 8 * k, vd + 2 * k, hi, o_idesc, 1u);
                    }
                    if (page && i + 1 == mine) umma_commit<false>(smem_u32(&o_done[t]));
                    if (page) umma_commit<false>(smem_u32(&v_free[s]));
                } else if (page) {
                    mbar_arrive(&v_free[s]);
                }
            }
            __syncwarp();
        };
        bool fine = wait(&q_full, 0) && wait(&k_full[0], 0);
        tc_fence_after();
        if (fine) scores(0);
        for (int i = 0; fine && i < count; ++i) {
            const int next = i + 1;
            fine = wait(&v_full[i % VS], (i / VS) & 1);
            for (int page = 0; fine && page < 2; ++page) {
                fine = i >= mine || wait(&p_full[t][page], i & 1);
                if (!fine) break;
                tc_fence_after();
                values(i, page);
            }
            if (!fine) break;
            if (next == count) break;
            fine = wait(&k_full[next % KS], (next / KS) & 1);
            if (!fine) break;
            tc_fence_after();
            scores(next);
        }
        }
    } else if (warp >= KP_SOFTMAX_WARPS) {
        // ---- converters
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KP_OTHER_REGS<DH>));
        const int ct = tid - KP_SOFTMAX_WARPS * 32;
        const size_t tail = kv8_unit(slot, c.layers, a.layer, 0, c.kv_heads, kvh);
        const uint16_t *tail_k = static_cast<const uint16_t *>(c.tail) + tail * HALF_PAGE, *tail_v = tail_k + static_cast<size_t>(c.kv_heads) * HALF_PAGE;
        const int rest = total - full_pages * KV8_BLOCK;
        // Tail values pass relative to a power of two; where the largest is not finite the scale is NaN and they are zeros (a
        // NaN here would reach rows that do not see the block).
        auto tail_inverse = [&](int values_part) {
            const uint32_t top = abs_bits(c.peak[tail + (values_part ? c.kv_heads : 0)]);
            return top < 0x7f800000u ? power_inverse(tail_scale(top)) : 0.f;
        };
        auto half_of = [&](uint32_t w, float inv) { return inv == 0.f ? 0u : tail_to_half<BF16>(w, inv); };
        auto page_at = [&](int block) {
            const int page = block < full_pages ? c.table[static_cast<size_t>(slot) * c.blocks + block] : 0;
            return page;
        };
        // a thread's sixteen-code pieces of half a page: (row, quarter) of 64-code rows
        using Half = uint4[SLABS * 2];
        auto fetch = [&](Half &w, int block, int page, bool keys) {
            if (block >= full_pages) return;
            page = page >= 0 && page < c.pages ? page : 0;       // (a table that lacks the page: not beyond the pool)
            const int8_t *from = c.codes + kv8_unit(page, c.layers, a.layer, keys ? 0 : 1, c.kv_heads, kvh) * HALF_PAGE;
#pragma unroll
            for (int j = 0; j < SLABS * 2; ++j)
                w[j] = *reinterpret_cast<const uint4 *>(from + (keys ? ((ct >> 2) + 32 * (j & 1)) * DH + (j >> 1) * 64 + (ct & 3) * 16 : (ct + 128 * j) * 16));
        };
        auto store = [&](const Half &w, int block, bool keys, uint8_t *to) {
            if (block < full_pages) {
#pragma unroll
                for (int j = 0; j < SLABS * 2; ++j) {
                    if (keys) convert16(w[j], to + (j >> 1) * K_SLAB, (ct >> 2) + 32 * (j & 1), ct & 3);
                    else convert16(w[j], to, (ct >> 2) + 32 * j, ct & 3);
                }
                return;
            }
            const int have = block == full_pages ? rest : 0;
            const float inv = have ? tail_inverse(!keys) : 0.f;
            // eight dimensions of a key at a time, four loads on their way
            constexpr int CHUNKS = DH / 8;
            const uint16_t *from = keys ? tail_k : tail_v;
#pragma unroll 1
            for (int id0 = ct; id0 < KV8_BLOCK * CHUNKS; id0 += 4 * 128) {
                uint4 x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int id = id0 + 128 * j, key = keys ? id / CHUNKS : id % KV8_BLOCK, chunk = keys ? id % CHUNKS : id / KV8_BLOCK;
                    x[j] = make_uint4(0u, 0u, 0u, 0u);
                    if (key < have) x[j] = *reinterpret_cast<const uint4 *>(from + key * DH + 8 * chunk);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int id = id0 + 128 * j, key = keys ? id / CHUNKS : id % KV8_BLOCK, chunk = keys ? id % CHUNKS : id / KV8_BLOCK;
                    const uint32_t w[4] = {half_of(x[j].x, inv), half_of(x[j].y, inv), half_of(x[j].z, inv), half_of(x[j].w, inv)};
                    if (keys) {
                        *reinterpret_cast<uint4 *>(to + (chunk >> 3) * K_SLAB + swizzled(key, chunk & 7)) = make_uint4(w[0], w[1], w[2], w[3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            *reinterpret_cast<uint16_t *>(to + swizzled(8 * chunk + e, key >> 3) + (key & 7) * 2) =
                                static_cast<uint16_t>(e & 1 ? w[e / 2] >> 16 : w[e / 2]);
                    }
                }
            }
        };
        auto publish = [&](uint64_t *bar) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        // asks L2 for a page: a thread for some of its 128-byte lines
        auto ask = [&](int block, int page) {
            if (block >= full_pages || page < 0 || page >= c.pages) return;
            const int8_t *from = c.codes + kv8_unit(page, c.layers, a.layer, 0, c.kv_heads, kvh) * HALF_PAGE;
            constexpr int LINES = HALF_PAGE / 128;           // of the keys; as many of the values
            if (ct < 2 * LINES)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(from + (ct < LINES ? ct : ct - LINES) * 128 + (ct < LINES ? 0 : static_cast<size_t>(c.kv_heads) * HALF_PAGE)));
        };
        static_assert(2 * HALF_PAGE / 128 <= KP_CONVERT_WARPS * 32, "one line per thread");
        // the tail is read late, by loads that are waited for: asked into L2 now
        if (rest && (u1 - 1) * 2 + 1 >= full_pages)
            for (int o = ct * 64; o < rest * DH; o += 128 * 64) {
                asm volatile("prefetch.global.L2 [%0];" ::"l"(tail_k + o));
                asm volatile("prefetch.global.L2 [%0];" ::"l"(tail_v + o));
            }
        Half even, odd;                          // the unit's first and second page: keys, then values
        int far0 = page_at(2 * (u0 + KP_AHEAD)), far1 = page_at(2 * (u0 + KP_AHEAD) + 1);
        int page0 = page_at(2 * u0), page1 = page_at(2 * u0 + 1);
        fetch(even, 2 * u0, page0, true);
        fetch(odd, 2 * u0 + 1, page1, true);
        for (int i = 0; i < count; ++i) {
            const int block = 2 * (u0 + i);
            const bool more = i + 1 < count;
            uint8_t *k_to = k_s + (i % KS) * Shape::K, *v_to = v_s + (i % VS) * Shape::K;
            const int next0 = more ? page_at(block + 2) : 0, next1 = more ? page_at(block + 3) : 0;
            if (i + KP_AHEAD < count) {
                ask(block + 2 * KP_AHEAD, far0);
                ask(block + 2 * KP_AHEAD + 1, far1);
            }
            far0 = page_at(block + 2 * KP_AHEAD + 2);
            far1 = page_at(block + 2 * KP_AHEAD + 3);
            if (i >= KS && !wait(&k_free[i % KS], (i / KS - 1) & 1)) break;
            store(even, block, true, k_to);
            fetch(even, block, page0, false);
            store(odd, block + 1, true, k_to + KV8_BLOCK * 128);
            fetch(odd, block + 1, page1, false);
            publish(&k_full[i % KS]);
            if (i >= VS && !wait(&v_free[i % VS], (i / VS - 1) & 1)) break;
            store(even, block, false, v_to);
            if (more) fetch(even, block + 2, next0, true);
            store(odd, block + 1, false, v_to + V_PAGE);
            if (more) fetch(odd, block + 3, next1, true);
            publish(&v_full[i % VS]);
            page0 = next0;
            page1 = next1;
        }
    } else {
        // ---- softmax: a thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(KP_SOFTMAX_REGS<DH>));
        const int t = warp >> 2, local = 32 * (warp & 3) + lane, row = row0 + t * KP_ROWS + local, mine = t ? count1 : count0;
        const bool valid = row < rows;
        const int token = valid ? row / p.group : 0, pos = start + token;
        const size_t out_row = static_cast<size_t>(first + token) * a.heads + kvh * p.group + (valid ? row - token * p.group : 0);
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        float m = -INFINITY, l = 0.f, product_m = -INFINITY;     // largest score and sum of the weights relative to it; log2 M
        bool fine = wait(&q_full, 0);
        const float factor = factor_s[t * KP_ROWS + local];
        const float *layer_scales = c.scales + kv8_unit(0, c.layers, a.layer, 0, c.kv_heads, kvh);
        const int page_scales = c.layers * 2 * c.kv_heads;
        // scales of a unit's two blocks, read a unit ahead (their pages two units ahead)
        auto page_at = [&](int block) { return block < full_pages ? c.table[static_cast<size_t>(slot) * c.blocks + block] : 0; };
        auto scales_at = [&](int block, int page, float &ks, float &vs) {
            if (block < full_pages) {
                const bool held = page >= 0 && page < c.pages;
                const float *from = layer_scales + static_cast<size_t>(held ? page : 0) * page_scales;
                ks = held ? from[0] : kv8_nan();
                vs = held ? from[c.kv_heads] : kv8_nan();
            } else if (block * KV8_BLOCK < total) {
                const size_t u = kv8_unit(slot, c.layers, a.layer, 0, c.kv_heads, kvh);
                ks = tail_scale(abs_bits(c.peak[u]));
                vs = tail_scale(abs_bits(c.peak[u + c.kv_heads]));
            } else {
                ks = vs = 0.f;
            }
        };
        float ks_next[2] = {0.f, 0.f}, vs_next[2] = {0.f, 0.f};
        int page_next[2] = {0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (mine) scales_at(2 * u0 + h, page_at(2 * u0 + h), ks_next[h], vs_next[h]);
            if (mine > 1) page_next[h] = page_at(2 * u0 + 2 + h);
        }
        for (int i = 0; fine && i < mine; ++i) {
            const int block = 2 * (u0 + i), key0 = block * KV8_BLOCK;
            float f[2], log_scale[2], alpha = 1.f;
            bool sees[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float ks = ks_next[h];
                log_scale[h] = log2_approx(vs_next[h]);
                if (i + 1 < mine) scales_at(block + 2 + h, page_next[h], ks_next[h], vs_next[h]);
                if (i + 2 < mine) page_next[h] = page_at(block + 4 + h);
                sees[h] = pos >= key0 + h * KV8_BLOCK;
                // (not below the smallest normal number, where a hidden key's -inf would meet a zero)
                f[h] = factor * ks;
                if (f[h] < KV8_MIN_SCALE || !sees[h]) f[h] = KV8_MIN_SCALE;
            }
            fine = wait(&s_full[t], i & 1);
            if (!fine) break;
            tc_fence_after();
            const uint32_t at = tmem + lanes + S_COL + 128 * t;
            uint32_t s[4][32];
#pragma unroll
            for (int q = 0; q < 4; ++q) tmem_ld32(at + 32 * q, s[q]);
            tmem_ld_wait();
            if (__any_sync(0xffffffffu, pos < key0 + KP_KEYS - 1)) {         // hidden keys
                const int limit = pos - key0;
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * q + e > limit) s[q][e] = 0xff800000u;
            }
            float tops[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                tops[q] = fmaxf(__uint_as_float(s[q][0]), __uint_as_float(s[q][1]));
#pragma unroll
                for (int e = 2; e < 32; e += 2) tops[q] = max3(tops[q], __uint_as_float(s[q][e]), __uint_as_float(s[q][e + 1]));
            }
            // (of a block that is hidden or not finite nothing comes through fmaxf)
            const float peak[2] = {fmaxf(tops[0], tops[1]) * f[0], fmaxf(tops[2], tops[3]) * f[1]};
            const float product[2] = {sees[0] ? peak[0] + log_scale[0] : -INFINITY, sees[1] ? peak[1] + log_scale[1] : -INFINITY};
            const float top = fmaxf(peak[0], peak[1]), top_product = fmaxf(product[0], product[1]);
            if (top > m + 8.f) {
                l *= exp2_approx(m - top);
                m = top;
            }
            if (top_product > product_m + KP_SLACK) {
                alpha = exp2_approx(product_m - top_product);
                product_m = top_product;
            }
            if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {            // (S of this unit follows the last value product)
#pragma unroll 1
                for (int d = 0; d < DH; d += 16) {
                    uint32_t o[16];
                    tmem_ld16(tmem + lanes + O_COL + DH * t + d, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                    tmem_st16(tmem + lanes + O_COL + DH * t + d, o);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool nothing = product[h] < product_m - KP_NOTHING || log_scale[h] == -INFINITY;
                const float move = !sees[h] ? 0.f : nothing ? -INFINITY : log_scale[h] - product_m + KP_RANGE;
                const float weigh = !sees[h] || nothing ? 0.f : exp2_approx(-move - m);
                if (__any_sync(0xffffffffu, nothing && sees[h])) {               // (rare; selected, so that the lanes stay together)
                    float only = 0.f;
#pragma unroll
                    for (int q = 0; q < 2; ++q)
#pragma unroll
                        for (int e = 0; e < 32; ++e) only += exp2_approx(fmaf(__uint_as_float(s[2 * h + q][e]), f[h], -peak[h]));
                    l += nothing && sees[h] ? only * exp2_approx(peak[h] - m) : 0.f;
                }
                const Pair f2 = pair(f[h], f[h]), move2 = pair(move, move);        // pairs: two per instruction
                Pair sums[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    uint32_t w[16], left[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const Pair exponents = pair_fma(pair(__uint_as_float(s[2 * h + q][e]), __uint_as_float(s[2 * h + q][e + 1])), f2, move2);
                        const float lo = exp2_approx(exponents.lo()), hi = exp2_approx(exponents.hi());
                        sums[e / 2 & 1] = pair_add(sums[e / 2 & 1], pair(lo, hi));
                        // (cut off at eleven bits, so that what is left is one exact subtraction)
                        auto minus_top = [](float x) { return __uint_as_float((__float_as_uint(x) & 0xffffe000u) | 0x80000000u); };
                        const Pair rest = pair_add(pair(lo, hi), pair(minus_top(lo), minus_top(hi)));
                        w[e / 2] = cut_half(lo, hi);
                        left[e / 2] = pack_half(rest.lo(), rest.hi());
                    }
                    tmem_st16(at + P_COL + 32 * h + 16 * q, w);
                    tmem_st16(at + 32 * h + 16 * q, left);
                }
                const Pair sum = pair_add(sums[0], sums[1]);
                l = fmaf(sum.lo() + sum.hi(), weigh, l);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t][h]);
            }
        }
        // ---- results
        if (mine && fine && wait(&o_done[t], 0)) {
            tc_fence_after();
            // (in two factors: M and the largest weight may lie 2^126 apart; a part of which the row sees no key adds nothing)
            const float half_gain = m == -INFINITY ? 0.f : exp2_approx(0.5f * (product_m - KP_RANGE - m));
            const float gain = p.splits == 1 ? __fdiv_rn(half_gain, l) : half_gain;
            float *to = p.splits == 1 ? nullptr : p.partial + ((static_cast<size_t>(part) * a.rows) * a.heads + out_row) * (DH + 2);
#pragma unroll 1
            for (int d = 0; d < DH; d += 32) {
                uint32_t o[32];
                __syncwarp();                    // (lanes whose rows do not exist)
                tmem_ld32(tmem + lanes + O_COL + DH * t + d, o);
                tmem_ld_wait();
                if (!valid) continue;
                float v[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(o[e]) * half_gain * gain;
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
    const int all = (start + (end - 1) / p.group) / KP_KEYS + 1;         // units of the row's CTA
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
// Parts of the keys, and the time that is estimated for them, in us: CTAs (one per SM; where they do not all start at once, half a
// CTA's time is lost at the end), each with its beginning and end and its units, and, for more than one part, the results on their way
// through memory and the joining kernel. Measured with one CTA per SM for a head dimension of 128: 25 us for one tile of rows and four
// units, 31 with two tiles, 37 and 48 for eight units. 128 CTAs of 63 units (16 sequences of 8000 keys) took 218 us in three parts, so in three rounds, when they
// took 196 in one (215 since the weights have remainders); 32 of 32 units 87 in eight parts, 59 in four. A further part has to gain a twentieth: three instead of two for
// the 192 CTAs of three chunks of 512 tokens behind up to 16000 took 369 us instead of 336.
struct PromptPlan {
    int splits;
    double time;
};
static PromptPlan prompt_plan(const b200q_kv8_cache *c, int heads, int batch, int rows, int max_new, int max_keys) {
    const long long list = static_cast<long long>(max_new) * (heads / c->kv_heads), units = (max_keys + KP_KEYS - 1) / KP_KEYS;
    const double ctas = static_cast<double>((list + KP_CTA_ROWS - 1) / KP_CTA_ROWS) * c->kv_heads * batch / sm_count();      // per SM
    const bool two = list > KP_ROWS, wide = c->head_dim == 128;
    const double once = two ? (wide ? 10.5 : 8.1) : (wide ? 5.7 : 4.8), unit = two ? (wide ? 5.2 : 3.7) : (wide ? 3.7 : 3.);
    const double part_bytes = 2. * rows * heads * (c->head_dim + 2) * 4.;
    PromptPlan best{1, 0.};
    for (int s = 1; s <= std::min(64ll, std::max(1ll, units / 2)); ++s) {
        const double rounds = ctas * s <= 1. ? 1. : ctas * s + 0.5;
        const double time = 3. + rounds * (once + unit * ((units + s - 1) / s)) + (s > 1 ? 4. + s * part_bytes * 2e-7 : 0.);
        if (s == 1 || time < 0.95 * best.time) best = {s, time};
    }
    return best;
}
static int prompt_splits(const b200q_kv8_cache *c, int heads, int batch, int rows, int max_new, int max_keys) {
    return prompt_plan(c, heads, batch, rows, max_new, max_keys).splits;
}
double kv8_prompt_time(const b200q_kv8_cache *c, int heads, int batch, int rows, int max_new, int max_keys) {
    return prompt_plan(c, heads, batch, rows, max_new, max_keys).time;
}

long long kv8_prompt_workspace(const b200q_kv8_cache *c, int heads, int batch, int rows, int max_new, int max_keys) {
    const int splits = prompt_splits(c, heads, batch, rows, max_new, max_keys);
    return splits == 1 ? 0 : static_cast<long long>(splits) * rows * heads * (c->head_dim + 2) * 4;
}

int kv8_prompt(const b200q_kv8_cache *c, const Kv8Attention &a, int max_new, int max_keys, void *workspace, long long workspace_bytes,
               cudaStream_t stream) {
    Kv8Prompt p{};
    p.a = a;
    p.group = a.heads / c->kv_heads;
    p.splits = prompt_splits(c, a.heads, a.batch, a.rows, max_new, max_keys);
    const long long bytes = kv8_prompt_workspace(c, a.heads, a.batch, a.rows, max_new, max_keys);
    if (bytes > workspace_bytes || (bytes && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15))))
        return fail(B200Q_EINVAL, "kv8_attention: workspace of %lld bytes, 16-byte aligned, needed", bytes);
    p.partial = static_cast<float *>(workspace);
    p.status = device_status_word();
    if (!p.status) return fail(B200Q_ECUDA, "kv8_attention: no CUDA device");
    const long long blocks = (static_cast<long long>(max_new) * p.group + KP_CTA_ROWS - 1) / KP_CTA_ROWS;
    const long long across = static_cast<long long>(c->kv_heads) * p.splits;
    const long long joins = (static_cast<long long>(a.rows) * a.heads + 7) / 8;
    if (a.batch > 65535 || blocks > 65535 || across > 0x7fffffffll || joins > 0x7fffffffll || static_cast<long long>(max_new) * p.group > 0x40000000ll)
        return fail(B200Q_EUNSUPPORTED, "kv8_attention: too many rows");
    const bool bf16 = c->dtype == B200Q_BF16;
    auto kernel = c->head_dim == 64 ? (bf16 ? kv8_prompt_kernel<64, true> : kv8_prompt_kernel<64, false>)
                                    : (bf16 ? kv8_prompt_kernel<128, true> : kv8_prompt_kernel<128, false>);
    const int smem = 1024 + (c->head_dim == 64 ? PromptShape<64>::BYTES : PromptShape<128>::BYTES);
    if (int rc = allow_large_shared_memory(reinterpret_cast<const void *>(kernel))) return rc;
    launch_chained(kernel, dim3(static_cast<unsigned>(across), a.batch, static_cast<unsigned>(blocks)), dim3(KP_THREADS), smem, stream, *c, p);
    if (int rc = check_launch("kv8_attention")) return rc;
    if (p.splits == 1) return B200Q_OK;
    launch_chained(c->head_dim == 64 ? kv8_prompt_join_kernel<64> : kv8_prompt_join_kernel<128>, dim3(static_cast<unsigned>(joins)), dim3(256), 0,
                   stream, *c, p);
    return check_launch("kv8_attention (join)");
}

}  // namespace b200q
