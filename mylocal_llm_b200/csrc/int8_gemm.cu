// Matrix product in 8-bit integers with one scale per token and per output channel, and the quantiser of its operands.
#include <algorithm>
#include <type_traits>

#include "kv8_cache.cuh"
#include "umma.cuh"

namespace b200q {

// Eight consecutive values of type IN as they are loaded. VEC: 16-byte loads are possible.
template <int IN> struct Raw8 {
    uint4 w;
    __device__ __forceinline__ void values(float (&f)[8]) const {
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 v = IN == B200Q_BF16 ? make_float2(__uint_as_float(x[e] << 16), __uint_as_float(x[e] & 0xffff0000u))
                                              : __half22float2(*reinterpret_cast<const __half2 *>(&x[e]));
            f[2 * e] = v.x;
            f[2 * e + 1] = v.y;
        }
    }
};
template <> struct Raw8<B200Q_F32> {
    float4 w[2];
    __device__ __forceinline__ void values(float (&f)[8]) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f[4 * h] = w[h].x; f[4 * h + 1] = w[h].y; f[4 * h + 2] = w[h].z; f[4 * h + 3] = w[h].w;
        }
    }
};
template <int IN, bool VEC>
__device__ __forceinline__ Raw8<IN> load8(const void *p, size_t base, int c, int k) {
    Raw8<IN> r;
    if constexpr (IN == B200Q_F32) {
        const float *q = static_cast<const float *>(p) + base + c;
        if (VEC && c + 8 <= k) {
            r.w[0] = reinterpret_cast<const float4 *>(q)[0];
            r.w[1] = reinterpret_cast<const float4 *>(q)[1];
        } else {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = c + e < k ? q[e] : 0.f;
            r.w[0] = make_float4(f[0], f[1], f[2], f[3]);
            r.w[1] = make_float4(f[4], f[5], f[6], f[7]);
        }
    } else {
        const uint16_t *q = static_cast<const uint16_t *>(p) + base + c;
        if (VEC && c + 8 <= k) {
            r.w = *reinterpret_cast<const uint4 *>(q);
        } else {
            uint32_t x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[e] = (c + 2 * e < k ? q[2 * e] : 0u) | (c + 2 * e + 1 < k ? static_cast<uint32_t>(q[2 * e + 1]) << 16 : 0u);
            r.w = make_uint4(x[0], x[1], x[2], x[3]);
        }
    }
    return r;
}
// Largest magnitude of eight values, as the bits of a float (16-bit integers order 16-bit floats, NaN and infinities on top).
template <int IN>
__device__ __forceinline__ uint32_t peak8(const Raw8<IN> &r) {
    if constexpr (IN == B200Q_F32) {
        uint32_t top = 0u;
#pragma unroll
        for (int h = 0; h < 2; ++h) top = max(max(top, max(abs_bits(r.w[h].x), abs_bits(r.w[h].y))), max(abs_bits(r.w[h].z), abs_bits(r.w[h].w)));
        return top;
    } else {
        constexpr uint32_t SIGNS = 0x7fff7fffu;
        const uint32_t top = __vmaxu2(__vmaxu2(r.w.x & SIGNS, r.w.y & SIGNS), __vmaxu2(r.w.z & SIGNS, r.w.w & SIGNS));
        return max(top & 0xffffu, top >> 16);
    }
}
template <int IN>
__device__ __forceinline__ uint32_t peak_bits(uint32_t peak) {
    if (IN == B200Q_F32) return peak;
    if (IN == B200Q_BF16) return peak << 16;
    return abs_bits(__half2float(__ushort_as_half(static_cast<unsigned short>(peak))));
}

// Eight values on their way: VEC rows as they are, other rows (whose beginning is no multiple of 16 bytes) as the aligned 16-byte
// words around them, `off` bytes in front of the first. The words may hold bytes of the rows before and behind, which do not
// count; where they would begin before the first row or end behind the last one, the values are fetched one by one (`get`).
template <int IN, bool VEC> struct Piece {
    Raw8<IN> r;
    __device__ __forceinline__ void load(const void *x, size_t base, int c, int k, const char *, const char *, bool wanted) {
        r = Raw8<IN>{};
        if (wanted) r = load8<IN, VEC>(x, base, c, k);
    }
    __device__ __forceinline__ Raw8<IN> get(const void *, size_t, int, int) const { return r; }
};
template <int IN> struct Piece<IN, false> {
    static constexpr int E = IN == B200Q_F32 ? 4 : 2, WORDS = 2 * E + 4;
    uint32_t w[WORDS];
    int off;                                             // -1: nothing was requested
    __device__ __forceinline__ void load(const void *x, size_t base, int c, int, const char *first, const char *end, bool wanted) {
        const char *q = static_cast<const char *>(x) + (base + c) * E;
        off = static_cast<int>(reinterpret_cast<uintptr_t>(q) & 15);
        const char *from = q - off;
        if (!wanted || from < first || from + 4 * WORDS > end) {
            off = -1;
            return;
        }
#pragma unroll
        for (int i = 0; i < WORDS / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4 *>(from)[i];
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    }
    __device__ __forceinline__ Raw8<IN> get(const void *x, size_t base, int c, int k) const {
        if (off < 0) return load8<IN, false>(x, base, c, k);
        uint32_t a[WORDS - 2], b[WORDS - 3], v[2 * E];
#pragma unroll
        for (int i = 0; i < WORDS - 2; ++i) a[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
        for (int i = 0; i < WORDS - 3; ++i) b[i] = off & 4 ? a[i + 1] : a[i];
#pragma unroll
        for (int i = 0; i < 2 * E; ++i) v[i] = E == 4 ? b[i] : __funnelshift_r(b[i], b[i + 1 < WORDS - 3 ? i + 1 : i], 8 * (off & 2));
        if (c + 8 > k)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e >= k) v[e * E / 4] &= E == 4 || e % 2 == 0 ? 0u : 0xffffu;
        Raw8<IN> r;
        if constexpr (IN == B200Q_F32) {
            r.w[0] = make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
            r.w[1] = make_float4(__uint_as_float(v[4]), __uint_as_float(v[5]), __uint_as_float(v[6]), __uint_as_float(v[7]));
        } else {
            r.w = make_uint4(v[0], v[1], v[2], v[3]);
        }
        return r;
    }
};

constexpr int I8_MAX_SIZE = 1 << 30;                 // rows and columns: sums of an index and a step fit 32 bits

// A team of `team` warps takes a row at a time: the largest magnitude, then the codes. The row's pieces of eight values stay in
// registers, as they were loaded, between the two up to 256 * team * KEEP columns (longer rows are read again), and the next row's
// are on their way meanwhile. Teams are as small as the row allows: warps that need not meet (6992 x 706 FP32, cold: by whole CTAs
// 37 us, by small teams 17). 4096 x 8192 BF16 take 26 us (held as floats instead of as loaded 34 us), 15 at the measured bandwidth:
// bound by issue slots (0.69 of them, some 19 instructions per value).
constexpr int I8_QUANTIZE_KEEP = 4;                  // pieces of 16-bit values (of FP32: half as many)
template <int IN, bool VEC>
__global__ void __launch_bounds__(256, VEC ? 4 : 2) int8_quantize_kernel(const void *x, int rows, int k, long long x_row, int8_t *codes,
                                                                         long long codes_row, float *scales, int team, int early) {
    constexpr int KEEP = IN == B200Q_F32 ? I8_QUANTIZE_KEEP / 2 : I8_QUANTIZE_KEEP;
    __shared__ uint32_t peaks[8];
    chain_wait();
    if (early) chain_trigger();                          // (only now: what the next kernel reads early was written before this one)
    const int warp = threadIdx.x >> 5, mine = warp & (team - 1), first_warp = warp - mine;
    const int c0 = (32 * mine + (threadIdx.x & 31)) * 8, width = 256 * team, padded = (k + 15) & ~15;
    const int row0 = (blockIdx.x * 8 + warp) / team, step = gridDim.x * 8 / team;
    auto meet = [&] {                                    // (barrier 0 is the CTA's)
        if (team > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + first_warp / team), "r"(32 * team) : "memory");
    };
    const char *first = static_cast<const char *>(x);
    const char *end = first + ((rows - 1) * static_cast<size_t>(x_row) + k) * (IN == B200Q_F32 ? 4 : 2);
    // (a row of which the thread has KEEP whole pieces needs no looking at their ends)
    const bool whole = VEC && c0 + width * (KEEP - 1) + 8 <= k;
    Piece<IN, VEC> next[KEEP];
    auto load_row = [&](int row) {
        if constexpr (VEC)
            if (whole && row < rows) {
                const char *from = first + (row * static_cast<size_t>(x_row) + c0) * (IN == B200Q_F32 ? 4 : 2);
#pragma unroll
                for (int j = 0; j < KEEP; ++j) next[j].r = *reinterpret_cast<const Raw8<IN> *>(from + static_cast<size_t>(width * j) * (IN == B200Q_F32 ? 4 : 2));
                return;
            }
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            const int c = c0 + width * j;
            next[j].load(x, row * static_cast<size_t>(x_row), c, k, first, end, row < rows && c < k);
        }
    };
    load_row(row0);
    for (int row = row0; row < rows; row += step) {
        const size_t base = row * static_cast<size_t>(x_row);
        Raw8<IN> kept[KEEP];
        uint32_t peak = 0u;
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            kept[j] = next[j].get(x, base, c0 + width * j, k);
            peak = max(peak, peak8<IN>(kept[j]));
        }
        load_row(row + step);
        auto again = [&](int c) {
            Piece<IN, VEC> piece;
            piece.load(x, base, c, k, first, end, true);
            return piece.get(x, base, c, k);
        };
        for (int c = c0 + width * KEEP; c < k; c += width) peak = max(peak, peak8<IN>(again(c)));
        peak = __reduce_max_sync(0xffffffffu, peak);
        if (team > 1) {
            meet();                                      // (the previous row's peaks have been read)
            if ((threadIdx.x & 31) == 0) peaks[warp] = peak;
            meet();
            peak = __reduce_max_sync(0xffffffffu, peaks[first_warp + (threadIdx.x & (team - 1))]);
        }
        const float s = int8_scale(peak_bits<IN>(peak)), inv = __fdiv_rn(1.f, s);
        if (c0 == 0) scales[row] = s;
        int8_t *to = codes + row * static_cast<size_t>(codes_row);
        auto put = [&](int c, const Raw8<IN> &r) {
            float f[8];
            r.values(f);
            const float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
            *reinterpret_cast<uint2 *>(to + c) = make_uint2(int8_codes(lo, s, inv), int8_codes(hi, s, inv));
        };
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            const int c = c0 + width * j;
            if (whole || c < padded) put(c, kept[j]);
        }
        for (int c = c0 + width * KEEP; c < padded; c += width) put(c, c < k ? again(c) : Raw8<IN>{});
    }
}

// ---------------------------------------------------------------------------------------------
// The product. Tokens are the M dimension of tcgen05.mma (kind::i8, signed by signed into 32-bit integers), output channels the
// N dimension; both operands are K-major slabs of 128 codes a row, brought by TMA with the 128-byte swizzle (rows and codes past
// the end arrive as zeros). One warp issues the loads, one the MMAs, four or eight read the sums back from tensor memory, scale and
// store them. There are two kernels:
//   int8_tile_kernel  one tile of 128 tokens x NT channels per CTA. Few tiles (few tokens, few channels): the K range is
//                     divided among the 2, 4 or 8 CTAs of a cluster, whose integer sums meet in shared memory - exact, so the
//                     division does not show in the result. Behind the quantiser of the activations (`early`), which lets this
//                     kernel start when everything in front of it is complete, weights are requested before it has ended.
//   int8_pair_kernel  many tokens: CTAs 2p and 2p + 1 are one tensor-core unit (cta_group::2) and own 256 x 256 tiles, each
//                     with half of both operands in its shared memory; the pairs walk the tiles in turn, and the sums of a tile
//                     are stored while the next one is computed (two accumulators fill the tensor memory).
// With few tokens the weights' bytes bound the product, with many the tensor cores.
//
// Every wait is bounded as in umma_gemm.cu: on expiry the status word tells, all roles leave their loops, copies in flight get
// time to land, the tensor memory is freed and the CTAs return.
// ---------------------------------------------------------------------------------------------
constexpr int I8_BM = 128, I8_BK = 128;              // tokens per CTA; codes per slab (one 128-byte swizzle row)
constexpr int I8_A_BYTES = I8_BM * I8_BK;
constexpr int I8_THREADS = 6 * 32;                   // TMA, MMA, four epilogue warps
constexpr int I8_PAIR_THREADS = 10 * 32;             // TMA, MMA, eight epilogue warps
constexpr int I8_MAX_STAGES = 8;
constexpr int STATUS_INT8_WAIT_TMA = 121, STATUS_INT8_WAIT_MMA = 122, STATUS_INT8_WAIT_EPILOGUE = 123;

struct Int8Gemm {
    const float *w_scales, *x_scales;
    int n, k, m;
    void *y;
    int y_dtype;
    int x_rows;               // rows of the activation box (a multiple of 8)
    int stages, slabs;        // slabs of K
    int tiles_m, tiles_n;     // int8_pair_kernel
    bool early;               // int8_tile_kernel: the preceding kernel does not write the weights, and what did is complete
    int *status;
};

// Instruction descriptor of kind::i8: 32-bit integer accumulator (bits [4,6) = 2), A and B signed (bits [7,10) and [10,13) = 1),
// both K-major, N >> 3 in [17,23), M >> 4 in [24,29).
__host__ __device__ constexpr uint32_t umma_idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

template <bool PAIR>
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
}

// A warp's 32 tokens x 32 channels: each lane's sums of one token, times that token's scale, pass through 4 KB of shared memory so
// that a lane has one channel of all tokens, whose scale is `w`, and the warp stores a token's 32 outputs together, whatever n and
// the alignment of rows (lanes that stored their own token's 64 bytes, one by one where rows are not 16-byte aligned: 1262 x 8231 x
// 2000 with its quantiser 140 us, so 39 us; 1993 x 12581 x 317 257 and 37 us). `at`: element of the first token, this lane's channel; `rows`: tokens that exist.
template <typename T>
__device__ __forceinline__ void store_channel(T *y, size_t n, int rows, uint32_t stage, int lane, float w) {
    auto put = [&](int r) {                              // (r * 128 + 4 * (lane ^ r): one exclusive or where r is a constant)
        float v;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"((stage ^ (4u * (lane ^ r))) + r * 128u));
        v *= w;
        T *to = y + r * n;
        if constexpr (sizeof(T) == 4) *to = v;
        else if constexpr (std::is_same_v<T, __half>) *to = __float2half_rn(v);
        else *to = __float2bfloat16_rn(v);
    };
    if (rows == 32) {
#pragma unroll
        for (int r = 0; r < 32; ++r) put(r);
    } else {
#pragma unroll 1
        for (int r = 0; r < rows; ++r) put(r);
    }
}
// `stage`: 4 KB, on a multiple of 128 bytes.
__device__ __forceinline__ void store_outputs(void *y, int y_dtype, size_t at, int n, bool exists, int rows, const uint32_t (&sums)[32], float xs,
                                              float w, uint32_t stage, int lane) {
    __syncwarp();                                        // (the previous outputs have been read)
    const uint32_t mine = stage + lane * 132u;           // lane * 128 + 4 * (e ^ lane)
#pragma unroll
    for (int e = 0; e < 32; ++e)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine ^ (4u * e)), "f"(static_cast<float>(static_cast<int>(sums[e])) * xs) : "memory");
    __syncwarp();
    if (!exists) return;
    if (y_dtype == B200Q_F32) store_channel(static_cast<float *>(y) + at, n, rows, stage, lane, w);
    else if (y_dtype == B200Q_F16) store_channel(static_cast<__half *>(y) + at, n, rows, stage, lane, w);
    else store_channel(static_cast<__nv_bfloat16 *>(y) + at, n, rows, stage, lane, w);
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

// grid (channel tiles * SPLIT, token tiles), clusters of SPLIT along x: CTA r of a cluster owns slabs [slabs * r / SPLIT, ...).
template <int NT, int SPLIT>
__global__ void __launch_bounds__(I8_THREADS, 1) int8_tile_kernel(const __grid_constant__ CUtensorMap xmap,
                                                                  const __grid_constant__ CUtensorMap wmap, const Int8Gemm a) {
    constexpr int STAGE = I8_A_BYTES + NT * I8_BK;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[I8_MAX_STAGES], free_bar[I8_MAX_STAGES], acc_done;
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile int abort_flag;
    __shared__ float w_scale[NT];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = SPLIT > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
    const int n0 = (blockIdx.x / SPLIT) * NT, m0 = blockIdx.y * I8_BM, S = a.stages;
    const int slab0 = a.slabs * rank / SPLIT, nslab = a.slabs * (rank + 1) / SPLIT - slab0;
    if (tid == 0) {
        for (int s = 0; s < I8_MAX_STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&free_bar[s], 1);
        }
        mbar_init(&acc_done, 1);
        abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0) {
        tmem_alloc<false>(&tmem_base_slot, NT);
        tmem_relinquish<false>();
    }
    if (!a.early) chain_wait();
    for (int i = tid; i < NT; i += I8_THREADS) w_scale[i] = n0 + i < a.n ? a.w_scales[n0 + i] : 0.f;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    chain_trigger();                     // (with the tensor memory in hand: the next kernel may allocate some before it waits)
    const uint32_t tmem_d = tmem_base_slot;

    if (warp == 0) {
        // ---- loads: `early`, the first stages' weights do not wait for the preceding kernel, whose result the activations are
        const uint32_t bytes = static_cast<uint32_t>(a.x_rows * I8_BK + NT * I8_BK);
        const int early = min(S, nslab);
        if (elect_one())
            for (int i = 0; i < early; ++i) {
                mbar_arrive_expect_tx(&full_bar[i], bytes);
                tma_load_2d(smem + i * STAGE + I8_A_BYTES, &wmap, (slab0 + i) * I8_BK, n0, &full_bar[i]);
            }
        __syncwarp();
        chain_wait();
        int issued = early, s = 0, wraps = 0;
        if (elect_one())
            for (int i = 0; i < early; ++i) tma_load_2d(smem + i * STAGE, &xmap, (slab0 + i) * I8_BK, m0, &full_bar[i]);
        __syncwarp();
        for (int i = early; i < nslab; ++i) {
            if (__any_sync(0xffffffffu, abort_flag != 0)) break;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&free_bar[s], wraps & 1, a.status, STATUS_INT8_WAIT_MMA))) {
                abort_flag = 1;
                break;
            }
            if (elect_one()) {
                mbar_arrive_expect_tx(&full_bar[s], bytes);
                tma_load_2d(smem + s * STAGE + I8_A_BYTES, &wmap, (slab0 + i) * I8_BK, n0, &full_bar[s]);
                tma_load_2d(smem + s * STAGE, &xmap, (slab0 + i) * I8_BK, m0, &full_bar[s]);
            }
            __syncwarp();
            ++issued;
            if (++s == S) {
                s = 0;
                ++wraps;
            }
        }
        if (abort_flag) {
            // copies already requested still write shared memory; they complete on their own within microseconds
            const uint64_t t0 = global_timer_ns();
            while (issued > 0 && global_timer_ns() - t0 < 100000) {
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMAs (the whole warp walks the loop, one elected lane issues)
        constexpr uint32_t idesc = umma_idesc_i8(I8_BM, NT);
        const uint64_t desc0 = smem_desc_sw128(smem);
        int done = 0, s = 0, phase = 0;
        for (int i = 0; i < nslab; ++i) {
            if (__any_sync(0xffffffffu, abort_flag != 0)) break;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full_bar[s], phase, a.status, STATUS_INT8_WAIT_TMA))) {
                abort_flag = 1;
                break;
            }
            tc_fence_after();
            if (elect_one()) {
                const uint64_t x_desc = desc0 + static_cast<uint32_t>(s * STAGE >> 4), w_desc = x_desc + (I8_A_BYTES >> 4);
#pragma unroll
                for (int q = 0; q < 4; ++q)            // 32 codes = 32 bytes per step: +2 in the address field
                    umma_i8<false>(tmem_d, x_desc + 2 * q, w_desc + 2 * q, idesc, i + q > 0);
                umma_commit<false>(smem_u32(&free_bar[s]));
            }
            __syncwarp();
            done = i + 1;
            if (++s == S) {
                s = 0;
                phase ^= 1;
            }
        }
        if (done == nslab && elect_one()) umma_commit<false>(smem_u32(&acc_done));
        __syncwarp();
    }
    // ---- the sums
    bool ok = !abort_flag;
    if (ok && !mbar_wait_bounded(&acc_done, 0, a.status, STATUS_INT8_WAIT_MMA)) {
        abort_flag = 1;
        ok = false;
    }
    ok = __syncthreads_and(ok) != 0;
    const int quarter = warp & 3, row = 32 * quarter + lane, rows = min(I8_BM, a.m - m0);
    if constexpr (SPLIT == 1) {
        if (ok && warp >= 2 && 32 * quarter < rows) {
            tc_fence_after();
            chain_wait();                // y may still be read by what precedes this kernel; the scales are its result
            const float xs = row < rows ? a.x_scales[m0 + row] : 0.f;
            const uint32_t stage = smem_u32(smem) + warp % 4 * 4096u;            // (the operands have been read)
#pragma unroll 1
            for (int c = 0; c < NT / 32; ++c) {
                const int col = n0 + 32 * c + lane;
                uint32_t r[32];
                __syncwarp();                            // (lanes whose outputs do not exist)
                tmem_ld32(tmem_d + (static_cast<uint32_t>(32 * quarter) << 16) + 32 * c, r);
                tmem_ld_wait();
                store_outputs(a.y, a.y_dtype, static_cast<size_t>(m0 + 32 * quarter) * a.n + col, a.n, col < a.n, min(32, rows - 32 * quarter),
                              r, xs, w_scale[32 * c + lane], stage, lane);
            }
        }
        tc_fence_before();
        __syncthreads();
    } else {
        // the cluster's partial sums, [row][NT + 1] integers where the stages were
        constexpr int LD = NT + 1;
        uint32_t *part = reinterpret_cast<uint32_t *>(smem);
        if (ok && warp >= 2 && 32 * quarter < rows) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < NT / 32; ++c) {
                uint32_t r[32];
                __syncwarp();                            // (lanes whose outputs do not exist)
                tmem_ld32(tmem_d + (static_cast<uint32_t>(32 * quarter) << 16) + 32 * c, r);
                tmem_ld_wait();
                if (row < rows)
#pragma unroll
                    for (int e = 0; e < 32; ++e) part[row * LD + 32 * c + e] = r[e];
            }
        }
        tc_fence_before();
        cluster_sync_all();
        if (ok) {
            chain_wait();
            const int total = rows * NT, from = total * rank / SPLIT, to = total * (rank + 1) / SPLIT;
            uint32_t base[SPLIT];
#pragma unroll
            for (int q = 0; q < SPLIT; ++q) base[q] = cluster_map(smem_u32(part), q);
            for (int i = from + tid; i < to; i += I8_THREADS) {
                const int rr = i / NT, col = i - rr * NT;
                int sum = 0;
#pragma unroll
                for (int q = 0; q < SPLIT; ++q) sum += static_cast<int>(ld_cluster_u32(base[q] + 4u * (rr * LD + col)));
                if (n0 + col < a.n)
                    store_from_float(a.y, a.y_dtype, static_cast<size_t>(m0 + rr) * a.n + n0 + col,
                                     static_cast<float>(sum) * a.x_scales[m0 + rr] * w_scale[col]);
            }
        }
        cluster_sync_all();              // nobody leaves while its sums may still be read
    }
    if (warp == 0) tmem_dealloc<false>(tmem_d, NT);
}

// 256 tokens x 256 channels per pair of CTAs; tiles are numbered in bands of eight token tiles, so that the pairs at work share
// the weights and activations that L2 holds.
constexpr int I8_PAIR_STAGE = 2 * I8_A_BYTES;        // 128 rows of each operand
__device__ __forceinline__ void pair_tile(const Int8Gemm &a, int tile, int &m0, int &n0) {
    constexpr int BAND = 8;
    const int per_band = BAND * a.tiles_n, band = tile / per_band, in = tile - band * per_band;
    const int high = min(BAND, a.tiles_m - band * BAND);
    const int tn = in / high;
    m0 = (band * BAND + in - tn * high) * 256;
    n0 = tn * 256;
}

__global__ void __launch_bounds__(I8_PAIR_THREADS, 1) int8_pair_kernel(const __grid_constant__ CUtensorMap xmap,
                                                                  const __grid_constant__ CUtensorMap wmap, const Int8Gemm a) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[I8_MAX_STAGES], free_bar[I8_MAX_STAGES], acc_full[2], acc_free[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile int abort_flag;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, S = a.stages;
    const uint32_t rank = cluster_cta_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, tiles = a.tiles_m * a.tiles_n;
    if (tid == 0) {
        for (int s = 0; s < I8_MAX_STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&free_bar[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_free[i], 16);             // eight epilogue warps of both CTAs
        }
        abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0) {
        tmem_alloc<true>(&tmem_base_slot, 512);
        tmem_relinquish<true>();
    }
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    chain_trigger();
    const uint32_t tmem_d = tmem_base_slot;

    if (warp == 0) {
        chain_wait();
        const uint32_t full0 = cluster_map(smem_u32(&full_bar[0]), 0);
        int issued = 0, s = 0, wraps = 0;
        for (int tile = pair; tile < tiles; tile += pairs) {
            int m0, n0;
            pair_tile(a, tile, m0, n0);
            m0 += 128 * static_cast<int>(rank);
            n0 += 128 * static_cast<int>(rank);
            for (int i = 0; i < a.slabs; ++i) {
                if (__any_sync(0xffffffffu, abort_flag != 0)) break;
                if (wraps > 0 && !__all_sync(0xffffffffu, mbar_wait_bounded(&free_bar[s], (wraps - 1) & 1, a.status, STATUS_INT8_WAIT_MMA))) {
                    abort_flag = 1;
                    break;
                }
                if (elect_one()) {
                    // the first CTA announces the bytes of both; either half may land first
                    if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * I8_PAIR_STAGE);
                    tma_load_2d_pair(smem + s * I8_PAIR_STAGE, &xmap, i * I8_BK, m0, full0 + 8u * s);
                    tma_load_2d_pair(smem + s * I8_PAIR_STAGE + I8_A_BYTES, &wmap, i * I8_BK, n0, full0 + 8u * s);
                }
                __syncwarp();
                issued = 1;
                if (++s == S) {
                    s = 0;
                    ++wraps;
                }
            }
            if (abort_flag) break;
        }
        if (abort_flag) {
            const uint64_t t0 = global_timer_ns();
            while (issued > 0 && global_timer_ns() - t0 < 100000) {
            }
        }
        __syncwarp();
    } else if (warp == 1 && rank == 0) {
        constexpr uint32_t idesc = umma_idesc_i8(256, 256);
        const uint32_t free0 = smem_u32(&free_bar[0]), free0_peer = cluster_map(free0, 1);
        const uint32_t done0 = smem_u32(&acc_full[0]), done0_peer = cluster_map(done0, 1);
        const uint64_t desc0 = smem_desc_sw128(smem);
        int s = 0, phase = 0, turn = 0;
        for (int tile = pair; tile < tiles; tile += pairs, ++turn) {
            const int acc = turn & 1;
            bool fine = !__any_sync(0xffffffffu, abort_flag != 0);
            if (fine && turn >= 2)
                fine = __all_sync(0xffffffffu, mbar_wait_bounded_cluster(&acc_free[acc], ((turn >> 1) - 1) & 1, a.status, STATUS_INT8_WAIT_EPILOGUE));
            tc_fence_after();
            for (int i = 0; fine && i < a.slabs; ++i) {
                if (__any_sync(0xffffffffu, abort_flag != 0) ||
                    !__all_sync(0xffffffffu, mbar_wait_bounded_cluster(&full_bar[s], phase, a.status, STATUS_INT8_WAIT_TMA))) {
                    fine = false;
                    break;
                }
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t x_desc = desc0 + static_cast<uint32_t>(s * I8_PAIR_STAGE >> 4), w_desc = x_desc + (I8_A_BYTES >> 4);
#pragma unroll
                    for (int q = 0; q < 4; ++q) umma_i8<true>(tmem_d + 256 * acc, x_desc + 2 * q, w_desc + 2 * q, idesc, i + q > 0);
                    umma_commit<true>(free0 + 8u * s);
                    umma_commit<true>(free0_peer + 8u * s);
                }
                __syncwarp();
                if (++s == S) {
                    s = 0;
                    phase ^= 1;
                }
            }
            if (!fine) {
                abort_flag = 1;
                break;
            }
            if (elect_one()) {
                umma_commit<true>(done0 + 8u * acc);
                umma_commit<true>(done0_peer + 8u * acc);
            }
            __syncwarp();
        }
    } else if (warp >= 2) {
        // two warps per quarter of the rows, 128 channels each
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const uint32_t stage = smem_u32(smem + S * I8_PAIR_STAGE) + (warp - 2) * 4096u;
        const uint32_t acc_free0 = cluster_map(smem_u32(&acc_free[0]), 0);
        chain_wait();
        int turn = 0;
        for (int tile = pair; tile < tiles; tile += pairs, ++turn) {
            int m0, n0;
            pair_tile(a, tile, m0, n0);
            const int acc = turn & 1, row0 = m0 + 128 * static_cast<int>(rank) + 32 * quarter, col0 = n0 + 128 * half + lane;
            const float xs = row0 + lane < a.m ? a.x_scales[row0 + lane] : 0.f;
            float w_next = col0 < a.n ? a.w_scales[col0] : 0.f;
            bool fine = !__any_sync(0xffffffffu, abort_flag != 0);
            if (fine) fine = __all_sync(0xffffffffu, mbar_wait_bounded(&acc_full[acc], (turn >> 1) & 1, a.status, STATUS_INT8_WAIT_MMA));
            if (!fine) {
                abort_flag = 1;
                break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                const int col = col0 + 32 * c;
                const float w = w_next;
                if (c < 3) w_next = col + 32 < a.n ? a.w_scales[col + 32] : 0.f;
                uint32_t r[32];
                __syncwarp();                        // (lanes whose outputs do not exist)
                tmem_ld32(tmem_d + (static_cast<uint32_t>(32 * quarter) << 16) + 256 * acc + 128 * half + 32 * c, r);
                tmem_ld_wait();
                if (c == 3) {                        // the accumulator is read: the next tile but one may have it
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(acc_free0 + 8u * acc);
                }
                if (row0 < a.m)
                    store_outputs(a.y, a.y_dtype, static_cast<size_t>(row0) * a.n + col, a.n, col < a.n, min(32, a.m - row0), r, xs, w, stage, lane);
            }
        }
    }
    tc_fence_before();
    cluster_sync_all();                  // both CTAs are done with the pair's barriers, operands and tensor memory
    if (warp == 0) tmem_dealloc<true>(tmem_d, 512);
}

// ----------------------------------------------------------------------------------------------------------- host side
// A [rows][row] int8 matrix, read in boxes of 128 codes x box_rows rows; codes from `columns` on read as zeros.
static int int8_map(CUtensorMap *map, EncodeTiledFn encode, const int8_t *codes, int columns, long long row, int rows, int box_rows) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row)};
    const cuuint32_t box[2] = {I8_BK, static_cast<cuuint32_t>(box_rows)}, steps[2] = {1, 1};
    const CUresult res = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(codes), dims, strides, box, steps,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return res == CUDA_SUCCESS ? B200Q_OK : fail(B200Q_ECUDA, "int8_gemm: cuTensorMapEncodeTiled failed (%d)", static_cast<int>(res));
}

using Int8Fn = void (*)(const CUtensorMap, const CUtensorMap, const Int8Gemm);
template <int NT>
static Int8Fn tile_kernel(int split) {
    return split == 1 ? int8_tile_kernel<NT, 1> : split == 2 ? int8_tile_kernel<NT, 2> : split == 4 ? int8_tile_kernel<NT, 4> : int8_tile_kernel<NT, 8>;
}

static int int8_gemm(const int8_t *w, long long w_row, const int8_t *x, long long x_row, Int8Gemm a, cudaStream_t stream) {
    EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) return fail(B200Q_ECUDA, "int8_gemm: the driver does not provide cuTensorMapEncodeTiled");
    a.status = device_status_word();
    if (!a.status) return fail(B200Q_ECUDA, "int8_gemm: no CUDA device");
    const int sms = sm_count(), columns = (a.k + 15) & ~15;
    a.slabs = (a.k + I8_BK - 1) / I8_BK;
    CUtensorMap xmap, wmap;
    a.tiles_m = (a.m + 255) / 256;
    a.tiles_n = (a.n + 255) / 256;
    const long long big = static_cast<long long>(a.tiles_m) * a.tiles_n;
    const int token_tiles = (a.m + I8_BM - 1) / I8_BM;
    // The tile kernel's CTAs have one tile each: it is the faster one while all of them run at once (K 4096: 512 tokens x 4096 channels,
    // 128 tiles, 18 us against 20 by pairs; 256 x 8192 20 against 22), the pairs with more tiles (512 x 6144 22 against 33, 1024 x 8192
    // 33 against 61, 64 x 24576 37 against 39).
    if (static_cast<long long>((a.n + 127) / 128) * token_tiles > sms) {
        if (big > 0x3fffffff) return fail(B200Q_EUNSUPPORTED, "int8_gemm: too many tiles");
        if (int rc = int8_map(&xmap, encode, x, columns, x_row, a.m, 128)) return rc;
        if (int rc = int8_map(&wmap, encode, w, columns, w_row, a.n, 128)) return rc;
        a.stages = 6;
        const int smem = a.stages * I8_PAIR_STAGE + 8 * 4096 + 1024, pairs = static_cast<int>(std::min<long long>(big, sms / 2));
        if (int rc = allow_large_shared_memory(reinterpret_cast<const void *>(int8_pair_kernel))) return rc;
        launch_chained_cluster(int8_pair_kernel, dim3(2 * pairs), dim3(I8_PAIR_THREADS), smem, stream, 2, xmap, wmap, a);
        return check_launch("int8_gemm");
    }
    // Tiles of 64 channels where those of 128 would leave half of the SMs idle (K 4096: one token x 4096 channels 16 us by both, 128 x
    // 8192 18 against 20, but one token x 12288 29 against 20).
    int nt = 128;
    if (static_cast<long long>((a.n + 127) / 128) * token_tiles * 2 <= sms) nt = 64;
    const int tiles_n = (a.n + nt - 1) / nt;
    const long long tiles = static_cast<long long>(tiles_n) * token_tiles;
    // K in parts of at least four slabs, as long as all CTAs run at once; eight only for a handful of tiles (one token, tiles of 64, in 1,
    // 2, 4 and 8 parts: 512 x 2048 12, 10, 10 and 8 us; 1024 x 4096 16, 12, 10 and 14; 2048 x 8192 25, 18, 14 and 25; 4096 x 8192 25,
    // 18, 22 and 37).
    int split = 1;
    while (split < (tiles <= 8 ? 8 : 4) && tiles * split * 2 <= sms && a.slabs >= split * 4) split *= 2;
    a.x_rows = a.m < I8_BM ? (a.m + 7) / 8 * 8 : I8_BM;
    const int stage = I8_A_BYTES + nt * I8_BK;
    a.stages = std::min(I8_MAX_STAGES, 200 * 1024 / stage);
    if (int rc = int8_map(&xmap, encode, x, columns, x_row, a.m, a.x_rows)) return rc;
    if (int rc = int8_map(&wmap, encode, w, columns, w_row, a.n, nt)) return rc;
    const Int8Fn fn = nt == 64 ? tile_kernel<64>(split) : tile_kernel<128>(split);
    const int smem = a.stages * stage + 1024;
    if (int rc = allow_large_shared_memory(reinterpret_cast<const void *>(fn))) return rc;
    const dim3 grid(tiles_n * split, token_tiles);
    if (split > 1) launch_chained_cluster(fn, grid, dim3(I8_THREADS), smem, stream, split, xmap, wmap, a);
    else launch_chained(fn, grid, dim3(I8_THREADS), smem, stream, xmap, wmap, a);
    return check_launch("int8_gemm");
}

}  // namespace b200q

using namespace b200q;

extern "C" int b200q_int8_quantize(const void *x, int x_dtype, int rows, int k, int64_t x_row, int8_t *codes,
                                   int64_t codes_row, float *scales, int early, void *stream) {
    if (rows == 0) return B200Q_OK;
    if (!x || !codes || !scales) return fail(B200Q_EINVAL, "int8_quantize: NULL pointer");
    if (!dtype_valid(x_dtype)) return fail(B200Q_EINVAL, "int8_quantize: bad dtype");
    if (rows < 0 || k < 1 || x_row < k || codes_row % 16 || codes_row < k)
        return fail(B200Q_EINVAL, "int8_quantize: bad shape rows=%d k=%d (code rows are multiples of 16 bytes)", rows, k);
    if (rows > I8_MAX_SIZE || k > I8_MAX_SIZE) return fail(B200Q_EUNSUPPORTED, "int8_quantize: at most %d rows and columns", I8_MAX_SIZE);
    if (reinterpret_cast<uintptr_t>(codes) & 15) return fail(B200Q_EINVAL, "int8_quantize: codes must be 16-byte aligned");
    const size_t e = dtype_size(x_dtype);
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && x_row * e % 16 == 0;
    auto kernel = x_dtype == B200Q_F32   ? (vec ? int8_quantize_kernel<B200Q_F32, true> : int8_quantize_kernel<B200Q_F32, false>)
                  : x_dtype == B200Q_F16 ? (vec ? int8_quantize_kernel<B200Q_F16, true> : int8_quantize_kernel<B200Q_F16, false>)
                                         : (vec ? int8_quantize_kernel<B200Q_BF16, true> : int8_quantize_kernel<B200Q_BF16, false>);
    int team = 1;
    const int keep = x_dtype == B200Q_F32 ? I8_QUANTIZE_KEEP / 2 : I8_QUANTIZE_KEEP;
    // (few rows: as many warps as there are, one row of 2048 took 1 us longer by two)
    while (team < 8 && (256 * team * keep < k || static_cast<long long>(rows) * team <= 2 * sm_count())) team *= 2;
    const int teams = 8 / team, ctas = std::min((rows + teams - 1) / teams, (vec ? 4 : 2) * sm_count());
    launch_chained(kernel, dim3(ctas), dim3(256), 0, static_cast<cudaStream_t>(stream), x, rows, k, static_cast<long long>(x_row), codes,
                   static_cast<long long>(codes_row), scales, team, early);
    return check_launch("int8_quantize");
}

static int checked_gemm(const int8_t *w_codes, int64_t w_row, const float *w_scales, int n, int k, const int8_t *x_codes, int64_t x_row,
                        const float *x_scales, int m, void *y, int y_dtype, bool early, void *stream) {
    if (m == 0) return B200Q_OK;
    if (!w_codes || !w_scales || !x_codes || !x_scales || !y) return fail(B200Q_EINVAL, "int8_gemm: NULL pointer");
    if (!dtype_valid(y_dtype)) return fail(B200Q_EINVAL, "int8_gemm: bad dtype");
    if (m < 0 || n < 1 || k < 1) return fail(B200Q_EINVAL, "int8_gemm: bad shape m=%d n=%d k=%d", m, n, k);
    if (m > I8_MAX_SIZE || n > I8_MAX_SIZE) return fail(B200Q_EUNSUPPORTED, "int8_gemm: at most %d rows and channels", I8_MAX_SIZE);
    if (k > 131071) return fail(B200Q_EUNSUPPORTED, "int8_gemm: sums of more than 131071 products do not fit 32 bits");
    if (w_row % 16 || x_row % 16 || w_row < k || x_row < k ||
        ((reinterpret_cast<uintptr_t>(w_codes) | reinterpret_cast<uintptr_t>(x_codes)) & 15))
        return fail(B200Q_EINVAL, "int8_gemm: code rows must be 16-byte aligned and at least k long");
    Int8Gemm a{};
    a.w_scales = w_scales; a.x_scales = x_scales; a.n = n; a.k = k; a.m = m; a.y = y; a.y_dtype = y_dtype; a.early = early;
    return int8_gemm(w_codes, w_row, x_codes, x_row, a, static_cast<cudaStream_t>(stream));
}

extern "C" int b200q_int8_gemm(const int8_t *w_codes, int64_t w_row, const float *w_scales, int n, int k,
                               const int8_t *x_codes, int64_t x_row, const float *x_scales, int m, void *y, int y_dtype,
                               void *stream) {
    return checked_gemm(w_codes, w_row, w_scales, n, k, x_codes, x_row, x_scales, m, y, y_dtype, false, stream);
}

extern "C" int b200q_int8_gemm_behind_quantize(const int8_t *w_codes, int64_t w_row, const float *w_scales, int n, int k,
                                               const int8_t *x_codes, int64_t x_row, const float *x_scales, int m, void *y,
                                               int y_dtype, void *stream) {
    return checked_gemm(w_codes, w_row, w_scales, n, k, x_codes, x_row, x_scales, m, y, y_dtype, true, stream);
}
