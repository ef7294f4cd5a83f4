// Fragments of the attention over the paged 8-bit cache: how codes, tails and queries become operands of
// mma.m16n8k16 (FP16 x FP16 -> FP32).
//
// The instruction fixes which lane holds which (row, k) of an operand, not which key or dimension stands behind a row or k. With
// g = lane / 4 and t = lane % 4 the kernels choose
//   scores: k index 2t + e (+ 8) of step s      <-> dimension 64 h + 16 t + 4 s' + e (+ 2),  s = 4 h + s'
//           column n of score tile j            <-> key 16 (n / 2) + 2 j + n % 2
//   values: k index 2t + e (+ 8) of step s      <-> key 16 t + 4 s + e (+ 2),   column n of tile i <-> dimension 8 i + n
// so that a lane's codes for four steps are 16 consecutive bytes of a key's row (of a dimension's row of the transposed
// values), one load, and the softmax weights of two score tiles are, in the registers they are in, one operand of the value
// product. Codes are exact in FP16: (c + 128) under the exponent byte 0x64 is 1024 + 128 + c, minus 1152.
//
// The instruction has sixteen rows. Where memory bounds the kernel a tile is eight rows of queries: rows 0..7 hold the FP16
// parts of queries and softmax weights, rows 8..15 what is left of them, again as FP16, and the two results are added. That
// keeps 22 bits of both for no additional instruction, down to FP16's smallest normal number (rows of queries and weights are scaled
// to the top of its range).
#pragma once

#include "kv8_cache.cuh"

namespace b200q {

struct Kv8Attention {
    const void *q;
    long long q_row;
    int q_dtype, layer, heads;
    const int32_t *slots, *offsets, *starts;
    int batch, rows;
    const float *cos_t, *sin_t;
    float scale;
    bool vec;                     // rows of q can be read 16 bytes at a time
    void *out;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first of a sum: d = a * b.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// Four codes -> two pairs of FP16 numbers.
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t x = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const __half2 ra = __hsub2(*reinterpret_cast<const __half2 *>(&a), off), rb = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
    lo = *reinterpret_cast<const uint32_t *>(&ra);
    hi = *reinterpret_cast<const uint32_t *>(&rb);
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&p);
}

// 2^x with a relative error of 2^-22; 0 for -inf.
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The power of two at or below a magnitude (its exponent field), at least 2^-126; NaN for what is not finite.
__device__ __forceinline__ float power_of(uint32_t bits) {
    if (bits >= 0x7f800000u) return kv8_nan();
    return __uint_as_float(max(bits & 0x7f800000u, 0x00800000u));
}
// Its reciprocal, exact (2^-127 is a subnormal number); of NaN: NaN.
__device__ __forceinline__ float power_inverse(float p) {
    const uint32_t e = __float_as_uint(p) >> 23;
    return __uint_as_float(e < 254 ? (254 - e) << 23 : e == 254 ? 0x00400000u : 0x7fc00000u);
}

// Scale of a row of queries: a power of two, by which its values are below 2^15, the top of FP16's range, so that a number and its
// remainder keep 22 bits of values down to 2^-28 of the largest; NaN for what is not finite.
__device__ __forceinline__ float query_scale(uint32_t top) {
    return power_of(top >= 0x7f800000u ? top : max(top, 0x07800000u)) * (1.f / 16384.f);          // (2^-112: the scale is a normal number)
}

// Scale of a tail whose largest magnitude has the bits `peak`: a power of two, by which its values are below 128 like codes. What a
// value loses as FP16 number is then 2^-31 of the largest at most, so nothing of an FP16 tail of magnitudes below 128; NaN for what is not finite.
__device__ __forceinline__ float tail_scale(uint32_t peak) {
    return power_of(peak >= 0x7f800000u ? peak : max(peak, 0x08800000u)) * (1.f / 64.f);         // (2^-110: the inverse is finite)
}

// Two 16-bit values of the tail (as stored) times a power of two, as FP16.
template <bool BF16>
__device__ __forceinline__ uint32_t tail_to_half(uint32_t w, float inv) {
    float lo, hi;
    if (BF16) {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xffff0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        lo = f.x;
        hi = f.y;
    }
    return pack_half(lo * inv, hi * inv);
}

// Four consecutive values as floats.
__device__ __forceinline__ void load4f(const void *p, int dtype, size_t i, bool vec, float (&f)[4]) {
    if (vec && dtype == B200Q_F32) {
        const float4 q = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
        f[0] = q.x; f[1] = q.y; f[2] = q.z; f[3] = q.w;
    } else if (vec) {
        const uint2 q = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i);
        const uint32_t w[2] = {q.x, q.y};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float2 v = dtype == B200Q_BF16 ? make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u))
                                                 : __half22float2(*reinterpret_cast<const __half2 *>(&w[e]));
            f[2 * e] = v.x;
            f[2 * e + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = load_as_float(p, dtype, i + e);
    }
}

// Sixteen consecutive values as floats; `vec`: base and strides are such that 16-byte loads can fetch them.
__device__ __forceinline__ void load16f(const void *p, int dtype, size_t i, bool vec, float (&f)[16]) {
    if (vec && dtype == B200Q_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float4 q = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i + 4 * e);
            f[4 * e] = q.x; f[4 * e + 1] = q.y; f[4 * e + 2] = q.z; f[4 * e + 3] = q.w;
        }
    } else if (vec) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 q = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i + 8 * h);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 v = dtype == B200Q_BF16 ? make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u))
                                                     : __half22float2(*reinterpret_cast<const __half2 *>(&w[e]));
                f[8 * h + 2 * e] = v.x;
                f[8 * h + 2 * e + 1] = v.y;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = load_as_float(p, dtype, i + e);
    }
}

// Rotated query values of a lane, FP32: dimensions 64 h + 16 t .. + 15 for every h.
template <int DH>
__device__ __forceinline__ void load_query(const Kv8Attention &a, size_t base, int t, int pos, float (&x)[DH / 4]) {
    constexpr int HALF = DH / 2;
    const int i = (16 * t) % HALF;                           // (head dimension 64: lanes t and t ^ 2 hold partners)
    float x0[16], x1[16];
    load16f(a.q, a.q_dtype, base + i, a.vec, x0);
    load16f(a.q, a.q_dtype, base + i + HALF, a.vec, x1);
    if (a.cos_t) {
        float c[16], s[16];
        load16f(a.cos_t, B200Q_F32, static_cast<size_t>(pos) * HALF + i, true, c);
        load16f(a.sin_t, B200Q_F32, static_cast<size_t>(pos) * HALF + i, true, s);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float lo = x0[e] * c[e] - x1[e] * s[e], hi = x0[e] * s[e] + x1[e] * c[e];
            x0[e] = lo;
            x1[e] = hi;
        }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        x[e] = DH == 64 && 16 * t >= HALF ? x1[e] : x0[e];
        if (DH == 128) x[DH / 4 - 16 + e] = x1[e];
    }
}

// x as an FP16 number and what is left of it as another, for pairs.
__device__ __forceinline__ void split_half(float x0, float x1, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = pack_half(x0 - f.x, x1 - f.y);
}

// The lane's part of the query operand of an eight-row tile, for row g of it, relative to the row's scale; the result is that scale
// times |scale| times log2(e), which turns sums of products into base-2 exponents (a negative scale's sign is in the query: larger
// sums are larger scores). base < 0: a row that does not exist (zeros).
template <int DH>
__device__ __forceinline__ float query_split(const Kv8Attention &a, long long base, int pos, int t, uint32_t (&qf)[DH / 16][4]) {
    float x[DH / 4];
    uint32_t top = 0u;
#pragma unroll
    for (int e = 0; e < DH / 4; ++e) x[e] = 0.f;
    if (base >= 0) load_query<DH>(a, base, t, pos, x);
#pragma unroll
    for (int e = 0; e < DH / 4; ++e) top = max(top, abs_bits(x[e]));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float p = query_scale(top), inv = a.scale < 0.f ? -power_inverse(p) : power_inverse(p);
#pragma unroll
    for (int s = 0; s < DH / 16; ++s) {
        split_half(x[4 * s] * inv, x[4 * s + 1] * inv, qf[s][0], qf[s][1]);
        split_half(x[4 * s + 2] * inv, x[4 * s + 3] * inv, qf[s][2], qf[s][3]);
    }
    return p * (fabsf(a.scale) * 1.4426950408889634f);
}

// Scores of a block of 64 keys (codes, in shared memory) for RT row tiles: acc[r][j] is score tile j. Four tiles at a time, so
// that neighbouring instructions do not depend on one another.
template <int DH, int RT>
__device__ __forceinline__ void score_codes(const uint8_t *k, const uint32_t (&qf)[RT][DH / 16][4], int g, int t, float (&acc)[RT][8][4]) {
    const uint8_t *row = k + (16 * (g >> 1) + (g & 1)) * DH + 16 * t;
#pragma unroll
    for (int j0 = 0; j0 < 8; j0 += 4) {
#pragma unroll
        for (int h = 0; h < DH / 64; ++h) {
            uint32_t word[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint4 w = *reinterpret_cast<const uint4 *>(row + 2 * (j0 + j) * DH + 64 * h);
                word[j][0] = w.x; word[j][1] = w.y; word[j][2] = w.z; word[j][3] = w.w;
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t b0, b1;
                    codes_to_half(word[j][s], b0, b1);
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        if (h + s == 0) mma_f16_first(acc[r][j0 + j], qf[r][0], b0, b1);
                        else mma_f16(acc[r][j0 + j], qf[r][4 * h + s], b0, b1);
                    }
                }
        }
    }
}

// The same for the tail (16-bit values in shared memory): keys from `rest` on count as zeros.
template <int DH, bool BF16, int RT>
__device__ __forceinline__ void score_tail(const uint8_t *k, float inv, int rest, const uint32_t (&qf)[RT][DH / 16][4], int g, int t,
                                           float (&acc)[RT][8][4]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int key = 16 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
        for (int h = 0; h < DH / 64; ++h) {
            uint4 w[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
            if (key < rest) {
                const uint4 *p = reinterpret_cast<const uint4 *>(k + (key * DH + 64 * h + 16 * t) * 2);
                w[0] = p[0];
                w[1] = p[1];
            }
            const uint32_t word[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const uint32_t b0 = tail_to_half<BF16>(word[2 * s], inv), b1 = tail_to_half<BF16>(word[2 * s + 1], inv);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    if (h + s == 0) mma_f16_first(acc[r][j], qf[r][0], b0, b1);
                    else mma_f16(acc[r][j], qf[r][4 * h + s], b0, b1);
                }
            }
        }
    }
}

// The lane's part of the value operand of the tail (rows of 16-bit values in shared memory) for tile i, steps s and s + 1: keys
// 16 t + 4 s .. + 7 of dimension 8 i + g. One transposing load of four 8 x 8 matrices; a matrix row is a key's dimensions 8 i ..
// 8 i + 7, lane l naming row l % 8 of matrix l / 8. Keys from `rest` on count as zeros.
template <int DH, bool BF16>
__device__ __forceinline__ void tail_values(uint32_t v, float inv, int rest, int i, int s, int lane, uint32_t (&b)[4]) {
    const int r = lane & 7, key = 16 * (r >> 1) + 4 * s + 2 * (lane >> 3) + (r & 1);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3])
                 : "r"(v + (key * DH + 8 * i) * 2)
                 : "memory");
    const int first = 16 * (lane & 3) + 4 * s;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (first + 2 * e + 1 >= rest) b[e] &= 0xffffu;
        if (first + 2 * e >= rest) b[e] = 0u;
        b[e] = tail_to_half<BF16>(b[e], inv);
    }
}

}  // namespace b200q
