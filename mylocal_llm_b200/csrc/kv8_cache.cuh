// Paged key/value cache in 8 bits: what the kernels of kv8_cache.cu (append, page operations) and kv8_attention.cu share.
//
// A block is 64 consecutive tokens of a sequence, and a page holds one full block of every layer. codes [pages][layers][2]
// [kv_heads][64 * head_dim] int8: the keys of a block as [64 tokens][head_dim], the values as [head_dim][64 tokens], so that
// both products of the attention read rows of consecutive bytes. scales [pages][layers][2][kv_heads] FP32: value = code *
// scale. The tokens behind the last full block of a sequence wait in tail [sequences][layers][2][kv_heads][64][head_dim] in
// the model's 16-bit type; peak [sequences][layers][2][kv_heads] is the largest magnitude among them. A page is written once,
// when its block becomes full, and never again: sequences can share it, and the content of a cache does not depend on how
// many tokens arrived per call. table [sequences][blocks] names the page of every full block, refs counts the sequences that
// refer to a page, free_bits has a bit set for every page without any.
#pragma once

#include "common.cuh"

namespace b200q {

constexpr int KV8_BLOCK = 64;
constexpr int KV8_MAX_SEQUENCES = 65536;
constexpr int KV8_MAX_PAGES = 1 << 20;
constexpr int KV8_MAX_STEP = 65535;        // sequences of a step: what a grid holds along z
constexpr int STATUS_KV8_POOL = 501;       // extend: the pool has too few free pages (nothing was taken)
constexpr int STATUS_KV8_LENGTH = 502;     // extend: a sequence would pass max_length, or a slot is out of range
constexpr int STATUS_KV8_SLOTS = 503;      // fork / free: a slot out of range, named twice, or a target that is not empty
constexpr int STATUS_KV8_FOLLOWS = 504;    // extend_after: the step before was refused
constexpr int KV8_REFUSED = -1;            // starts of a refused step

// Smallest scale: the smallest normal number, so that no quotient by it overflows and no scale is zero.
constexpr float KV8_MIN_SCALE = 1.17549435e-38f;

__device__ __forceinline__ float kv8_nan() { return __uint_as_float(0x7fc00000u); }

// Scale of values whose largest magnitude has the bits `peak` (sign cleared; NaN and infinities compare above every finite
// number): peak / 127 correctly rounded. A block with a value that is not finite has no scale: NaN, which shows in
// everything computed from it.
__device__ __forceinline__ float int8_scale(uint32_t peak) {
    if (peak >= 0x7f800000u) return kv8_nan();
    return fmaxf(__fdiv_rn(__uint_as_float(peak), 127.0f), KV8_MIN_SCALE);
}

// Two FP32 values in one 64-bit register, and the instructions that work on both at once.
struct Pair {
    uint64_t v;
    __device__ __forceinline__ float lo() const { return __uint_as_float(static_cast<uint32_t>(v)); }
    __device__ __forceinline__ float hi() const { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
};
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
    return p;
}
__device__ __forceinline__ Pair pair_fma(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
__device__ __forceinline__ Pair pair_add(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}

// The integer nearest to x / s, ties to even, of the exact quotient, for scales near the smallest normal number.
static __device__ __noinline__ uint32_t int8_code_tiny(float x, float s) {
    return static_cast<uint32_t>(__double2int_rn(static_cast<double>(x) / static_cast<double>(s)));
}

// The codes of four values as bytes of a word: the integers nearest to x / s, ties to even, of the exact quotients.
// x * inv + 1.5 * 2^23 has the nearest integer of x * inv in its low bits, and that is the code unless x * inv lies within 2^-16 of
// a border (x / s does not differ from it by more than 2^-17 there). Then only the neighbours can be nearer, and the sign of
// x - (q +- 1/2) s as one FMA tells (an FMA rounds once, so its sign is that of the exact difference, which does not underflow
// from 7.9e-31 on). Values of few bits and scales of few bits meet borders often: one group of 128 BF16 values in seven.
__device__ __forceinline__ uint32_t int8_codes(const float (&x)[4], float s, float inv) {
    constexpr float MAGIC = 12582912.f, TINY = 7.8886e-31f;
    uint32_t t[4];
    Pair q[2];
    float far = s < TINY ? 1.f : 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const Pair v = pair(x[2 * e], x[2 * e + 1]), k = pair(inv, inv);
        const Pair y = pair_fma(v, k, pair(MAGIC, MAGIC));
        q[e] = pair_add(y, pair(-MAGIC, -MAGIC));
        const Pair negative{q[e].v ^ 0x8000000080000000ull};
        const Pair r = pair_fma(v, k, negative);
        far = fmaxf(far, fmaxf(fabsf(r.lo()), fabsf(r.hi())));
        t[2 * e] = static_cast<uint32_t>(y.v);
        t[2 * e + 1] = static_cast<uint32_t>(y.v >> 32);
    }
    if (far > 0.49998f) {
        if (s < TINY) {
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = int8_code_tiny(x[e], s);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float whole = e & 1 ? q[e >> 1].hi() : q[e >> 1].lo();
                const float up = __fmaf_rn(-(whole + 0.5f), s, x[e]), down = __fmaf_rn(-(whole - 0.5f), s, x[e]);
                const bool odd = t[e] & 1u;
                if (up > 0.f || (up == 0.f && odd)) ++t[e];
                else if (down < 0.f || (down == 0.f && odd)) --t[e];
            }
        }
    }
    return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Index of the first element of (page, layer, part, head) in units of [64 * head_dim].
__device__ __forceinline__ size_t kv8_unit(size_t page, int layers, int layer, int part, int kv_heads, int head) {
    return ((page * layers + layer) * 2 + part) * kv_heads + head;
}

}  // namespace b200q
