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
constexpr int STATUS_KV8_POOL = 501;       // extend: the pool has too few free pages (nothing was taken)
constexpr int STATUS_KV8_LENGTH = 502;     // extend: a sequence would pass max_length, or a slot is out of range
constexpr int STATUS_KV8_SLOTS = 503;      // fork / free: a slot out of range, named twice, or a target that is not empty

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

// The integer nearest to x / s, ties to even, of the exact quotient: the product with the reciprocal is off by less than
// 2^-15 (|x / s| < 128), so only the neighbours can be nearer, and the sign of x - (q +- 1/2) s as one FMA tells (an FMA
// rounds once, so its sign is that of the exact difference). Scales near the smallest normal number, where that difference
// can underflow, divide in 64 bits instead.
static __device__ __noinline__ int int8_code_exact(float x, float s, float inv) {
    if (s < 7.8886e-31f) return __double2int_rn(static_cast<double>(x) / static_cast<double>(s));
    const float q = rintf(__fmul_rn(x, inv));
    const float up = __fmaf_rn(-(q + 0.5f), s, x), down = __fmaf_rn(-(q - 0.5f), s, x);
    int code = __float2int_rn(q);                        // (NaN: 0, and the scale is NaN)
    if (up > 0.f || (up == 0.f && (code & 1))) ++code;
    else if (down < 0.f || (down == 0.f && (code & 1))) --code;
    return code;
}

// The codes of four values as bytes of a word. x * inv + 1.5 * 2^23 has the nearest integer of x * inv in its low bits, and that
// is the code unless x * inv lies within 2^-16 of a border (x / s does not differ from it by more than 2^-17 there): then, in
// one of 2^13 groups or so, each of the four is looked at exactly.
__device__ __forceinline__ uint32_t int8_codes(const float (&x)[4], float s, float inv) {
    constexpr float MAGIC = 12582912.f;
    uint32_t t[4];
    float far = s < 7.8886e-31f ? 1.f : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float y = __fmaf_rn(x[e], inv, MAGIC);
        far = fmaxf(far, fabsf(__fmaf_rn(x[e], inv, -__fadd_rn(y, -MAGIC))));
        t[e] = __float_as_uint(y);
    }
    if (far > 0.49998f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = static_cast<uint32_t>(int8_code_exact(x[e], s, inv));
    }
    return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Index of the first element of (page, layer, part, head) in units of [64 * head_dim].
__device__ __forceinline__ size_t kv8_unit(size_t page, int layers, int layer, int part, int kv_heads, int head) {
    return ((page * layers + layer) * 2 + part) * kv_heads + head;
}

}  // namespace b200q
