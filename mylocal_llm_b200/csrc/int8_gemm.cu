// Matrix product in 8-bit integers with one scale per token and per output channel, and the quantiser of its operands.
#include "kv8_cache.cuh"

namespace b200q {

// One CTA per row. The row's pieces of eight values stay in registers between the two passes (the largest magnitude, then
// the codes) up to 256 * 8 * KEEP columns; longer rows are read again. VEC: 16-byte loads are possible.
template <bool VEC>
__device__ __forceinline__ void load8(const void *p, int dtype, size_t base, int c, int k, float (&f)[8]) {
    if (VEC && c + 8 <= k) {
        if (dtype == B200Q_F32) {
            const float4 *q = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + base + c);
            const float4 lo = q[0], hi = q[1];
            f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w;
            f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
        } else {
            const uint4 q = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + base + c);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (dtype == B200Q_BF16) {
                    f[2 * e] = __uint_as_float(w[e] << 16);
                    f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                } else {
                    const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&w[e]));
                    f[2 * e] = h.x;
                    f[2 * e + 1] = h.y;
                }
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = c + e < k ? load_as_float(p, dtype, base + c + e) : 0.f;
}

template <bool VEC>
__global__ void __launch_bounds__(256) int8_quantize_kernel(const void *x, int dtype, int k, long long x_row, int8_t *codes,
                                                            long long codes_row, float *scales) {
    constexpr int KEEP = 4;
    __shared__ uint32_t peaks[8];
    chain_trigger();
    chain_wait();
    const int tid = threadIdx.x;
    const size_t base = blockIdx.x * static_cast<size_t>(x_row);
    const int padded = (k + 15) & ~15;
    float kept[KEEP][8];
    uint32_t peak = 0u;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        const int c = (tid + 256 * j) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) kept[j][e] = 0.f;
        if (c < k) load8<VEC>(x, dtype, base, c, k, kept[j]);
    }
#pragma unroll
    for (int j = 0; j < KEEP; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) peak = max(peak, abs_bits(kept[j][e]));
    for (int c = (tid + 256 * KEEP) * 8; c < k; c += 256 * 8) {
        float f[8];
        load8<VEC>(x, dtype, base, c, k, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) peak = max(peak, abs_bits(f[e]));
    }
    peak = __reduce_max_sync(0xffffffffu, peak);
    if ((tid & 31) == 0) peaks[tid >> 5] = peak;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) peak = max(peak, peaks[w]);
    const float s = int8_scale(peak), inv = __fdiv_rn(1.f, s);
    if (tid == 0) scales[blockIdx.x] = s;
    auto put = [&](int c, const float (&f)[8]) {
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e >> 2] |= (static_cast<uint32_t>(int8_code(f[e], s, inv)) & 0xffu) << (8 * (e & 3));
        *reinterpret_cast<uint2 *>(codes + blockIdx.x * static_cast<size_t>(codes_row) + c) = make_uint2(w[0], w[1]);
    };
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        const int c = (tid + 256 * j) * 8;
        if (c < padded) put(c, kept[j]);
    }
    for (int c = (tid + 256 * KEEP) * 8; c < padded; c += 256 * 8) {
        float f[8];
        load8<VEC>(x, dtype, base, c, k, f);
        put(c, f);
    }
}

struct Int8Gemm {
    const int8_t *w, *x;
    long long w_row, x_row;
    const float *w_scales, *x_scales;
    int n, k, m;
    void *y;
    int y_dtype;
};

// A CTA computes 64 tokens x 64 channels with 4-way integer dots; a thread 4 x 4 of them.
__global__ void __launch_bounds__(256) int8_gemm_simple_kernel(const Int8Gemm a) {
    __shared__ int x_s[64][17], w_s[64][17];
    chain_trigger();
    chain_wait();
    const int tid = threadIdx.x, m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tx = tid & 15, ty = tid >> 4;
    const int padded = (a.k + 15) & ~15;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < padded; k0 += 64) {
        const int r = tid >> 2, c = k0 + 16 * (tid & 3);
        int4 xv = make_int4(0, 0, 0, 0), wv = xv;
        if (c < padded && m0 + r < a.m) xv = *reinterpret_cast<const int4 *>(a.x + (m0 + r) * a.x_row + c);
        if (c < padded && n0 + r < a.n) wv = *reinterpret_cast<const int4 *>(a.w + (n0 + r) * a.w_row + c);
        __syncthreads();
        int *xs = &x_s[r][4 * (tid & 3)], *ws = &w_s[r][4 * (tid & 3)];
        xs[0] = xv.x; xs[1] = xv.y; xs[2] = xv.z; xs[3] = xv.w;
        ws[0] = wv.x; ws[1] = wv.y; ws[2] = wv.z; ws[3] = wv.w;
        __syncthreads();
        for (int i = 0; i < 16; ++i)
            for (int u = 0; u < 4; ++u)
                for (int v = 0; v < 4; ++v) acc[u][v] = __dp4a(x_s[ty + 16 * u][i], w_s[tx + 16 * v][i], acc[u][v]);
    }
    for (int u = 0; u < 4; ++u)
        for (int v = 0; v < 4; ++v) {
            const int m = m0 + ty + 16 * u, n = n0 + tx + 16 * v;
            if (m < a.m && n < a.n)
                store_from_float(a.y, a.y_dtype, static_cast<size_t>(m) * a.n + n,
                                 static_cast<float>(acc[u][v]) * a.x_scales[m] * a.w_scales[n]);
        }
}

}  // namespace b200q

using namespace b200q;

extern "C" int b200q_int8_quantize(const void *x, int x_dtype, int rows, int k, int64_t x_row, int8_t *codes,
                                   int64_t codes_row, float *scales, void *stream) {
    if (rows == 0) return B200Q_OK;
    if (!x || !codes || !scales) return fail(B200Q_EINVAL, "int8_quantize: NULL pointer");
    if (!dtype_valid(x_dtype)) return fail(B200Q_EINVAL, "int8_quantize: bad dtype");
    if (rows < 0 || k < 1 || x_row < k || codes_row % 16 || codes_row < k)
        return fail(B200Q_EINVAL, "int8_quantize: bad shape rows=%d k=%d (code rows are multiples of 16 bytes)", rows, k);
    if (reinterpret_cast<uintptr_t>(codes) & 15) return fail(B200Q_EINVAL, "int8_quantize: codes must be 16-byte aligned");
    const size_t e = dtype_size(x_dtype);
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && x_row * e % 16 == 0;
    launch_chained(vec ? int8_quantize_kernel<true> : int8_quantize_kernel<false>, dim3(rows), dim3(256), 0,
                   static_cast<cudaStream_t>(stream), x, x_dtype, k, static_cast<long long>(x_row), codes,
                   static_cast<long long>(codes_row), scales);
    return check_launch("int8_quantize");
}

extern "C" int b200q_int8_gemm(const int8_t *w_codes, int64_t w_row, const float *w_scales, int n, int k,
                               const int8_t *x_codes, int64_t x_row, const float *x_scales, int m, void *y, int y_dtype,
                               void *stream) {
    if (m == 0) return B200Q_OK;
    if (!w_codes || !w_scales || !x_codes || !x_scales || !y) return fail(B200Q_EINVAL, "int8_gemm: NULL pointer");
    if (!dtype_valid(y_dtype)) return fail(B200Q_EINVAL, "int8_gemm: bad dtype");
    if (m < 0 || n < 1 || k < 1) return fail(B200Q_EINVAL, "int8_gemm: bad shape m=%d n=%d k=%d", m, n, k);
    if (k > 131071) return fail(B200Q_EUNSUPPORTED, "int8_gemm: sums of more than 131071 products do not fit 32 bits");
    if (w_row % 16 || x_row % 16 || w_row < k || x_row < k ||
        ((reinterpret_cast<uintptr_t>(w_codes) | reinterpret_cast<uintptr_t>(x_codes)) & 15))
        return fail(B200Q_EINVAL, "int8_gemm: code rows must be 16-byte aligned and at least k long");
    Int8Gemm a{};
    a.w = w_codes; a.x = x_codes; a.w_row = w_row; a.x_row = x_row; a.w_scales = w_scales; a.x_scales = x_scales;
    a.n = n; a.k = k; a.m = m; a.y = y; a.y_dtype = y_dtype;
    launch_chained(int8_gemm_simple_kernel, dim3((n + 63) / 64, (m + 63) / 64), dim3(256), 0,
                   static_cast<cudaStream_t>(stream), a);
    return check_launch("int8_gemm");
}
