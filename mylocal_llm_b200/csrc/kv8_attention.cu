// Causal attention over the paged 8-bit key/value cache (layout: kv8_cache.cuh).
#include "kv8_attention.cuh"

namespace b200q {

int kv8_check(const char *what, const b200q_kv8_cache *c);       // kv8_cache.cu

// kv8_decode.cu
long long kv8_decode_workspace(const b200q_kv8_cache *c, int heads, int batch, int max_new, int max_keys);
int kv8_decode(const b200q_kv8_cache *c, const Kv8Attention &a, int max_new, int max_keys, void *workspace,
               long long workspace_bytes, cudaStream_t stream);

// Whether a step goes to the kernel for few tokens per sequence: all rows of a key/value head are one tile of 16, or single
// tokens.
static bool few_rows(const b200q_kv8_cache *c, int heads, int max_new) { return max_new == 1 || max_new * (heads / c->kv_heads) <= 16; }

// One CTA = one row of one head: a block of 64 keys at a time, a thread per key for the scores and a thread per dimension
// for the values, with the running maximum and sum of the softmax.
template <int DH>
__global__ void __launch_bounds__(128) kv8_attention_simple_kernel(const b200q_kv8_cache c, const Kv8Attention a) {
    __shared__ float q_s[DH], p_s[KV8_BLOCK];
    __shared__ float red[2];
    chain_trigger();
    chain_wait();
    const int tid = threadIdx.x, row = blockIdx.x, head = blockIdx.y, kvh = head / (a.heads / c.kv_heads);
    int b = 0;
    for (int lo = 0, hi = a.batch - 1; lo <= hi;) {
        const int mid = (lo + hi) >> 1;
        if (a.offsets[mid] <= row) { b = mid; lo = mid + 1; } else { hi = mid - 1; }
    }
    const int start = a.starts[b], slot = a.slots[b], pos = start + row - a.offsets[b];
    const int total = start + a.offsets[b + 1] - a.offsets[b];
    const size_t at_out = (static_cast<size_t>(row) * a.heads + head) * DH;
    if (start < 0) {
        if (tid < DH) store_from_float(a.out, c.dtype, at_out + tid, kv8_nan());
        return;
    }
    if (tid < DH) {
        const size_t base = row * a.q_row + static_cast<size_t>(head) * DH;
        const int i = tid % (DH / 2);
        const float x0 = load_as_float(a.q, a.q_dtype, base + i), x1 = load_as_float(a.q, a.q_dtype, base + i + DH / 2);
        float v = tid < DH / 2 ? x0 : x1;
        if (a.cos_t) {
            const float cc = a.cos_t[static_cast<size_t>(pos) * (DH / 2) + i], ss = a.sin_t[static_cast<size_t>(pos) * (DH / 2) + i];
            v = tid < DH / 2 ? x0 * cc - x1 * ss : x0 * ss + x1 * cc;
        }
        q_s[tid] = v * a.scale;
    }
    float m = -INFINITY, l = 0.f, acc = 0.f;
    const size_t tail = kv8_unit(slot, c.layers, a.layer, 0, c.kv_heads, kvh);
    for (int block = 0; block * KV8_BLOCK <= pos; ++block) {
        const bool full = (block + 1) * KV8_BLOCK <= total;
        size_t u = tail;
        if (full) u = kv8_unit(c.table[static_cast<size_t>(slot) * c.blocks + block], c.layers, a.layer, 0, c.kv_heads, kvh);
        __syncthreads();
        if (tid < KV8_BLOCK) {
            float s = -INFINITY;
            if (block * KV8_BLOCK + tid <= pos) {
                s = 0.f;
                for (int d = 0; d < DH; ++d)
                    s += q_s[d] * (full ? static_cast<float>(c.codes[u * (KV8_BLOCK * DH) + tid * DH + d])
                                        : load_as_float(c.tail, c.dtype, u * (KV8_BLOCK * DH) + tid * DH + d));
                if (full) s *= c.scales[u];
            }
            p_s[tid] = s;
        }
        __syncthreads();
        if (tid < 32) {
            float x = fmaxf(p_s[tid], p_s[tid + 32]);
            for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            const float mn = fmaxf(m, x);
            const float e0 = __expf(p_s[tid] - mn), e1 = __expf(p_s[tid + 32] - mn);
            const float sum = warp_sum(e0 + e1);
            p_s[tid] = e0;
            p_s[tid + 32] = e1;
            if (tid == 0) {
                red[0] = mn;
                red[1] = sum;
            }
        }
        __syncthreads();
        const float mn = red[0], alpha = __expf(m - mn);
        m = mn;
        l = l * alpha + red[1];
        acc *= alpha;
        if (tid < DH) {
            float o = 0.f;
            const size_t v = (u + c.kv_heads) * (KV8_BLOCK * DH);
            const int keys = min(KV8_BLOCK, pos + 1 - block * KV8_BLOCK);
            for (int t = 0; t < keys; ++t)
                o += p_s[t] * (full ? static_cast<float>(c.codes[v + tid * KV8_BLOCK + t]) : load_as_float(c.tail, c.dtype, v + t * DH + tid));
            acc += full ? o * c.scales[u + c.kv_heads] : o;
        }
    }
    if (tid < DH) store_from_float(a.out, c.dtype, at_out + tid, acc / l);
}

}  // namespace b200q

using namespace b200q;

extern "C" long long b200q_kv8_attention_workspace(const b200q_kv8_cache *cache, int heads, int batch, int rows, int max_new,
                                                   int max_keys) {
    if (!cache || heads < 1 || cache->kv_heads < 1 || heads % cache->kv_heads || max_new < 1) return 0;
    return few_rows(cache, heads, max_new) ? kv8_decode_workspace(cache, heads, batch, max_new, max_keys) : 0;
}

extern "C" int b200q_kv8_attention(const b200q_kv8_cache *cache, int layer, const void *q, int q_dtype, int64_t q_row,
                                   int heads, const int32_t *slots, const int32_t *offsets, const int32_t *starts, int batch,
                                   int rows, int max_new, int max_keys, const float *cos_table, const float *sin_table,
                                   int rope_rows, float scale, void *out, void *workspace, long long workspace_bytes,
                                   void *stream) {
    if (int rc = kv8_check("kv8_attention", cache)) return rc;
    if (batch == 0 || rows == 0) return B200Q_OK;
    if (!q || !slots || !offsets || !starts || !out) return fail(B200Q_EINVAL, "kv8_attention: NULL pointer");
    if (layer < 0 || layer >= cache->layers) return fail(B200Q_EINVAL, "kv8_attention: layer %d out of range", layer);
    if (!dtype_valid(q_dtype)) return fail(B200Q_EINVAL, "kv8_attention: bad dtype");
    if (heads < 1 || heads % cache->kv_heads) return fail(B200Q_EINVAL, "kv8_attention: heads %d are no multiple of %d", heads, cache->kv_heads);
    if (batch < 0 || batch > cache->sequences || rows < 0 || max_new < 1 || max_new > cache->max_length || max_new > rows ||
        max_keys < 1 || max_keys > cache->max_length)
        return fail(B200Q_EINVAL, "kv8_attention: batch %d, rows %d, new tokens %d, keys %d out of range", batch, rows, max_new, max_keys);
    if (q_row < static_cast<int64_t>(heads) * cache->head_dim) return fail(B200Q_EINVAL, "kv8_attention: row stride below heads * head_dim");
    if (!cos_table != !sin_table) return fail(B200Q_EINVAL, "kv8_attention: one of the two RoPE tables is NULL");
    if (cos_table && rope_rows < cache->max_length)
        return fail(B200Q_EINVAL, "kv8_attention: RoPE tables of %d rows for sequences of up to %d tokens", rope_rows, cache->max_length);
    if ((reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) & 15)
        return fail(B200Q_EINVAL, "kv8_attention: RoPE tables must be 16-byte aligned");
    if (heads > 65535) return fail(B200Q_EUNSUPPORTED, "kv8_attention: too many heads");
    Kv8Attention a{};
    a.q = q; a.q_row = q_row; a.q_dtype = q_dtype; a.layer = layer; a.heads = heads;
    a.slots = slots; a.offsets = offsets; a.starts = starts; a.batch = batch; a.rows = rows;
    a.cos_t = cos_table; a.sin_t = sin_table; a.scale = scale; a.out = out;
    a.vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && q_row * dtype_size(q_dtype) % 16 == 0;
    if (few_rows(cache, heads, max_new))
        return kv8_decode(cache, a, max_new, max_keys, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
    launch_chained(cache->head_dim == 64 ? kv8_attention_simple_kernel<64> : kv8_attention_simple_kernel<128>,
                   dim3(rows, heads), dim3(128), 0, static_cast<cudaStream_t>(stream), *cache, a);
    return check_launch("kv8_attention");
}
