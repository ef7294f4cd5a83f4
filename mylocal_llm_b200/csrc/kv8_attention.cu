// Causal attention over the paged 8-bit key/value cache (layout: kv8_cache.cuh): the entry point, which looks the arguments over
// and chooses between the kernel for few tokens per sequence (kv8_decode.cu) and the one for many (kv8_prompt.cu).
#include "kv8_attention.cuh"

namespace b200q {

int kv8_check(const char *what, const b200q_kv8_cache *c);       // kv8_cache.cu

// kv8_decode.cu
long long kv8_decode_workspace(const b200q_kv8_cache *c, int heads, int batch, int max_new, int max_keys);
double kv8_decode_time(const b200q_kv8_cache *c, int heads, int batch, int max_new, int max_keys);
int kv8_decode(const b200q_kv8_cache *c, const Kv8Attention &a, int max_new, int max_keys, void *workspace,
               long long workspace_bytes, cudaStream_t stream);
// kv8_prompt.cu
long long kv8_prompt_workspace(const b200q_kv8_cache *c, int heads, int batch, int rows, int max_new, int max_keys);
double kv8_prompt_time(const b200q_kv8_cache *c, int heads, int batch, int rows, int max_new, int max_keys);
int kv8_prompt(const b200q_kv8_cache *c, const Kv8Attention &a, int max_new, int max_keys, void *workspace, long long workspace_bytes,
               cudaStream_t stream);

// Whether a step goes to the kernel for few tokens per sequence: single tokens, and where it is estimated to take less time, as for
// chunks that are short next to their context: tiles of 16 rows against tiles of 128 (16 sequences of 8000 keys, 8 heads shared by
// 4: 8 new tokens each 160 us against 203, 16 new tokens 294 against 214).
static bool few_rows(const b200q_kv8_cache *c, int heads, int batch, int rows, int max_new, int max_keys) {
    return max_new == 1 || kv8_decode_time(c, heads, batch, max_new, max_keys) < kv8_prompt_time(c, heads, batch, rows, max_new, max_keys);
}

}  // namespace b200q

using namespace b200q;

extern "C" long long b200q_kv8_attention_workspace(const b200q_kv8_cache *cache, int heads, int batch, int rows, int max_new,
                                                   int max_keys) {
    if (!cache || heads < 1 || cache->kv_heads < 1 || heads % cache->kv_heads || max_new < 1) return 0;
    return few_rows(cache, heads, batch, rows, max_new, max_keys) ? kv8_decode_workspace(cache, heads, batch, max_new, max_keys)
                                               : kv8_prompt_workspace(cache, heads, batch, rows, max_new, max_keys);
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
    if (reinterpret_cast<uintptr_t>(out) & 15) return fail(B200Q_EINVAL, "kv8_attention: out must be 16-byte aligned");
    if (heads > 65535) return fail(B200Q_EUNSUPPORTED, "kv8_attention: too many heads");
    Kv8Attention a{};
    a.q = q; a.q_row = q_row; a.q_dtype = q_dtype; a.layer = layer; a.heads = heads;
    a.slots = slots; a.offsets = offsets; a.starts = starts; a.batch = batch; a.rows = rows;
    a.cos_t = cos_table; a.sin_t = sin_table; a.scale = scale; a.out = out;
    a.vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && q_row * dtype_size(q_dtype) % 16 == 0;
    if (few_rows(cache, heads, batch, rows, max_new, max_keys))
        return kv8_decode(cache, a, max_new, max_keys, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
    return kv8_prompt(cache, a, max_new, max_keys, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
