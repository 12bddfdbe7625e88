// Attention of a step of several requests over a paged cache, behind a prefix that they share.
#include "common.hpp"

namespace l2 {

struct BatchAttnArgs {
    uint16_t* out;
    const uint16_t* q;
    const uint16_t* key;
    const uint16_t* value;
    const int* prefix_table;
    const int* block_tables;
    const int* query_starts;
    const int* positions;
    long long block_stride;
    int n_requests, n_tokens, table_stride, prefix_length, max_rows;
    int n_blocks, shift, n_kv_heads, group, out_stride, q_stride;
    float scale;
};

// One wavefront per token and head: 64 / (D / 8) rows at a time, D / 8 lanes each.
template <int D>
__global__ __launch_bounds__(64) void batch_attn_simple_kernel(BatchAttnArgs a)
{
    constexpr int L = D / 8;
    const int t = blockIdx.x, h = blockIdx.y, kvh = h / a.group;
    const int lane = threadIdx.x, c = lane % L, sub = lane / L;
    const int position = a.positions[t];
    if (position < 0)
        return;
    int b = 0;
    while (b + 1 < a.n_requests && a.query_starts[b + 1] <= t)
        ++b;
    const int own = min(max(position - a.prefix_length + 1, 0), a.max_rows);
    float q[8], o[8] = {};
    for (int i = 0; i < 8; ++i)
        q[i] = half_bits_to_float(a.q[static_cast<size_t>(t) * a.q_stride + h * D + c * 8 + i]);
    float m = -INFINITY, sum = 0.0f;
    for (int r = sub; r < a.prefix_length + own; r += 64 / L) {
        const bool shared = r < a.prefix_length;
        const int row = shared ? r : r - a.prefix_length;
        const int block = shared ? a.prefix_table[row >> a.shift]
                                 : a.block_tables[static_cast<size_t>(b) * a.table_stride + (row >> a.shift)];
        if (static_cast<unsigned>(block) >= static_cast<unsigned>(a.n_blocks))
            continue;
        const size_t at = block * a.block_stride +
                          (static_cast<size_t>(row & ((1 << a.shift) - 1)) * a.n_kv_heads + kvh) * D + c * 8;
        float s = 0.0f;
        for (int i = 0; i < 8; ++i)
            s += q[i] * half_bits_to_float(a.key[at + i]);
        for (int x = L / 2; x; x >>= 1)
            s += __shfl_xor(s, x, 64);
        s *= a.scale;
        const float nm = fmaxf(m, s), base = nm == -INFINITY ? 0.0f : nm;
        const float alpha = expf(m - base), p = expf(s - base);
        m = nm;
        sum = sum * alpha + p;
        for (int i = 0; i < 8; ++i)
            o[i] = o[i] * alpha + p * half_bits_to_float(a.value[at + i]);
    }
    for (int x = L; x < 64; x <<= 1) {
        const float om = __shfl_xor(m, x, 64), nm = fmaxf(m, om), base = nm == -INFINITY ? 0.0f : nm;
        const float wa = expf(m - base), wb = expf(om - base);
        sum = sum * wa + __shfl_xor(sum, x, 64) * wb;
        for (int i = 0; i < 8; ++i)
            o[i] = o[i] * wa + __shfl_xor(o[i], x, 64) * wb;
        m = nm;
    }
    if (sub == 0)
        for (int i = 0; i < 8; ++i)
            a.out[static_cast<size_t>(t) * a.out_stride + h * D + c * 8 + i] =
                float_to_half_bits(sum == 0.0f ? 0.0f : o[i] / sum);
}

} // namespace l2

using namespace l2;

extern "C" {

int llama2_batch_attention(llama2_half* output, const llama2_half* query, const llama2_batch* batch,
                           const llama2_paged_cache* cache, int n_heads, int output_stride, int query_stride, float scale)
{
    const char* fn = "llama2_batch_attention";
    L2_REQUIRE_INIT();
    if (int rc = check_batch(fn, batch))
        return rc;
    if (int rc = check_paged_cache(fn, cache, n_heads))
        return rc;
    const llama2_batch& b = *batch;
    L2_CHECK(output && query && b.block_tables && b.query_starts && b.positions && (b.prefix_table || b.prefix_length == 0),
             "%s: null pointer", fn);
    L2_CHECK(aligned(output, 16) && aligned(query, 16), "%s: pointers must be 16-byte aligned", fn);
    const int row = n_heads * cache->head_size;
    L2_CHECK(output_stride >= row && query_stride >= row && output_stride % 8 == 0 && query_stride % 8 == 0,
             "%s: strides %d, %d must be multiples of 8 and hold a row of %d", fn, output_stride, query_stride, row);
    L2_CHECK(!overlap(output, (static_cast<size_t>(b.n_tokens - 1) * output_stride + row) * 2, query,
                      (static_cast<size_t>(b.n_tokens - 1) * query_stride + row) * 2), "%s: output overlaps query", fn);
    L2_CHECK(b.table_stride > 0 && b.max_length > 0 && b.max_length <= (0x7FFFFFFF - 4096 - b.prefix_length),
             "%s: table_stride=%d and max_length=%d must be positive, and below 2^31 rows with the prefix", fn, b.table_stride,
             b.max_length);
    const long long table_rows = static_cast<long long>(b.table_stride) * cache->block_size;
    BatchAttnArgs a = {};
    a.out = output;
    a.q = query;
    a.key = cache->key;
    a.value = cache->value;
    a.prefix_table = b.prefix_table;
    a.block_tables = b.block_tables;
    a.query_starts = b.query_starts;
    a.positions = b.positions;
    a.block_stride = cache->block_stride ? cache->block_stride
                                         : static_cast<long long>(cache->block_size) * cache->n_kv_heads * cache->head_size;
    a.n_requests = b.n_requests;
    a.n_tokens = b.n_tokens;
    a.table_stride = b.table_stride;
    a.prefix_length = b.prefix_length;
    a.max_rows = table_rows < b.max_length ? static_cast<int>(table_rows) : b.max_length;
    a.n_blocks = cache->n_blocks;
    for (a.shift = 3; (1 << a.shift) < cache->block_size; ++a.shift) {
    }
    a.n_kv_heads = cache->n_kv_heads;
    a.group = n_heads / cache->n_kv_heads;
    a.out_stride = output_stride;
    a.q_stride = query_stride;
    a.scale = scale;
    const dim3 grid(b.n_tokens, n_heads);
    if (cache->head_size == 128)
        hipLaunchKernelGGL(batch_attn_simple_kernel<128>, grid, dim3(64), 0, ctx().stream, a);
    else
        hipLaunchKernelGGL(batch_attn_simple_kernel<64>, grid, dim3(64), 0, ctx().stream, a);
    L2_LAUNCH_CHECK(fn);
    return LLAMA2_OK;
}

} // extern "C"
