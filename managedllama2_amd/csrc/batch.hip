// The operators in front of the attention of a step of several requests: block tables and slots from the requests'
// lengths, and the rotation of queries and keys (normed, where the model does that) with the store into the paged cache.
#include "common.hpp"
#include "batch_plan.hpp"

#include <cmath>

namespace l2 {

// ---------------------------------------------------------------- block tables
struct TablesArgs {
    int* block_tables;
    int* lengths;
    int* query_starts;
    int* positions;
    int* slots;
    const int* cached;
    const int* counts;
    const int* free_blocks;
    const int* taken;
    int* new_taken;
    unsigned* arrivals; // zero between launches
    bool apart;         // lengths and new_taken are not what is read
    int n_requests, n_tokens, table_stride, prefix_length, n_free, shift;
};

constexpr int kTablesBlock = 1024;

// Inclusive prefix sum over the workgroup, each sum cut off at `most` (which keeps it associative for terms >= 0).
__device__ __forceinline__ int block_scan(int v, int most, int* lds /* 16 */)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d, 64);
        v = lane >= d ? min(v + o, most) : v;
    }
    if (lane == 63)
        lds[wave] = v;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < wave; ++w)
        before = min(before + lds[w], most);
    __syncthreads();
    return min(v + before, most);
}

// A block of 1024 requests at a time, lane by lane, two prefix sums (tokens, blocks); then their tokens, each of which
// finds its request in the sums.  A new block holds at least one new token, and the one in its first row writes the
// table entry.  Latency bounds it: lengths, sums, entries and stores follow each other.
//
// Workgroups of several compute the same sums and take every so many thousandth token each (14579 tokens: one workgroup 15.6
// us, 15 workgroups 5.8).  Where lengths or the number of taken blocks are updated in place, the last workgroup to have
// read them writes them.
__global__ __launch_bounds__(kTablesBlock) void batch_tables_kernel(TablesArgs a)
{
    __shared__ int sums[16];
    __shared__ int begin[kTablesBlock], rows[kTablesBlock], from[kTablesBlock]; // from: first free block, -1: refused
    __shared__ int most_taken;
    __shared__ unsigned arrived;
    const int size = 1 << a.shift, tid = threadIdx.x;
    const int limit = a.table_stride > (0x7FFFFFFF >> a.shift) ? 0x7FFFFFFF : a.table_stride << a.shift;
    const int taken = a.taken[0];
    const bool list = taken >= 0 && taken <= a.n_free; // else it counts as empty
    const int left = list ? a.n_free - taken : 0;
    const int every = static_cast<int>(gridDim.x) * kTablesBlock;
    int t = static_cast<int>(blockIdx.x) * kTablesBlock + tid; // this thread's next token
    bool lengths = gridDim.x == 1 || (a.apart && blockIdx.x == 0), starts = blockIdx.x == 0;
    for (;;) {
        if (tid == 0)
            most_taken = 0;
        int tokens_before = 0, need_before = 0; // the tokens cut off one above what there is
        for (int first = 0; first < a.n_requests; first += kTablesBlock) {
            const int b = first + tid, in_block = min(a.n_requests - first, kTablesBlock);
            const int c = b < a.n_requests ? a.cached[b] : 0, n = b < a.n_requests ? a.counts[b] : 0;
            const int tokens = min(max(n, 0), a.n_tokens + 1);
            const int end = min(block_scan(tokens, a.n_tokens + 1, sums) + tokens_before, a.n_tokens + 1);
            const bool fits = b < a.n_requests && c >= 0 && n >= 0 && c <= limit && n <= limit - c && end <= a.n_tokens;
            const int have = fits ? (c >> a.shift) + ((c & (size - 1)) != 0) : 0;
            const int total = fits ? ((c + n) >> a.shift) + (((c + n) & (size - 1)) != 0) : 0;
            const int need = total - have;
            const int upto = block_scan(need, kMaxBatchTokens, sums) + need_before; // a new block holds a new token: no more of them
            const bool admitted = fits && (need == 0 || upto <= left);
            begin[tid] = end;
            rows[tid] = c;
            from[tid] = !admitted ? -1 : need > 0 ? taken + upto - need : 0;
            const unsigned long long who = __ballot(admitted); // the sums never fall: a wavefront's last one has its largest
            if (admitted && (who >> (tid & 63)) == 1)
                atomicMax(&most_taken, upto);
            if (b < a.n_requests) {
                if (starts)
                    a.query_starts[b + 1] = min(end, a.n_tokens);
                if (lengths)
                    a.lengths[b] = admitted ? c + n : c;
            }
            if (b == 0 && starts)
                a.query_starts[0] = 0;
            if (tid == kTablesBlock - 1)
                sums[0] = upto;
            __syncthreads();
            need_before = sums[0];
            const int last = min(begin[kTablesBlock - 1], a.n_tokens);
            for (; t < last; t += every) {
                int lo = 0, hi = in_block - 1; // the first request whose tokens end behind t
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (begin[mid] > t)
                        hi = mid;
                    else
                        lo = mid + 1;
                }
                const int start_of = lo ? begin[lo - 1] : tokens_before;
                const int cb = rows[lo], f = from[lo];
                int position = -1, slot = -1;
                if (f >= 0) {
                    const int row = cb + (t - start_of), page = row >> a.shift;
                    const int had = (cb >> a.shift) + ((cb & (size - 1)) != 0);
                    int* entry = a.block_tables + static_cast<size_t>(first + lo) * a.table_stride + page;
                    const int block = page >= had ? a.free_blocks[f + page - had] : *entry;
                    if ((row & (size - 1)) == 0)
                        *entry = block;
                    position = a.prefix_length + row;
                    if (block >= 0 && block <= 0x7FFFFFFF >> a.shift) // else its slots are no ints, and would alias others
                        slot = (block << a.shift) + (row & (size - 1));
                }
                a.positions[t] = position;
                a.slots[t] = slot;
            }
            tokens_before = begin[kTablesBlock - 1];
            __syncthreads();
        }
        for (; t < a.n_tokens; t += every) {
            a.positions[t] = -1;
            a.slots[t] = -1;
        }
        if (lengths) {
            if (tid == 0)
                a.new_taken[0] = list ? taken + most_taken : taken;
            return;
        }
        if (a.apart)
            return;
        if (tid == 0)
            arrived = add_agent(a.arrivals, 1);
        __syncthreads();
        if (arrived + 1 != gridDim.x)
            return;
        if (tid == 0)
            store_agent(a.arrivals, 0u);
        lengths = true; // once more, for the lengths alone
        starts = false;
        __syncthreads();
    }
}

// ---------------------------------------------------------------- norm, rotation, store
struct RopeArgs {
    uint16_t* q_output;
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const uint16_t* q_gamma;
    const uint16_t* k_gamma;
    const int* positions;
    const int* slots;
    uint16_t* key;
    uint16_t* value;
    long long block_stride;
    long long n_slots;
    int n_heads, n_kv_heads, per, q_output_stride, q_stride, kv_stride, shift; // per: heads per workgroup
    float eps;
    unsigned long long powers[6]; // theta^(-2 i / head_size) for i = 1, 2, 4 .. 32, in units of 2^-64
};

// Turns per position of pair i, theta^(-2 i / head_size) / 2 pi, in 64 bits of fixed point: times a position, the bits above are
// whole turns and drop out by themselves.  Six products, and powers that are off by
// up to 2^-59 after their squarings, leave less than 2^-28 of a turn at 2^31 positions; the rounding to fp32 behind it is 2^-26.
__device__ __forceinline__ unsigned long long turns_of(const unsigned long long (&powers)[6], int i)
{
    unsigned long long v = 0x28BE60DB9391054Bull; // 1 / 2 pi
#pragma unroll
    for (int k = 0; k < 6; ++k)
        v = (i >> k) & 1 ? __umul64hi(v, powers[k]) : v;
    return v;
}

// The value of the lane that holds the other half's elements of the same pairs.
template <int D>
__device__ __forceinline__ float other_half(float v)
{
    if constexpr (D == 128)
        return dpp_f32<DPP_ROW_ROR8>(v);
    else
        return dpp_f32<DPP_QUAD_XOR3>(dpp_f32<DPP_ROW_HALF_MIRROR>(v)); // lane ^ 7, then ^ 3
}

template <int D>
__device__ __forceinline__ float head_sum(float v)
{
    v += dpp_f32<DPP_QUAD_XOR1>(v);
    v += dpp_f32<DPP_QUAD_XOR2>(v);
    v += dpp_f32<DPP_ROW_HALF_MIRROR>(v);
    if constexpr (D == 128)
        v += dpp_f32<DPP_ROW_MIRROR>(v);
    return v;
}

// A workgroup takes `per` heads of one token (of its queries, keys and values side by side), D / 8 lanes per head with 16
// bytes each; norms and the exchange of halves are row operations.  Sine and cosine of a token's angles are
// computed once per workgroup, one pair per thread, while the heads are on their way: kRopeDeep loads per lane at a time.
constexpr int kRopeDeep = 4;

template <int D>
__global__ __launch_bounds__(256) void batch_rope_kernel(RopeArgs a)
{
    constexpr int L = D / 8, HEADS = 256 / L; // lanes per head, heads side by side
    __shared__ __align__(16) float cosines[D / 2];
    __shared__ __align__(16) float sines[D / 2];
    const int t = blockIdx.x, tid = threadIdx.x, c = tid % L;
    const int position = a.positions[t], slot = a.slots[t];
    const int units = a.n_heads + 2 * a.n_kv_heads, first = blockIdx.y * a.per + tid / L, end = min(units, (static_cast<int>(blockIdx.y) + 1) * a.per);
    const bool stores = slot >= 0 && slot < a.n_slots;
    const long long to = stores ? (slot >> a.shift) * a.block_stride +
                                      static_cast<long long>(slot & ((1 << a.shift) - 1)) * a.n_kv_heads * D : 0;
    u32x4 x[kRopeDeep];
    auto load = [&](int u0) {
#pragma unroll
        for (int i = 0; i < kRopeDeep; ++i) {
            const int u = u0 + i * HEADS;
            if (u < end) {
                const uint16_t* p = u < a.n_heads ? a.q + static_cast<size_t>(t) * a.q_stride + u * D
                                    : u < a.n_heads + a.n_kv_heads
                                        ? a.k + static_cast<size_t>(t) * a.kv_stride + (u - a.n_heads) * D
                                        : a.v + static_cast<size_t>(t) * a.kv_stride + (u - a.n_heads - a.n_kv_heads) * D;
                x[i] = *reinterpret_cast<const u32x4*>(p + c * 8);
            }
        }
    };
    load(first);
    u32x4 gq = {}, gk = {};
    if (a.q_gamma)
        gq = *reinterpret_cast<const u32x4*>(a.q_gamma + c * 8);
    if (a.k_gamma)
        gk = *reinterpret_cast<const u32x4*>(a.k_gamma + c * 8);
    if (position < 0)
        return; // the whole workgroup
    if (tid < D / 2) {
        const int turn = static_cast<int>((static_cast<unsigned long long>(position) * turns_of(a.powers, tid)) >> 32);
        float s, cs;
        sincospif(static_cast<float>(turn) * 0x1p-31f, &s, &cs);
        cosines[tid] = cs;
        sines[tid] = s;
    }
    __syncthreads();
    float cs[8], sn[8]; // of this lane's pairs; the first half subtracts
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        cs[k] = cosines[c % (L / 2) * 8 + k];
        sn[k] = c < L / 2 ? -sines[c % (L / 2) * 8 + k] : sines[c % (L / 2) * 8 + k];
    }
    for (int u0 = first; u0 - tid / L < end; u0 += kRopeDeep * HEADS) {
        if (u0 != first)
            load(u0);
#pragma unroll
        for (int i = 0; i < kRopeDeep; ++i) {
            const int u = u0 + i * HEADS;
            const bool is_q = u < a.n_heads, is_v = u >= a.n_heads + a.n_kv_heads;
            u32x4 w = x[i];
            if (!is_v) {
                float f[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    f[2 * k] = static_cast<float>(as_h2(w[k])[0]);
                    f[2 * k + 1] = static_cast<float>(as_h2(w[k])[1]);
                }
                if (is_q ? a.q_gamma != nullptr : a.k_gamma != nullptr) {
                    float ss = 0.0f;
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        ss = __builtin_fmaf(f[k], f[k], ss);
                    const float r = 1.0f / sqrtf(head_sum<D>(ss) / static_cast<float>(D) + a.eps);
                    const u32x4 g = is_q ? gq : gk;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        f[2 * k] *= r * static_cast<float>(as_h2(g[k])[0]);
                        f[2 * k + 1] *= r * static_cast<float>(as_h2(g[k])[1]);
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float y0 = __builtin_fmaf(f[2 * k], cs[2 * k], other_half<D>(f[2 * k]) * sn[2 * k]);
                    const float y1 = __builtin_fmaf(f[2 * k + 1], cs[2 * k + 1], other_half<D>(f[2 * k + 1]) * sn[2 * k + 1]);
                    w[k] = static_cast<uint32_t>(float_to_half_bits(y0)) | static_cast<uint32_t>(float_to_half_bits(y1)) << 16;
                }
            }
            if (u < end) {
                if (is_q)
                    *reinterpret_cast<u32x4*>(a.q_output + static_cast<size_t>(t) * a.q_output_stride + u * D + c * 8) = w;
                else if (stores)
                    *reinterpret_cast<u32x4*>((is_v ? a.value + (u - a.n_heads - a.n_kv_heads) * D : a.key + (u - a.n_heads) * D) +
                                              to + c * 8) = w;
            }
        }
    }
}

// ---------------------------------------------------------------- host side
} // namespace l2

using namespace l2;

extern "C" {

int llama2_batch_tables(const llama2_batch* batch, const int* cached, const int* counts, const int* free_blocks, int n_free,
                        const int* taken, int* new_taken, int block_size)
{
    L2_REQUIRE_INIT();
    if (int rc = check_batch_tables(batch, cached, counts, free_blocks, n_free, taken, new_taken, block_size))
        return rc;
    const llama2_batch& b = *batch;
    TablesArgs a = {b.block_tables, b.lengths, b.query_starts, b.positions, b.slots, cached, counts, free_blocks, taken,
                    new_taken, ctx().batch_counters + kMaxBatchCounters, b.lengths != cached && new_taken != taken, b.n_requests, b.n_tokens, b.table_stride, b.prefix_length, n_free, log2_of(block_size)};
    const int groups = ceil_div(b.n_tokens, kTablesBlock);
    hipLaunchKernelGGL(batch_tables_kernel, dim3(groups < 64 ? groups : 64), dim3(kTablesBlock), 0, ctx().stream, a);
    L2_LAUNCH_CHECK("llama2_batch_tables");
    return LLAMA2_OK;
}

int llama2_batch_qk_norm_rope(llama2_half* q_output, const llama2_half* q, const llama2_half* k, const llama2_half* v,
                              const llama2_half* q_gamma, const llama2_half* k_gamma, const llama2_batch* batch,
                              const llama2_paged_cache* cache, int n_heads, int q_output_stride, int q_stride, int kv_stride,
                              float eps, float theta)
{
    const char* fn = "llama2_batch_qk_norm_rope";
    L2_REQUIRE_INIT();
    if (int rc = check_batch_rope(q_output, q, k, v, q_gamma, k_gamma, batch, cache, n_heads, q_output_stride, q_stride, kv_stride, eps,
                                  theta))
        return rc;
    const int d = cache->head_size;
    RopeArgs a = {};
    a.q_output = q_output;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_gamma = q_gamma;
    a.k_gamma = k_gamma;
    a.positions = batch->positions;
    a.slots = batch->slots;
    a.key = cache->key;
    a.value = cache->value;
    a.block_stride = block_halfs(*cache);
    a.n_slots = static_cast<long long>(cache->n_blocks) * cache->block_size;
    a.n_heads = n_heads;
    a.n_kv_heads = cache->n_kv_heads;
    a.q_output_stride = q_output_stride;
    a.q_stride = q_stride;
    a.kv_stride = kv_stride;
    a.shift = log2_of(cache->block_size);
    a.eps = eps;
    long double power = powl(static_cast<long double>(theta), -2.0L / d);
    for (unsigned long long& p : a.powers) { // of theta 1: the largest number below 1
        p = power >= 1.0L ? ~0ull : static_cast<unsigned long long>(power * 0x1p64L);
        power *= power;
    }
    // Few tokens: as few heads per workgroup as are side by side, which is quickest; many: a workgroup computes the
    // angles of a token once for all its heads.
    const int units = n_heads + 2 * a.n_kv_heads, side = 256 / (d / 8);
    const int parts = ceil_div(units, side), want = ceil_div(4 * ctx().num_cus, batch->n_tokens);
    a.per = ceil_div(parts, parts < want ? parts : want) * side;
    const dim3 grid(batch->n_tokens, ceil_div(units, a.per));
    if (d == 128)
        hipLaunchKernelGGL(batch_rope_kernel<128>, grid, dim3(256), 0, ctx().stream, a);
    else
        hipLaunchKernelGGL(batch_rope_kernel<64>, grid, dim3(256), 0, ctx().stream, a);
    L2_LAUNCH_CHECK(fn);
    return LLAMA2_OK;
}

} // extern "C"
