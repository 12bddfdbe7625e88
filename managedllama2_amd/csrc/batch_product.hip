// Products of the rows of many tokens with int4 tensors, low-rank adapters of the tokens' requests beside them, and the first
// half of the gated feed-forward block.
//
//   y[t][n] = sum_g s[n][g] sum_{k in g} x[t][k] (w[n][k] - z[n][g])  +  f_a sum_r up_a[n][r] h[t][r],   h[t][r] = sum_k down_a[r][k] x[t][k]
//
// w - z is an exact fp16 integer, its products with x are summed in fp32 over a group of 128 and scaled in fp32.  h is summed in
// fp32 and leaves as two fp16 numbers and a power of two (22 bits of the token's largest), which the matrix cores take as 16 ranks a product.
#include "common.hpp"
#include "batch_product_plan.hpp"

#include <cmath>

namespace l2 {

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

struct ProductTensor {
    const uint32_t* w;
    const uint32_t* z;
    const uint16_t* s;
    uint16_t* out;
    const uint16_t* residual;
    const uint16_t* down; // null: no adapters
    const uint16_t* up;
    const float* scales;
    const int* ranks;
    long long down_stride, up_stride;
    uint16_t* low;  // [n_tokens][max_rank / 8][2][8]: what the ranks received, upper and lower part
    float* factors; // [n_tokens]: scale of the adapter and power of two of the token
    int n_adapters, max_rank, cols, out_stride, residual_stride;
    int first; // first block of rows of this tensor
};

struct ProductArgs {
    ProductTensor m[LLAMA2_MAX_BATCH_MATRICES];
    const uint16_t* x;
    const int* positions;
    const int* token_adapters;
    int n_matrices, K, groups, ws, ss, zs, x_stride, n_tokens, row_blocks, token_blocks;
};

// The arguments as they lie in memory: a tensor chosen by an index is then a scalar load (chosen among registers it is a hundred
// instructions).
typedef __attribute__((address_space(4))) const ProductArgs KernelArgs;
__device__ __forceinline__ KernelArgs& kernel_args()
{
    return *(KernelArgs*)__builtin_amdgcn_kernarg_segment_ptr();
}

constexpr int kNoAdapter = -1, kNoToken = -2;

// Adapter of token t: one of 0 .. n - 1, kNoAdapter, or kNoToken where there is no token.
__device__ __forceinline__ int adapter_of(KernelArgs& a, int t)
{
    if (t >= a.n_tokens || a.positions[t] < 0)
        return kNoToken;
    const int id = a.token_adapters ? a.token_adapters[t] : kNoAdapter;
    return id < 0 ? kNoAdapter : id;
}

// Which of 16 tokens in LDS are the first with their adapter, as bits; the same in every wavefront.
__device__ __forceinline__ unsigned first_of_adapter(const int* ids, int n_adapters)
{
    const int l = threadIdx.x & 15, id = ids[l];
    bool first = id >= 0 && id < n_adapters;
#pragma unroll
    for (int j = 0; j < 15; ++j)
        first = first && !(j < l && ids[j] == id);
    return static_cast<unsigned>(__ballot(first)) & 0xFFFFu;
}

__device__ __forceinline__ int nth_bit(unsigned mask, int n) // of the set ones
{
    for (; n > 0; --n)
        mask &= mask - 1;
    return __builtin_ctz(mask);
}

__device__ __forceinline__ int rank_of(const int* ranks, int a, int max_rank)
{
    const int r = __builtin_amdgcn_readfirstlane(ranks[a]);
    return r < 0 ? 0 : r > max_rank ? max_rank : r;
}

__device__ __forceinline__ f4_t mfma16(h8_t a, h8_t b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Elements k .. k + 7 of a row of which n exist.
__device__ __forceinline__ h8_t load8(const uint16_t* row, int k, int n)
{
    u32x4 v = {};
    if (k < n)
        v = *reinterpret_cast<const u32x4*>(row + k);
    return __builtin_bit_cast(h8_t, v);
}

// ---------------------------------------------------------------- what the ranks receive
// A workgroup takes 16 tokens and one of the adapters that they use; its wavefronts split the inputs.  Columns of other tokens are
// computed with it and dropped: columns of a matrix product do not mix.
constexpr int kLowWaves = 8, kLowTiles = 4; // rank tiles of 16 at a time

__global__ __launch_bounds__(kLowWaves * 64) void batch_low_kernel(ProductArgs)
{
    constexpr int kStride = kLowTiles * 16 + 4;
    __shared__ int ids[16];
    __shared__ __align__(16) float red[kLowWaves * 16 * kStride];
    __shared__ __align__(16) float sums[16 * (kMaxRank + 4)];
    KernelArgs& a = kernel_args();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, c = lane >> 4;
    const int t0 = blockIdx.x * 16;
    __attribute__((address_space(4))) const ProductTensor& m = a.m[blockIdx.z];
    if (!m.down)
        return;
    if (threadIdx.x < 16)
        ids[threadIdx.x] = adapter_of(a, t0 + threadIdx.x);
    __syncthreads();
    const unsigned firsts = first_of_adapter(ids, m.n_adapters);
    if (static_cast<int>(blockIdx.y) >= __builtin_popcount(firsts))
        return;
    const int id = __builtin_amdgcn_readfirstlane(ids[nth_bit(firsts, blockIdx.y)]);
    const int rank = rank_of(m.ranks, id, m.max_rank);
    const int token = t0 + l15 < a.n_tokens ? t0 + l15 : a.n_tokens - 1;
    const uint16_t* x = a.x + static_cast<size_t>(token) * a.x_stride;
    const uint16_t* down = m.down + id * m.down_stride;
    for (int r0 = 0; r0 < rank; r0 += kLowTiles * 16) {
        f4_t acc[kLowTiles] = {};
        const int tiles = min((rank - r0 + 15) / 16, kLowTiles);
        for (int k0 = wave * 128; k0 < a.K; k0 += kLowWaves * 128) {
            h8_t xf[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                xf[j] = load8(x, k0 + 32 * j + 8 * c, a.K);
#pragma unroll
            for (int i = 0; i < kLowTiles; ++i)
                if (i < tiles) {
                    const int r = r0 + i * 16 + l15;
                    const uint16_t* row = down + static_cast<size_t>(r < rank ? r : rank - 1) * a.K;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[i] = mfma16(xf[j], load8(row, k0 + 32 * j + 8 * c, a.K), acc[i]);
                }
        }
#pragma unroll
        for (int i = 0; i < kLowTiles; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                red[(wave * 16 + 4 * c + e) * kStride + i * 16 + l15] = acc[i][e];
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * kLowTiles * 16; e += kLowWaves * 64) {
            const int t = e / (kLowTiles * 16), r = e % (kLowTiles * 16);
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kLowWaves; ++w)
                v += red[(w * 16 + t) * kStride + r];
            sums[t * (kMaxRank + 4) + r0 + r] = r0 + r < rank ? v : 0.0f;
        }
        __syncthreads();
    }
    // 32 threads a token, 4 ranks a thread
    const int t = threadIdx.x >> 5, r = (threadIdx.x & 31) * 4;
    if (ids[t] != id)
        return;
    float v[4] = {}, most = 0.0f;
    if (r < rank) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = sums[t * (kMaxRank + 4) + r + e];
            most = fmaxf(most, fabsf(v[e]));
        }
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1)
        most = fmaxf(most, __shfl_xor(most, d, 64));
    // the largest between 2^14 and 2^15; nothing to scale where all are 0 or one is infinite
    int e2 = 0;
    if (most > 0.0f && most < INFINITY)
        e2 = 14 - ilogbf(most);
    if (r < (rank + 7) / 8 * 8) {
        uint32_t hi[2] = {}, lo[2] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float s = ldexpf(v[e], e2);
            const uint16_t h = float_to_half_bits(s);
            hi[e >> 1] |= static_cast<uint32_t>(h) << (16 * (e & 1));
            lo[e >> 1] |= static_cast<uint32_t>(float_to_half_bits(s - half_bits_to_float(h))) << (16 * (e & 1));
        }
        uint16_t* to = m.low + (static_cast<size_t>(t0 + t) * m.max_rank + r / 8 * 8) * 2 + (r & 4);
        *reinterpret_cast<u32x2*>(to) = u32x2{hi[0], hi[1]};
        *reinterpret_cast<u32x2*>(to + 8) = u32x2{lo[0], lo[1]};
    }
    if (r == 0)
        m.factors[t0 + t] = ldexpf(m.scales[id], -e2);
}

// ---------------------------------------------------------------- the products
// The eight weights of a word as fp16 n - z, in order: a byte into both halves, the lower nibble of one and the upper nibble
// of the other into the mantissa of 1024, then 1024 + n - (1024 + z) and (1024 + 16 n) / 16 - (64 + z).
__device__ __forceinline__ h8_t weights_of(uint32_t w, h2_t minus)
{
    const h2_t times = {static_cast<_Float16>(1.0f), static_cast<_Float16>(0.0625f)};
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = __builtin_amdgcn_perm(0u, w, 0x0C000C00u | i | i << 16);
        v[i] = as_u32(__builtin_elementwise_fma(as_h2((u & 0x00F0000Fu) | 0x64006400u), times, minus));
    }
    return __builtin_bit_cast(h8_t, v);
}

// Lane group c of 16 holds words 4 c .. 4 c + 3 of a group's 16 in v; afterwards words c, 4 + c, 8 + c and 12 + c.
__device__ __forceinline__ u32x4 words_by_product(u32x4 v)
{
    const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
    const auto lo = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

constexpr int kProductWaves = 8;

// A workgroup takes R tiles of 16 outputs (GATED: half of them of the gate, half of the up projection) and T tiles of 16
// tokens; its wavefronts take the groups of 128 inputs in turn and add up through LDS.
template <int R, int T, bool GATED>
__global__ __launch_bounds__(kProductWaves * 64) void batch_product_kernel(ProductArgs)
{
    constexpr int kTokens = T * 16, kRows = R * 16, kStride = kRows + 4;
    __shared__ __align__(16) float red[kProductWaves * kTokens * kStride];
    __shared__ int ids[kTokens];
    __shared__ __align__(16) float factors[2][kTokens];
    KernelArgs& a = kernel_args();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, c = lane >> 4;
    // the token blocks of one block of rows follow each other on one XCD
    const int slot = blockIdx.x >> 3, rb = slot / a.token_blocks * 8 + (blockIdx.x & 7), t0 = slot % a.token_blocks * kTokens;
    if (rb >= a.row_blocks)
        return;
    int which = 0;
    if (!GATED)
        while (which + 1 < a.n_matrices && rb >= a.m[which + 1].first)
            ++which;
    auto& m0 = a.m[which];
    auto& m1 = a.m[GATED ? 1 : which];
    const int n0 = (rb - (GATED ? 0 : m0.first)) * (GATED ? kRows / 2 : kRows);
    auto row_of = [&](int r) { return n0 + (GATED ? r % (R / 2) : r) * 16; };
    if (threadIdx.x < kTokens) {
        const int t = t0 + threadIdx.x, id = adapter_of(a, t);
        ids[threadIdx.x] = id;
        factors[0][threadIdx.x] = m0.down && id >= 0 && id < m0.n_adapters ? m0.factors[t] : 0.0f;
        if (GATED)
            factors[1][threadIdx.x] = m1.down && id >= 0 && id < m1.n_adapters ? m1.factors[t] : 0.0f;
    }

    const uint32_t* w[R];
    const uint32_t* z[R];
    const uint16_t* s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        auto& m = GATED && r >= R / 2 ? m1 : m0;
        const int n = min(row_of(r) + l15, m.cols - 1);
        w[r] = m.w + static_cast<size_t>(n) * a.ws;
        z[r] = m.z + static_cast<size_t>(n) * a.zs;
        s[r] = m.s + static_cast<size_t>(n) * a.ss;
    }
    const uint16_t* x[T];
#pragma unroll
    for (int t = 0; t < T; ++t)
        x[t] = a.x + static_cast<size_t>(min(t0 + t * 16 + l15, a.n_tokens - 1)) * a.x_stride;

    f4_t acc[T][R] = {};
    for (int g = wave; g < a.groups; g += kProductWaves) {
        h8_t wf[R][4];
        float sc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            // words behind the end of a row meet zeros of x
            const u32x4 v = words_by_product(*reinterpret_cast<const u32x4*>(w[r] + min(16 * g + 4 * c, a.ws - 4)));
            const float zero = static_cast<float>(z[r][g >> 3] >> (4 * (g & 7)) & 15u);
            const h2_t minus = {static_cast<_Float16>(-1024.0f - zero), static_cast<_Float16>(-64.0f - zero)};
            sc[r] = half_bits_to_float(s[r][g]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                wf[r][j] = weights_of(v[j], minus);
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            h8_t xf[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                xf[j] = load8(x[t], 128 * g + 32 * j + 8 * c, a.K);
            f4_t p[R] = {};
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    p[r] = mfma16(xf[j], wf[r][j], p[r]);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[t][r][e] = __builtin_fmaf(p[r][e], sc[r], acc[t][r][e]);
        }
    }
    __syncthreads(); // ids and factors
    // The adapters, each added to the tokens that use it (an adapter with infinite weights must not reach the others).
#pragma unroll
    for (int h = 0; h < (GATED ? 2 : 1); ++h) {
        auto& m = h ? m1 : m0;
        if (!m.down)
            continue;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const unsigned firsts = first_of_adapter(ids + t * 16, m.n_adapters);
            const int count = __builtin_popcount(firsts);
            for (int i = wave; i < count; i += kProductWaves) {
                const int id = __builtin_amdgcn_readfirstlane(ids[t * 16 + nth_bit(firsts, i)]);
                const int rank = rank_of(m.ranks, id, m.max_rank), token = min(t0 + t * 16 + l15, a.n_tokens - 1);
                f4_t p[R] = {};
                for (int r0 = 0; r0 < rank; r0 += 16) {
                    // lane groups 0 and 1: the upper parts of ranks 0 .. 7 and 8 .. 15; 2 and 3: the lower ones
                    const int at = r0 + (c & 1) * 8, have = rank - at;
                    u32x4 h4 = {};
                    if (have > 0)
                        h4 = *reinterpret_cast<const u32x4*>(m.low + (static_cast<size_t>(token) * m.max_rank + at) * 2 + (c >> 1) * 8);
#pragma unroll
                    for (int r = h * (R / 2); r < (GATED && !h ? R / 2 : R); ++r) {
                        u32x4 u = {};
                        if (have > 0)
                            u = *reinterpret_cast<const u32x4*>(m.up + id * m.up_stride +
                                                                static_cast<size_t>(min(row_of(r) + l15, m.cols - 1)) * m.max_rank + at);
                        if (rank & 7)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                u[k] &= have >= 2 * k + 2 ? ~0u : have == 2 * k + 1 ? 0xFFFFu : 0u;
                        p[r] = mfma16(__builtin_bit_cast(h8_t, h4), __builtin_bit_cast(h8_t, u), p[r]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool own = ids[t * 16 + 4 * c + e] == id;
                    const float f = factors[h][t * 16 + 4 * c + e];
#pragma unroll
                    for (int r = h * (R / 2); r < (GATED && !h ? R / 2 : R); ++r)
                        acc[t][r][e] = own ? __builtin_fmaf(p[r][e], f, acc[t][r][e]) : acc[t][r][e];
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                red[(wave * kTokens + t * 16 + 4 * c + e) * kStride + r * 16 + l15] = acc[t][r][e];
    __syncthreads();
    constexpr int kOut = GATED ? kRows / 2 : kRows, kPieces = kOut / 8;
    for (int i = threadIdx.x; i < kTokens * kPieces; i += kProductWaves * 64) {
        const int t = i / kPieces, piece = i % kPieces * 8, n = n0 + piece;
        if (ids[t] == kNoToken || n >= m0.cols)
            continue;
        float v[2][8] = {};
#pragma unroll
        for (int h = 0; h < (GATED ? 2 : 1); ++h)
            for (int q = 0; q < kProductWaves; ++q)
#pragma unroll
                for (int k = 0; k < 8; k += 4) {
                    const f4_t y = *reinterpret_cast<const f4_t*>(red + (q * kTokens + t) * kStride + h * kOut + piece + k);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[h][k + e] += y[e];
                }
        u32x4 o;
        if (GATED) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[0][k] = v[0][k] / (1.0f + expf(-v[0][k])) * v[1][k];
        } else if (m0.residual) {
            const u32x4 y = *reinterpret_cast<const u32x4*>(m0.residual + static_cast<size_t>(t0 + t) * m0.residual_stride + n);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[0][k] += half_bits_to_float(static_cast<uint16_t>(y[k >> 1] >> (16 * (k & 1))));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            o[k] = static_cast<uint32_t>(float_to_half_bits(v[0][2 * k])) | static_cast<uint32_t>(float_to_half_bits(v[0][2 * k + 1])) << 16;
        *reinterpret_cast<u32x4*>(m0.out + static_cast<size_t>(t0 + t) * m0.out_stride + n) = o;
    }
}

template <int R, int T, bool GATED>
static void launch_product(ProductArgs& a)
{
    constexpr int kRows = GATED ? R * 8 : R * 16;
    a.row_blocks = 0;
    for (int i = 0; i < (GATED ? 1 : a.n_matrices); ++i) {
        a.m[i].first = a.row_blocks;
        a.row_blocks += ceil_div(a.m[i].cols, kRows);
    }
    a.token_blocks = ceil_div(a.n_tokens, T * 16);
    const dim3 grid(static_cast<unsigned>(ceil_div(a.row_blocks, 8)) * 8 * a.token_blocks);
    hipLaunchKernelGGL((batch_product_kernel<R, T, GATED>), grid, dim3(kProductWaves * 64), 0, ctx().stream, a);
}

template <bool GATED>
static int run_product(const char* fn, ProductArgs& a)
{
    size_t bytes = 0;
    int most = 0;
    for (int i = 0; i < a.n_matrices; ++i)
        if (a.m[i].down) {
            bytes += static_cast<size_t>(a.n_tokens) * (a.m[i].max_rank * 4 + 4);
            most = a.m[i].n_adapters > most ? a.m[i].n_adapters : most;
        }
    if (bytes) {
        if (int rc = ensure_attn_partials(bytes))
            return rc;
        char* p = reinterpret_cast<char*>(ctx().attn_partials);
        for (int i = 0; i < a.n_matrices; ++i)
            if (a.m[i].down) {
                a.m[i].low = reinterpret_cast<uint16_t*>(p);
                p += static_cast<size_t>(a.n_tokens) * a.m[i].max_rank * 4;
            }
        for (int i = 0; i < a.n_matrices; ++i)
            if (a.m[i].down) {
                a.m[i].factors = reinterpret_cast<float*>(p);
                p += static_cast<size_t>(a.n_tokens) * 4;
            }
        hipLaunchKernelGGL(batch_low_kernel, dim3(ceil_div(a.n_tokens, 16), most < 16 ? most : 16, a.n_matrices), dim3(kLowWaves * 64), 0,
                           ctx().stream, a);
        L2_LAUNCH_CHECK(fn);
    }
    if (a.n_tokens <= 16)
        launch_product<2, 1, GATED>(a);
    else if (a.n_tokens <= 32)
        launch_product<2, 2, GATED>(a);
    else
        launch_product<2, 4, GATED>(a);
    L2_LAUNCH_CHECK(fn);
    return LLAMA2_OK;
}

static ProductArgs product_args(const llama2_half* input, int rows, int input_stride, const int* token_adapters, const llama2_batch& batch)
{
    ProductArgs a = {};
    a.x = input;
    a.positions = batch.positions;
    a.token_adapters = token_adapters;
    a.K = rows;
    a.groups = weight_groups(rows);
    a.ws = weight_words(rows);
    a.ss = a.groups;
    a.zs = zero_words(rows);
    a.x_stride = input_stride;
    a.n_tokens = batch.n_tokens;
    return a;
}

static void put_tensor(ProductTensor& m, const llama2_qweight& w, const llama2_adapters* a, int rows, int cols)
{
    m.w = w.weight;
    m.z = w.zeros;
    m.s = w.scales;
    m.cols = cols;
    if (a) {
        m.down = a->down;
        m.up = a->up;
        m.scales = a->scales;
        m.ranks = a->ranks;
        m.down_stride = down_halfs(*a, rows);
        m.up_stride = up_halfs(*a, cols);
        m.n_adapters = a->n_adapters;
        m.max_rank = a->max_rank;
    }
}

} // namespace l2

using namespace l2;

extern "C" {

int llama2_batch_mat_mul_int4(const llama2_batch_matrix* matrices, int n_matrices, const llama2_half* input, int rows, int input_stride,
                              const int* token_adapters, const llama2_batch* batch)
{
    L2_REQUIRE_INIT();
    if (int rc = check_batch_mat_mul(matrices, n_matrices, input, rows, input_stride, token_adapters, batch))
        return rc;
    ProductArgs a = product_args(input, rows, input_stride, token_adapters, *batch);
    a.n_matrices = n_matrices;
    for (int i = 0; i < n_matrices; ++i) {
        const llama2_batch_matrix& m = matrices[i];
        put_tensor(a.m[i], m.weight, m.adapters, rows, m.cols);
        a.m[i].out = m.output;
        a.m[i].residual = m.residual;
        a.m[i].out_stride = m.output_stride;
        a.m[i].residual_stride = m.residual_stride;
    }
    return run_product<false>("llama2_batch_mat_mul_int4", a);
}

int llama2_batch_mat_mul_swiglu(llama2_half* output, const llama2_half* input, const llama2_qweight* gate, const llama2_qweight* up, int rows,
                                int cols, int output_stride, int input_stride, const llama2_adapters* gate_adapters,
                                const llama2_adapters* up_adapters, const int* token_adapters, const llama2_batch* batch)
{
    L2_REQUIRE_INIT();
    if (int rc = check_batch_swiglu(output, input, gate, up, rows, cols, output_stride, input_stride, gate_adapters, up_adapters,
                                    token_adapters, batch))
        return rc;
    ProductArgs a = product_args(input, rows, input_stride, token_adapters, *batch);
    a.n_matrices = 2;
    put_tensor(a.m[0], *gate, gate_adapters, rows, cols);
    put_tensor(a.m[1], *up, up_adapters, rows, cols);
    a.m[0].out = output;
    a.m[0].out_stride = output_stride;
    return run_product<true>("llama2_batch_mat_mul_swiglu", a);
}

} // extern "C"
