// What the products of many tokens share with the kernels of the prompt's products: operands from nibbles and rows, the tokens' adapters in
// groups that the matrix cores take together, and small device helpers.
#pragma once

#include "common.hpp"
#include "batch_product_plan.hpp"

namespace l2 {

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

// An int4 tensor of a product.  Arguments lie in memory, and a kernel that asks for them one after the other waits for each: a tensor's
// are neighbours.
struct alignas(64) ProductTensor {
    const uint32_t* w;
    const uint32_t* z;
    const uint16_t* s;
    uint16_t* out;
    const uint16_t* residual;
    const uint16_t* up; // null: no adapters
    const void* low;
    const TokenAdapter* info;
    long long up_stride;
    int cols, out_stride, residual_stride, n_adapters, max_rank;
};

// A step of one token, where the kernels of a decode step take its shape; false where they do not.
struct ProductArgs;
bool launch_one_token(const ProductArgs& call, int n_matrices, bool gated);

struct alignas(64) ProductArgs {
    const uint16_t* x;
    const int* positions;
    const int* token_adapters;
    int K, x_stride, n_tokens, most_adapters; // of any tensor
    int token_blocks;
    ProductTensor t[LLAMA2_MAX_BATCH_MATRICES];
};

// The arguments as they lie in memory: a tensor chosen by an index is then a few scalar loads (chosen among registers it is a hundred
// instructions).
template <class A>
using Constant = __attribute__((address_space(4))) const A;

template <class A>
__device__ __forceinline__ Constant<A>& kernel_args()
{
    return *(Constant<A>*)__builtin_amdgcn_kernarg_segment_ptr();
}

template <class V>
__device__ __forceinline__ void needed(const V& v)
{
    asm volatile("" : : "s"(v));
}

template <class... V>
__device__ __forceinline__ void loaded(const V&... v) // here, together
{
    (needed(v), ...);
}

constexpr int kNoAdapter = -1, kNoToken = -2;

__device__ __forceinline__ int known_adapter(int position, int id, int most_adapters)
{
    return position < 0 ? kNoToken : id < 0 || id >= most_adapters ? kNoAdapter : id;
}

// Adapter of token t: one that some tensor has, kNoAdapter, or kNoToken where there is no token.
__device__ __forceinline__ int adapter_of(const int* positions, const int* token_adapters, int t, int n_tokens, int most_adapters)
{
    int position = -1, id = kNoAdapter;
    if (t < n_tokens) {
        position = positions[t];
        if (token_adapters)
            id = token_adapters[t];
    }
    return known_adapter(position, id, most_adapters);
}

// Tokens of a block of up to 64 that use the same adapter, by up to 16 of them: an item.  Items are numbered in the order of their
// first tokens.  Tokens are stored, and what stands behind several blocks' items is read, 16 bytes at a time.
struct alignas(16) Items {
    int ids[64];            // adapter of a token, kNoAdapter, kNoToken
    int adapter[64];        // of an item
    uint8_t tokens[64][16]; // of an item, kNobody behind the last
    int count;
};
static_assert(sizeof(Items) % 16 == 0 && offsetof(Items, tokens) % 16 == 0, "16 bytes at a time");
constexpr uint8_t kNobody = 255;

// By one wavefront, from the first `tokens` of items.ids, which are below `most`; everyone may read the items after the next barrier.
__device__ __forceinline__ void find_items(Items& items, int tokens, int most)
{
    const int lane = threadIdx.x & 63, id = lane < tokens ? items.ids[lane] : kNoToken;
    unsigned long long same = __ballot(id >= 0); // the lanes with this lane's adapter, bit by bit
    for (int bits = most - 1, b = 0; bits >> b; ++b) {
        const unsigned long long set = __ballot((id >> b) & 1);
        same &= (id >> b) & 1 ? set : ~set;
    }
    const int before = __builtin_popcountll(same & ((1ULL << lane) - 1));
    for (int n = before & ~15; n > 0; --n) // what the sixteens in front hold
        same &= same - 1;
    const int lead = __builtin_ctzll(same | 1ULL << 63); // the first of this lane's sixteen
    const unsigned long long leads = __ballot(id >= 0 && lead == lane);
    reinterpret_cast<u32x4*>(items.tokens)[lane] = u32x4{~0u, ~0u, ~0u, ~0u};
    if (id >= 0) {
        const int item = __builtin_popcountll(leads & ((1ULL << lead) - 1));
        items.tokens[item][before & 15] = static_cast<uint8_t>(lane);
        if (lead == lane)
            items.adapter[item] = id;
    }
    if (lane == 0)
        items.count = __builtin_popcountll(leads);
}

__device__ __forceinline__ f4_t mfma16(h8_t a, h8_t b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// A buffer whose reads beyond `bytes` return zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const void* p, size_t bytes)
{
    return make_rsrc(p, bytes > 0x7FFFFFFFu ? 0x7FFFFFFFu : static_cast<uint32_t>(bytes));
}

constexpr int kBehind = static_cast<int>(0x80000000u); // an offset behind the end of every buffer: reads zero, moves nothing

// ---------------------------------------------------------------- inputs of the prompt's products
constexpr int kGroup = 128;       // quantisation group along K
constexpr int kFragBytes = 1024;  // one operand fragment: 64 lanes of 16 bytes
constexpr int kBlockBytes = 8 * kFragBytes; // a token tile times a group

// Fragment order of an activation matrix [m][k]: the lane (k / 64 % 2) * 32 + m % 32 of fragment
// (m / 32, k / 128, k / 8 % 8) holds 8 consecutive k, in the order in which the weights' nibbles come out of
// a word (0 4 1 5 2 6 3 7).  The word of weights that goes with them is word k / 8 of its row, so a lane's 8
// words of a group are 32 contiguous bytes, and every fragment is one fully coalesced load.
__device__ __forceinline__ uint32_t frag_offset(int m, int k, int groups)
{
    return static_cast<uint32_t>(((m >> 5) * groups + (k >> 7)) * 8 + ((k >> 3) & 7)) * kFragBytes +
           ((((k >> 6) & 1) << 5) + (m & 31)) * 16;
}

__device__ __forceinline__ u32x4 frag_order(u32x4 v) // 8 consecutive values -> 0 4 1 5 2 6 3 7
{
    u32x4 o;
    o[0] = (v[0] & 0xFFFFu) | (v[2] << 16);
    o[1] = (v[0] >> 16) | (v[2] & 0xFFFF0000u);
    o[2] = (v[1] & 0xFFFFu) | (v[3] << 16);
    o[3] = (v[1] >> 16) | (v[3] & 0xFFFF0000u);
    return o;
}

// Pair k of the 8 nibbles of a word as fp16 n - z, exact: n sits in the mantissa of 1024 + n (bits 0-3 of a half) or
// 1024 + 16 n (bits 4-7).
__device__ __forceinline__ uint32_t dequant_pair(uint32_t w, int k, h2_t zlo /* 1024 + z */, h2_t zhi /* -(64 + z) */)
{
    const h2_t sixteenth = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
    uint32_t magic = 0x64006400u; // in a vector register: (w & mask) | magic is one instruction then
    asm("" : "+v"(magic));
    const uint32_t v = k >= 2 ? w >> 8 : w;
    return k & 1 ? as_u32(__builtin_elementwise_fma(as_h2((v & 0x00F000F0u) | magic), sixteenth, zhi))
                 : as_u32(as_h2((v & 0x000F000Fu) | magic) - zlo);
}

// Rows into fragment order, zeros behind the end of a row and in rows behind the last: by 512 threads of `worker` of `workers`, a token tile and
// a group at a time.
__device__ __forceinline__ void pack_fragments(uint16_t* xf, const uint16_t* x, int K, int x_stride, int n_tokens, int worker, int workers)
{
    const int groups = (K + kGroup - 1) / kGroup, units = (n_tokens + 31) / 32 * groups;
    if (threadIdx.x >= 512)
        return;
    for (int u = worker; u < units; u += workers) {
        const int m = u / groups * 32 + (threadIdx.x >> 4), k = u % groups * kGroup + (threadIdx.x & 15) * 8;
        u32x4 v = {};
        if (m < n_tokens && k < K)
            v = *reinterpret_cast<const u32x4*>(x + static_cast<size_t>(m) * x_stride + k);
        *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(xf) + frag_offset(m, k, groups)) = frag_order(v);
    }
}

// ---------------------------------------------------------------- adapters beside the prompt's products
// What a product needs of a tensor's adapters.
struct AdapterPart {
    const uint16_t* up; // null: no adapters
    const void* low;
    const TokenAdapter* info;
    long long up_stride;
    int n_adapters, max_rank;
};

__device__ __forceinline__ AdapterPart adapter_part(Constant<ProductTensor>& t)
{
    return AdapterPart{t.up, t.low, t.info, t.up_stride, t.n_adapters, t.max_rank};
}

// The adapter's part of the tokens of an item for RT tiles of 16 outputs from n0 on (of which `rows` exist), by a wavefront: sink(token,
// tile, value) for output lane % 16 of a tile.  t0: first token of the block that the items are of; lds: (RT + 1) / 2 KB of this wavefront's.
// Columns of a matrix product do not mix, so that what one adapter or token holds stays with it.
template <int RT, class Sink>
__device__ __forceinline__ void add_item(const Items& items, int item, const AdapterPart& m, int t0, int n0, int rows, char* lds, Sink sink)
{
    const int lane = threadIdx.x & 63, l15 = lane & 15, c = lane >> 4, id = __builtin_amdgcn_readfirstlane(items.adapter[item]);
    if (!m.up || id >= m.n_adapters)
        return;
    // tokens of the places that this lane's row of inputs, and its four rows of results, stand for
    const int own = items.tokens[item][l15], lead = items.tokens[item][0];
    const size_t blocks = (m.max_rank + 15) / 16, mine = (t0 + (own == kNobody ? lead : own)) * blocks;
    const __amdgpu_buffer_rsrc_t ru =
        rows_buffer(m.up + id * m.up_stride + static_cast<size_t>(n0) * m.max_rank, static_cast<size_t>(rows) * m.max_rank * 2);
    int of[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        of[e] = items.tokens[item][4 * c + e];
    const int rank = __builtin_amdgcn_readfirstlane(m.info[(t0 + lead) * blocks].rank);
    f4_t sum[RT] = {};
    for (int b = 0; b * 16 < rank; ++b) {
        // lane groups 0 and 1: the upper parts of ranks 0 .. 7 and 8 .. 15 of the block; 2 and 3: the lower ones
        const int have = rank - b * 16 - (c & 1) * 8;
        const u32x4 hf = static_cast<const u32x4*>(m.low)[(mine + b) * 4 + c];
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            f[e] = m.info[(t0 + (of[e] == kNobody ? lead : of[e])) * blocks + b].factor;
        u32x4 u[(RT + 1) / 2];
#pragma unroll
        for (int r = 0; r < (RT + 1) / 2; ++r) { // 32 rows of 16 ranks, a row by two lanes
            const int row = r * 32 + (lane >> 1), r8 = b * 16 + (lane & 1) * 8;
            u[r] = __builtin_amdgcn_raw_buffer_load_b128(ru, r8 < rank && row < RT * 16 ? (row * m.max_rank + r8) * 2 : kBehind, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < (RT + 1) / 2; ++r)
            *reinterpret_cast<u32x4*>(lds + r * 1024 + lane * 16) = u[r];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            u32x4 v = *reinterpret_cast<const u32x4*>(lds + (r * 16 + l15) * 32 + (c & 1) * 16);
            if (rank & 7)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    v[k] &= have >= 2 * k + 2 ? ~0u : have == 2 * k + 1 ? 0xFFFFu : 0u;
            const f4_t p = mfma16(__builtin_bit_cast(h8_t, hf), __builtin_bit_cast(h8_t, v), f4_t{});
#pragma unroll
            for (int e = 0; e < 4; ++e)
                sum[r][e] = __builtin_fmaf(p[e], f[e], sum[r][e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (of[e] != kNobody)
#pragma unroll
            for (int r = 0; r < RT; ++r)
                sink(of[e], r, sum[r][e]);
}

} // namespace l2
