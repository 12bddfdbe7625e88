// Products of the rows of many tokens with int4 tensors, low-rank adapters of the tokens' requests beside them, and the first
// half of the gated feed-forward block.
//
//   y[t][n] = sum_g s[n][g] sum_{k in g} x[t][k] (w[n][k] - z[n][g])  +  f_a sum_r up_a[n][r] h[t][r],   h[t][r] = sum_k down_a[r][k] x[t][k]
//
// w - z is an exact fp16 integer, its products with x are summed in fp32 over a group of 128 and scaled in fp32.  h is summed in
// fp32; in the tiles here it meets the adapter's halfs in fp32 too, for the prompt's kernels it leaves as two fp16 numbers and a power of two (22
// bits of the token's largest of 16), which the matrix cores take as 16 ranks a product.
#include "batch_product.hpp"
#include "prefill.hpp"

#include <cmath>

namespace l2 {

// Arguments lie in memory, and a kernel that asks for them one after the other waits for each: a tensor's are neighbours, chosen by
// an index that the first cache line holds.
struct alignas(64) LowTensor {
    const uint16_t* down; // null: no adapters
    const float* scales;
    const int* ranks;
    void* low;          // [n_tokens][blocks] of 64 bytes: what the ranks received, 16 floats or the upper and lower parts of 16 numbers
    TokenAdapter* info; // [n_tokens][blocks]
    long long down_stride;
    int n_adapters, max_rank;
};

struct alignas(64) LowArgs {
    const uint16_t* x;
    const int* positions;
    const int* token_adapters;
    int K, x_stride, n_tokens, most_adapters;
    uint16_t* packed; // non-null: the rows as operands, by the workgroups behind those of the tensors
    int n_matrices;
    LowTensor t[LLAMA2_MAX_BATCH_MATRICES];
};

// 16 rows of 128 halfs, requested in the order of memory (a compute unit looks up 64 bytes at a time, and only neighbouring lanes share a
// lookup: lanes that read 16 bytes of a row each, as the matrix cores want them, cost four times as many) and turned around through
// LDS that belongs to the wavefront.  Load i: rows 4 i + lane / 16, elements 8 (lane % 16) on.
struct HalfTile {
    u32x4 v[4];
};

// Lane's place in a row of the tile, or kBehind where the row of n elements has ended; k0: first element of the tile.
__device__ __forceinline__ int tile_column(int k0, int n)
{
    const int k = k0 + 8 * (threadIdx.x & 15);
    return k < n ? 2 * k : kBehind;
}

constexpr int kTileBytes = 16 * 256;

template <bool NIBBLES> // eight elements in the order in which nibbles come out of a word
__device__ __forceinline__ void put_tile(char* lds, const HalfTile& t)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 4 * i + (lane >> 4);
        *reinterpret_cast<u32x4*>(lds + row * 256 + ((lane & 15) ^ row) * 16) = NIBBLES ? frag_order(t.v[i]) : t.v[i];
    }
}

// Operand m of four: lane group c holds elements 32 c + 8 m on of row lane % 16.
__device__ __forceinline__ h8_t tile_operand(const char* lds, int m)
{
    const int row = threadIdx.x & 15, c = (threadIdx.x & 63) >> 4;
    return *reinterpret_cast<const h8_t*>(lds + row * 256 + ((4 * c + m) ^ row) * 16);
}

// ---------------------------------------------------------------- rows as operands
// 16 tokens and a group of 128 inputs are the four operands of 16 x 16 x 32 products, 1 KB each: lane group c of operand m holds elements
// 32 c + 8 m on of token lane % 16, in the order of a word's nibbles, zeros behind the end of a row.  Tokens behind the last one repeat it.
// `worker` of `workers` takes pairs of such tiles with 512 threads.
__device__ __forceinline__ void pack_rows(uint16_t* packed, const uint16_t* x, int K, int x_stride, int n_tokens, int worker, int workers)
{
    const int groups = (K + 127) / 128, units = (n_tokens + 15) / 16 * groups, lane = threadIdx.x & 63, part = threadIdx.x >> 6;
    for (int u = worker * 2 + (part >> 2); u < units; u += workers * 2) {
        const int tile = u / groups, g = u % groups, m = part & 3;
        const int token = min(tile * 16 + (lane & 15), n_tokens - 1), k = g * 128 + 32 * (lane >> 4) + 8 * m;
        u32x4 v = {};
        if (k < K)
            v = *reinterpret_cast<const u32x4*>(x + static_cast<size_t>(token) * x_stride + k);
        reinterpret_cast<u32x4*>(packed)[(static_cast<size_t>(u) * 4 + m) * 64 + lane] = frag_order(v);
    }
}

__global__ __launch_bounds__(512) void batch_pack_kernel(uint16_t* packed, const uint16_t* x, int K, int x_stride, int n_tokens)
{
    pack_rows(packed, x, K, x_stride, n_tokens, blockIdx.x, gridDim.x);
}

// ---------------------------------------------------------------- what the ranks receive
// Block `to` of 16 ranks, one in each of 16 lanes, as two fp16 numbers and a power of two, which the matrix cores take.
__device__ __forceinline__ void put_parts(void* lows, TokenAdapter* info, size_t to, float v, float scale, int rank, bool write)
{
    const int l15 = threadIdx.x & 15;
    const float most = row16_max(fabsf(v));
    // the largest between 2^14 and 2^15; nothing to scale where all are 0 or one is infinite
    const int e2 = most > 0.0f && most < INFINITY ? 14 - ilogbf(most) : 0;
    const float scaled = ldexpf(v, e2);
    const uint16_t h = float_to_half_bits(scaled);
    if (!write)
        return;
    uint16_t* const low = static_cast<uint16_t*>(lows);
    low[to * 32 + l15] = h;
    low[to * 32 + 16 + l15] = float_to_half_bits(scaled - half_bits_to_float(h));
    if (l15 == 0)
        info[to] = TokenAdapter{ldexpf(scale, -e2), rank};
}

// Few tokens: a wavefront takes a rank of a token's adapter, whose row of the adapter it sums up with the token's inputs in fp32; tokens that
// share an adapter find it in the caches.  A chain of loads bounds it, so nothing waits but the adapter's number for the arguments and its row
// for the number: ranks and scales of small pools and the inputs are requested together with the number.  4096 inputs, one token, 16 ranks 2.7 us;
// 5120 inputs, 64 tokens with an adapter each through two tensors 6.0 (taken in items, as below, 6.6 and 11.9).
// WIDE: as the prompt's products take them, a block of 16 ranks per workgroup.
constexpr int kRankLoads = 4; // at a time, which leaves room for 32 wavefronts on a CU (8: 1 .. 2 % longer steps)
constexpr int rank_waves(bool wide) { return wide ? 16 : 8; }

template <bool WIDE>
__global__ __launch_bounds__(rank_waves(WIDE) * 64) void batch_ranks_kernel(LowArgs)
{
    __shared__ float received[rank_waves(WIDE)];
    auto& a = kernel_args<LowArgs>();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), token = blockIdx.x;
    const int K = a.K, x_stride = a.x_stride, n_tokens = a.n_tokens, most_adapters = a.most_adapters;
    const uint16_t* const x = a.x;
    const int *const positions = a.positions, *const token_adapters = a.token_adapters;
    if (static_cast<int>(blockIdx.z) == a.n_matrices) {
        const int worker = blockIdx.y * gridDim.x + blockIdx.x, workers = gridDim.x * gridDim.y;
        if constexpr (WIDE)
            pack_fragments(a.packed, x, K, x_stride, n_tokens, worker, workers);
        else
            pack_rows(a.packed, x, K, x_stride, n_tokens, worker, workers);
        return;
    }
    auto& t = a.t[blockIdx.z];
    const uint16_t* const down = t.down;
    const float* const scales = t.scales;
    const int* const ranks = t.ranks;
    void* const low = t.low;
    TokenAdapter* const info = t.info;
    const long long down_stride = t.down_stride;
    const int n_adapters = t.n_adapters, max_rank = t.max_rank;
    loaded(K, x_stride, n_tokens, most_adapters, x, positions, token_adapters, down, scales, ranks, low, info, down_stride, n_adapters, max_rank);
    const int r = blockIdx.y * rank_waves(WIDE) + wave;
    if (!down || r >= (max_rank + 15) / 16 * 16)
        return;
    const int position = positions[token], given = token_adapters[token];
    int rank_table = 0;
    float scale_table = 0.0f;
    if (lane < n_adapters) {
        rank_table = ranks[lane];
        scale_table = scales[lane];
    }
    const __amdgpu_buffer_rsrc_t rx = rows_buffer(x + static_cast<size_t>(token) * x_stride, static_cast<size_t>(K) * 2);
    u32x4 xv[kRankLoads], dv[kRankLoads];
    auto request = [&](u32x4(&v)[kRankLoads], const __amdgpu_buffer_rsrc_t& row, int k0) { // elements behind the end are zero
#pragma unroll
        for (int i = 0; i < kRankLoads; ++i)
            v[i] = __builtin_amdgcn_raw_buffer_load_b128(row, k0 * 2 + i * 1024 + lane * 16, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    request(xv, rx, 0);
    const int id = __builtin_amdgcn_readfirstlane(known_adapter(position, given, most_adapters));
    if (id < 0 || id >= n_adapters)
        return;
    const int rank = min(max(id < 64 ? __builtin_amdgcn_readlane(rank_table, id) : ranks[id], 0), max_rank);
    const float scale = id < 64 ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale_table), id)) : scales[id];
    float sum = 0.0f;
    if (r < rank) {
        const __amdgpu_buffer_rsrc_t rd = rows_buffer(down + id * down_stride + static_cast<size_t>(r) * K, static_cast<size_t>(K) * 2);
        for (int k0 = 0; k0 < K; k0 += kRankLoads * 512) {
            if (k0 > 0)
                request(xv, rx, k0);
            request(dv, rd, k0);
#pragma unroll
            for (int i = 0; i < kRankLoads; ++i)
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    sum = __builtin_fmaf(half_bits_to_float(static_cast<uint16_t>(dv[i][k >> 1] >> (16 * (k & 1)))),
                                         half_bits_to_float(static_cast<uint16_t>(xv[i][k >> 1] >> (16 * (k & 1)))), sum);
        }
        sum = wave_sum(sum);
    }
    const size_t to = static_cast<size_t>(token) * ((max_rank + 15) / 16) + r / 16;
    if constexpr (WIDE) {
        if (lane == 0)
            received[wave] = sum;
        __syncthreads();
        if (wave == 0)
            put_parts(low, info, to, received[lane & 15], scale, rank, lane < 16);
    } else {
        if (lane == 0 && r < (rank + 15) / 16 * 16)
            static_cast<float*>(low)[to * 16 + r % 16] = sum * scale;
        if (lane == 0 && r % 16 == 0)
            info[to] = TokenAdapter{scale, rank};
    }
}

// Many tokens, for whom adapters would be looked up too often that way: a workgroup takes items of a block of 64 tokens, so that an adapter is
// read once for up to 16 tokens that use it, and ranks by 16; its wavefronts split the inputs.  Ranks and scales of small pools are
// requested together with the tokens' adapters.  1100 tokens of 4096 inputs through three tensors of 64 ranks 19.6 us: look-ups of the adapters and
// their turn through LDS, 5 us each, behind the chain of tokens, items and rows.
// CHUNKS of 128 inputs that a wavefront has requested; KEEP: they are all that there are, and the inputs stay for all ranks.
constexpr int kLowWaves = 8, kLowTable = kLowWaves * 64;

template <int CHUNKS, bool KEEP>
__global__ __launch_bounds__(kLowWaves * 64) void batch_low_kernel(LowArgs)
{
    constexpr int kStride = 16 + 4;
    __shared__ Items items;
    __shared__ int table[kLowTable];
    __shared__ float scale_table[kLowTable];
    __shared__ __align__(16) char tiles[kLowWaves * kTileBytes];
    __shared__ __align__(16) float red[kLowWaves * 16 * kStride];
    auto& a = kernel_args<LowArgs>();
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, c = lane >> 4;
    const int t0 = blockIdx.x * 64, K = a.K, x_stride = a.x_stride, n_tokens = a.n_tokens, most_adapters = a.most_adapters;
    const uint16_t* const x = a.x;
    const int *const positions = a.positions, *const token_adapters = a.token_adapters;
    if (static_cast<int>(blockIdx.z) == a.n_matrices) {
        pack_fragments(a.packed, x, K, x_stride, n_tokens, blockIdx.y * gridDim.x + blockIdx.x, gridDim.x * gridDim.y);
        return;
    }
    auto& t = a.t[blockIdx.z];
    const uint16_t* const down = t.down;
    const float* const scales = t.scales;
    const int* const ranks = t.ranks;
    void* const lows = t.low;
    TokenAdapter* const info = t.info;
    const long long down_stride = t.down_stride;
    const int n_adapters = t.n_adapters, max_rank = t.max_rank;
    loaded(K, x_stride, n_tokens, most_adapters, x, positions, token_adapters, down, scales, ranks, lows, info, down_stride, n_adapters, max_rank);
    if (!down)
        return;
    int mine = 0;
    float mine_scale = 0.0f;
    if (tid < n_adapters) {
        mine = ranks[tid];
        mine_scale = scales[tid];
    }
    if (wave == 0) {
        items.ids[lane] = adapter_of(positions, token_adapters, t0 + lane, n_tokens, most_adapters);
        find_items(items, min(64, n_tokens - t0), most_adapters);
    }
    table[tid] = mine;
    scale_table[tid] = mine_scale;
    __syncthreads();
    const __amdgpu_buffer_rsrc_t rx = rows_buffer(x + static_cast<size_t>(t0) * x_stride,
                                                  (static_cast<size_t>(min(64, n_tokens - t0) - 1) * x_stride + K) * 2);
    char* const lds = tiles + wave * kTileBytes;
    for (int item = blockIdx.y; item < items.count; item += gridDim.y) {
        const int id = __builtin_amdgcn_readfirstlane(items.adapter[item]);
        if (id >= n_adapters)
            continue;
        const int rank = min(max(__builtin_amdgcn_readfirstlane(id < kLowTable ? table[id] : ranks[id]), 0), max_rank);
        const float scale = id < kLowTable ? scale_table[id] : scales[id];
        const __amdgpu_buffer_rsrc_t rd = rows_buffer(down + id * down_stride, static_cast<size_t>(rank) * K * 2); // ranks beyond are zero
        int xoff[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int own = items.tokens[item][4 * i + c];
            xoff[i] = own == kNobody ? kBehind : own * x_stride * 2;
        }
        HalfTile xt[CHUNKS], dt[CHUNKS];
        h8_t xf[KEEP ? CHUNKS : 1][4];
        auto chunk = [&](int q) { return (wave + q * kLowWaves) * 128; };
        auto request_x = [&](int q, int k0) {
            const int column = tile_column(k0, K);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                xt[q].v[i] = __builtin_amdgcn_raw_buffer_load_b128(rx, column < 0 || xoff[i] < 0 ? kBehind : xoff[i] + column, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        };
        auto request_d = [&](int q, int k0, int block) { // blocks behind the rank lie behind the end
            const int column = tile_column(k0, K);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                dt[q].v[i] = __builtin_amdgcn_raw_buffer_load_b128(rd, column < 0 ? kBehind : (block * 16 + 4 * i + c) * K * 2 + column, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int q = 0; q < CHUNKS; ++q) {
            request_x(q, chunk(q));
            request_d(q, chunk(q), 0);
        }
        if constexpr (KEEP) {
#pragma unroll
            for (int q = 0; q < CHUNKS; ++q) {
                put_tile<false>(lds, xt[q]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    xf[q][j] = tile_operand(lds, j);
            }
        }
        for (int block = 0; block == 0 || block * 16 < rank; ++block) { // the first one says that there are no ranks at all
            f4_t acc = {};
            for (int k0 = wave * 128; k0 < K; k0 += CHUNKS * kLowWaves * 128) {
#pragma unroll
                for (int q = 0; q < CHUNKS; ++q) { // behind the last elements both are zero
                    const int next = k0 + (q + CHUNKS) * kLowWaves * 128;
                    const bool on = next - q * kLowWaves * 128 < K; // else the next block from the front
                    h8_t df[4];
                    if constexpr (!KEEP) {
                        put_tile<false>(lds, xt[q]);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            xf[0][j] = tile_operand(lds, j);
                        request_x(q, on ? next : chunk(q));
                    }
                    put_tile<false>(lds, dt[q]);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        df[j] = tile_operand(lds, j);
                    request_d(q, on ? next : chunk(q), on ? block : block + 1);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc = mfma16(xf[KEEP ? q : 0][j], df[j], acc);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                red[(wave * 16 + 4 * c + e) * kStride + l15] = acc[e];
            __syncthreads();
            if (wave < 4) { // 16 lanes a token, a rank each
                const int place = tid >> 4, m = items.tokens[item][place];
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < kLowWaves; ++w)
                    v += red[(w * 16 + place) * kStride + l15];
                v = block * 16 + l15 < rank ? v : 0.0f;
                const size_t to = static_cast<size_t>(t0 + (m == kNobody ? 0 : m)) * ((max_rank + 15) / 16) + block;
                put_parts(lows, info, to, v, scale, rank, m != kNobody);
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------- the products
// 16 rows of the 16 words of a group, requested in the order of memory (row lane / 4, words 4 (lane % 4) on) and turned around through
// LDS: afterwards lane group c holds words 4 c .. 4 c + 3 of row lane % 16, which go with operand m of a tile of inputs word by word.
__device__ __forceinline__ u32x4 turned_words(char* lds, u32x4 v)
{
    const int lane = threadIdx.x & 63, row = lane & 15, c = lane >> 4;
    *reinterpret_cast<u32x4*>(lds + (lane >> 2) * 64 + ((lane & 3) ^ (lane >> 4)) * 16) = v;
    return *reinterpret_cast<const u32x4*>(lds + row * 64 + (c ^ (row >> 2)) * 16);
}

// 16 bytes that are aligned as halfs, or as words
struct __attribute__((packed, aligned(2))) AnyHalfs {
    u32x4 v;
};
struct __attribute__((packed, aligned(4))) AnyWords {
    u32x4 v;
};

constexpr int kScaleBytes = 20480; // of LDS for the scales and zero points of a workgroup's rows

// A workgroup takes R tiles of 16 outputs (GATED: half of them of the gate, half of the up projection) and T tiles of 16
// tokens; its W wavefronts take the groups of 128 inputs in turn, D of them requested ahead, and add up through LDS.  Every weight is read
// once and unpacked once for all tokens of a tile.
//
// What bounds it: a group's inputs are T / R * 4 times the bytes of its weights, and a CU looks up 64 bytes per cycle, so higher tiles read
// less and leave CUs without a workgroup; in front and behind stand the arguments, the adapters' chain of loads, scales through LDS and the sums, about
// 5 us.  48 tokens, 12288 columns of 4096 inputs with adapters 18.6 us (2.4 TB/s of weights and adapters), 64 tokens, gated 2 * 13824
// columns of 5120 with an adapter each 50 (35 without: 432 workgroups are two rounds), 24 tokens, 5120 columns of 13824 20.5.  K cut
// over several workgroups won 7 % on long rows and is not here.
template <int W, int R, int T, int D, bool GATED, bool ADAPTERS>
__global__ __launch_bounds__(W * 64, 2) void batch_product_kernel(ProductArgs)
{
    constexpr int kTokens = T * 16, kRows = R * 16, kStride = kRows + 4, kTensors = GATED ? 2 : 1, RT = R / kTensors;
    constexpr int kRing = T * D <= 4 && !(R == 4 && T == 4) ? T * D : 2; // tiles of tokens whose inputs are on their way or in use
    static_assert(T * D % kRing == 0 && kRing <= T * D, "a tile has one place in the ring");
    constexpr bool PACKED = T > 2; // the inputs come as operands; of few tokens in rows, which saves the launch that packs them
    constexpr int kWaveBytes = (PACKED ? 0 : kTileBytes) + R * 1024, kWordsAt = kWaveBytes - R * 1024;
    constexpr int kSums = W * kTokens * kStride * 4, kExtraAt = W * kWaveBytes + kScaleBytes, kFront = kExtraAt + (ADAPTERS ? kTokens * kStride * 4 : 0);
    __shared__ __align__(16) char pool[kFront > kSums ? kFront : kSums]; // the sums come where tiles, scales and the adapters' part were
    __shared__ int live[kTokens];
    auto& a = kernel_args<ProductArgs>();
    auto& t = a.t[GATED ? 0 : blockIdx.y];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, c = lane >> 4;
    const int K = a.K, x_stride = a.x_stride, n_tokens = a.n_tokens, most_adapters = a.most_adapters, token_blocks = a.token_blocks;
    const uint16_t* const x = a.x;
    const int *const positions = a.positions, *const token_adapters = a.token_adapters;
    struct Tensor : AdapterPart {
        const uint32_t* w;
        const uint32_t* z;
        const uint16_t* s;
    } m[kTensors];
    m[0] = {adapter_part(t), t.w, t.z, t.s};
    if constexpr (GATED)
        m[1] = {adapter_part(a.t[1]), a.t[1].w, a.t[1].z, a.t[1].s};
    const int cols = t.cols, out_stride = t.out_stride, residual_stride = t.residual_stride;
    uint16_t* const out = t.out;
    const uint16_t* const residual_rows = t.residual;
    loaded(K, x_stride, n_tokens, most_adapters, token_blocks, x, positions, token_adapters, m[0].w, m[0].z, m[0].s, m[kTensors - 1].w,
           m[kTensors - 1].z, m[kTensors - 1].s, cols, out_stride, residual_stride, out, residual_rows);
    if (ADAPTERS)
        loaded(m[0].up, m[0].low, m[0].info, m[0].up_stride, m[0].n_adapters, m[0].max_rank, m[kTensors - 1].up, m[kTensors - 1].low,
               m[kTensors - 1].info, m[kTensors - 1].up_stride, m[kTensors - 1].n_adapters, m[kTensors - 1].max_rank);
    // the token blocks of one block of rows follow each other on one XCD
    const int slot = blockIdx.x >> 3, rb = slot / token_blocks * 8 + (blockIdx.x & 7), t0 = slot % token_blocks * kTokens, n0 = rb * RT * 16;
    if (n0 >= cols)
        return;
    const int ws = (K + 31) / 32 * 4, groups = (K + 127) / 128, zs = (groups + 7) / 8;

    // The threads of a token, its adapter and that one's ranks: asked for first, since more hangs on them.
    constexpr int kThreads = (W < 8 ? W : 8) * 64 / kTokens; // the other wavefronts take none
    const int my_token = tid / kThreads, token_at = t0 + my_token;
    int position = -1, adapter = kNoAdapter, rank[kTensors] = {};
    if (my_token < kTokens && token_at < n_tokens) {
        position = positions[token_at];
        if (token_adapters)
            adapter = token_adapters[token_at];
        if constexpr (ADAPTERS)
#pragma unroll
            for (int h = 0; h < kTensors; ++h)
                if (m[h].up)
                    rank[h] = m[h].info[static_cast<size_t>(token_at) * ((m[h].max_rank + 15) / 16)].rank; // of no adapter: not used
    }

    // Rows and tokens that do not exist lie behind the ends of the buffers.
    const int rows = min(RT * 16, cols - n0), here = min(kTokens, n_tokens - t0);
    __amdgpu_buffer_rsrc_t rw[kTensors];
#pragma unroll
    for (int h = 0; h < kTensors; ++h)
        rw[h] = rows_buffer(m[h].w + static_cast<size_t>(n0) * ws, static_cast<size_t>(rows) * ws * 4);
    const int tiles = (here + 15) / 16;
    const __amdgpu_buffer_rsrc_t rx = PACKED ? rows_buffer(x + static_cast<size_t>(t0) * groups * 128, static_cast<size_t>(tiles) * groups * 4096)
                                             : rows_buffer(x + static_cast<size_t>(t0) * x_stride, (static_cast<size_t>(here - 1) * x_stride + K) * 2);
    const int woff = (lane >> 2) * ws * 4 + 16 * (lane & 3), xoff = c * x_stride * 2;

    // A group's weights and inputs.  A group that does not exist is requested behind the ends too: loads that come and go would make
    // every wait one for all of them.
    u32x4 raw[D][R];
    HalfTile xt[kRing];
    auto load_w = [&](int d, int g) {
        const int k = g < groups ? 64 * g : kBehind;
#pragma unroll
        for (int r = 0; r < R; ++r)
            raw[d][r] = __builtin_amdgcn_raw_buffer_load_b128(rw[r / RT], woff + (r % RT) * ws * 64 + k, 0, 0);
        __builtin_amdgcn_sched_barrier(0); // loads keep one order from the first group on: waits count them
    };
    auto load_x = [&](int q, int i, int g) { // tile i into place q
        if constexpr (PACKED) {
            const int at = g < groups ? (i * groups + g) * 4096 + lane * 16 : kBehind;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                xt[q].v[e] = __builtin_amdgcn_raw_buffer_load_b128(rx, at + e * 1024, 0, 0);
        } else {
            const int column = tile_column(128 * g, K), at = column < 0 ? kBehind : column + xoff;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                xt[q].v[e] = __builtin_amdgcn_raw_buffer_load_b128(rx, at + (i * 16 + 4 * e) * x_stride * 2, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int d = 0; d < D; ++d) {
        load_w(d, wave + d * W);
#pragma unroll
        for (int i = 0; i < T; ++i)
            if (d * T + i < kRing)
                load_x(d * T + i, i, wave + d * W);
    }
    // Scales and zero points of all rows: they are neighbours in memory, and multiples of 8.
    char* const lds = pool + wave * kWaveBytes; // of this wavefront
    uint16_t* const scales = reinterpret_cast<uint16_t*>(pool + W * kWaveBytes);
    uint32_t* const zeros = reinterpret_cast<uint32_t*>(scales + kRows * groups);
#pragma unroll
    for (int h = 0; h < kTensors; ++h) {
        const AnyHalfs* const s = reinterpret_cast<const AnyHalfs*>(m[h].s + static_cast<size_t>(n0) * groups);
        const AnyWords* const z = reinterpret_cast<const AnyWords*>(m[h].z + static_cast<size_t>(n0) * zs);
        const int ns = rows * groups / 8, nz = rows * zs / 4;
        for (int i = tid; i < ns + nz; i += W * 64)
            if (i < ns)
                reinterpret_cast<u32x4*>(scales + h * RT * 16 * groups)[i] = s[i].v;
            else
                reinterpret_cast<u32x4*>(zeros + h * RT * 16 * zs)[i - ns] = z[i - ns].v;
    }
    const int id = known_adapter(position, adapter, most_adapters);
    if (tid % kThreads == 0 && my_token < kTokens)
        live[my_token] = id != kNoToken;
    f4_t acc[T][R] = {};
    if constexpr (ADAPTERS) {
        // The adapters' part, into the first wavefront's sums.  A thread takes every so many outputs of one token: with few tokens of an
        // adapter the matrix cores would compute 16 for one.
        float* const extra = reinterpret_cast<float*>(pool + kExtraAt);
        constexpr int kOwn = kRows > kThreads ? kRows / kThreads : 1, kPer = kOwn / kTensors ? kOwn / kTensors : 1;
        constexpr int kBoth = kOwn < kTensors ? 1 : kTensors; // tensors of a thread's outputs; a token may have as many threads as outputs
        static_assert(kOwn * kThreads >= kRows, "all outputs of a token");
        const int mine = tid % kThreads;
        AdapterPart part[kBoth];
        int ranks[kBoth], first[kBoth], column[kBoth], most = 0; // rows first + i * kThreads of a tensor
#pragma unroll
        for (int h = 0; h < kBoth; ++h) {
            const int of = kBoth < kTensors ? min(mine / (RT * 16), kTensors - 1) : h;
            first[h] = kBoth < kTensors ? mine - of * RT * 16 : mine;
            column[h] = of * RT * 16 + first[h];
            part[h] = of == 0 ? AdapterPart(m[0]) : AdapterPart(m[kTensors - 1]);
            ranks[h] = id >= 0 && id < part[h].n_adapters && first[h] < RT * 16 ? (of == 0 ? rank[0] : rank[kTensors - 1]) : 0;
            most = max(most, ranks[h]);
        }
        float sum[kBoth][kPer] = {};
        for (int r0 = 0; r0 < most; r0 += 16) {
            f4_t x[kBoth][4] = {};
            u32x4 u[kBoth][kPer][2] = {};
#pragma unroll
            for (int h = 0; h < kBoth; ++h) {
                const uint16_t* const up = part[h].up + id * part[h].up_stride + static_cast<size_t>(n0 + first[h]) * part[h].max_rank + r0;
                const f4_t* const low = static_cast<const f4_t*>(part[h].low) + (static_cast<size_t>(token_at) * ((part[h].max_rank + 15) / 16) * 16 + r0) / 4;
                if (r0 < ranks[h])
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        x[h][k] = low[k]; // zeros behind the rank
#pragma unroll
                for (int i = 0; i < kPer; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (first[h] + i * kThreads < rows && r0 + 8 * k < ranks[h])
                            u[h][i][k] = *reinterpret_cast<const u32x4*>(up + static_cast<size_t>(i) * kThreads * part[h].max_rank + 8 * k);
            }
#pragma unroll
            for (int h = 0; h < kBoth; ++h) {
                if (ranks[h] - r0 < 16 && (ranks[h] & 7))
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int have = ranks[h] - r0 - 2 * k;
                        const uint32_t mask = have >= 2 ? ~0u : have == 1 ? 0xFFFFu : 0u;
#pragma unroll
                        for (int i = 0; i < kPer; ++i)
                            u[h][i][k >> 2][k & 3] &= mask;
                    }
#pragma unroll
                for (int i = 0; i < kPer; ++i)
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        sum[h][i] = __builtin_fmaf(half_bits_to_float(static_cast<uint16_t>(u[h][i][k >> 3][(k & 7) >> 1] >> (16 * (k & 1)))),
                                                   x[h][k >> 2][k & 3], sum[h][i]);
            }
        }
#pragma unroll
        for (int h = 0; h < kBoth; ++h)
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (my_token < kTokens && first[h] + i * kThreads < RT * 16)
                    extra[my_token * kStride + column[h] + i * kThreads] = sum[h][i];
        __syncthreads();
        if (wave == 0)
#pragma unroll
            for (int i = 0; i < T; ++i)
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[i][r][e] = extra[(i * 16 + 4 * c + e) * kStride + r * 16 + l15];
    } else {
        __syncthreads();
    }

    for (int g0 = wave; g0 < groups; g0 += W * D) {
#pragma unroll
        for (int d = 0; d < D; ++d) { // groups that do not exist are zeros
            const int g = g0 + d * W, gs = min(g, groups - 1);
            h8_t wf[R][4];
            float sc[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const u32x4 v = turned_words(lds + kWordsAt + r * 1024, raw[d][r]);
                const int row = r * 16 + l15;
                const float zero = static_cast<float>(zeros[row * zs + (gs >> 3)] >> (4 * (gs & 7)) & 15u);
                const _Float16 lo = static_cast<_Float16>(1024.0f + zero), hi = static_cast<_Float16>(-64.0f - zero);
                const h2_t zlo = {lo, lo}, zhi = {hi, hi};
                sc[r] = half_bits_to_float(scales[row * groups + gs]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    wf[r][j] = __builtin_bit_cast(h8_t, u32x4{dequant_pair(v[j], 0, zlo, zhi), dequant_pair(v[j], 1, zlo, zhi),
                                                               dequant_pair(v[j], 2, zlo, zhi), dequant_pair(v[j], 3, zlo, zhi)});
            }
            __builtin_amdgcn_sched_barrier(0);
            load_w(d, g + W * D);
#pragma unroll
            for (int i = 0; i < T; ++i) {
                const int q = (d * T + i) % kRing, next = d * T + i + kRing; // the tile that comes into this place
                h8_t xf[4];
                if constexpr (PACKED) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        xf[j] = __builtin_bit_cast(h8_t, xt[q].v[j]);
                } else {
                    put_tile<true>(lds, xt[q]);
                    __builtin_amdgcn_sched_barrier(0);
                    load_x(q, next % T, g0 + next / T * W);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        xf[j] = tile_operand(lds, j);
                }
                f4_t p[R] = {};
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        p[r] = mfma16(xf[j], wf[r][j], p[r]);
                if constexpr (PACKED) {
                    __builtin_amdgcn_sched_barrier(0);
                    load_x(q, next % T, g0 + next / T * W);
                }
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[i][r][e] = __builtin_fmaf(p[r][e], sc[r], acc[i][r][e]);
            }
        }
    }
    __syncthreads(); // everyone is through with tiles and scales
    float* const red = reinterpret_cast<float*>(pool);
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                red[(wave * kTokens + i * 16 + 4 * c + e) * kStride + r * 16 + l15] = acc[i][r][e];
    __syncthreads();
    constexpr int kPieces = RT * 2; // of 8 outputs
    for (int i = tid; i < kTokens * kPieces; i += W * 64) {
        const int token = i / kPieces, piece = i % kPieces * 8, n = n0 + piece;
        if (!live[token] || n >= cols)
            continue;
        u32x4 residual = {};
        if (!GATED && residual_rows)
            residual = *reinterpret_cast<const u32x4*>(residual_rows + static_cast<size_t>(t0 + token) * residual_stride + n);
        float v[kTensors][8] = {};
#pragma unroll
        for (int h = 0; h < kTensors; ++h)
#pragma unroll
            for (int q = 0; q < W; ++q)
#pragma unroll
                for (int k = 0; k < 8; k += 4) {
                    const f4_t y = *reinterpret_cast<const f4_t*>(red + (q * kTokens + token) * kStride + h * RT * 16 + piece + k);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[h][k + e] += y[e];
                }
        u32x4 o;
        if constexpr (GATED) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[0][k] = v[0][k] / (1.0f + expf(-v[0][k])) * v[1][k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[0][k] += half_bits_to_float(static_cast<uint16_t>(residual[k >> 1] >> (16 * (k & 1))));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            o[k] = static_cast<uint32_t>(float_to_half_bits(v[0][2 * k])) | static_cast<uint32_t>(float_to_half_bits(v[0][2 * k + 1])) << 16;
        *reinterpret_cast<u32x4*>(out + static_cast<size_t>(t0 + token) * out_stride + n) = o;
    }
}

// ---------------------------------------------------------------- host side
struct Product { // a call of either entry point
    ProductArgs a;
    LowArgs low;
    int n_matrices;
    bool adapters;
};

template <int W, int R, int T, int D, bool GATED>
static void launch_product(Product& p)
{
    ProductArgs& a = p.a;
    int cols = 0;
    for (int i = 0; i < p.n_matrices; ++i)
        cols = a.t[i].cols > cols ? a.t[i].cols : cols;
    a.token_blocks = ceil_div(a.n_tokens, T * 16);
    const dim3 grid(static_cast<unsigned>(round_up(ceil_div(cols, GATED ? R * 8 : R * 16), 8)) * a.token_blocks, GATED ? 1 : p.n_matrices), block(W * 64);
    if (p.adapters)
        hipLaunchKernelGGL((batch_product_kernel<W, R, T, D, GATED, true>), grid, block, 0, ctx().stream, a);
    else
        hipLaunchKernelGGL((batch_product_kernel<W, R, T, D, GATED, false>), grid, block, 0, ctx().stream, a);
}

constexpr int kMostTokens = 4096; // of a launch
constexpr int kMostGroups = 256; // of rows whose inputs are packed; of more one tile of outputs has room for its scales

// Tiles by how many columns all tensors of a call have beside the CUs: as few workgroups as have something for every CU, since every one
// reads the inputs of its tokens, and as many wavefronts in them as the CU has room for.  Measured in us with 256 CUs (W wavefronts, R
// tiles of outputs; 4096 inputs and no adapters where nothing else is said):
//   tokens  columns          chosen          others
//   4       4096             W 8, R 1  5.7   W 12, R 2 6.6;  W 4, R 2  7.5
//   4       5120 of 13824    W 12, R 2 14.2  W 8, R 1 16.9;  W 4, R 2 18.9
//   16      12288            W 4, R 2 10.4   W 8, R 1 12.2;  W 4, R 2 with two groups requested ahead (D 2) 10.8
//   16      32000            W 4, R 4 16.8   W 4, R 2 17.5;  W 8, R 1 25.4
//   8       gated 2 * 11008  W 4, R 2 15.6   D 2 16.0;  W 8, R 2 17.0;  W 4, R 4 16.4
//   8       gated 2 * 13824 of 5120   W 4, R 4 20.0   W 4, R 2 22.1
//   32      4096             W 8, R 1  7.3   W 12, R 2 8.3;  W 8, R 4 11.7
//   32      6144             W 12, R 2 9.1   W 8, R 1 11.1;  W 8, R 4 12.2
//   32      12288            W 8, R 4 13.5   W 4, R 4 14.8;  W 8, R 1 15.6
//   32      gated 2 * 11008, an adapter each   W 4, R 4 28.0   W 8, R 4 32.6;  W 4, R 2 30.1
//   64      4096             two blocks of 32 tokens, W 12, R 2 8.5   one of 64, W 8, R 2 12.6;  R 4 15.5
//   64      6144             W 8, R 2 12.8   R 4 15.4;  two blocks 16.1
//   64      12288            W 8, R 4 17.0   R 2 20.7;  two blocks (48 tokens) 22.7
// Inputs that come as operands (a launch more, or workgroups of the adapters' first kernel) pay off in blocks of 64 tokens (48 tokens of 12288
// columns with adapters 23.8 against 27.2 with inputs in rows), not below (32 tokens of 4096 columns 8.3 against 7.3).
// Scales and zero points of a workgroup's rows fit up to R * groups = 512.
constexpr int kFewColumns = 16; // of a CU

template <bool GATED>
static void launch_shape(Product& p, bool packed, int per_cu, int groups)
{
    const int n = p.a.n_tokens;
    const bool high = groups <= kMostGroups / 2;
    if (packed)
        return per_cu > 24 && high ? launch_product<8, 4, 4, 1, GATED>(p) : launch_product<8, 2, 4, 1, GATED>(p);
    if constexpr (!GATED) { // a gated tile is one of both tensors
        if (groups > kMostGroups || (n <= 16 && per_cu <= kFewColumns))
            return launch_product<8, 1, 1, 2, false>(p);
        if (n <= 32 && per_cu <= kFewColumns)
            return launch_product<8, 1, 2, 1, false>(p);
    }
    if (n <= 16 && per_cu <= 32)
        launch_product<12, 2, 1, 1, GATED>(p);
    else if (n <= 16)
        per_cu >= 100 && high ? launch_product<4, 4, 1, 1, GATED>(p) : launch_product<4, 2, 1, 1, GATED>(p);
    else if (per_cu <= 24 || !high)
        launch_product<12, 2, 2, 1, GATED>(p);
    else
        per_cu < 64 ? launch_product<8, 4, 2, 1, GATED>(p) : launch_product<4, 4, 2, 1, GATED>(p);
}

template <bool GATED>
static int run_product(const char* fn, Product& p)
{
    ProductArgs& a = p.a;
    LowArgs& l = p.low;
    const int all = a.n_tokens, groups = weight_groups(a.K);
    int columns = 0, max_rank = 0, max_ranks[LLAMA2_MAX_BATCH_MATRICES] = {};
    bool fits = true, adapters = false; // the prompt's products hold a tensor's offsets in 31 bits
    for (int i = 0; i < p.n_matrices; ++i) {
        columns += a.t[i].cols; // at most 2^22
        fits = fits && static_cast<long long>(a.t[i].cols) * weight_words(a.K) * 4 <= 0x7FFFFFFFLL;
        if (!l.t[i].down)
            continue;
        adapters = true;
        max_ranks[i] = l.t[i].max_rank;
        max_rank = l.t[i].max_rank > max_rank ? l.t[i].max_rank : max_rank;
        a.most_adapters = l.t[i].n_adapters > a.most_adapters ? l.t[i].n_adapters : a.most_adapters;
    }
    const int per_cu = columns / ctx().num_cus;
    // More than 64 tokens go through the kernels of the prompt's products, and more than 16 where these have tiles for every CU and no
    // adapters, of which each tile reads those of all its tokens one after the other (gated 2 * 11008 columns of 4096 inputs, 32 tokens
    // 23.2 -> 18.6 us, 64 29.5 -> 24.2; with an adapter each 49 against 122; 2 * 8192 columns, 64 tokens 18.4 against 20.7).
    // For the same reason up to 192 tokens with many adapters of few ranks do not (in us, prompt's kernels against these tiles: 128 tokens through
    // q, k and v of 4096 with 128 adapters of 16 ranks 53.8, 40.2, 4 of 16 36.1, 35.4, 32 of 32 55.6, 47.8, 4 of 64 46.0, 71.5; 192 with 64 of 16
    // 80.0, 56.7; gated 2 * 11008, 100 with 16 of 32 82.3, 62.6; 256 through one of 4096 with 64 of 16 33.9, 39.9).  The pool's size stands for the
    // adapters in use, which only the device knows: one prompt with one adapter out of a large pool is 0 .. 6 % slower that way at 16 ranks up to 128
    // tokens (of 64: 100 tokens through q, k and v 32.4, 33.3, gated 46.0, 49.0) and up to 46 % at the rule's end (192 gated with one of 16 of 32 ranks
    // 68.0, 99.1), where all 64 in use would cost twice the time the other way (100 tokens 62.9, 36.0; gated 107, 52.5).  Nor do up to 128 for a few columns
    // (2048 of 2048 inputs 10.5, 6.0; 128 tokens through 4096 of 4096 15.4, 16.1).
    const int tile_tokens = adapters ? (max_rank <= 32 && 2 * a.most_adapters >= max_rank ? 192 : 64) : per_cu <= 8 ? 128 : 64;
    const bool wide = fits && (all > tile_tokens || (all > 16 && !adapters && per_cu >= 80));
    const bool packed = !wide && all > 32 && per_cu > kFewColumns && groups <= kMostGroups;
    const int step = groups <= kMostGroups ? kMostTokens : kMostTokens / 8; // threads of a launch in 32 bits
    const int most = all < step ? all : step;
    // More than 64 tokens: what the ranks receive token by token while that looks up little, else in items of tokens that share an adapter, more
    // reluctantly where those read their inputs again for every 16 ranks (100 tokens of 16 adapters through gated 2 * 11008 columns of 4096, 16
    // ranks, 52 MB: 66.3 us against 71.4; 200 through q, k and v of 4096, 32 ranks, 315 MB: 91.4 against 86.7; 128 of 13824 inputs, 64 ranks, 453 MB:
    // 72.6 against 96.8).
    const bool keeps = a.K <= 5 * kLowWaves * 128;
    double looked_up = 0.0; // bytes
    for (int i = 0; i < p.n_matrices; ++i)
        if (l.t[i].down)
            looked_up += 4.0 * all * a.K * l.t[i].max_rank;
    const bool each = looked_up <= (keeps ? 2e8 : 5e8);
    const size_t fragments = wide ? batch_gemm_bytes(most, a.K) : packed ? static_cast<size_t>(ceil_div(most, 16)) * groups * 4096 : 0;
    p.adapters = adapters;
    const LowScratch scratch = low_scratch(fragments, most, max_ranks, p.n_matrices);
    if (scratch.bytes)
        if (int rc = ensure_attn_partials(scratch.bytes))
            return rc;
    char* const base = reinterpret_cast<char*>(ctx().attn_partials);
    for (int i = 0; i < p.n_matrices; ++i) {
        LowTensor& t = l.t[i];
        if (!t.down)
            continue;
        t.low = base + scratch.low[i];
        t.info = reinterpret_cast<TokenAdapter*>(base + scratch.info[i]);
        a.t[i].low = t.low;
        a.t[i].info = t.info;
        a.t[i].n_adapters = t.n_adapters;
        a.t[i].max_rank = t.max_rank;
    }
    for (int done = 0; done < all; done += step) {
        a.n_tokens = all - done < step ? all - done : step;
        if (p.adapters) {
            l.x = a.x;
            l.positions = a.positions;
            l.token_adapters = a.token_adapters;
            l.K = a.K;
            l.x_stride = a.x_stride;
            l.n_tokens = a.n_tokens;
            l.most_adapters = a.most_adapters;
            l.n_matrices = p.n_matrices;
            l.packed = packed || wide ? reinterpret_cast<uint16_t*>(base) : nullptr;
            const hipStream_t st = ctx().stream;
            const int tensors = p.n_matrices + (l.packed ? 1 : 0);
            if (!wide) {
                hipLaunchKernelGGL(batch_ranks_kernel<false>, dim3(a.n_tokens, round_up(max_rank, 16) / 8, tensors), dim3(512), 0, st, l);
            } else if (each) {
                hipLaunchKernelGGL(batch_ranks_kernel<true>, dim3(a.n_tokens, ceil_div(max_rank, 16), tensors), dim3(1024), 0, st, l);
            } else {
                // Items of a block of 64 tokens: one for each adapter in use, and one more for every 16 tokens.  A workgroup takes several
                // where there are many, since those with nothing to do cost as well.
                int items = a.n_tokens < 64 ? a.n_tokens : 64;
                items = a.most_adapters + 3 < items ? a.most_adapters + 3 : items;
                const dim3 grid(ceil_div(a.n_tokens, 64), items < 8 ? items : 8, tensors), threads(kLowWaves * 64);
                if (a.K <= 4 * kLowWaves * 128)
                    hipLaunchKernelGGL((batch_low_kernel<4, true>), grid, threads, 0, st, l);
                else if (keeps)
                    hipLaunchKernelGGL((batch_low_kernel<5, true>), grid, threads, 0, st, l);
                else
                    hipLaunchKernelGGL((batch_low_kernel<4, false>), grid, threads, 0, st, l);
            }
            L2_LAUNCH_CHECK(fn);
        }
        const uint16_t* const rows = a.x;
        if (packed) {
            if (!p.adapters) {
                const int units = ceil_div(a.n_tokens, 16) * groups;
                hipLaunchKernelGGL(batch_pack_kernel, dim3(ceil_div(units, 2)), dim3(512), 0, ctx().stream, reinterpret_cast<uint16_t*>(base), a.x,
                                   a.K, a.x_stride, a.n_tokens);
                L2_LAUNCH_CHECK(fn);
            }
            a.x = reinterpret_cast<const uint16_t*>(base);
        }
        if (wide) {
            if (int rc = launch_batch_gemm(fn, a, p.n_matrices, GATED, p.adapters, p.adapters, base))
                return rc;
        } else {
            if (all > 1 || !launch_one_token(a, p.n_matrices, GATED))
                launch_shape<GATED>(p, packed, per_cu, groups);
            L2_LAUNCH_CHECK(fn);
        }
        a.x = rows + static_cast<size_t>(a.n_tokens) * a.x_stride;
        a.positions += a.n_tokens;
        if (a.token_adapters)
            a.token_adapters += a.n_tokens;
        for (int i = 0; i < (GATED ? 1 : p.n_matrices); ++i) {
            a.t[i].out += static_cast<size_t>(a.n_tokens) * a.t[i].out_stride;
            if (a.t[i].residual)
                a.t[i].residual += static_cast<size_t>(a.n_tokens) * a.t[i].residual_stride;
        }
    }
    return LLAMA2_OK;
}

static Product product_of(const llama2_half* input, int rows, int input_stride, const int* token_adapters, const llama2_batch& batch)
{
    Product p = {};
    p.a.x = input;
    p.a.positions = batch.positions;
    p.a.token_adapters = token_adapters;
    p.a.K = rows;
    p.a.x_stride = input_stride;
    p.a.n_tokens = batch.n_tokens;
    return p;
}

static void put_tensor(Product& p, int i, const llama2_qweight& w, const llama2_adapters* a, int cols)
{
    ProductTensor& t = p.a.t[i];
    t.w = w.weight;
    t.z = w.zeros;
    t.s = w.scales;
    t.cols = cols;
    if (!a)
        return;
    t.up = a->up;
    t.up_stride = up_halfs(*a, cols);
    LowTensor& l = p.low.t[i];
    l.down = a->down;
    l.scales = a->scales;
    l.ranks = a->ranks;
    l.down_stride = down_halfs(*a, p.a.K);
    l.n_adapters = a->n_adapters;
    l.max_rank = a->max_rank;
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
    Product p = product_of(input, rows, input_stride, token_adapters, *batch);
    p.n_matrices = n_matrices;
    for (int i = 0; i < n_matrices; ++i) {
        const llama2_batch_matrix& m = matrices[i];
        put_tensor(p, i, m.weight, m.adapters, m.cols);
        p.a.t[i].out = m.output;
        p.a.t[i].residual = m.residual;
        p.a.t[i].out_stride = m.output_stride;
        p.a.t[i].residual_stride = m.residual_stride;
    }
    return run_product<false>("llama2_batch_mat_mul_int4", p);
}

int llama2_batch_mat_mul_swiglu(llama2_half* output, const llama2_half* input, const llama2_qweight* gate, const llama2_qweight* up, int rows,
                                int cols, int output_stride, int input_stride, const llama2_adapters* gate_adapters,
                                const llama2_adapters* up_adapters, const int* token_adapters, const llama2_batch* batch)
{
    L2_REQUIRE_INIT();
    if (int rc = check_batch_swiglu(output, input, gate, up, rows, cols, output_stride, input_stride, gate_adapters, up_adapters,
                                    token_adapters, batch))
        return rc;
    Product p = product_of(input, rows, input_stride, token_adapters, *batch);
    p.n_matrices = 2;
    put_tensor(p, 0, *gate, gate_adapters, cols);
    put_tensor(p, 1, *up, up_adapters, cols);
    p.a.t[0].out = output;
    p.a.t[0].out_stride = output_stride;
    return run_product<true>("llama2_batch_mat_mul_swiglu", p);
}

} // extern "C"
