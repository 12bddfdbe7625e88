// Attention of a step of several requests over a paged cache, behind a prefix that they share.
//
// out = sum_r softmax_r(scale q.k_r) v_r over the shared rows and the request's own, by the running maximum and sum.  The
// queries of one key/value head (all of a group, all tokens that see the same rows) are the columns of
//   S^T = K Q^T,   O^T = V^T P^T
// on the matrix cores: with rows of the cache along the first operand, a lane ends up with the scores of ONE query, and
// its probabilities are already the second operand of the second product.  A workgroup takes one item:
//   own      a tile of columns of one request x a piece of its own rows, behind the prefix where that is not shared;
//   shared   a tile of columns out of all tokens, of any request, x a piece of the prefix: a shared row is read once per
//            tile instead of once per request.
// Pieces leave fp32 sums, maximum and denominator, which are joined in order.
//
// Tiles of up to 16 columns (few_rows) are bound by reading the cache: 1059 MB of four long documents in 201 us, 5.3 TB/s, HBM
// traffic 1.00 times that; 594 MB of 64 conversations in 119 .. 124 us, 5.0 TB/s, 1.02 times (a plain read of 1 GiB reaches 5.9 .. 6.3).
// Tiles of up to 128 columns (many_rows) are bound by products and power: with all compute units in their passes two of them
// take 3200 cycles, 2048 of them matrix products, at a clock that falls from 2.4 to 1.73 GHz; 16384 tokens of 8 heads 830
// TFLOP/s, where a library product of 8192^3 reaches 1235.
#include "common.hpp"
#include "batch_plan.hpp"

namespace l2 {

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f16v_t __attribute__((ext_vector_type(16)));

// Probabilities enter the matrix cores as fp16, relative to a reference m that follows the running maximum only when that is
// more than 2^8 above it (rescaling the sums is a fifth of a wide pass's vector work, and one of 32 columns has a new
// maximum in nearly every pass): 2^6 exp2(score - m) is at most 2^14, and one of 2^-30 is still a number.  The sum carries
// the same factors, so that they drop out of the quotient.  Narrow tiles, which wait for
// the cache, take what that rounding left in a second product: 22 bits in all, and against 64 bits 2.1e-4, which is the output's own
// rounding, instead of 2.5e-4 .. 2.9e-4 (one request of 777 rows 8.1 -> 8.2 us, 16 samples 16.9 -> 17.0, 64 conversations 121.4 -> 121.8,
// 128 behind 8192 rows 92.1 -> 92.6, four documents 201.4).  Wide tiles are bound by the matrix cores, which it would give half as many
// products again: there the sum is of the rounded ones, so that the weights add up to 1.
constexpr float kProbShift = 6.0f;
constexpr float kSlack = 8.0f;

struct BatchAttnArgs {
    uint16_t* out;
    const uint16_t* q;
    const uint16_t* key;
    const uint16_t* value;
    const int* prefix_table;
    const int* block_tables;
    const int* query_starts;
    const int* positions;
    float* parts; // [slot][token][head][D] sums, then (maximum, denominator) of each; null: one piece, straight to `out`
    float2* stats;
    unsigned* counters; // [token][key/value head], zero between launches: pieces are joined by whoever leaves the last one; or null
    uint32_t parts_bytes;
    long long block_stride;
    int n_requests, n_tokens, table_stride, prefix_length, max_rows;
    int n_blocks, shift, n_kv_heads, group, out_stride, q_stride;
    float scale; // its absolute value times log2(e), positive
    uint32_t q_sign; // what turns the queries over where the scale is negative
    // items: [shared_splits x n_kv_heads, by eights][shared_tiles][of the eight], and [own_splits][own_tiles][n_kv_heads]
    int shared_items, shared_tiles, shared_splits, shared_piece;
    Divisor by_eights, by_heads, by_tiles, by_group, by_guess; // 8 shared_tiles, n_kv_heads, own_tiles, group, a tile's columns + group
    Divisor by_piece, by_all; // own_piece, all heads
    int own_items, own_tiles, own_piece, own_prefix, spread; // own_prefix: prefix rows in front of a request's own, a multiple of kPass, or 0
};

__device__ __forceinline__ int div_by(int n, Divisor d) { return static_cast<int>(__umulhi(2u * static_cast<uint32_t>(n), d.m) >> d.shift); }

// What a workgroup computes; the same in all its lanes.
struct Item {
    int token, row0, rows, kv_head; // column c: query head kv_head * group + (row0 + c) % group of token `token` + (row0 + c) / group
    int tokens;                 // that the columns belong to
    int least;                  // own rows that all columns attend
    int p0, p1;                 // shared rows
    int r0, r1;                 // own rows
    const int* table;           // of the own rows
    int slot;
    int split;                  // which piece of the own rows
};

__device__ __forceinline__ f4_t mfma16(h8_t x, h8_t y, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0); }
__device__ __forceinline__ f16v_t mfma32(h8_t x, h8_t y, f16v_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0); }

__device__ __forceinline__ float max_xor16(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_xor32(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// One value for the whole wavefront, through the scalar cache: it does not queue behind the cache rows that the vector
// memory path is busy with.
__device__ __forceinline__ int uniform_load(const int* p, int i)
{
    typedef const int __attribute__((address_space(4))) * Scalar;
    return ((Scalar)p)[__builtin_amdgcn_readfirstlane(i)];
}

// Largest of the wavefront's values, the same in all lanes; by row operations, shuffles are round trips through LDS.
__device__ __forceinline__ int wave_max_int(int v)
{
#define L2_MAX_STEP(ctrl, rows) v = max(v, __builtin_amdgcn_update_dpp(v, v, ctrl, rows, 0xF, false))
    L2_MAX_STEP(DPP_QUAD_XOR1, 0xF);
    L2_MAX_STEP(DPP_QUAD_XOR2, 0xF);
    L2_MAX_STEP(DPP_ROW_HALF_MIRROR, 0xF);
    L2_MAX_STEP(DPP_ROW_MIRROR, 0xF);
    L2_MAX_STEP(DPP_ROW_BCAST15, 0xA);
    L2_MAX_STEP(DPP_ROW_BCAST31, 0xC);
#undef L2_MAX_STEP
    return __builtin_amdgcn_readlane(v, 63);
}

// Own rows that a token at position p attends.
__device__ __forceinline__ int own_rows_of(const BatchAttnArgs& a, int p)
{
    return p < a.prefix_length ? 0 : min(p - a.prefix_length, a.max_rows - 1) + 1;
}

// The pieces that hold what a token at position p attends of the request's own rows (and of the prefix, where that lies in front).
__device__ __forceinline__ int pieces_of(const BatchAttnArgs& a, int p)
{
    return div_by(a.own_prefix + own_rows_of(a, p) + a.own_piece - 1, a.by_piece);
}

// exp2(v - base) is the probability times 2^6; without any score above -infinity everything is 0, not NaN.
__device__ __forceinline__ float prob_base(float most) { return most == -INFINITY ? 0.0f : most - kProbShift; }
// Is 2^24 reached, where fp32 numbers are so far apart that the rounding of m and of base alone could take exponents beyond what fp16
// holds?  Then exponents are those of the rounded scores, cut off at what they are without base's rounding.
__device__ __forceinline__ bool far_out(float base) { return __any(fabsf(base) >= 0x1p24f); }
__device__ __forceinline__ float far_exponent(float score, float scale, float base)
{
#pragma clang fp contract(off)
    const float v = score * scale, e = v - base;
    return e > kProbShift + kSlack ? kProbShift + kSlack : e; // NaN stays
}
// Has some column a score so far above its reference that the reference has to follow?  As a difference: m + kSlack would be rounded.
__device__ __forceinline__ bool has_to_follow(float most, float m) { return __any(most - m > kSlack); }
__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float weight_of(float m, float most) { return m == -INFINITY ? 0.0f : exp2_of(m - most); }

// Any element infinite or NaN?  (bits 15 and 31 of the sum: all exponent bits set)
__device__ __forceinline__ uint32_t not_finite(uint32_t v) { return ((v & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }

// Elements of a head (D of them) in row `row` of a table; 64-bit offsets: a cache may be larger than 4 GB.
template <int D>
__device__ __forceinline__ const uint16_t* row_address(const BatchAttnArgs& a, const uint16_t* cache, int block, int row, int kv_head)
{
    return cache + block * a.block_stride + ((row & ((1 << a.shift) - 1)) * a.n_kv_heads + kv_head) * static_cast<long long>(D);
}

// What an infinite or NaN value adds to a sum that it is a part of.
__device__ __forceinline__ float special_part(uint16_t h)
{
    return (h & 0x7C00u) == 0x7C00u ? half_bits_to_float(h) : 0.0f;
}

__device__ __forceinline__ bool in_cache(const BatchAttnArgs& a, int block)
{
    return static_cast<unsigned>(block) < static_cast<unsigned>(a.n_blocks);
}

__device__ __forceinline__ h8_t load_query(const BatchAttnArgs& a, int token, int at)
{
    u32x4 v = *reinterpret_cast<const u32x4*>(a.q + static_cast<size_t>(token) * a.q_stride + at);
#pragma unroll
    for (int k = 0; k < 4; ++k)
        v[k] ^= a.q_sign;
    return __builtin_bit_cast(h8_t, v);
}

// ---------------------------------------------------------------- joining pieces
template <int D>
__device__ __forceinline__ void store_joined(const BatchAttnArgs& a, int token, int head, int x, float sum, const float (&o)[8])
{
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        w[k] = static_cast<uint32_t>(float_to_half_bits(o[2 * k] * inv)) | static_cast<uint32_t>(float_to_half_bits(o[2 * k + 1] * inv)) << 16;
    *reinterpret_cast<u32x4*>(a.out + static_cast<size_t>(token) * a.out_stride + head * D + x * 8) = w;
}

// What the groups of D / 8 lanes of a wavefront have, as one.
template <int D>
__device__ __forceinline__ void join_lanes(const BatchAttnArgs& a, int token, int head, float m, float sum, float (&o)[8])
{
    constexpr int SIDE = D / 8;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = SIDE; d < 64; d <<= 1) {
        const float om = __shfl_xor(m, d, 64), most = fmaxf(m, om), wa = weight_of(m, most), wb = weight_of(om, most);
        const bool lower = (lane & d) == 0; // the same order of the two terms on both sides
        const float os = __shfl_xor(sum, d, 64);
        sum = lower ? fmaf(wb, os, sum * wa) : fmaf(wa, sum, os * wb);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float ov = __shfl_xor(o[i], d, 64);
            o[i] = lower ? fmaf(wb, ov, o[i] * wa) : fmaf(wa, o[i], ov * wb);
        }
        m = most;
    }
    if (lane < SIDE)
        store_joined<D>(a, token, head, lane, sum, o);
}

// One token's head by a wavefront: D / 8 lanes side by side (8 elements each), the others with every 512 / D-th piece.
template <int D>
__device__ void join_pieces(const BatchAttnArgs& a, int token, int head, int slots, __amdgpu_buffer_rsrc_t parts)
{
    constexpr int SIDE = D / 8, DEEP = 64 / SIDE;
    const int lane = threadIdx.x & 63, x = lane % SIDE, deep = lane / SIDE;
    const int heads = a.n_kv_heads * a.group, rows = a.n_tokens * heads;
    float m = -INFINITY, sum = 0.0f, o[8] = {};
    for (int s = deep; s < slots; s += DEEP) {
        const int part = s * rows + token * heads + head; // parts_bytes < 2^31
        const float pm = load_agent(&a.stats[part].x), ps = load_agent(&a.stats[part].y);
        const u32x4 v0 = __builtin_amdgcn_raw_buffer_load_b128(parts, (part * D + x * 8) * 4, 0, kAuxAgent);
        const u32x4 v1 = __builtin_amdgcn_raw_buffer_load_b128(parts, (part * D + x * 8) * 4 + 16, 0, kAuxAgent);
        const float most = fmaxf(m, pm), wa = weight_of(m, most), wb = weight_of(pm, most);
        m = most;
        sum = fmaf(wb, ps, sum * wa);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o[i] = fmaf(wb, __uint_as_float(i < 4 ? v0[i] : v1[i - 4]), o[i] * wa);
    }
    join_lanes<D>(a, token, head, m, sum, o);
}

// ---------------------------------------------------------------- few columns
// Up to 16 columns.  Each of 4 wavefronts takes every fourth tile of 32 rows (each of 8 every eighth, or one wavefront all of them), straight from
// memory into the operands' registers: no row is used twice, so LDS would only be a detour.  Lane (g, c), g = lane / 16: keys of
// row 16 t + c, elements 32 j + 8 g .. + 7 (64 consecutive bytes of a row per load and row); values of the rows 16 t + 4 g .. + 3,
// whose scores the same lane holds, 1/16 of a row each (4 whole rows per load), turned by byte permutations into columns:
// operand i holds elements c * D/16 + i.  16 KB are on their way per wavefront, 12 wavefronts per compute unit; with the
// next tile requested ahead the registers allow fewer of them, and it was slower (64 conversations 136 -> 162 us), with 16
// wavefronts registers spill (123 -> 162).
template <int D, int WAVES>
__device__ void few_rows(const BatchAttnArgs& a, const Item& it, char* lds)
{
    constexpr int kStep = 32 * WAVES;
    constexpr int KS = D / 32, VE = D / 16, VW = VE / 2; // k steps; elements and words of a value row per lane
    const int lane = threadIdx.x & 63, wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, c = lane & 15;
    const int r = min(c, it.rows - 1);
    const int of_tokens = div_by(it.row0 + r, a.by_group), token = it.token + of_tokens;
    const int head = it.kv_head * a.group + it.row0 + r - of_tokens * a.group;
    const int position = a.positions[token];
    const int limit = own_rows_of(a, position);
    const int least = it.least;
    h8_t qf[KS];
#pragma unroll
    for (int j = 0; j < KS; ++j)
        qf[j] = load_query(a, token, head * D + j * 32 + g * 8);

    f4_t o[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i)
        o[i] = f4_t{};
    float m = -INFINITY, sum = 0.0f;

    for (int seg = 0; seg < 2; ++seg) {
        const int* table = seg ? it.table : a.prefix_table;
        const int begin = seg ? it.r0 : it.p0, end = seg ? it.r1 : it.p1;
        const int seen = seg ? limit : end, all_see = seg ? least : end;
        if (begin + wave * 32 >= end)
            continue;
        const int last4 = (end - 1) & ~3;
        auto block_of = [&](int row) { return table[min(row, last4) >> a.shift]; };
        int kid[2], vid[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            kid[t] = block_of(begin + wave * 32 + 16 * t + (c & ~3));
            vid[t] = block_of(begin + wave * 32 + 16 * t + 4 * g);
        }
        for (int tb = begin + wave * 32; tb < end; tb += kStep) {
            h8_t kf[2][KS];
            uint32_t vr[8][VW];
            bool ok[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int row = min(tb + 16 * t + (c & ~3), last4) + (c & 3);
                const uint16_t* p = row_address<D>(a, a.key, in_cache(a, kid[t]) ? kid[t] : 0, row, it.kv_head) + g * 8;
#pragma unroll
                for (int j = 0; j < KS; ++j)
                    kf[t][j] = *reinterpret_cast<const h8_t*>(p + j * 32);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                ok[t] = in_cache(a, vid[t]);
                const int row = min(tb + 16 * t + 4 * g, last4);
                const uint16_t* p = row_address<D>(a, a.value, ok[t] ? vid[t] : 0, row, it.kv_head) + c * VE;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t* w = reinterpret_cast<const uint32_t*>(p + static_cast<size_t>(i) * a.n_kv_heads * D);
                    if constexpr (VW == 4) {
                        const u32x4 x = *reinterpret_cast<const u32x4*>(w);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            vr[4 * t + i][k] = x[k];
                    } else {
                        const u32x2 x = *reinterpret_cast<const u32x2*>(w);
                        vr[4 * t + i][0] = x[0];
                        vr[4 * t + i][1] = x[1];
                    }
                }
            }
            if (tb + kStep < end) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    kid[t] = block_of(tb + kStep + 16 * t + (c & ~3));
                    vid[t] = block_of(tb + kStep + 16 * t + 4 * g);
                }
            }
            f4_t s[2] = {};
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    s[t] = mfma16(kf[t][j], qf[j], s[t]);
            const bool whole = tb + 32 <= all_see && !__any(!ok[0] || !ok[1]);
            float most = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = s[t][i] * a.scale;
                    s[t][i] = whole || (tb + 16 * t + 4 * g + i < seen && ok[t]) ? v : -INFINITY;
                    most = fmaxf(most, s[t][i]);
                }
            most = max_xor32(max_xor16(most));
            if (has_to_follow(most, m)) {
                most = fmaxf(m, most);
                const float alpha = weight_of(m, most);
                sum *= alpha;
#pragma unroll
                for (int i = 0; i < VE; ++i)
                    o[i] *= alpha;
                m = most;
            }
            float base = prob_base(m);
            if (far_out(base)) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        s[t][i] = far_exponent(s[t][i], 1.0f, base);
                base = 0.0f;
            }
            h8_t p, rest; // the probabilities, and what their rounding left
            float less = -1.0f; // kept from the compiler: a fused multiply-add takes the fp16 number as it is and rounds to fp16
            asm volatile("" : "+s"(less));
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float e0 = exp2_of(s[t][i] - base), e1 = exp2_of(s[t][i + 1] - base);
                    sum += e0;
                    sum += e1;
                    uint32_t both = as_u32(h2_t{static_cast<_Float16>(e0), static_cast<_Float16>(e1)});
                    asm volatile("" : "+v"(both)); // rounded once: the compiler would round one by one for the differences, too
                    const h2_t e = as_h2(both);
                    p[4 * t + i] = e[0];
                    p[4 * t + i + 1] = e[1];
                    rest[4 * t + i] = static_cast<_Float16>(__builtin_fmaf(static_cast<float>(e[0]), less, e0));
                    rest[4 * t + i + 1] = static_cast<_Float16>(__builtin_fmaf(static_cast<float>(e[1]), less, e1));
                }
            float check[2] = {}; // sums of products of neighbours, not finite where one of them is not: two words at a time
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int k = 0; k < VW; k += 2)
                    check[i & 1] = dot2(vr[i][k], vr[i][k + 1], check[i & 1]);
            bool special = false;
            if (!whole || __any(!__builtin_isfinite(check[0]) || !__builtin_isfinite(check[1]))) {
                // What lies behind the last row, or in a block that is none, and what is infinite or NaN (in rows that some
                // columns attend and others do not, or beside a product of 0 or less), must not reach a sum through the products.
                uint32_t bad = 0;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool keep = tb + 16 * t + 4 * g + i < end && ok[t];
#pragma unroll
                        for (int k = 0; k < VW; ++k) {
                            const uint32_t v = keep ? vr[4 * t + i][k] : 0u, b = not_finite(v);
                            vr[4 * t + i][k] = v & ~((b >> 15) * 0xFFFFu);
                            bad |= b;
                        }
                    }
                special = __any(bad != 0);
            }
            h8_t w[2];
#pragma unroll
            for (int i = 0; i <= VE; ++i) {
                if (i < VE) {
                    u32x4 x;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        x[k] = __builtin_amdgcn_perm(vr[2 * k + 1][i >> 1], vr[2 * k][i >> 1], (i & 1) ? 0x07060302u : 0x05040100u);
                    w[i & 1] = __builtin_bit_cast(h8_t, x);
                    o[i] = mfma16(w[i & 1], p, o[i]);
                }
                if (i > 0) // one behind: it waits for the product above
                    o[i - 1] = mfma16(w[(i - 1) & 1], rest, o[i - 1]);
            }
            if (special) // to the columns that attend them
                for (int row = tb; row < min(tb + 32, end); ++row) {
                    const int block = uniform_load(table, row >> a.shift);
                    if (!in_cache(a, block))
                        continue;
                    const uint16_t* v = row_address<D>(a, a.value, block, row, it.kv_head);
#pragma unroll
                    for (int i = 0; i < VE; ++i)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            o[i][k] += row < seen ? special_part(v[(g * 4 + k) * VE + i]) : 0.0f;
                }
        }
    }
    sum = add_xor32(add_xor16(sum));

    if constexpr (WAVES == 1) { // the whole of the rows: the output
        if (c >= it.rows || position < 0)
            return;
        typedef _Float16 Halfs __attribute__((ext_vector_type(VE)));
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            Halfs h;
#pragma unroll
            for (int x = 0; x < VE; ++x)
                h[x] = __builtin_bit_cast(_Float16, float_to_half_bits(o[x][k] * inv));
            *reinterpret_cast<Halfs*>(a.out + static_cast<size_t>(token) * a.out_stride + head * D + (g * 4 + k) * VE) = h;
        }
        return;
    }

    // The wavefronts' sums through LDS, then each of the first four adds up a quarter of the elements: those with k == wave, which are
    // VE neighbours in each lane.
    constexpr int QUADS = VE / 4;
    f4_t* all = reinterpret_cast<f4_t*>(lds);
    float2* stat = reinterpret_cast<float2*>(lds + WAVES * VE * 64 * 16);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int x = 0; x < QUADS; ++x)
            all[((wave * 4 + k) * QUADS + x) * 64 + lane] = f4_t{o[4 * x][k], o[4 * x + 1][k], o[4 * x + 2][k], o[4 * x + 3][k]};
    if (g == 0)
        stat[wave * 16 + c] = float2{m, sum};
    __syncthreads();
    float most = -INFINITY, total = 0.0f, weight[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
        most = fmaxf(most, stat[w * 16 + c].x);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float2 st = stat[w * 16 + c];
        weight[w] = weight_of(st.x, most);
        total = fmaf(weight[w], st.y, total);
    }
    if (WAVES > 4 && wave >= 4)
        return; // there is no barrier behind this one: a.counters is null
    f4_t e[QUADS];
#pragma unroll
    for (int x = 0; x < QUADS; ++x) {
        e[x] = f4_t{};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const f4_t y = all[((w * 4 + wave) * QUADS + x) * 64 + lane];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                e[x][k] = fmaf(weight[w], y[k], e[x][k]);
        }
    }
    const bool live = c < it.rows && position >= 0;
    const int rows = a.n_tokens * a.n_kv_heads * a.group, d = (g * 4 + wave) * VE; // rows < 2^26
    const size_t part = static_cast<size_t>(it.slot) * rows + static_cast<size_t>(token) * a.n_kv_heads * a.group + head;
    if (live && !a.parts) {
        typedef _Float16 Halfs __attribute__((ext_vector_type(VE)));
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        Halfs h;
#pragma unroll
        for (int x = 0; x < VE; ++x)
            h[x] = __builtin_bit_cast(_Float16, float_to_half_bits(e[x / 4][x % 4] * inv));
        *reinterpret_cast<Halfs*>(a.out + static_cast<size_t>(token) * a.out_stride + head * D + d) = h;
    }
    const __amdgpu_buffer_rsrc_t parts = make_rsrc(a.parts, a.parts_bytes); // of pieces that are joined in this launch
    if (live && a.parts) {
#pragma unroll
        for (int x = 0; x < QUADS; ++x) {
            if (a.counters) // written through, for the workgroup that joins the pieces; parts_bytes < 2^31
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, e[x]), parts,
                                                       static_cast<int>((part * D + d + 4 * x) * sizeof(float)), 0, kAuxAgent);
            else
                *reinterpret_cast<f4_t*>(a.parts + part * D + d + 4 * x) = e[x];
        }
        if (wave == 0 && g == 0) {
            store_agent(&a.stats[part].x, most);
            store_agent(&a.stats[part].y, total);
        }
    }
    if (WAVES != 4 || !a.counters)
        return;

    // Tokens whose last piece this was; nothing is shared, and their columns lie in one tile each: the group divides 16.
    wait_agent_stores();
    __syncthreads();
    int* const slots_of = reinterpret_cast<int*>(lds); // per token of the tile: pieces to join, 0: not by this workgroup
    if (wave == 0) {
        const int p = __shfl(position, (lane * a.group) & 15, 64); // of token `lane` of the tile: that of its first column
        int slots = 0;
        if (lane * a.group < it.rows && p >= 0) {
            const int pieces = pieces_of(a, p);
            unsigned* const counter = a.counters + (it.token + div_by(it.row0, a.by_group) + lane) * a.n_kv_heads + it.kv_head;
            if (it.split < pieces && add_agent(counter, 1) + 1 == static_cast<unsigned>(pieces)) {
                store_agent(counter, 0);
                slots = pieces;
            }
        }
        if (lane < 16)
            slots_of[lane] = slots;
    }
    __syncthreads();
    for (int k = wave; k < it.rows; k += 4) {
        const int t = div_by(k, a.by_group), slots = __builtin_amdgcn_readfirstlane(slots_of[t]);
        if (slots)
            join_pieces<D>(a, it.token + div_by(it.row0, a.by_group) + t, it.kv_head * a.group + k - t * a.group, slots, parts);
    }
}

// ---------------------------------------------------------------- many columns
// 17 to 128 columns, 32 per wavefront: passes of 64 rows through LDS, read by all four.  The rows of the next pass go
// straight from memory into the other of two LDS buffers while this one is computed, so a pass has one barrier and no
// register holds rows in flight.  With two halves (8 wavefronts, the columns twice) each half has buffers of its own and takes
// every other pass, and their sums are joined at the end.  Rows lie in LDS as in the cache, their 16-byte pieces exchanged by row so that reads have
// no bank conflicts; values come out transposed (ds_read_b64_tr_b16: 4 rows of 16 elements per 16 lanes, a column each), in
// the order in which a lane holds their probabilities (4 rows of one half of the lanes, 4 of the other).
template <int D>
struct ManyLds {
    static constexpr int kRow = D * 2, kPieces = D / 8;      // bytes and 16-byte pieces of a row
    static constexpr int kTensor = kPass * kRow;             // keys, or values, of a pass
    static constexpr int kBuffer = 2 * kTensor, kFlags = 2 * kBuffer, kTotal = kFlags + 32;
    // A wavefront reads keys of 16 rows at the same piece at a time, values of 8 rows at 2 x 2 neighbouring pieces.
    static __device__ __forceinline__ int key_piece(int row, int piece) { return piece ^ (D == 128 ? row & 15 : (row >> 1) & 7); }
    static __device__ __forceinline__ int value_piece(int row, int piece) { return piece ^ (D == 128 ? (row & 7) * 2 : ((row >> 1) & 3) * 2); }
};

// 64 lanes x 16 bytes from base + offset (per lane) straight into LDS at `lds` + 16 lane.  Inline assembly because the
// compiler would wait for it in front of the next read of any LDS; whoever reads the data waits for vmcnt.
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t lds)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "{m0}"(lds), "v"(offset), "s"(base) : "memory");
}

typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ h4_t read_transposed(const char* p)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(h4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p)));
}

template <int D, int HALVES>
__device__ void many_rows(const BatchAttnArgs& a, const Item& it, char* all_lds)
{
    using L = ManyLds<D>;
    constexpr int QS = D / 16, DT = D / 32; // k steps, tiles of output elements
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    const int half = HALVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8); // takes every other pass
    char* const lds = all_lds + half * L::kTotal;
    const int hl = lane >> 5, l31 = lane & 31;
    const int r = wave * 32 + l31, rq = min(r, it.rows - 1);
    const bool idle = wave * 32 >= it.rows;
    const int of_tokens = div_by(it.row0 + rq, a.by_group), token = it.token + of_tokens;
    const int head = it.kv_head * a.group + it.row0 + rq - of_tokens * a.group;
    h8_t qf[QS];
#pragma unroll
    for (int j = 0; j < QS; ++j)
        qf[j] = load_query(a, token, head * D + j * 16 + hl * 8);
    const int position = a.positions[token];
    bool first_rows = true; // what follows is computed behind the first request
    int limit = 0, most_rows = 0, least = 0;
    f16v_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
        o[d] = f16v_t{};
    float m = -INFINITY, sum = 0.0f; // m: the exponents' reference, at most kSlack below the largest score

    // A wavefront loads rows 16 wave .. + 15 of a pass, 8 at a time: those lie in one block.
    constexpr int AT_ONCE = 1024 / L::kRow, LOADS = 8 / AT_ONCE; // rows per load, loads per 8 rows
    const uint32_t row_bytes = static_cast<uint32_t>(a.n_kv_heads) * D * 2;
    const int in_load = lane / L::kPieces, piece = lane % L::kPieces;
    int* const flags = reinterpret_cast<int*>(lds + L::kFlags); // [buffer][wavefront]: bits 0, 1: which of its blocks are none, 2: not finite
    const uint32_t lds_base = __builtin_amdgcn_readfirstlane(
        static_cast<int>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds)));
    // address of the values that a lane reads transposed: row (lane / 16 / 2) * 4 + lane % 16 / 4 of 8, elements lane / 16 % 2 * 16 + lane % 4 * 4
    const int tr_row = hl * 4 + ((lane & 15) >> 2), tr_piece = ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1), tr_byte = (lane & 1) * 8;

    for (int seg = 0; seg < 2; ++seg) {
        const int* table = seg ? it.table : a.prefix_table;
        const int begin = seg ? it.r0 : it.p0, end = seg ? it.r1 : it.p1;
        if (begin >= end)
            continue;
        const int wg_all_see = min(seg ? it.least : end, end);
        const int last8 = (end - 1) & ~7;
        auto block_of = [&](int row) { return uniform_load(table, min(row, last8) >> a.shift); };
        int block[2]; // of the pass that is requested next
        auto look_up = [&](int tb) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                block[h] = block_of(tb + wave * 16 + h * 8);
        };
        auto request = [&](int tb, int buffer) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int first = wave * 16 + h * 8;
                const long long at = (in_cache(a, block[h]) ? block[h] : 0) * a.block_stride +
                                     ((min(tb + first, last8) & ((1 << a.shift) - 1)) * a.n_kv_heads + it.kv_head) * static_cast<long long>(D);
                const uint32_t to = lds_base + buffer * L::kBuffer + first * L::kRow;
#pragma unroll
                for (int x = 0; x < LOADS; ++x) {
                    const int row = x * AT_ONCE + in_load; // of the 8; first is a multiple of 8, and of 16 for h = 0
                    load_to_lds(a.key + at, row * row_bytes + L::key_piece(h * 8 + row, piece) * 16, to + x * 1024);
                }
#pragma unroll
                for (int x = 0; x < LOADS; ++x) {
                    const int row = x * AT_ONCE + in_load;
                    load_to_lds(a.value + at, row * row_bytes + L::value_piece(h * 8 + row, piece) * 16, to + L::kTensor + x * 1024);
                }
            }
        };
        __syncthreads(); // the last pass of the shared rows has been read
        look_up(begin + half * kPass);
        int no_block = (!in_cache(a, block[0]) ? 1 : 0) | (!in_cache(a, block[1]) ? 2 : 0); // of the pass that is on its way
        if (HALVES == 1 || begin + half * kPass < end)
            request(begin + half * kPass, 0);
        look_up(begin + (half + HALVES) * kPass);
        if (first_rows) {
            limit = own_rows_of(a, position);
            most_rows = wave_max_int(limit);
            least = -wave_max_int(-limit);
            first_rows = false;
        }
        const int seen = seg ? limit : end, all_see = seg ? least : end, any_sees = seg ? most_rows : end;
        int buffer = 0;
        for (int first = begin; first < end; first += HALVES * kPass, buffer ^= 1) {
            const int tb = first + half * kPass;
            const bool here = HALVES == 1 || tb < end;
            char* const ks = lds + buffer * L::kBuffer;
            char* const vs = ks + L::kTensor;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // this wavefront's share of the pass lies in LDS
            int found = 0;
            if (here && (no_block || tb + kPass > wg_all_see)) {
                // What lies behind the last row, or in a block that is none, and what is infinite or NaN in rows that some
                // columns attend and others do not, must not reach a sum through a probability of 0.
                for (int x = lane; x < 16 * L::kPieces; x += 64) {
                    const int row = x / L::kPieces;
                    u32x4* at = reinterpret_cast<u32x4*>(vs + (wave * 16 + row) * L::kRow + x % L::kPieces * 16);
                    u32x4 v = *at;
                    if (tb + wave * 16 + row >= end || ((no_block >> (row >> 3)) & 1))
                        v = u32x4{};
                    uint32_t bad = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t b = not_finite(v[k]);
                        v[k] &= ~((b >> 15) * 0xFFFFu);
                        bad |= b;
                    }
                    *at = v;
                    found |= bad ? 4 : 0;
                }
                found = __any(found) ? 4 : 0;
            }
            if (lane == 0)
                flags[buffer * 4 + wave] = no_block | found;
            __syncthreads(); // everybody's share does, and the other buffer has been read
            if (tb + HALVES * kPass < end) {
                no_block = (!in_cache(a, block[0]) ? 1 : 0) | (!in_cache(a, block[1]) ? 2 : 0);
                request(tb + HALVES * kPass, buffer ^ 1);
                look_up(tb + 2 * HALVES * kPass);
            }
            if (!here || idle || tb >= any_sees)
                continue;
            int no_rows = 0, said = 0; // no_rows: a bit per 8 rows
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int f = flags[buffer * 4 + w];
                no_rows |= (f & 3) << (2 * w);
                said |= f;
            }
            no_rows = __builtin_amdgcn_readfirstlane(no_rows);
            said = __builtin_amdgcn_readfirstlane(said);

            f16v_t s[2] = {};
#pragma unroll
            for (int j = 0; j < QS; ++j)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int row = t * 32 + l31;
                    s[t] = mfma32(*reinterpret_cast<const h8_t*>(ks + row * L::kRow + L::key_piece(row, j * 2 + hl) * 16), qf[j], s[t]);
                }
            if (tb + kPass > all_see || no_rows) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int row = t * 32 + 8 * (i >> 2) + 4 * hl + (i & 3);
                        s[t][i] = tb + row < seen && !((no_rows >> (row >> 3)) & 1) ? s[t][i] : -INFINITY;
                    }
            }
            float most = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    most = fmaxf(most, s[t][i]);
            most = max_xor32(most) * a.scale;
            if (has_to_follow(most, m)) {
                most = fmaxf(m, most);
                const float alpha = weight_of(m, most);
                sum *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    o[d] *= alpha;
                m = most;
            }
            const float base = prob_base(m);
            // Exponents are s * scale - base with one rounding.
            float factor = a.scale, minus = base;
            if (far_out(base)) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        s[t][i] = far_exponent(s[t][i], a.scale, base);
                factor = 1.0f;
                minus = 0.0f;
            }
            h8_t p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    h2_t e;
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        e[x] = static_cast<_Float16>(exp2_of(__builtin_fmaf(s[u >> 1][8 * (u & 1) + i + x], factor, -minus)));
                    p[u][i] = e[0];
                    p[u][i + 1] = e[1];
                    sum = dot2(as_u32(e), 0x3C003C00u, sum); // of the rounded ones, in fp32
                }
            auto values = [&](int d, int u) { // elements 32 d + lane % 32 of rows 16 u + 8 (j / 4) + 4 hl + j % 4
                h8_t v;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int row = u * 16 + half * 8 + tr_row;
                    const h4_t x = read_transposed(vs + row * L::kRow + L::value_piece(row, d * 4 + tr_piece) * 16 + tr_byte);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        v[half * 4 + k] = x[k];
                }
                return v;
            };
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    o[d] = mfma32(values(d, u), p[u], o[d]);
            if (said & 4) // values that are not finite, taken out above: to the columns that attend them
                for (int row = tb; row < min(tb + kPass, end); ++row) {
                    const int block_id = uniform_load(table, row >> a.shift);
                    if (!in_cache(a, block_id))
                        continue;
                    const uint16_t* v = row_address<D>(a, a.value, block_id, row, it.kv_head) + 4 * hl;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            o[d][x] += row < seen ? special_part(v[d * 32 + 8 * (x >> 2) + (x & 3)]) : 0.0f;
                }
        }
    }
    sum += __shfl_xor(sum, 32, 64);
    if constexpr (HALVES == 2) { // the other half's sums through LDS
        f4_t* const others = reinterpret_cast<f4_t*>(all_lds) + wave * DT * 4 * 64;
        float2* const other = reinterpret_cast<float2*>(all_lds + 4 * DT * 4 * 64 * 16) + wave * 64;
        __syncthreads();
        if (half == 1) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    others[(d * 4 + k) * 64 + lane] = f4_t{o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]};
            other[lane] = float2{m, sum};
        }
        __syncthreads();
        if (half == 1)
            return;
        const float2 st = other[lane];
        const float most = fmaxf(m, st.x), wa = weight_of(m, most), wb = weight_of(st.x, most);
        m = most;
        sum = fmaf(wb, st.y, sum * wa);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f4_t y = others[(d * 4 + k) * 64 + lane];
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    o[d][4 * k + x] = fmaf(wb, y[x], o[d][4 * k + x] * wa);
            }
    }
    if (r >= it.rows || position < 0)
        return;
    if (a.parts) {
        const size_t row = static_cast<size_t>(token) * a.n_kv_heads * a.group + head;
        const size_t part = static_cast<size_t>(it.slot) * a.n_tokens * a.n_kv_heads * a.group + row;
        float* out = a.parts + part * D + 4 * hl;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<float4*>(out + d * 32 + 8 * k) = float4{o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]};
        if (hl == 0)
            a.stats[part] = float2{m, sum};
        return;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t* out = a.out + static_cast<size_t>(token) * a.out_stride + head * D + 4 * hl;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            u32x2 w;
#pragma unroll
            for (int x = 0; x < 2; ++x)
                w[x] = static_cast<uint32_t>(float_to_half_bits(o[d][4 * k + 2 * x] * inv)) |
                       static_cast<uint32_t>(float_to_half_bits(o[d][4 * k + 2 * x + 1] * inv)) << 16;
            *reinterpret_cast<u32x2*>(out + d * 32 + 8 * k) = w;
        }
}

// The first of a request's tiles of columns: room for every request to end with a tile that is not full.
template <int TILE>
__device__ __forceinline__ int first_tile(const BatchAttnArgs& a, int start, int request)
{
    return start * a.group / TILE + request;
}

__device__ __forceinline__ int request_start(const BatchAttnArgs& a, int request)
{
    return min(max(uniform_load(a.query_starts, request), 0), a.n_tokens);
}

template <int D, int WAVES>
constexpr int kFewLds = WAVES * ((D / 16) * 1024 + 128);
template <int D, int HALVES>
constexpr int kManyLds = HALVES * ManyLds<D>::kTotal > kFewLds<D, 4 * HALVES> ? HALVES * ManyLds<D>::kTotal : kFewLds<D, 4 * HALVES>;

// kNarrow: a workgroup per tile of up to 16 columns.  kSingle: a wavefront per tile, for many tiles of few rows, where most
// of a workgroup would have no rows; no sharing and no pieces.  kWide: a workgroup per tile of up to 128 columns.  kTall: the same
// with two halves of the workgroup that take turns with the passes, where there are no more tiles than compute units.
template <int D, BatchAttnKernel KIND>
__global__ __launch_bounds__(KIND == BatchAttnKernel::kTall ? 512 : 256, KIND == BatchAttnKernel::kWide || KIND == BatchAttnKernel::kTall ? 2 : 3) void batch_attn_kernel(BatchAttnArgs a)
{
    constexpr bool TALL = KIND == BatchAttnKernel::kTall, MANY = KIND == BatchAttnKernel::kWide || TALL, SINGLE = KIND == BatchAttnKernel::kSingle;
    constexpr int kTileRows = MANY ? kManyRows : kFewRows;
    __shared__ __align__(16) char lds[MANY ? kManyLds<D, TALL ? 2 : 1> : SINGLE ? 16 : kFewLds<D, 4>];
    Item it = {};
    const int shared_items = a.shared_items;
    // Wide tiles of shared rows first, they take longest; narrow ones last, to fill up what long requests leave idle (64
    // conversations 133 -> 125 us).
    int index = blockIdx.x;
    if (KIND == BatchAttnKernel::kNarrow)
        index = index < a.own_items ? index + shared_items : index - a.own_items;
    if (SINGLE) {
        index = index * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (index >= a.own_items)
            return;
    }
    if (index < shared_items) {
        // The tiles of a piece to one XCD: they read the same rows.
        const int eight = div_by(index, a.by_eights), tile = (index - eight * 8 * a.shared_tiles) / 8, rest = eight * 8 + index % 8;
        if (rest >= a.shared_splits * a.n_kv_heads)
            return;
        it.slot = div_by(rest, a.by_heads);
        it.kv_head = rest - it.slot * a.n_kv_heads;
        it.p0 = it.slot * a.shared_piece;
        it.p1 = min(it.p0 + a.shared_piece, a.prefix_length);
        it.row0 = tile * kTileRows;
        it.rows = min(a.n_tokens * a.group - it.row0, kTileRows);
        it.tokens = 1; // all see the same rows
    } else {
        index -= shared_items;
        const int of_heads = div_by(index, a.by_heads);
        const int split = div_by(of_heads, a.by_tiles), turn = of_heads - split * a.own_tiles;
        // wide tiles from the last one on: of a prompt, later tiles see more rows (3827 prompt tokens 102 -> 92 us)
        const int tile = MANY ? a.own_tiles - 1 - turn : turn;
        // An XCD gets every eighth workgroup: the same heads every time, or all of them in turn.
        it.kv_head = a.spread ? index + of_heads : index;
        it.kv_head -= div_by(it.kv_head, a.by_heads) * a.n_kv_heads;
        // The request: the one it would be if all brought one token, else (and always among prompts) by counting, 64 at a time.
        int request = 0, start = 0, stop = 0;
        const bool guess = !MANY || a.spread;
        if (guess) {
            request = min(div_by((tile + 1) * kTileRows - 1, a.by_guess), a.n_requests - 1);
            start = request_start(a, request);
            stop = request_start(a, request + 1);
        }
        if (!guess || first_tile<kTileRows>(a, start, request) > tile || first_tile<kTileRows>(a, stop, request + 1) <= tile) {
            const int lane = threadIdx.x & 63;
            for (int first = 0; first < a.n_requests; first += 64) { // the last one whose first tile is not behind `tile`
                const int b = min(first + lane, a.n_requests - 1);
                const int from = min(max(a.query_starts[b], 0), a.n_tokens), to = min(max(a.query_starts[b + 1], 0), a.n_tokens);
                const int n = __popcll(__ballot(first + lane < a.n_requests && first_tile<kTileRows>(a, from, b) <= tile));
                if (n > 0) {
                    request = first + n - 1;
                    start = __builtin_amdgcn_readlane(from, n - 1);
                    stop = __builtin_amdgcn_readlane(to, n - 1);
                }
                if (n < 64)
                    break;
            }
        }
        it.row0 = (tile - first_tile<kTileRows>(a, start, request)) * kTileRows;
        it.rows = min((stop - start) * a.group - it.row0, kTileRows);
        if (it.rows <= 0 || it.row0 < 0)
            return;
        it.token = start;
        const int t0 = start + div_by(it.row0, a.by_group), t1 = start + div_by(it.row0 + it.rows - 1, a.by_group);
        it.tokens = t1 - t0 + 1; // 16 at most, 128 of wide tiles
        int most;
        if (it.tokens == 1) {
            it.least = most = own_rows_of(a, uniform_load(a.positions, t1));
        } else {
            const int t = t0 + static_cast<int>(threadIdx.x & 63);
            const int x = own_rows_of(a, a.positions[min(t, t1)]), y = MANY ? own_rows_of(a, a.positions[min(t + 64, t1)]) : x;
            most = wave_max_int(max(x, y));
            it.least = -wave_max_int(-min(x, y));
        }
        const int from = split * a.own_piece, to = from + a.own_piece; // of the shared rows in front and its own
        if (a.own_prefix) {
            it.p0 = min(from, a.prefix_length);
            it.p1 = min(to, a.prefix_length);
        }
        it.r0 = max(from - a.own_prefix, 0);
        it.r1 = min(max(to - a.own_prefix, 0), most);
        it.slot = a.shared_splits + split;
        it.split = split;
        it.table = a.block_tables + static_cast<size_t>(request) * a.table_stride;
        if (it.p0 >= it.p1 && it.r0 >= it.r1 && a.parts)
            return;
    }
    if constexpr (MANY) {
        if (it.rows > kFewRows) {
            many_rows<D, TALL ? 2 : 1>(a, it, lds);
            return;
        }
    }
    few_rows<D, SINGLE ? 1 : TALL ? 8 : 4>(a, it, lds);
}

// Joins the pieces of a token's head, in order, where no workgroup of the attention does: LANES lanes per row, D / 8 of
// them side by side (8 elements each), the others with every LANES * 8 / D-th piece.
template <int D, int LANES>
__global__ __launch_bounds__(256) void batch_attn_merge_kernel(BatchAttnArgs a)
{
    constexpr int SIDE = D / 8, DEEP = LANES / SIDE;
    __shared__ float lds[LANES > 64 ? DEEP * SIDE * 8 : 1];
    __shared__ float2 stat[LANES > 64 ? DEEP : 1];
    const int heads = a.n_kv_heads * a.group, rows = a.n_tokens * heads; // < 2^26: checked on the host
    const int row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES, x = lane % SIDE, deep = lane / SIDE;
    const int token = div_by(min(row, rows - 1), a.by_all), head = row - token * heads, position = a.positions[token];
    if (row >= rows || position < 0)
        return; // a whole wavefront at least, the whole workgroup where it has barriers
    const int slots = a.shared_splits + pieces_of(a, position);
    float m = -INFINITY, sum = 0.0f, o[8] = {};
    for (int s = deep; s < slots; s += DEEP) {
        const size_t part = static_cast<size_t>(s) * rows + row;
        const float2 st = a.stats[part];
        const float4* p = reinterpret_cast<const float4*>(a.parts + part * D + x * 8);
        const float4 v0 = p[0], v1 = p[1];
        const float most = fmaxf(m, st.x), wa = weight_of(m, most), wb = weight_of(st.x, most);
        m = most;
        sum = fmaf(wb, st.y, sum * wa);
        const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o[i] = fmaf(wb, v[i], o[i] * wa);
    }
    if constexpr (LANES == 64) {
        join_lanes<D>(a, token, head, m, sum, o);
    } else {
        if (x == 0)
            stat[deep] = float2{m, sum};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            lds[(i * DEEP + deep) * SIDE + x] = o[i];
        __syncthreads();
        if (deep > 0)
            return;
        for (int d = 0; d < DEEP; ++d)
            m = fmaxf(m, stat[d].x);
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o[i] = 0.0f;
        for (int d = 0; d < DEEP; ++d) {
            const float w = weight_of(stat[d].x, m);
            sum = fmaf(w, stat[d].y, sum);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                o[i] = fmaf(w, lds[(i * DEEP + d) * SIDE + x], o[i]);
        }
        store_joined<D>(a, token, head, x, sum, o);
    }
}

template <int D>
static void batch_attn_launch(const BatchAttnArgs& a, BatchAttnKernel kind, int items, int slots)
{
    if (kind == BatchAttnKernel::kWide)
        hipLaunchKernelGGL((batch_attn_kernel<D, BatchAttnKernel::kWide>), dim3(items), dim3(256), 0, ctx().stream, a);
    else if (kind == BatchAttnKernel::kTall)
        hipLaunchKernelGGL((batch_attn_kernel<D, BatchAttnKernel::kTall>), dim3(items), dim3(512), 0, ctx().stream, a);
    else if (kind == BatchAttnKernel::kSingle)
        hipLaunchKernelGGL((batch_attn_kernel<D, BatchAttnKernel::kSingle>), dim3(ceil_div(items, 4)), dim3(256), 0, ctx().stream, a);
    else
        hipLaunchKernelGGL((batch_attn_kernel<D, BatchAttnKernel::kNarrow>), dim3(items), dim3(256), 0, ctx().stream, a);
    if (!a.parts || a.counters)
        return;
    const int rows = a.n_tokens * a.n_kv_heads * a.group;
    if (slots <= 16 || rows >= 1 << 24) // of threads there are less than 2^32
        hipLaunchKernelGGL((batch_attn_merge_kernel<D, 64>), dim3(ceil_div(rows, 4)), dim3(256), 0, ctx().stream, a);
    else
        hipLaunchKernelGGL((batch_attn_merge_kernel<D, 256>), dim3(rows), dim3(256), 0, ctx().stream, a);
}

} // namespace l2

using namespace l2;

extern "C" {

int llama2_batch_attention(llama2_half* output, const llama2_half* query, const llama2_batch* batch,
                           const llama2_paged_cache* cache, int n_heads, int output_stride, int query_stride, float scale)
{
    const char* fn = "llama2_batch_attention";
    L2_REQUIRE_INIT();
    if (int rc = check_batch_attention(output, query, batch, cache, n_heads, output_stride, query_stride, scale))
        return rc;
    const llama2_batch& b = *batch;
    const int max_rows = batch_own_rows(b, cache->block_size), group = n_heads / cache->n_kv_heads;
    const BatchAttnPlan p = batch_attn_plan(b, cache->n_kv_heads, group, max_rows, ctx().num_cus > 0 ? ctx().num_cus : 256);
    if (int rc = check_batch_attn_plan(p, b.n_tokens, n_heads, cache->n_kv_heads))
        return rc;
    const long long rows = static_cast<long long>(b.n_tokens) * n_heads, items = p.items(cache->n_kv_heads);
    BatchAttnArgs a = {};
    a.out = output;
    a.q = query;
    a.key = cache->key;
    a.value = cache->value;
    a.prefix_table = b.prefix_table;
    a.block_tables = b.block_tables;
    a.query_starts = b.query_starts;
    a.positions = b.positions;
    a.block_stride = block_halfs(*cache);
    a.n_requests = b.n_requests;
    a.n_tokens = b.n_tokens;
    a.table_stride = b.table_stride;
    a.prefix_length = b.prefix_length;
    a.max_rows = max_rows;
    a.n_blocks = cache->n_blocks;
    a.shift = log2_of(cache->block_size);
    a.n_kv_heads = cache->n_kv_heads;
    a.group = group;
    a.out_stride = output_stride;
    a.q_stride = query_stride;
    // powers of two from here on; never 0, which would make NaN of a score that is masked with -infinity
    a.scale = fmaxf(fabsf(scale) * 1.44269504088896340736f, 1.17549435e-38f);
    a.q_sign = scale < 0.0f ? 0x80008000u : 0u;
    a.shared_tiles = p.shared_tiles;
    a.shared_splits = p.shared_splits;
    a.shared_piece = p.shared_piece;
    a.shared_items = static_cast<int>(p.shared_items(a.n_kv_heads));
    a.own_items = static_cast<int>(items) - a.shared_items;
    a.own_tiles = p.own_tiles;
    a.own_piece = p.own_piece;
    a.own_prefix = p.own_prefix;
    a.by_eights = divisor(8 * (p.shared_tiles > 0 ? p.shared_tiles : 1));
    a.by_heads = divisor(a.n_kv_heads);
    a.by_tiles = divisor(p.own_tiles);
    a.by_group = divisor(group);
    a.by_guess = divisor((p.kernel == BatchAttnKernel::kWide || p.kernel == BatchAttnKernel::kTall ? kManyRows : kFewRows) + group);
    a.by_piece = divisor(p.own_piece);
    a.by_all = divisor(n_heads);
    a.spread = p.spread;
    if (p.slots() > 1) {
        const size_t part = static_cast<size_t>(p.slots()) * rows;
        if (int rc = ensure_attn_partials(part * (cache->head_size + 2) * sizeof(float)))
            return rc;
        a.parts = ctx().attn_partials;
        a.stats = reinterpret_cast<float2*>(a.parts + part * cache->head_size);
        // Joined in the same launch: few pieces of few columns, which one wavefront per column has done sooner than another
        // launch begins.
        const size_t bytes = part * cache->head_size * sizeof(float);
        if (p.kernel == BatchAttnKernel::kNarrow && p.shared_splits == 0 && p.slots() <= 16 && kFewRows % group == 0 && rows / group <= kMaxBatchCounters && bytes < (1u << 31)) {
            a.counters = ctx().batch_counters;
            a.parts_bytes = static_cast<uint32_t>(bytes);
        }
    }
    if (cache->head_size == 128)
        batch_attn_launch<128>(a, p.kernel, static_cast<int>(items), p.slots());
    else
        batch_attn_launch<64>(a, p.kernel, static_cast<int>(items), p.slots());
    L2_LAUNCH_CHECK(fn);
    return LLAMA2_OK;
}

} // extern "C"
