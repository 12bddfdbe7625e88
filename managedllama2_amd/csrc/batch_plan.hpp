// Host side of the operators of a step of several requests, without a GPU call in it: what arguments are refused, and how
// the attention is cut into workgroups.  Uses L2_CHECK, fail, aligned, overlap and ceil_div of whoever includes it.
#pragma once

#include <cstddef>
#include <cstdint>
#include <utility>

#include "../../include/llama2_hip.h"

namespace l2 {

constexpr int kMaxBatchTokens = 1 << 20; // tokens and requests of a step
constexpr int kMaxBatchHeads = 1024;
constexpr int kMaxBatchRows = 1 << 29; // that a token attends: sums of two such numbers are ints

constexpr int kManyRows = 128; // columns (token, head of the group) of a workgroup's widest tile
constexpr int kFewRows = 16;   // at most this many: the wavefronts split the cache rows instead of the columns
constexpr int kPass = 64;      // cache rows per pass of wide tiles; pieces are multiples of it
constexpr int kMaxPieces = 256; // of a request's rows, and of the prefix
constexpr long long kMaxBatchScratch = 512LL << 20; // bytes of sums of all pieces

inline int round_up(int v, int to) { return ceil_div(v, to) * to; }

inline int log2_of(int power)
{
    int s = 0;
    while ((1 << s) < power)
        ++s;
    return s;
}

// n / d for 0 <= n < 2^31 as the upper half of a product (a division by a number known only at run time is 20 instructions
// that wait for one another, and a workgroup has six in front of its first load): 2 n m / 2^(32 + shift).  m = ceil(2^(31 + shift) / d)
// is off by less than 1, so the quotient by less than n / 2^(31 + shift) < 2^-shift <= 1 / d.
struct Divisor {
    uint32_t m, shift;
};

inline Divisor divisor(int d)
{
    uint32_t shift = 0;
    while ((1LL << shift) < d)
        ++shift;
    return {static_cast<uint32_t>(((1ULL << (31 + shift)) + d - 1) / d), shift};
}

// ---------------------------------------------------------------- refusals
inline int check_block_size(const char* fn, int block_size)
{
    L2_CHECK(block_size >= 8 && block_size <= 1024 && (block_size & (block_size - 1)) == 0,
             "%s: block_size=%d must be a power of two from 8 to 1024", fn, block_size);
    return LLAMA2_OK;
}

inline int check_batch(const char* fn, const llama2_batch* b)
{
    L2_CHECK(b, "%s: null batch", fn);
    L2_CHECK(b->n_requests > 0 && b->n_requests <= kMaxBatchTokens && b->n_tokens > 0 && b->n_tokens <= kMaxBatchTokens,
             "%s: n_requests=%d and n_tokens=%d must be 1 .. %d", fn, b->n_requests, b->n_tokens, kMaxBatchTokens);
    L2_CHECK(b->prefix_length >= 0, "%s: prefix_length=%d is negative", fn, b->prefix_length);
    L2_CHECK(aligned(b->block_tables, 4) && aligned(b->lengths, 4) && aligned(b->query_starts, 4) && aligned(b->positions, 4) &&
                 aligned(b->slots, 4) && aligned(b->prefix_table, 4), "%s: misaligned array in the batch", fn);
    return LLAMA2_OK;
}

inline long long block_halfs(const llama2_paged_cache& c)
{
    return c.block_stride ? c.block_stride : static_cast<long long>(c.block_size) * c.n_kv_heads * c.head_size;
}

inline size_t cache_bytes(const llama2_paged_cache& c) // of keys, or of values
{
    return (static_cast<size_t>(c.n_blocks - 1) * block_halfs(c) + static_cast<size_t>(c.block_size) * c.n_kv_heads * c.head_size) * 2;
}

inline int check_paged_cache(const char* fn, const llama2_paged_cache* c, int n_heads)
{
    L2_CHECK(c && c->key && c->value, "%s: null cache", fn);
    L2_CHECK(aligned(c->key, 16) && aligned(c->value, 16), "%s: cache pointers must be 16-byte aligned", fn);
    if (c->head_size != 64 && c->head_size != 128)
        return fail(LLAMA2_ERR_UNSUPPORTED, "%s: head_size=%d must be 64 or 128", fn, c->head_size);
    if (int rc = check_block_size(fn, c->block_size))
        return rc;
    L2_CHECK(c->n_kv_heads > 0 && n_heads > 0 && n_heads % c->n_kv_heads == 0,
             "%s: n_heads=%d must be a positive multiple of n_kv_heads=%d", fn, n_heads, c->n_kv_heads);
    if (n_heads > kMaxBatchHeads)
        return fail(LLAMA2_ERR_UNSUPPORTED, "%s: n_heads=%d exceeds %d", fn, n_heads, kMaxBatchHeads);
    const long long block = static_cast<long long>(c->block_size) * c->n_kv_heads * c->head_size;
    L2_CHECK(c->n_blocks > 0 && c->n_blocks <= 0x7FFFFFFF / c->block_size,
             "%s: n_blocks=%d must be positive, and n_blocks * block_size below 2^31", fn, c->n_blocks);
    L2_CHECK(c->block_stride == 0 || (c->block_stride >= block && c->block_stride % 8 == 0 && c->block_stride <= (1LL << 45) / c->n_blocks),
             "%s: block_stride=%lld must be 0 or a multiple of 8 of at least %lld halfs", fn, c->block_stride, block);
    return LLAMA2_OK;
}

// `n` rows of a_width halfs from `a` on and as many of b_width from `b` on, both `stride` halfs apart (no less than the
// widths): does one of the first overlap one of the others?
inline bool rows_overlap(const void* a, long long a_width, const void* b, long long b_width, long long n, long long stride)
{
    uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    if (x > y) {
        std::swap(x, y);
        std::swap(a_width, b_width);
    }
    const uintptr_t s = static_cast<uintptr_t>(stride) * 2, of = (y - x) / s, rest = (y - x) % s; // only these two rows of the first can
    const uintptr_t last = static_cast<uintptr_t>(n - 1);
    return (of <= last && rest < static_cast<uintptr_t>(a_width) * 2) || (of + 1 <= last && s - rest < static_cast<uintptr_t>(b_width) * 2);
}

// Does an array of `bytes` at p overlap one of `n` rows of `width` halfs from `a` on, `stride` halfs apart?
inline bool touches_rows(const void* p, size_t bytes, const void* a, long long width, long long n, long long stride)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(p);
    if (!p || bytes == 0)
        return false;
    if (y < x)
        return bytes > x - y;
    const uintptr_t s = static_cast<uintptr_t>(stride) * 2, of = (y - x) / s, rest = (y - x) % s, last = static_cast<uintptr_t>(n - 1);
    return (of <= last && rest < static_cast<uintptr_t>(width) * 2) || (of < last && bytes > s - rest);
}

inline size_t rows_bytes(int rows, int stride, int width) { return (static_cast<size_t>(rows - 1) * stride + width) * 2; }

inline int check_batch_tables(const llama2_batch* batch, const int* cached, const int* counts, const int* free_blocks, int n_free,
                              const int* taken, const int* new_taken, int block_size)
{
    const char* fn = "llama2_batch_tables";
    if (int rc = check_batch(fn, batch))
        return rc;
    const llama2_batch& b = *batch;
    L2_CHECK(b.block_tables && b.lengths && b.query_starts && b.positions && b.slots && cached && counts && taken && new_taken,
             "%s: null pointer", fn);
    L2_CHECK(aligned(cached, 4) && aligned(counts, 4) && aligned(free_blocks, 4) && aligned(taken, 4) && aligned(new_taken, 4),
             "%s: misaligned pointer", fn);
    L2_CHECK(n_free >= 0 && n_free < 0x7FFFFFFF - kMaxBatchTokens && (free_blocks || n_free == 0), "%s: n_free=%d free_blocks=%p", fn, n_free,
             static_cast<const void*>(free_blocks));
    if (int rc = check_block_size(fn, block_size))
        return rc;
    L2_CHECK(b.table_stride > 0 && b.table_stride <= (0x7FFFFFFF - b.prefix_length) / block_size,
             "%s: table_stride=%d must be positive, and prefix_length=%d + table_stride * block_size below 2^31", fn, b.table_stride,
             b.prefix_length);
    const size_t requests = static_cast<size_t>(b.n_requests) * 4, tokens = static_cast<size_t>(b.n_tokens) * 4;
    const struct {
        const void* p;
        size_t bytes;
    } written[] = {{b.block_tables, requests * b.table_stride}, {b.lengths, requests}, {b.query_starts, requests + 4},
                   {b.positions, tokens}, {b.slots, tokens}, {new_taken, 4}},
      read[] = {{cached, requests}, {counts, requests}, {free_blocks, static_cast<size_t>(n_free) * 4}, {taken, 4}};
    for (int i = 0; i < 6; ++i) {
        for (int j = 0; j < i; ++j)
            L2_CHECK(!overlap(written[i].p, written[i].bytes, written[j].p, written[j].bytes), "%s: output arrays overlap", fn);
        for (int j = 0; j < 4; ++j) {
            const bool in_place = written[i].p == read[j].p && ((i == 1 && j == 0) || (i == 5 && j == 3));
            L2_CHECK(in_place || !overlap(written[i].p, written[i].bytes, read[j].p, read[j].bytes),
                     "%s: an output overlaps an input (lengths may be cached, and new_taken taken)", fn);
        }
    }
    return LLAMA2_OK;
}

inline int check_batch_rope(const llama2_half* q_output, const llama2_half* q, const llama2_half* k, const llama2_half* v,
                            const llama2_half* q_gamma, const llama2_half* k_gamma, const llama2_batch* batch,
                            const llama2_paged_cache* cache, int n_heads, int q_output_stride, int q_stride, int kv_stride, float eps,
                            float theta)
{
    const char* fn = "llama2_batch_qk_norm_rope";
    if (int rc = check_batch(fn, batch))
        return rc;
    if (int rc = check_paged_cache(fn, cache, n_heads))
        return rc;
    L2_CHECK(q_output && q && k && v && batch->positions && batch->slots, "%s: null pointer", fn);
    L2_CHECK(aligned(q_output, 16) && aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(q_gamma, 16) &&
                 aligned(k_gamma, 16), "%s: pointers must be 16-byte aligned", fn);
    const int q_row = n_heads * cache->head_size, kv_row = cache->n_kv_heads * cache->head_size, t = batch->n_tokens;
    L2_CHECK(q_stride >= q_row && q_output_stride >= q_row && kv_stride >= kv_row && q_stride % 8 == 0 && q_output_stride % 8 == 0 &&
                 kv_stride % 8 == 0, "%s: strides %d, %d, %d must be multiples of 8 and hold a row of %d, %d, %d", fn, q_output_stride,
             q_stride, kv_stride, q_row, q_row, kv_row);
    L2_CHECK(theta >= 1.0f && theta <= 3.0e38f, "%s: theta=%g must be at least 1", fn, static_cast<double>(theta));
    L2_CHECK(eps >= 0.0f && eps <= 3.0e38f, "%s: eps=%g must not be negative", fn, static_cast<double>(eps));
    const size_t out_bytes = rows_bytes(t, q_output_stride, q_row), kv_bytes = rows_bytes(t, kv_stride, kv_row);
    const bool in_place = q_output == q && q_output_stride == q_stride;
    L2_CHECK(in_place || !overlap(q_output, out_bytes, q, rows_bytes(t, q_stride, q_row)), "%s: q_output overlaps q without being it", fn);
    for (const llama2_half* x : {k, v}) { // in place, their rows may lie between those of q
        const bool between = in_place && kv_stride == q_stride && !rows_overlap(q, q_row, x, kv_row, t, q_stride);
        L2_CHECK(between || !overlap(q_output, out_bytes, x, kv_bytes), "%s: q_output overlaps k or v", fn);
    }
    // blocks of keys and values may take turns
    L2_CHECK(!rows_overlap(cache->key, static_cast<long long>(cache->block_size) * kv_row, cache->value,
                           static_cast<long long>(cache->block_size) * kv_row, cache->n_blocks, block_halfs(*cache)),
             "%s: the cache's keys and values overlap", fn);
    const void* written[] = {cache->key, cache->value};
    for (const void* c : written)
        L2_CHECK(!overlap(c, cache_bytes(*cache), q, rows_bytes(t, q_stride, q_row)) && !overlap(c, cache_bytes(*cache), k, kv_bytes) &&
                     !overlap(c, cache_bytes(*cache), v, kv_bytes) && !overlap(c, cache_bytes(*cache), q_output, out_bytes),
                 "%s: the cache overlaps q, k, v or q_output", fn);
    const struct {
        const void* p;
        size_t bytes;
    } read[] = {{q_gamma, static_cast<size_t>(cache->head_size) * 2}, {k_gamma, static_cast<size_t>(cache->head_size) * 2},
                {batch->positions, static_cast<size_t>(t) * 4}, {batch->slots, static_cast<size_t>(t) * 4}};
    for (const auto& r : read) {
        L2_CHECK(!touches_rows(r.p, r.bytes, q_output, q_row, t, q_output_stride), "%s: q_output overlaps a gamma, positions or slots", fn);
        for (const void* c : written)
            L2_CHECK(!touches_rows(r.p, r.bytes, c, static_cast<long long>(cache->block_size) * kv_row, cache->n_blocks, block_halfs(*cache)),
                     "%s: the cache overlaps a gamma, positions or slots", fn);
    }
    return LLAMA2_OK;
}

// The most own rows that a request can have.
inline int batch_own_rows(const llama2_batch& b, int block_size)
{
    const long long rows = static_cast<long long>(b.table_stride) * block_size;
    return rows < b.max_length ? static_cast<int>(rows) : b.max_length;
}

inline int check_batch_attention(const llama2_half* output, const llama2_half* query, const llama2_batch* batch,
                                 const llama2_paged_cache* cache, int n_heads, int output_stride, int query_stride, float scale)
{
    const char* fn = "llama2_batch_attention";
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
    L2_CHECK(scale >= -3.0e37f && scale <= 3.0e37f, "%s: scale=%g is not a finite number", fn, static_cast<double>(scale));
    const size_t out_bytes = rows_bytes(b.n_tokens, output_stride, row);
    L2_CHECK(!overlap(output, out_bytes, query, rows_bytes(b.n_tokens, query_stride, row)) &&
                 !overlap(output, out_bytes, cache->key, cache_bytes(*cache)) && !overlap(output, out_bytes, cache->value, cache_bytes(*cache)),
             "%s: output overlaps query or the cache", fn);
    L2_CHECK(b.table_stride > 0 && b.max_length > 0, "%s: table_stride=%d and max_length=%d must be positive", fn, b.table_stride,
             b.max_length);
    if (b.prefix_length > kMaxBatchRows || batch_own_rows(b, cache->block_size) > kMaxBatchRows - b.prefix_length)
        return fail(LLAMA2_ERR_UNSUPPORTED, "%s: prefix_length=%d and %d own rows exceed %d", fn, b.prefix_length,
                    batch_own_rows(b, cache->block_size), kMaxBatchRows);
    const struct {
        const void* p;
        size_t ints;
    } read[] = {{b.positions, static_cast<size_t>(b.n_tokens)}, {b.query_starts, static_cast<size_t>(b.n_requests) + 1},
                {b.block_tables, static_cast<size_t>(b.n_requests) * b.table_stride},
                {b.prefix_table, (static_cast<size_t>(b.prefix_length) + cache->block_size - 1) / cache->block_size}};
    for (const auto& r : read)
        L2_CHECK(!touches_rows(r.p, r.ints * 4, output, row, b.n_tokens, output_stride),
                 "%s: output overlaps positions, query_starts or a block table", fn);
    return LLAMA2_OK;
}

// ---------------------------------------------------------------- how the attention is cut
enum class BatchAttnKernel { kNarrow, kSingle, kWide, kTall };

struct BatchAttnPlan {
    BatchAttnKernel kernel = BatchAttnKernel::kNarrow;
    int shared_tiles = 0, shared_splits = 0, shared_piece = kPass;
    int own_tiles = 0, own_splits = 1, own_piece = kPass;
    bool spread = false; // the requests' heads over all XCDs
    int own_prefix = 0; // prefix rows in front of a request's own, a multiple of kPass; 0: none, or shared
    int slots() const { return shared_splits + own_splits; }
    // (piece, key/value head) pairs by eights, one for each XCD
    long long shared_items(int n_kv_heads) const { return (static_cast<long long>(shared_splits) * n_kv_heads + 7) / 8 * 8 * shared_tiles; }
    long long items(int n_kv_heads) const { return shared_items(n_kv_heads) + static_cast<long long>(own_tiles) * own_splits * n_kv_heads; }
};

// Pieces of `rows` cache rows, for `items` of them in each piece: up to `want` workgroups altogether, but pieces not shorter
// than `shortest` nor longer than `longest`, and no more than `room` of them.
inline int batch_attn_piece(long long items, int rows, int shortest, int longest, long long want, long long room)
{
    const long long enough = want > items ? want / items : 1, most = ceil_div(rows, shortest), least = ceil_div(rows, longest);
    long long n = enough < most ? enough : most;
    n = n > least ? n : least;
    n = n < kMaxPieces ? n : kMaxPieces;
    n = n < room ? n : room;
    return round_up(ceil_div(rows, static_cast<int>(n)), kPass);
}

// Sharing pays while a request has fewer than 64 columns of its own (more fill a workgroup's columns anyway, and the
// prefix becomes the front of every request's rows: 40 requests of 32 heads, up to 2000 own rows behind 1024, 48 tokens each: shared
// 143 us, not 150; 96 tokens: 223, 178), and where the prefix, read once more for every other request, is
// more than joining the pieces costs: about 2^15 rows of a head, and a pass at least (98 requests of 40 heads behind 10
// rows: shared 36 us, not 30; 19 of 8 heads behind 333: 13.1, 15.6).
//
// Narrow tiles: pieces so that every compute unit has 4 workgroups, of 128 rows at least (one round of the 4 wavefronts;
// 777 rows of 32 heads: 64 rows 11.5 us, 128 9.9, 256 11.0) and 1024 at most, so that a long request ends with the others
// (64 conversations: 512 rows 133 us, 1024 133, 4096 170; four documents of up to 131000 rows: 215, 203, 218).
// Wide tiles are bound by the matrix cores, and the sums of their pieces weigh more than the cache.  Of prompts (64 columns
// per request): 2 workgroups per compute unit, of 1024 rows at least (40 requests of 64 tokens, nothing shared: 81 us, cut as
// below 114; of 48 tokens, cut as below, 100, so 75).  Where prompts and single tokens mix: 2 per compute unit of 128 to 1024 rows
// while a piece of all has fewer workgroups than there are compute units (a mixed step: 1 per compute unit 76 us, 2 60, 3 69;
// another one: 44, 53, 53), else 4 of 512 to 1024 rows.
//
// Wide tiles where a request has more than 16 columns on average (40 requests of 32 heads: 12 tokens narrow 60 us, wide 58; 16: 66, 61;
// 24: 90, 71).  The average stands for all: one prompt of 2048 tokens beside 255 single ones is computed in narrow tiles, 545 us where
// wide ones take 344.
//
// Rows are cut by the bounds that the host knows, not by the lengths: one request of 777 rows 8.2 us, with a max_length of 4096 9.9, of
// 131072 19.4.
inline BatchAttnPlan batch_attn_plan(const llama2_batch& b, int n_kv_heads, int group, int max_rows, int cus)
{
    BatchAttnPlan p;
    const long long columns = static_cast<long long>(b.n_tokens) * group;
    const bool fill = columns >= 64LL * b.n_requests;
    // Every piece leaves sums, a maximum and a denominator for every query row (room for heads of 128), used or not: there are no more
    // pieces than kMaxBatchScratch holds, and where it does not hold two, nothing is shared and nothing cut (200 requests of 50 tokens of
    // 32 heads, up to 8050 own rows: 1.3 GB of sums 1060 us, 0.5 GB 980; with a max_length of 131072 21.3 GB 3100, 0.5 GB 900).
    const long long room = kMaxBatchScratch / (columns * n_kv_heads * (128 + 2) * 4);
    const bool shared = !fill && static_cast<long long>(b.n_requests - 1) * b.prefix_length * n_kv_heads >= 1 << 15 && b.prefix_length >= kPass && room >= 2;
    const long long own_room = shared ? room / 2 : room > 1 ? room : 1;
    // Up to 128 shared columns are cheaper as tiles of 16 that read the prefix out of the L2 again, if that is little next to
    // the requests' own rows: the kernel without the wide tiles has 3 wavefronts per SIMD instead of 2 (72 columns, 1024
    // shared rows, up to 4000 own ones: 121 us, 130; 75 columns, 2558 and 84: 54, 42).
    const long long again = (columns + kFewRows - 1) / kFewRows - 1;
    const bool wide = columns > 128 || again * b.prefix_length * 16 > static_cast<long long>(b.n_requests) * max_rows;
    const bool many = columns > static_cast<long long>(kFewRows) * b.n_requests || (shared && wide);
    const int tile = many ? kManyRows : kFewRows;
    p.own_tiles = static_cast<int>(columns / tile) + b.n_requests;
    p.own_prefix = shared ? 0 : round_up(b.prefix_length, kPass);
    const int own_rows = p.own_prefix + max_rows;
    const long long items = static_cast<long long>(p.own_tiles) * n_kv_heads;
    if (fill)
        p.own_piece = batch_attn_piece(items, own_rows, 1024, own_rows, 2LL * cus, own_room);
    else if (many && items >= cus)
        p.own_piece = batch_attn_piece(items, own_rows, 512, 1024, 4LL * cus, own_room);
    else
        p.own_piece = batch_attn_piece(items, own_rows, 128, 1024, many ? 2LL * cus : 4LL * cus, own_room);
    p.own_splits = ceil_div(own_rows, p.own_piece);
    // A head's rows lie in few of an XCD's L2 channels: where every row is read once, an XCD takes all heads in turn; where
    // tiles read the same rows, all of a head go to one XCD, whose L2 then serves them (128 requests of 4 columns beside a wide
    // prefix: in turn 96 us, 101; 8 prompts: 102, 94).
    p.spread = columns <= static_cast<long long>(kFewRows) * b.n_requests;
    // More tiles than the GPU holds workgroups, of few rows each: a wavefront per tile (98 requests of 40 heads, 10 shared and 6 own
    // rows: 31.1 us, 16.6; 64 of 32 heads: 60 rows 16.9, 16.5; 120 rows 22.9, 27.4).
    if (many)
        // No more pieces than compute units: twice the wavefronts, which take turns with the passes, from 4 passes on (5 prompts of up
        // to 609 tokens of 8 heads 24.4 us, 21.9; 17 requests of up to 43 tokens behind 5000 rows 27.2, 23.8; two of 21 behind 388, in
        // pieces of 2 passes: 12.0, 13.6).
        p.kernel = !shared && items * p.own_splits <= cus && p.own_piece >= 4 * kPass ? BatchAttnKernel::kTall : BatchAttnKernel::kWide;
    else if (!shared && p.own_splits == 1 && b.prefix_length + max_rows <= kPass && items >= 3LL * cus)
        p.kernel = BatchAttnKernel::kSingle;
    if (shared) {
        p.shared_tiles = static_cast<int>((columns + tile - 1) / tile);
        // A workgroup per compute unit (16 samples behind 2048 rows 17.2 us, twice as many workgroups 20.8); of wide tiles half a
        // one beside long rows of the requests' own, which need the rest (128 requests behind 8192 rows, up to 2001 own ones: 92 us,
        // 98; 25 behind 11736, at most 24 own ones: 25.7, 20.2), and up to 2048 rows, whose sums weigh less (the first case
        // with 1024: 97; 109 behind 7911 52 -> 46, with up to 4096: 74).
        p.shared_piece = batch_attn_piece(static_cast<long long>(p.shared_tiles) * n_kv_heads, b.prefix_length, 128, many ? 2048 : 1024,
                                          many && max_rows > 2 * kPass ? cus / 2 : cus, room - p.own_splits);
        p.shared_splits = ceil_div(b.prefix_length, p.shared_piece);
    }
    return p;
}

// Launches hold less than 2^32 threads.
inline int check_batch_attn_plan(const BatchAttnPlan& p, int n_tokens, int n_heads, int n_kv_heads)
{
    if (p.items(n_kv_heads) >= 1 << 24 || static_cast<long long>(n_tokens) * n_heads >= 1 << 26)
        return fail(LLAMA2_ERR_UNSUPPORTED, "llama2_batch_attention: %d tokens of %d heads in %lld pieces are too many", n_tokens, n_heads,
                    p.items(n_kv_heads));
    return LLAMA2_OK;
}

} // namespace l2
