// Host side of the products, norms and log probabilities of a step of several requests, without a GPU call in it: what
// arguments are refused, and how the products are cut into workgroups.  Uses L2_CHECK, fail, aligned, overlap and ceil_div of
// whoever includes it.
#pragma once

#include "batch_plan.hpp"

namespace l2 {

constexpr int kMaxProductRows = 1 << 16; // inputs of a tensor
constexpr int kMaxGatedRows = 1 << 15; // of a gate and an up projection, whose scales a workgroup holds side by side
constexpr int kMaxProductCols = 1 << 20; // outputs of a tensor
constexpr int kMaxStride = 1 << 24; // of the input: offsets within 64 rows are ints
constexpr int kMaxAdapters = 1 << 20;
constexpr int kMaxRank = 128;
constexpr int kMaxNormSize = 1 << 16;
constexpr int kMaxVocab = 1 << 20; // 32 segments of 32768
constexpr int kMaxGiven = 1024;

inline int weight_words(int rows) { return ceil_div(rows, 32) * 4; } // of an output
inline int weight_groups(int rows) { return ceil_div(rows, 128); }
inline int zero_words(int rows) { return ceil_div(weight_groups(rows), 8); }

inline long long down_halfs(const llama2_adapters& a, int rows)
{
    return a.down_stride ? a.down_stride : static_cast<long long>(a.max_rank) * rows;
}
inline long long up_halfs(const llama2_adapters& a, int cols) { return a.up_stride ? a.up_stride : static_cast<long long>(cols) * a.max_rank; }

inline size_t pool_bytes(int n, long long stride, long long halfs) { return static_cast<size_t>((n - 1) * stride + halfs) * 2; }

// Rows of halfs that a call writes, or reads beside them.
struct HalfRows {
    const void* p;
    int width, stride;
};

inline bool half_rows_overlap(const HalfRows& a, const HalfRows& b, int n)
{
    if (a.stride == b.stride)
        return rows_overlap(a.p, a.width, b.p, b.width, n, a.stride);
    return overlap(a.p, rows_bytes(n, a.stride, a.width), b.p, rows_bytes(n, b.stride, b.width));
}

inline int check_adapters(const char* fn, const llama2_adapters* a, int rows, int cols, const int* token_adapters)
{
    if (!a)
        return LLAMA2_OK;
    L2_CHECK(a->down && a->up && a->scales && a->ranks && token_adapters, "%s: null pointer in the adapters, or no token_adapters", fn);
    L2_CHECK(aligned(a->down, 16) && aligned(a->up, 16) && aligned(a->scales, 4) && aligned(a->ranks, 4) && aligned(token_adapters, 4),
             "%s: misaligned array of adapters", fn);
    L2_CHECK(a->n_adapters > 0 && a->n_adapters <= kMaxAdapters, "%s: n_adapters=%d must be 1 .. %d", fn, a->n_adapters, kMaxAdapters);
    L2_CHECK(a->max_rank > 0 && a->max_rank <= kMaxRank && a->max_rank % 8 == 0, "%s: max_rank=%d must be a multiple of 8 up to %d", fn,
             a->max_rank, kMaxRank);
    const long long down = static_cast<long long>(a->max_rank) * rows, up = static_cast<long long>(a->max_rank) * cols;
    const long long most = (1LL << 45) / a->n_adapters;
    L2_CHECK(a->down_stride == 0 || (a->down_stride >= down && a->down_stride % 8 == 0 && a->down_stride <= most),
             "%s: down_stride=%lld must be 0 or a multiple of 8 of at least %lld halfs", fn, a->down_stride, down);
    L2_CHECK(a->up_stride == 0 || (a->up_stride >= up && a->up_stride % 8 == 0 && a->up_stride <= most),
             "%s: up_stride=%lld must be 0 or a multiple of 8 of at least %lld halfs", fn, a->up_stride, up);
    return LLAMA2_OK;
}

// What the products of many rows share: the input, a tensor and its adapters, and that `out` overlaps none of them.
inline int check_product_input(const char* fn, const llama2_half* input, int rows, int most_rows, int input_stride,
                               const int* token_adapters, const llama2_batch* batch)
{
    if (int rc = check_batch(fn, batch))
        return rc;
    L2_CHECK(input && batch->positions, "%s: null pointer", fn);
    L2_CHECK(aligned(input, 16), "%s: input must be 16-byte aligned", fn);
    L2_CHECK(aligned(token_adapters, 4), "%s: misaligned token_adapters", fn);
    L2_CHECK(rows > 0 && rows % 8 == 0, "%s: rows=%d must be a positive multiple of 8", fn, rows);
    if (rows > most_rows)
        return fail(LLAMA2_ERR_UNSUPPORTED, "%s: rows=%d exceeds %d", fn, rows, most_rows);
    L2_CHECK(input_stride >= rows && input_stride % 8 == 0, "%s: input_stride=%d must be a multiple of 8 and hold a row of %d", fn,
             input_stride, rows);
    if (input_stride > kMaxStride)
        return fail(LLAMA2_ERR_UNSUPPORTED, "%s: input_stride=%d exceeds %d", fn, input_stride, kMaxStride);
    return LLAMA2_OK;
}

inline int check_product_tensor(const char* fn, const llama2_qweight& w, int cols)
{
    L2_CHECK(w.weight && w.zeros && w.scales, "%s: null pointer in a tensor", fn);
    L2_CHECK(aligned(w.weight, 16) && aligned(w.zeros, 4) && aligned(w.scales, 2),
             "%s: weights must be 16-byte aligned, zeros and scales to their size", fn);
    L2_CHECK(cols > 0 && cols % 8 == 0, "%s: cols=%d must be a positive multiple of 8", fn, cols);
    if (cols > kMaxProductCols)
        return fail(LLAMA2_ERR_UNSUPPORTED, "%s: cols=%d exceeds %d", fn, cols, kMaxProductCols);
    return LLAMA2_OK;
}

inline int check_output_apart(const char* fn, const HalfRows& out, const llama2_qweight& w, const llama2_adapters* a, int rows, int cols,
                              const llama2_half* input, int input_stride, const int* token_adapters, const llama2_batch& b)
{
    const int t = b.n_tokens;
    L2_CHECK(!half_rows_overlap(out, {input, rows, input_stride}, t), "%s: an output overlaps the input", fn);
    const size_t n = static_cast<size_t>(cols);
    const struct {
        const void* p;
        size_t bytes;
    } read[] = {{w.weight, n * weight_words(rows) * 4}, {w.zeros, n * zero_words(rows) * 4}, {w.scales, n * weight_groups(rows) * 2},
                {b.positions, static_cast<size_t>(t) * 4}, {token_adapters, static_cast<size_t>(t) * 4},
                {a ? a->scales : nullptr, a ? static_cast<size_t>(a->n_adapters) * 4 : 0},
                {a ? a->ranks : nullptr, a ? static_cast<size_t>(a->n_adapters) * 4 : 0},
                {a ? a->down : nullptr, a ? pool_bytes(a->n_adapters, down_halfs(*a, rows), static_cast<long long>(a->max_rank) * rows) : 0},
                {a ? a->up : nullptr, a ? pool_bytes(a->n_adapters, up_halfs(*a, cols), static_cast<long long>(a->max_rank) * cols) : 0}};
    for (const auto& r : read)
        L2_CHECK(!touches_rows(r.p, r.bytes, out.p, out.width, t, out.stride),
                 "%s: an output overlaps a tensor, adapters, positions or token_adapters", fn);
    return LLAMA2_OK;
}

inline int check_batch_mat_mul(const llama2_batch_matrix* m, int n_matrices, const llama2_half* input, int rows, int input_stride,
                               const int* token_adapters, const llama2_batch* batch)
{
    const char* fn = "llama2_batch_mat_mul_int4";
    if (int rc = check_product_input(fn, input, rows, kMaxProductRows, input_stride, token_adapters, batch))
        return rc;
    L2_CHECK(m && n_matrices > 0 && n_matrices <= LLAMA2_MAX_BATCH_MATRICES, "%s: n_matrices=%d must be 1 .. %d, and matrices not null", fn,
             n_matrices, LLAMA2_MAX_BATCH_MATRICES);
    const int t = batch->n_tokens;
    for (int i = 0; i < n_matrices; ++i) {
        if (int rc = check_product_tensor(fn, m[i].weight, m[i].cols))
            return rc;
        L2_CHECK(m[i].output && aligned(m[i].output, 16) && aligned(m[i].residual, 16), "%s: null or misaligned output, or residual", fn);
        L2_CHECK(m[i].output_stride >= m[i].cols && m[i].output_stride % 8 == 0 &&
                     (!m[i].residual || (m[i].residual_stride >= m[i].cols && m[i].residual_stride % 8 == 0)),
                 "%s: strides %d, %d must be multiples of 8 and hold a row of %d", fn, m[i].output_stride, m[i].residual_stride, m[i].cols);
        if (int rc = check_adapters(fn, m[i].adapters, rows, m[i].cols, token_adapters))
            return rc;
    }
    for (int i = 0; i < n_matrices; ++i) {
        const HalfRows out = {m[i].output, m[i].cols, m[i].output_stride};
        for (int j = 0; j < n_matrices; ++j) {
            if (int rc = check_output_apart(fn, out, m[j].weight, m[j].adapters, rows, m[j].cols, input, input_stride, token_adapters, *batch))
                return rc;
            L2_CHECK(i == j || !half_rows_overlap(out, {m[j].output, m[j].cols, m[j].output_stride}, t), "%s: outputs overlap", fn);
            if (!m[j].residual || (i == j && m[j].residual == m[j].output && m[j].residual_stride == m[j].output_stride))
                continue;
            L2_CHECK(!half_rows_overlap(out, {m[j].residual, m[j].cols, m[j].residual_stride}, t),
                     "%s: an output overlaps a residual without being it", fn);
        }
    }
    return LLAMA2_OK;
}

inline int check_batch_swiglu(const llama2_half* output, const llama2_half* input, const llama2_qweight* gate, const llama2_qweight* up,
                              int rows, int cols, int output_stride, int input_stride, const llama2_adapters* gate_adapters,
                              const llama2_adapters* up_adapters, const int* token_adapters, const llama2_batch* batch)
{
    const char* fn = "llama2_batch_mat_mul_swiglu";
    if (int rc = check_product_input(fn, input, rows, kMaxGatedRows, input_stride, token_adapters, batch))
        return rc;
    L2_CHECK(output && aligned(output, 16) && gate && up, "%s: null pointer, or misaligned output", fn);
    const llama2_qweight* w[] = {gate, up};
    const llama2_adapters* a[] = {gate_adapters, up_adapters};
    for (int i = 0; i < 2; ++i) {
        if (int rc = check_product_tensor(fn, *w[i], cols))
            return rc;
        if (int rc = check_adapters(fn, a[i], rows, cols, token_adapters))
            return rc;
    }
    L2_CHECK(output_stride >= cols && output_stride % 8 == 0, "%s: output_stride=%d must be a multiple of 8 and hold a row of %d", fn,
             output_stride, cols);
    for (int i = 0; i < 2; ++i)
        if (int rc = check_output_apart(fn, {output, cols, output_stride}, *w[i], a[i], rows, cols, input, input_stride, token_adapters, *batch))
            return rc;
    return LLAMA2_OK;
}

inline int check_batch_norm(const llama2_half* output, const llama2_half* residual_output, const llama2_half* residual,
                            const llama2_half* input, const llama2_half* gamma, const llama2_half* input_gamma, const llama2_half* gate,
                            const llama2_batch* batch, int size, int output_stride, int residual_output_stride, int residual_stride,
                            int input_stride, float residual_scale, float eps)
{
    const char* fn = "llama2_batch_residual_rmsnorm";
    if (int rc = check_batch(fn, batch))
        return rc;
    const int t = batch->n_tokens;
    L2_CHECK(residual && batch->positions && (output || residual_output) && (gamma || !output),
             "%s: null pointer (residual, positions, an output and, with output, gamma are needed)", fn);
    L2_CHECK(input || (!input_gamma && !gate), "%s: input_gamma or gate without an input", fn);
    L2_CHECK(aligned(output, 16) && aligned(residual_output, 16) && aligned(residual, 16) && aligned(input, 16) && aligned(gamma, 16) &&
                 aligned(input_gamma, 16) && aligned(gate, 16), "%s: pointers must be 16-byte aligned", fn);
    L2_CHECK(size > 0 && size % 8 == 0, "%s: size=%d must be a positive multiple of 8", fn, size);
    if (size > kMaxNormSize)
        return fail(LLAMA2_ERR_UNSUPPORTED, "%s: size=%d exceeds %d", fn, size, kMaxNormSize);
    auto holds = [&](const void* p, int stride) { return !p || (stride >= size && stride % 8 == 0); };
    L2_CHECK(holds(output, output_stride) && holds(residual_output, residual_output_stride) && holds(residual, residual_stride) &&
                 holds(input, input_stride), "%s: strides %d, %d, %d, %d must be multiples of 8 and hold a row of %d", fn, output_stride,
             residual_output_stride, residual_stride, input_stride, size);
    L2_CHECK(residual_scale >= -3.0e38f && residual_scale <= 3.0e38f, "%s: residual_scale=%g is not a finite number", fn,
             static_cast<double>(residual_scale));
    L2_CHECK(eps >= 0.0f && eps <= 3.0e38f, "%s: eps=%g must not be negative", fn, static_cast<double>(eps));
    const HalfRows written[] = {{output, size, output_stride}, {residual_output, size, residual_output_stride}},
                   read[] = {{input, size, input_stride}, {residual, size, residual_stride}}; // each may be the output of its place
    for (int i = 0; i < 2; ++i) {
        if (!written[i].p)
            continue;
        if (i == 1 && output)
            L2_CHECK(!half_rows_overlap(written[0], written[1], t), "%s: outputs overlap", fn);
        for (int j = 0; j < 2; ++j) {
            const bool in_place = i == j && written[i].p == read[j].p && written[i].stride == read[j].stride;
            L2_CHECK(!read[j].p || in_place || !half_rows_overlap(written[i], read[j], t),
                     "%s: an output overlaps an input (output may be input, and residual_output residual)", fn);
        }
        const struct {
            const void* p;
            size_t bytes;
        } vectors[] = {{gamma, static_cast<size_t>(size) * 2}, {input_gamma, static_cast<size_t>(size) * 2},
                       {gate, static_cast<size_t>(size) * 2}, {batch->positions, static_cast<size_t>(t) * 4}};
        for (const auto& v : vectors)
            L2_CHECK(!touches_rows(v.p, v.bytes, written[i].p, size, t, written[i].stride), "%s: an output overlaps a gamma, the gate or positions",
                     fn);
    }
    return LLAMA2_OK;
}

inline int check_batch_log_probs(const float* log_probs, const float* entropies, const int* top_tokens, const float* top_log_probs,
                                 const llama2_half* logits, const int* tokens, const int* positions, int n_rows, int vocab_size,
                                 int logits_stride, int n_tokens, int n_top, float temperature)
{
    const char* fn = "llama2_batch_log_probs";
    L2_CHECK(logits && (log_probs || entropies || top_tokens), "%s: null logits, or nothing to compute", fn);
    L2_CHECK(aligned(logits, 2) && aligned(log_probs, 4) && aligned(entropies, 4) && aligned(top_tokens, 4) && aligned(top_log_probs, 4) &&
                 aligned(tokens, 4) && aligned(positions, 4), "%s: misaligned pointer", fn);
    L2_CHECK(n_rows > 0 && n_rows <= kMaxBatchTokens, "%s: n_rows=%d must be 1 .. %d", fn, n_rows, kMaxBatchTokens);
    L2_CHECK(vocab_size > 0, "%s: vocab_size=%d must be positive", fn, vocab_size);
    if (vocab_size > kMaxVocab)
        return fail(LLAMA2_ERR_UNSUPPORTED, "%s: vocab_size=%d exceeds %d", fn, vocab_size, kMaxVocab);
    L2_CHECK(logits_stride >= vocab_size, "%s: logits_stride=%d holds no row of %d", fn, logits_stride, vocab_size);
    L2_CHECK(n_tokens >= 0 && n_tokens <= kMaxGiven && (n_tokens > 0) == (log_probs != nullptr) && (tokens || n_tokens == 0),
             "%s: n_tokens=%d must be 0 .. %d, and 0 where log_probs is null", fn, n_tokens, kMaxGiven);
    L2_CHECK(n_top >= 0 && n_top <= LLAMA2_MAX_TOP_TOKENS && (n_top > 0) == (top_tokens != nullptr) && (top_tokens || !top_log_probs),
             "%s: n_top=%d must be 0 .. %d, and 0 where top_tokens is null", fn, n_top, LLAMA2_MAX_TOP_TOKENS);
    L2_CHECK(temperature > 1.0e-30f && temperature <= 1.0e30f, "%s: temperature=%g must be a positive number", fn,
             static_cast<double>(temperature));
    const size_t r = static_cast<size_t>(n_rows);
    const struct {
        const void* p;
        size_t bytes;
    } written[] = {{log_probs, r * n_tokens * 4}, {entropies, entropies ? r * 4 : 0}, {top_tokens, r * n_top * 4},
                   {top_log_probs, top_log_probs ? r * n_top * 4 : 0}},
      read[] = {{logits, rows_bytes(n_rows, logits_stride, vocab_size)}, {tokens, r * n_tokens * 4}, {positions, positions ? r * 4 : 0}};
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < i; ++j)
            L2_CHECK(!written[i].bytes || !written[j].bytes || !overlap(written[i].p, written[i].bytes, written[j].p, written[j].bytes),
                     "%s: outputs overlap", fn);
        for (const auto& x : read)
            L2_CHECK(!written[i].bytes || !x.bytes || !overlap(written[i].p, written[i].bytes, x.p, x.bytes), "%s: an output overlaps an input", fn);
    }
    return LLAMA2_OK;
}

// ---------------------------------------------------------------- scratch of the products
// What a tensor's adapters leave for its product, per token and 16 ranks (a block): the scale of the adapter with the block's power of
// two, and the adapter's rank.
struct TokenAdapter {
    float factor;
    int rank;
};

constexpr size_t kLowBytes = 64; // what 16 ranks of a token receive: looked up as one piece, on its multiples

// Where that lies behind the operands: what the ranks of all tensors receive first, which stays on multiples of kLowBytes whatever the
// number of tokens, then the factors.
struct LowScratch {
    size_t low[LLAMA2_MAX_BATCH_MATRICES], info[LLAMA2_MAX_BATCH_MATRICES], bytes;
};

// operands: bytes, a multiple of kLowBytes; max_ranks: of a tensor's adapters, 0 without.
inline LowScratch low_scratch(size_t operands, int tokens, const int* max_ranks, int n_matrices)
{
    LowScratch s = {};
    s.bytes = operands;
    for (int i = 0; i < n_matrices; ++i) {
        s.low[i] = s.bytes;
        s.bytes += static_cast<size_t>(tokens) * ceil_div(max_ranks[i], 16) * kLowBytes;
    }
    for (int i = 0; i < n_matrices; ++i) {
        s.info[i] = s.bytes;
        s.bytes += static_cast<size_t>(tokens) * ceil_div(max_ranks[i], 16) * sizeof(TokenAdapter);
    }
    return s;
}

// ---------------------------------------------------------------- how rows of logits are cut
constexpr int kLogProbRows = 1 << 15; // of a launch

struct LogProbShape {
    int segments, length, pieces; // length: of a segment; pieces: of 4096 logits that it takes at most, 1, 2, 4 or 8
};

// A workgroup holds up to 32768 logits.  Few rows are cut until there are as many workgroups as compute units, into pieces of 4096 at
// least; the likeliest of all segments are ranked by comparison with each other, 512 of them while there is a choice.
inline LogProbShape log_prob_shape(int rows, int vocab, int n_top, int cus)
{
    const int least = ceil_div(vocab, 1 << 15), most = ceil_div(vocab, 1 << 12);
    int n = cus / rows < most ? cus / rows : most;
    n = n < 64 ? n : 64; // a lane each puts them together
    n = n_top > 0 && n > 512 / n_top ? 512 / n_top : n;
    n = n > least ? n : least;
    LogProbShape s;
    s.length = round_up(ceil_div(vocab, n), 8);
    s.segments = ceil_div(vocab, s.length);
    const int pieces = ceil_div(s.length, 1 << 12);
    s.pieces = pieces <= 2 ? pieces : pieces <= 4 ? 4 : 8;
    return s;
}

} // namespace l2
