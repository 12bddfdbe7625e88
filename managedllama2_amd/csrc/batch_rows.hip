// Row operators of a step of several requests: the residual with the norms around it, and log probabilities with entropy and
// the most likely tokens.
#include "common.hpp"
#include "batch_product_plan.hpp"

#include <cmath>

namespace l2 {

// Sum over a workgroup of WAVES wavefronts, in every thread.
template <int WAVES>
__device__ __forceinline__ float block_sum(float v, float* lds /* WAVES */)
{
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0)
        lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = lds[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w)
        t += lds[w];
    __syncthreads();
    return t;
}

template <int WAVES>
__device__ __forceinline__ float block_max(float v, float* lds)
{
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0)
        lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = lds[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w)
        t = fmaxf(t, lds[w]);
    __syncthreads();
    return t;
}

// ---------------------------------------------------------------- residual and norms
struct NormRowsArgs {
    uint16_t* output;
    uint16_t* residual_output;
    const uint16_t* residual;
    const uint16_t* input;
    const uint16_t* gamma;
    const uint16_t* input_gamma;
    const uint16_t* gate;
    const int* positions;
    int size, output_stride, residual_output_stride, residual_stride, input_stride;
    float scale, eps;
};

// A workgroup per row, which stays in registers between its one reading and its writing: PIECES of 8 elements per thread.
template <int WAVES, int PIECES>
__global__ __launch_bounds__(WAVES * 64) void batch_norm_kernel(NormRowsArgs a)
{
    __shared__ float lds[WAVES];
    const int t = blockIdx.x;
    if (a.positions[t] < 0)
        return;
    const size_t row = static_cast<size_t>(t);
    auto at = [](int i) { return (threadIdx.x + i * WAVES * 64) * 8; };
    auto half_of = [](u32x4 v, int k) { return half_bits_to_float(static_cast<uint16_t>(v[k >> 1] >> (16 * (k & 1)))); };
    float r[PIECES][8];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        u32x4 v = {};
        if (at(i) < a.size)
            v = *reinterpret_cast<const u32x4*>(a.residual + row * a.residual_stride + at(i));
#pragma unroll
        for (int k = 0; k < 8; ++k)
            r[i][k] = half_of(v, k);
    }
    if (a.input) {
        u32x4 y[PIECES] = {};
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
            if (at(i) < a.size)
                y[i] = *reinterpret_cast<const u32x4*>(a.input + row * a.input_stride + at(i));
        float norm = 1.0f;
        if (a.input_gamma) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    ss = __builtin_fmaf(half_of(y[i], k), half_of(y[i], k), ss);
            norm = 1.0f / sqrtf(block_sum<WAVES>(ss, lds) / static_cast<float>(a.size) + a.eps);
        }
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if (at(i) >= a.size)
                continue;
            float f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                f[k] = half_of(y[i], k);
            if (a.input_gamma) {
                const u32x4 g = *reinterpret_cast<const u32x4*>(a.input_gamma + at(i));
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    f[k] *= norm * half_of(g, k);
            }
            if (a.gate) {
                const u32x4 g = *reinterpret_cast<const u32x4*>(a.gate + at(i));
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    f[k] *= half_of(g, k);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                r[i][k] = __builtin_fmaf(a.scale, f[k], r[i][k]);
        }
    }
    auto store = [&](uint16_t* p, int i, const float* f) {
        u32x4 o;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            o[k] = static_cast<uint32_t>(float_to_half_bits(f[2 * k])) | static_cast<uint32_t>(float_to_half_bits(f[2 * k + 1])) << 16;
        *reinterpret_cast<u32x4*>(p + at(i)) = o;
    };
    if (a.residual_output)
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
            if (at(i) < a.size)
                store(a.residual_output + row * a.residual_output_stride, i, r[i]);
    if (!a.output)
        return;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k)
            ss = __builtin_fmaf(r[i][k], r[i][k], ss);
    const float norm = 1.0f / sqrtf(block_sum<WAVES>(ss, lds) / static_cast<float>(a.size) + a.eps);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        if (at(i) >= a.size)
            continue;
        const u32x4 g = *reinterpret_cast<const u32x4*>(a.gamma + at(i));
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            f[k] = r[i][k] * (norm * half_of(g, k));
        store(a.output + row * a.output_stride, i, f);
    }
}

// ---------------------------------------------------------------- log probabilities
struct LogProbArgs {
    float* log_probs;
    float* entropies;
    int* top_tokens;
    float* top_log_probs;
    const uint16_t* logits;
    const int* tokens;
    const int* positions;
    int vocab, stride, n_tokens, n_top;
    float inverse, per_e; // 1 / temperature, and with log2(e)
};

// A number that orders as the logits do, NaN lowest: larger is likelier, equal numbers are equal (-0 as 0).
__device__ __forceinline__ unsigned order_of(uint16_t h)
{
    if ((h & 0x7FFFu) > 0x7C00u)
        return 0;
    if (h == 0x8000u)
        h = 0;
    return h & 0x8000u ? 0xFFFFu ^ h : h | 0x8000u; // -infinity: 0x03FF
}

constexpr int kLogProbThreads = 1024, kCandidates = 2048;

// A workgroup per row.  Its threads' largest logits bound the n_top-th largest from below (the n_top-th of 1024 maxima); what
// reaches that bound is collected and ranked by comparison.  Where more than kCandidates do (rows of equal logits), the bound is
// found bit by bit, and of the equal ones the first by their index are taken.
__global__ __launch_bounds__(kLogProbThreads) void batch_log_probs_kernel(LogProbArgs a)
{
    constexpr int WAVES = kLogProbThreads / 64;
    __shared__ float lds[WAVES];
    __shared__ unsigned maxima[kLogProbThreads];
    __shared__ unsigned long long found[kCandidates];
    __shared__ int count, bound;
    const int row = blockIdx.x, tid = threadIdx.x;
    if (a.positions && a.positions[row] < 0)
        return;
    const uint16_t* x = a.logits + static_cast<size_t>(row) * a.stride;
    float top = -INFINITY;
    unsigned largest = 0;
    bool nan = false;
    for (int i = tid; i < a.vocab; i += kLogProbThreads) {
        const float v = half_bits_to_float(x[i]);
        nan = nan || v != v;
        top = fmaxf(top, v);
        largest = max(largest, order_of(x[i]));
    }
    top = block_max<WAVES>(top, lds);
    float total = 0.0f, moment = 0.0f;
    if (top > -INFINITY && top < INFINITY) {
        for (int i = tid; i < a.vocab; i += kLogProbThreads) {
            const float d = half_bits_to_float(x[i]) - top;
            const float e = __builtin_amdgcn_exp2f(d * a.per_e);
            total += e;
            moment = e > 0.0f ? __builtin_fmaf(e, d, moment) : moment;
        }
    }
    total = block_sum<WAVES>(total, lds);
    moment = block_sum<WAVES>(moment, lds);
    const bool wrong = __syncthreads_or(nan) || top == INFINITY;
    const float log_total = logf(total);
    auto log_prob = [&](float v) {
        return wrong ? NAN : v == -INFINITY ? -INFINITY : (v - top) * a.inverse - log_total;
    };
    if (a.log_probs)
        for (int i = tid; i < a.n_tokens; i += kLogProbThreads) {
            const int token = a.tokens[static_cast<size_t>(row) * a.n_tokens + i];
            const bool there = token >= 0 && token < a.vocab;
            a.log_probs[static_cast<size_t>(row) * a.n_tokens + i] = there ? log_prob(half_bits_to_float(x[token])) : -INFINITY;
        }
    if (a.entropies && tid == 0)
        a.entropies[row] = wrong ? NAN : top == -INFINITY ? 0.0f : log_total - moment * a.inverse / total;
    if (a.n_top == 0)
        return;
    // the n_top-th largest of the threads' maxima (threads without a logit have 0, which bounds everything)
    const int want = min(a.n_top, a.vocab);
    maxima[tid] = largest;
    if (tid == 0)
        count = 0;
    __syncthreads();
    int above = 0;
    for (int j = 0; j < kLogProbThreads; ++j) {
        const unsigned o = maxima[j];
        above += o > largest || (o == largest && j < tid);
    }
    if (above == want - 1)
        bound = static_cast<int>(largest);
    __syncthreads();
    unsigned least = static_cast<unsigned>(bound);
    auto key = [&](unsigned order, int i) { return static_cast<unsigned long long>(order) << 32 | (0xFFFFFFFFu - i); };
    for (int i = tid; i < a.vocab; i += kLogProbThreads) {
        const unsigned o = order_of(x[i]);
        if (o >= least) {
            const int at = atomicAdd(&count, 1);
            if (at < kCandidates)
                found[at] = key(o, i);
        }
    }
    __syncthreads();
    int have = count;
    if (have > kCandidates) { // uniform
        // the largest bound that `want` logits reach, bit by bit
        unsigned reach = 0;
        for (int bit = 15; bit >= 0; --bit) {
            const unsigned probe = reach | 1u << bit;
            int n = 0;
            for (int i = tid; i < a.vocab; i += kLogProbThreads)
                n += order_of(x[i]) >= probe;
            __syncthreads();
            if (tid == 0)
                count = 0;
            __syncthreads();
            if (n)
                atomicAdd(&count, n);
            __syncthreads();
            if (count >= want)
                reach = probe;
        }
        __syncthreads();
        if (tid == 0)
            count = 0;
        __syncthreads();
        for (int i = tid; i < a.vocab; i += kLogProbThreads) {
            const unsigned o = order_of(x[i]);
            if (o > reach)
                found[atomicAdd(&count, 1)] = key(o, i); // fewer than `want`
        }
        __syncthreads();
        // the equal ones in order, a thousand at a time
        for (int first = 0; first < a.vocab; first += kLogProbThreads) {
            const int before = count;
            if (before >= want)
                break;
            const bool equal = first + tid < a.vocab && order_of(x[first + tid]) == reach;
            maxima[tid] = equal;
            __syncthreads();
            if (equal) {
                int at = before;
                for (int j = 0; j < tid; ++j)
                    at += maxima[j];
                if (at < want)
                    found[at] = key(reach, first + tid);
            }
            const int n = __syncthreads_count(equal);
            if (tid == 0)
                count = min(before + n, want);
            __syncthreads();
        }
        have = want;
    }
    for (int i = tid; i < have; i += kLogProbThreads) {
        int rank = 0;
        for (int j = 0; j < have; ++j)
            rank += found[j] > found[i];
        if (rank >= a.n_top)
            continue;
        const int token = static_cast<int>(0xFFFFFFFFu - static_cast<unsigned>(found[i]));
        a.top_tokens[static_cast<size_t>(row) * a.n_top + rank] = token;
        if (a.top_log_probs)
            a.top_log_probs[static_cast<size_t>(row) * a.n_top + rank] = log_prob(half_bits_to_float(x[token]));
    }
    for (int i = want + tid; i < a.n_top; i += kLogProbThreads) {
        a.top_tokens[static_cast<size_t>(row) * a.n_top + i] = -1;
        if (a.top_log_probs)
            a.top_log_probs[static_cast<size_t>(row) * a.n_top + i] = -INFINITY;
    }
}

} // namespace l2

using namespace l2;

extern "C" {

int llama2_batch_residual_rmsnorm(llama2_half* output, llama2_half* residual_output, const llama2_half* residual, const llama2_half* input,
                                  const llama2_half* gamma, const llama2_half* input_gamma, const llama2_half* gate, const llama2_batch* batch,
                                  int size, int output_stride, int residual_output_stride, int residual_stride, int input_stride,
                                  float residual_scale, float eps)
{
    L2_REQUIRE_INIT();
    if (int rc = check_batch_norm(output, residual_output, residual, input, gamma, input_gamma, gate, batch, size, output_stride,
                                  residual_output_stride, residual_stride, input_stride, residual_scale, eps))
        return rc;
    const NormRowsArgs a = {output, residual_output, residual, input, gamma, input_gamma, gate, batch->positions, size, output_stride,
                            residual_output_stride, residual_stride, input_stride, residual_scale, eps};
    const dim3 grid(batch->n_tokens);
    const hipStream_t st = ctx().stream;
    if (size <= 2048)
        hipLaunchKernelGGL((batch_norm_kernel<4, 1>), grid, dim3(256), 0, st, a);
    else if (size <= 8192)
        hipLaunchKernelGGL((batch_norm_kernel<16, 1>), grid, dim3(1024), 0, st, a);
    else if (size <= 16384)
        hipLaunchKernelGGL((batch_norm_kernel<16, 2>), grid, dim3(1024), 0, st, a);
    else
        hipLaunchKernelGGL((batch_norm_kernel<16, 8>), grid, dim3(1024), 0, st, a);
    L2_LAUNCH_CHECK("llama2_batch_residual_rmsnorm");
    return LLAMA2_OK;
}

int llama2_batch_log_probs(float* log_probs, float* entropies, int* top_tokens, float* top_log_probs, const llama2_half* logits,
                           const int* tokens, const int* positions, int n_rows, int vocab_size, int logits_stride, int n_tokens, int n_top,
                           float temperature)
{
    L2_REQUIRE_INIT();
    if (int rc = check_batch_log_probs(log_probs, entropies, top_tokens, top_log_probs, logits, tokens, positions, n_rows, vocab_size,
                                       logits_stride, n_tokens, n_top, temperature))
        return rc;
    const double inverse = 1.0 / static_cast<double>(temperature);
    const LogProbArgs a = {log_probs, entropies, top_tokens, top_log_probs, logits, tokens, positions, vocab_size, logits_stride, n_tokens,
                           n_top, static_cast<float>(inverse), static_cast<float>(inverse * 1.4426950408889634)};
    hipLaunchKernelGGL(batch_log_probs_kernel, dim3(n_rows), dim3(kLogProbThreads), 0, ctx().stream, a);
    L2_LAUNCH_CHECK("llama2_batch_log_probs");
    return LLAMA2_OK;
}

} // extern "C"
