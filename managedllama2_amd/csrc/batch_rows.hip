// Row operators of a step of several requests: the residual with the norms around it, and log probabilities with entropy and
// the most likely tokens.
#include "common.hpp"
#include "batch_product_plan.hpp"

#include <cmath>
#include <type_traits>

namespace l2 {

// Sum over a workgroup of up to 16 wavefronts, in every thread.
__device__ __forceinline__ float block_sum(float v, float* lds /* 16 */)
{
    v = wave_sum(v);
    const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
        lds[wave] = v;
    __syncthreads();
    float t = lds[0];
    for (int w = 1; w < waves; ++w)
        t += lds[w];
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
//
// HBM bounds many rows: 4000 rows of 5120 with both norms and a gate 28 us, 5.8 TB/s; with results that pass through the L2 (which
// cannot hold them) 39.6, with one piece per thread, and so ten wavefronts to a sum, 34.4.  Few rows are latency: 48 rows of 4096 3.9 us, with two
// pieces 4.3.
template <int PIECES, bool THROUGH>
__global__ __launch_bounds__(1024) void batch_norm_kernel(NormRowsArgs a)
{
    __shared__ float lds[16];
    const int t = blockIdx.x;
    if (a.positions[t] < 0)
        return;
    const size_t row = static_cast<size_t>(t);
    auto at = [](int i) { return static_cast<int>(threadIdx.x + i * blockDim.x) * 8; };
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
            norm = 1.0f / sqrtf(block_sum(ss, lds) / static_cast<float>(a.size) + a.eps);
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
        if constexpr (THROUGH)
            __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(p + at(i)));
        else
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
    const float norm = 1.0f / sqrtf(block_sum(ss, lds) / static_cast<float>(a.size) + a.eps);
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
    float* parts;       // several segments: [row][segment] of 4 floats (largest, sum, moment), then [row][segment][n_top] keys
    unsigned* counters; // per row, zero between launches
    int vocab, stride, n_tokens, n_top, segments, length; // length: of a segment, a multiple of 8
    float inverse, per_e; // 1 / temperature, and with log2(e)
};

// A number that orders as the logits do, NaN lowest: larger is likelier, equal numbers are equal (-0 as 0).
__device__ __forceinline__ unsigned order_of(uint16_t h)
{
    if ((h & 0x7FFFu) > 0x7C00u)
        return 0;
    if (h == 0x8000u)
        h = 0;
    return h & 0x8000u ? 0xFFFFu ^ h : h | 0x8000u;
}
constexpr unsigned kOrderOfNothing = 0x03FF; // -infinity

__device__ __forceinline__ float logit_of(unsigned order)
{
    return order == 0 ? NAN : half_bits_to_float(static_cast<uint16_t>(order & 0x8000u ? order & 0x7FFFu : 0xFFFFu ^ order));
}

// Likelier first, equal ones by index.
__device__ __forceinline__ unsigned long long key_of(unsigned order, int i) { return static_cast<unsigned long long>(order) << 32 | (0xFFFFFFFFu - i); }

__device__ __forceinline__ uint16_t element(const u32x4& v, int k) { return static_cast<uint16_t>(v[k >> 1] >> (16 * (k & 1))); }

constexpr int kNotThere = -1;

struct __attribute__((packed, aligned(2))) AnyHalfs { // 16 bytes of halfs
    u32x4 v;
};

constexpr int kLogProbWaves = 8, kLogProbThreads = kLogProbWaves * 64, kCandidates = 2048, kQuads = kLogProbThreads / 4;

struct LogProbLds {
    float sums[2][kLogProbWaves], largest[kLogProbWaves];
    unsigned quads[kQuads];
    unsigned long long found[kCandidates];
    int count, bound, scan[kLogProbWaves];
    unsigned arrived;
};

// Largest, sum and moment of a segment, or of all of them.
struct LogProbSums {
    float top, total, moment; // sum of e = exp((x - top) / T), and of e (x - top)
};

// What a row answers: by all threads, from its sums and its likeliest tokens in `found` (`have` of them, in any order).  given: the logit of the
// thread's first given token, kNotThere of one that is not.
__device__ __forceinline__ void answer_row(const LogProbArgs& a, int row, const LogProbSums& s, const unsigned long long* found, int have, int given)
{
    const uint16_t* const x = a.logits + static_cast<size_t>(row) * a.stride;
    const bool wrong = s.top == INFINITY || s.total != s.total;
    const float log_total = logf(s.total);
    auto log_prob = [&](float v) { return wrong ? NAN : v == -INFINITY ? -INFINITY : (v - s.top) * a.inverse - log_total; };
    if (a.log_probs)
        for (int i = threadIdx.x; i < a.n_tokens; i += kLogProbThreads) {
            if (i >= kLogProbThreads) {
                const int token = a.tokens[static_cast<size_t>(row) * a.n_tokens + i];
                given = token >= 0 && token < a.vocab ? x[token] : kNotThere;
            }
            a.log_probs[static_cast<size_t>(row) * a.n_tokens + i] = given == kNotThere ? -INFINITY : log_prob(half_bits_to_float(static_cast<uint16_t>(given)));
        }
    if (a.entropies && threadIdx.x == 0)
        a.entropies[row] = wrong ? NAN : s.top == -INFINITY ? 0.0f : log_total - s.moment * a.inverse / s.total;
    for (int i = threadIdx.x; i < have; i += kLogProbThreads) {
        const unsigned long long key = found[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < have; ++j)
            rank += found[j] > key;
        if (rank >= a.n_top)
            continue;
        a.top_tokens[static_cast<size_t>(row) * a.n_top + rank] = static_cast<int>(0xFFFFFFFFu - static_cast<unsigned>(key));
        if (a.top_log_probs)
            a.top_log_probs[static_cast<size_t>(row) * a.n_top + rank] = log_prob(logit_of(static_cast<unsigned>(key >> 32)));
    }
    for (int i = a.vocab + threadIdx.x; i < a.n_top; i += kLogProbThreads) { // more asked for than there are
        a.top_tokens[static_cast<size_t>(row) * a.n_top + i] = -1;
        if (a.top_log_probs)
            a.top_log_probs[static_cast<size_t>(row) * a.n_top + i] = -INFINITY;
    }
}

// Eight logits of a segment from index i on, -infinity behind its end.
__device__ __forceinline__ u32x4 load_logits(const uint16_t* row, int i, int end)
{
    u32x4 v = {0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u};
    if (i + 8 <= end)
        return reinterpret_cast<const AnyHalfs*>(row + i)->v;
    for (int k = 0; k < end - i; ++k) {
        const uint32_t h = row[i + k];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e == k >> 1)
                v[e] = k & 1 ? (v[e] & 0xFFFFu) | h << 16 : (v[e] & 0xFFFF0000u) | h;
    }
    return v;
}

// Those of eight logits that are of order `least` at least, with what is there already; the count goes on behind what fits.
__device__ __forceinline__ void collect(LogProbLds& lds, const u32x4& v, unsigned least, int i, int end)
{
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const unsigned o = order_of(element(v, k));
        if (o >= least && i + k < end) {
            const int at = atomicAdd(&lds.count, 1);
            if (at < kCandidates)
                lds.found[at] = key_of(o, i + k);
        }
    }
}

// The likeliest `want` of a segment into lds.found where the bound does not find them: the want-th largest order bit by bit (`reach`, or
// 0xFFFF: to be found), then what lies above it, then of those equal to it the first by their index.  Returns how many were found.  Reads the
// segment again for each of these: rows of many equal logits, or with NaN.
__device__ __noinline__ int likeliest_one_by_one(LogProbLds& lds, const uint16_t* row, int begin, int end, int want, unsigned reach)
{
    const int tid = threadIdx.x;
    auto count = [&](unsigned least) {
        __syncthreads();
        if (tid == 0)
            lds.count = 0;
        __syncthreads();
        int n = 0;
        for (int i = begin + tid * 8; i < end; i += kLogProbThreads * 8) {
            const u32x4 v = load_logits(row, i, end);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                n += order_of(element(v, k)) >= least && i + k < end;
        }
        if (n)
            atomicAdd(&lds.count, n);
        __syncthreads();
        return lds.count;
    };
    if (reach == 0xFFFF || count(reach + 1) > kCandidates || count(reach) < want) {
        reach = 0;
        for (int bit = 15; bit >= 0; --bit)
            if (count(reach | 1u << bit) >= want)
                reach |= 1u << bit;
    }
    __syncthreads();
    if (tid == 0)
        lds.count = 0;
    __syncthreads();
    for (int i = begin + tid * 8; i < end; i += kLogProbThreads * 8)
        collect(lds, load_logits(row, i, end), reach + 1, i, end);
    __syncthreads();
    int have = min(lds.count, kCandidates);
    for (int first = begin; first < end && have < want; first += kLogProbThreads * 8) {
        const int i = first + tid * 8, lane = tid & 63;
        const u32x4 v = load_logits(row, i, end);
        int n = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            n += order_of(element(v, k)) == reach && i + k < end;
        int upto = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(upto, d, 64);
            upto = lane >= d ? upto + o : upto;
        }
        __syncthreads();
        if (lane == 63)
            lds.scan[tid >> 6] = upto;
        __syncthreads();
        int at = have + upto - n, all = 0;
        for (int w = 0; w < kLogProbWaves; ++w) {
            at += w < (tid >> 6) ? lds.scan[w] : 0;
            all += lds.scan[w];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (order_of(element(v, k)) == reach && i + k < end) {
                if (at < want)
                    lds.found[at] = key_of(reach, i + k);
                ++at;
            }
        have = min(have + all, want);
    }
    __syncthreads();
    return have;
}

// A workgroup per segment of a row, which stays in registers.  One reading, packed maxima, one exponential per logit; with few
// rows a row is cut into segments, which the last one to arrive puts together.
//
// Instructions per logit bound many rows: 2000 rows of 32000 with four given and twenty likeliest 36.8 us, 3.5 TB/s (the reading alone would be 25).  14.9
// vector instructions per logit keep the vector units busy for 72 % of the time in which their CU has work; 73 registers leave room for three
// workgroups on a CU, 20 wavefronts on average, to fill the rest.  A chain of loads, sums, search and hand-over bounds few (48 rows 7.7 us, one
// row of 128000 in 32 segments 7.5; in one workgroup 97).
template <int PIECES>
__global__ __launch_bounds__(kLogProbThreads) void batch_log_probs_kernel(LogProbArgs a)
{
    __shared__ LogProbLds lds;
    const int row = blockIdx.y, segment = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (a.positions && a.positions[row] < 0)
        return;
    const int begin = segment * a.length, end = min(begin + a.length, a.vocab);
    const uint16_t* const row_at = a.logits + static_cast<size_t>(row) * a.stride;
    int token = -1; // of those given: its logit is looked up while the row is
    if (tid < a.n_tokens)
        token = a.tokens[static_cast<size_t>(row) * a.n_tokens + tid];
    u32x4 x[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int i = begin + (p * kLogProbThreads + tid) * 8;
        x[p] = load_logits(row_at, i, end);
    }
    h2_t m2 = as_h2(0xFC00FC00u);
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
        m2 = max_h2(m2, max_h2(max_h2(as_h2(x[p][0]), as_h2(x[p][1])), max_h2(as_h2(x[p][2]), as_h2(x[p][3]))));
    const int given = token >= 0 && token < a.vocab ? row_at[token] : kNotThere;
    const float most = fmaxf(static_cast<float>(m2[0]), static_cast<float>(m2[1]));
    float quad = fmaxf(most, dpp_f32<DPP_QUAD_XOR1>(most));
    quad = fmaxf(quad, dpp_f32<DPP_QUAD_XOR2>(quad));
    if ((lane & 3) == 0)
        lds.quads[tid >> 2] = order_of(float_to_half_bits(quad));
    const float of_wave = wave_max(most);
    if (lane == 0)
        lds.largest[wave] = of_wave;
    if (tid == 0)
        lds.count = 0;
    __syncthreads();
    LogProbSums s = {lds.largest[0], 0.0f, 0.0f};
#pragma unroll
    for (int w = 1; w < kLogProbWaves; ++w)
        s.top = fmaxf(s.top, lds.largest[w]);
    const int want = min(a.n_top, end - begin);
    if (wave == 0 && want > 0) { // the want-th largest of the quads
        const unsigned q0 = lds.quads[lane], q1 = lds.quads[lane + 64];
        unsigned bound = 0;
#pragma unroll
        for (int bit = 15; bit >= 0; --bit) {
            const unsigned probe = bound | 1u << bit;
            if (__builtin_popcountll(__ballot(q0 >= probe)) + __builtin_popcountll(__ballot(q1 >= probe)) >= want)
                bound = probe;
        }
        if (lane == 0)
            lds.bound = static_cast<int>(bound);
    }
    // of a row that holds nothing above -infinity, nothing; NaN makes its way into the sum
    const float base = s.top == -INFINITY ? 0.0f : s.top;
    float total[2] = {}, moment[2] = {};
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        asm volatile("" : "+v"(x[p]));
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float d = __builtin_fmaf(half_bits_to_float(element(x[p], k)), 1.0f, -base); // one instruction
            const float e = __builtin_amdgcn_exp2f(d * a.per_e);
            total[k & 1] += e;
            moment[k & 1] = __builtin_fmaf(e, __builtin_amdgcn_fmed3f(d, -3.0e38f, 0.0f), moment[k & 1]); // of a masked logit 0
        }
    }
    const float t = wave_sum(total[0] + total[1]), m = wave_sum(moment[0] + moment[1]);
    if (lane == 0) {
        lds.sums[0][wave] = t;
        lds.sums[1][wave] = m;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kLogProbWaves; ++w) {
        s.total += lds.sums[0][w];
        s.moment += lds.sums[1][w];
    }
    int have = 0;
    if (want > 0) {
        // The largest of every four threads bound the want-th largest from below (lds.bound, the want-th of these 128), and what reaches
        // that bound is collected.  Where that is nothing but -infinity, too much (many equal logits) or too little (NaN, which the
        // maxima leave out), in another way.
        const unsigned bound = static_cast<unsigned>(lds.bound);
        const float least = logit_of(bound);
        if (bound > kOrderOfNothing && most >= least)
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                asm volatile("" : "+v"(x[p])); // nothing is carried over from the exponentials, which would take a register per logit
                const h2_t m8 = max_h2(max_h2(as_h2(x[p][0]), as_h2(x[p][1])), max_h2(as_h2(x[p][2]), as_h2(x[p][3])));
                if (static_cast<float>(m8[0]) >= least || static_cast<float>(m8[1]) >= least)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int i = begin + (p * kLogProbThreads + tid) * 8 + k;
                        if (half_bits_to_float(element(x[p], k)) >= least && i < end) {
                            const int at = atomicAdd(&lds.count, 1);
                            if (at < kCandidates)
                                lds.found[at] = key_of(order_of(element(x[p], k)), i);
                        }
                    }
            }
        __syncthreads();
        have = lds.count;
        if (have < want || have > kCandidates)
            have = likeliest_one_by_one(lds, row_at, begin, end, want, bound > kOrderOfNothing ? 0xFFFFu : kOrderOfNothing);
    }
    if (a.segments == 1) {
        answer_row(a, row, s, lds.found, have, given);
        return;
    }
    // Several segments: sums and the likeliest of each go through memory that every XCD sees.
    const size_t at = static_cast<size_t>(row) * a.segments;
    float* const sums = a.parts + at * 4;
    unsigned* const keys = reinterpret_cast<unsigned*>(a.parts + static_cast<size_t>(gridDim.y) * a.segments * 4) + at * a.n_top * 2;
    if (tid == 0) {
        store_agent(sums + segment * 4, s.top);
        store_agent(sums + segment * 4 + 1, s.total);
        store_agent(sums + segment * 4 + 2, s.moment);
    }
    auto put = [&](int rank, unsigned long long key) {
        store_agent(keys + (static_cast<size_t>(segment) * a.n_top + rank) * 2, static_cast<unsigned>(key));
        store_agent(keys + (static_cast<size_t>(segment) * a.n_top + rank) * 2 + 1, static_cast<unsigned>(key >> 32));
    };
    for (int i = tid; i < have; i += kLogProbThreads) {
        const unsigned long long key = lds.found[i];
        int rank = 0;
        for (int j = 0; j < have; ++j)
            rank += lds.found[j] > key;
        if (rank < a.n_top)
            put(rank, key);
    }
    for (int i = want + tid; i < a.n_top; i += kLogProbThreads) // a segment shorter than that
        put(i, 0);
    wait_agent_stores();
    __syncthreads();
    if (tid == 0)
        lds.arrived = add_agent(a.counters + row, 1);
    __syncthreads();
    if (lds.arrived + 1 != static_cast<unsigned>(a.segments))
        return;
    if (tid == 0)
        store_agent(a.counters + row, 0u);
    // A lane per segment, and a thread per key.
    LogProbSums own = {-INFINITY, 0.0f, 0.0f};
    if (lane < a.segments)
        own = {load_agent(sums + lane * 4), load_agent(sums + lane * 4 + 1), load_agent(sums + lane * 4 + 2)};
    auto key_at = [&](int i) {
        const unsigned lo = load_agent(keys + i * 2), hi = load_agent(keys + i * 2 + 1);
        return static_cast<unsigned long long>(hi) << 32 | lo;
    };
    const int n = a.segments * a.n_top;
    const unsigned long long first = tid < n ? key_at(tid) : 0;
    if (n <= 64) {
        if (tid < n)
            lds.found[tid] = first;
    } else {
        // Each segment's keys are in order, so the largest of their last ones bounds the n_top-th of all from below: what does not reach it
        // need not be ranked (one row of 128000, five of each of 32 segments 8.4 -> 7.4 us; 48 rows of 25 keys would take 0.3 longer).
        unsigned last = 0;
        if (lane < a.segments)
            last = load_agent(keys + ((lane + 1) * a.n_top - 1) * 2 + 1);
        const unsigned least = static_cast<unsigned>(wave_max(static_cast<float>(last))); // 16 bits
        if (tid == 0)
            lds.count = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kLogProbThreads) {
            const unsigned long long key = i == tid ? first : key_at(i);
            if (key >> 32 >= least)
                lds.found[atomicAdd(&lds.count, 1)] = key;
        }
    }
    LogProbSums all = {wave_max(own.top), 0.0f, 0.0f};
    const float d = own.top - all.top, w = __builtin_amdgcn_exp2f(d * a.per_e);
    const bool nothing = own.top == -INFINITY; // but NaN, perhaps
    all.total = wave_sum(nothing ? own.total * 0.0f : own.total * w);
    all.moment = wave_sum(nothing ? 0.0f : w * __builtin_fmaf(own.total, d, own.moment));
    __syncthreads();
    answer_row(a, row, all, lds.found, n <= 64 ? n : lds.count, given);
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
    // Two pieces a thread where there are more rows than the card holds workgroups of one piece a thread.  What the L2 of all XCDs cannot
    // hold does not go through it.
    const int pieces_all = size / 8, written = (output != nullptr) + (residual_output != nullptr);
    int pieces = batch->n_tokens >= 2 * ctx().num_cus ? 2 : 1;
    while (ceil_div(pieces_all, pieces) > 1024)
        pieces *= 2;
    const bool through = static_cast<size_t>(batch->n_tokens) * size * 2 * written >= 32u << 20;
    const dim3 grid(batch->n_tokens), block(round_up(ceil_div(pieces_all, pieces), 64));
    const hipStream_t st = ctx().stream;
    auto launch = [&](auto p) {
        constexpr int P = decltype(p)::value;
        if (through)
            hipLaunchKernelGGL((batch_norm_kernel<P, true>), grid, block, 0, st, a);
        else
            hipLaunchKernelGGL((batch_norm_kernel<P, false>), grid, block, 0, st, a);
    };
    switch (pieces) {
    case 1: launch(std::integral_constant<int, 1>()); break;
    case 2: launch(std::integral_constant<int, 2>()); break;
    case 4: launch(std::integral_constant<int, 4>()); break;
    default: launch(std::integral_constant<int, 8>()); break;
    }
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
    LogProbArgs a = {log_probs, entropies, top_tokens, top_log_probs, logits, tokens, positions, nullptr, ctx().batch_counters, vocab_size,
                     logits_stride, n_tokens, n_top, 1, vocab_size, static_cast<float>(inverse), static_cast<float>(inverse * 1.4426950408889634)};
    const LogProbShape shape = log_prob_shape(n_rows, vocab_size, n_top, ctx().num_cus);
    a.segments = shape.segments;
    a.length = shape.length;
    for (int done = 0; done < n_rows; done += kLogProbRows) {
        const int rows = n_rows - done < kLogProbRows ? n_rows - done : kLogProbRows;
        if (a.segments > 1) {
            const size_t parts = static_cast<size_t>(rows) * a.segments;
            if (int rc = ensure_attn_partials(parts * (16 + 8 * static_cast<size_t>(n_top))))
                return rc;
            a.parts = ctx().attn_partials;
        }
        const dim3 grid(a.segments, rows), block(kLogProbThreads);
        switch (shape.pieces) {
        case 1: hipLaunchKernelGGL(batch_log_probs_kernel<1>, grid, block, 0, ctx().stream, a); break;
        case 2: hipLaunchKernelGGL(batch_log_probs_kernel<2>, grid, block, 0, ctx().stream, a); break;
        case 4: hipLaunchKernelGGL(batch_log_probs_kernel<4>, grid, block, 0, ctx().stream, a); break;
        default: hipLaunchKernelGGL(batch_log_probs_kernel<8>, grid, block, 0, ctx().stream, a); break;
        }
        L2_LAUNCH_CHECK("llama2_batch_log_probs");
        a.logits += static_cast<size_t>(rows) * logits_stride;
        a.positions += positions ? rows : 0;
        a.tokens += tokens ? static_cast<size_t>(rows) * n_tokens : 0;
        a.log_probs += log_probs ? static_cast<size_t>(rows) * n_tokens : 0;
        a.entropies += entropies ? rows : 0;
        a.top_tokens += top_tokens ? static_cast<size_t>(rows) * n_top : 0;
        a.top_log_probs += top_log_probs ? static_cast<size_t>(rows) * n_top : 0;
    }
    return LLAMA2_OK;
}

} // extern "C"
