/*
 * llama2_hip.h -- C ABI of libllama2_hip.so, the MI355X (gfx950) implementation
 * of ManagedLlama2's quantized batch-1 decode path.
 *
 * The library takes the place of ManagedCuda + the embedded PTX modules
 * underneath the reference's C# module classes: every entry point below names
 * the reference interface it replaces (paths relative to the reference
 * checkout).  Kernel entry points keep the argument order of the reference's
 * `extern "C" __global__` prototypes (the native/<kernel>.cuh headers); what the reference
 * encoded in the launch grid (number of heads / rows) is an explicit trailing
 * int here, because grid and block shapes are chosen inside the library.
 *
 * Conventions
 *   - plain C, no C++ or framework types in any signature;
 *   - every function returns 0 (LLAMA2_OK) on success, a negative LLAMA2_ERR_*
 *     for rejected arguments / state, or a positive hipError_t value when the
 *     HIP runtime failed; llama2_last_error() describes the last failure of
 *     the calling thread;
 *   - `llama2_half` is IEEE binary16 storage (C# System.Half, CUDA half);
 *   - all pointers named out/x/q/... are DEVICE pointers obtained from
 *     llama2_malloc (or any hipMalloc'ed memory of the same device);
 *   - kernels are enqueued asynchronously on one library-owned stream, in
 *     call order; llama2_memcpy_d2h and llama2_sync wait for them.  The
 *     reference runs on a single NULL stream from one host thread; here host
 *     threads may share the library: every entry point takes one lock and
 *     binds the calling thread to the library's device, so calls take turns.
 */
#ifndef LLAMA2_HIP_H
#define LLAMA2_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

typedef uint16_t llama2_half;

#define LLAMA2_OK 0
#define LLAMA2_ERR_INVALID_ARGUMENT (-1) /* null / misaligned pointer, bad size, aliasing */
#define LLAMA2_ERR_NOT_INITIALIZED (-2)  /* llama2_init not called                        */
#define LLAMA2_ERR_UNSUPPORTED (-3)      /* shape outside what the kernels implement      */
#define LLAMA2_ERR_NO_DEVICE (-4)        /* no usable gfx950 device                        */
#define LLAMA2_ERR_STEP_FAILED (-5)      /* a persistent decode step gave up a bounded wait */

/* Largest softmax row, as in the reference (native/softmax_kernel.cu:5). */
#define LLAMA2_MAX_SOFTMAX_SIZE 8192
/* Largest `size` of the sampler modules (softmax_logits, sort, cumulative_sum,
 * sample_top_p): the 1024 partial sums, whose order is that of one
 * workgroup, take up to 64 elements each; positions and ranks are 16 bits. */
#define LLAMA2_MAX_SAMPLER_SIZE 65536

/* ---------------------------------------------------------------- runtime */

/* new CudaContext(deviceID): src/Transformer.cs:48-49.  Idempotent per device. */
int llama2_init(int device);
/* Releases the stream and internal scratch.  Caller-owned buffers and decoders
 * stay valid and work again after the next llama2_init on the same device; graphs
 * that the caller captured from modules with scratch (llama2_vec_mat,
 * llama2_multi_head_attention, the sampler modules, llama2_batch_tables, llama2_batch_attention,
 * llama2_batch_mat_mul_int4, llama2_batch_mat_mul_swiglu, llama2_batch_log_probs) hold its address and do not. */
int llama2_shutdown(void);
/* Text of the calling thread's last error ("" if none).  Never NULL. */
const char* llama2_last_error(void);

/* new CudaDeviceVariable<T>(n): src/RunState.cs:41-53.  256-byte aligned. */
int llama2_malloc(void** ptr, size_t bytes);
/* CudaDeviceVariable.Dispose. */
int llama2_free(void* ptr);
/* implicit T[] -> CudaDeviceVariable<T> (src/TransformerWeights.cs:61-66) and
 * CopyToDevice(src, 0, dstByteOffset, bytes) (src/Extensions.cs:23-24,
 * src/Transformer.cs:93,127).  Ordered after previously enqueued kernels. */
int llama2_memcpy_h2d(void* dst, size_t dst_offset_bytes, const void* src, size_t bytes);
/* explicit CudaDeviceVariable<T> -> T[] and the 1-element indexer read
 * `runstate.tokens[nextPosition]` (src/Sampler.cs:69).  Waits for the stream. */
int llama2_memcpy_d2h(void* dst, const void* src, size_t src_offset_bytes, size_t bytes);
/* CudaDeviceVariable.CopyToDevice(CudaDeviceVariable): asynchronous device-to-
 * device copy by a plain copy kernel (16-byte granularity, no overlap). */
int llama2_memcpy_d2d(void* dst, const void* src, size_t bytes);
/* Asynchronous fill (tests and RunState set-up; ManagedCuda's Memset). */
int llama2_memset(void* dst, int byte_value, size_t bytes);
/* CudaContext.GetFreeDeviceMemorySize(): src/RunState.cs:34. */
int llama2_mem_info(size_t* free_bytes, size_t* total_bytes);
/* CudaContext.Synchronize(). */
int llama2_sync(void);
/* The hipStream_t every entry point launches on (for callers that time or
 * order their own work against it).  NULL before llama2_init. */
void* llama2_stream(void);

/* HIP events on the library's stream, for timing the enqueued kernels. */
int llama2_event_create(void** event);
int llama2_event_record(void* event);
int llama2_event_elapsed_ms(void* start, void* stop, float* ms); /* waits for `stop` */
int llama2_event_destroy(void* event);

/* Stream capture of the calls made between begin and end into a hipGraph that
 * llama2_graph_launch replays with a single submission (no counterpart in the
 * reference, which pays one cuLaunchKernel per module call, src/Module.cs:21-22).
 * Only kernel entry points may be called while capturing: no malloc / free /
 * memcpy / sync, and llama2_vec_mat / llama2_multi_head_attention /
 * llama2_batch_attention / llama2_batch_mat_mul_* / llama2_batch_log_probs only for shapes whose scratch already exists (call them once
 * eagerly first).  The captured calls keep the argument
 * values they were made with, the scratch address included: the library never
 * frees a scratch buffer before llama2_shutdown, so a later eager call that
 * needs a larger one leaves earlier graphs valid. */
int llama2_graph_begin_capture(void);
int llama2_graph_end_capture(void** graph);
int llama2_graph_launch(void* graph);
int llama2_graph_destroy(void* graph);

/* ------------------------------------------------- int4 tensors ("QWeight")
 * Layout per output row n of a K-input tensor (src/TransformerWeights.cs:54-69,
 * native/mat_vec_kernel.cu:98-134):
 *   weights_size = ceil(K/32)*4 uint32, element k in bits 4*(k%8).. of word k/8
 *   scales_size  = ceil(K/128)   fp16,  scale of group g = k/128
 *   zeros_size   = ceil(scales_size/8) uint32, zero of group g = nibble g%8 of word g/8
 *   value(n,k)   = (w - z) * scale
 * `rows` is the INPUT length K and `cols` the number of outputs N, as in the
 * reference (src/MatVecResidual.cs:15-22).  The three *_size arguments must be
 * the values above (they are what the reference's modules pass); weight rows
 * must be 16-byte aligned.
 */

/* src/QWeight.cs:5-10 */
typedef struct llama2_qweight {
    const uint32_t* weight;
    const uint32_t* zeros;
    const llama2_half* scales;
} llama2_qweight;

/* mat_vec_residual_int4_kernel (native/mat_vec_kernel.cuh:58-59), module
 * MatVecResidual.Forward (src/MatVecResidual.cs:15-22):
 *   output[n] = half(float(output[n]) + sum_k input[k]*(w-z)*s).
 * `output` must not overlap `input`. */
int llama2_mat_vec_residual_int4(llama2_half* output, const llama2_half* input,
                                 const uint32_t* weights, const uint32_t* zeros,
                                 const llama2_half* scales, int rows, int cols, int zeros_size,
                                 int scales_size, int weights_size);

/* The same dot product without the residual read (device function
 * mat_vec_int4, native/mat_vec_kernel.cu:166-177; one third of QKVMatVec). */
int llama2_mat_vec_int4(llama2_half* output, const llama2_half* input, const uint32_t* weights,
                        const uint32_t* zeros, const llama2_half* scales, int rows, int cols,
                        int zeros_size, int scales_size, int weights_size);

/* qkv_mat_vec_kernel (native/mat_vec_kernel.cuh:85-89), module QKVMatVec.Forward
 * (src/QKVMatVec.cs:19-31): three int4 mat-vecs of one input in one launch.
 * k_output / v_output are the KV-cache rows, i.e. the caller has already added
 * layerOffset + pos*kvDim (src/QKVMatVec.cs:25-26). */
int llama2_qkv_mat_vec(llama2_half* q_output, llama2_half* k_output, llama2_half* v_output,
                       const llama2_half* input, const uint32_t* q_weight, const uint32_t* q_zeros,
                       const llama2_half* q_scales, const uint32_t* k_weight,
                       const uint32_t* k_zeros, const llama2_half* k_scales,
                       const uint32_t* v_weight, const uint32_t* v_zeros,
                       const llama2_half* v_scales, int rows, int cols, int zeros_size,
                       int scales_size, int weights_size);

/* mat_vec_swiglu_kernel (native/mat_vec_kernel.cuh:113-116), module
 * MatVecSwiGLU.Forward (src/MatVecSwiGLU.cs:15-24):
 *   output[n] = half( silu(g.x) * (u.x) ),  silu(v) = v / (1 + expf(-v)). */
int llama2_mat_vec_swiglu(llama2_half* output, const llama2_half* input, const uint32_t* g_weight,
                          const uint32_t* g_zeros, const llama2_half* g_scales,
                          const uint32_t* u_weight, const uint32_t* u_zeros,
                          const llama2_half* u_scales, int rows, int cols, int zeros_size,
                          int scales_size, int weights_size);

/* ---------------------------------------------------------- fp16 mat-vecs */

/* mat_vec_kernel (native/mat_vec_kernel.cuh:17), module MatVec.Forward
 * (src/MatVec.cs:15-16): output[n] = sum_k matrix[n*rows + k] * vector[k];
 * rows % 8 == 0 as in the reference (native/mat_vec_kernel.cu:16,26). */
int llama2_mat_vec(llama2_half* output, const llama2_half* vector, const llama2_half* matrix,
                   int rows, int cols);

/* mat_vec_strided_kernel (native/mat_vec_kernel.cuh:37-38), module
 * MatVecStrided.Forward (src/MatVecStrided.cs:16-18); n_heads was gridDim.y:
 *   output[h*o_stride + t] = alpha * sum_{r<rows} vector[h*v_stride + r]
 *                                    * matrix[t*m_row_stride + h*m_col_stride + r]
 * for t < cols, h < n_heads. */
int llama2_mat_vec_strided(llama2_half* output, const llama2_half* vector,
                           const llama2_half* matrix, int rows, int cols, int v_stride,
                           int m_col_stride, int m_row_stride, int o_stride, float alpha,
                           int n_heads);

/* vec_mat_kernel (native/vec_mat_kernel.cuh:5-6), module VecMat.Forward
 * (src/VecMat.cs:17-19); n_heads was gridDim.y:
 *   output[h*o_stride + r] = sum_{t<cols} vector[h*cols + t]
 *                            * matrix[t*m_row_stride + h*m_col_stride + r],  r < rows. */
int llama2_vec_mat(llama2_half* output, const llama2_half* vector, const llama2_half* matrix,
                   int rows, int cols, int m_col_stride, int o_stride, int m_row_stride,
                   int n_heads);

/* llama2_vec_mat for callers that cannot allocate (code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc).  No counterpart in the reference.  Same
 * arguments, same kernels, same results bit for bit; but where llama2_vec_mat keeps the fp32
 * partial sums of a sequence split over workgroups in a buffer it allocates (and grows) on
 * demand, this entry point keeps them in a fixed array of LLAMA2_STATIC_VEC_MAT_BYTES inside
 * the library's code object (one copy per GPU, held until the process ends) and calls no
 * hipMalloc, hipFree or other allocating routine.  A call whose partial sums
 * (sequence blocks x n_heads x rows floats) do not fit returns LLAMA2_ERR_UNSUPPORTED
 * (32 heads of 128 rows fit at any sequence length; 40 heads up to about 3300 positions).
 * All calls on a GPU share the array: calls that overlap on one GPU (two streams, two
 * replaying graphs) race; calls on the library's one stream are in order and safe. */
#define LLAMA2_STATIC_VEC_MAT_BYTES 2097152
int llama2_vec_mat_static(llama2_half* output, const llama2_half* vector, const llama2_half* matrix,
                   int rows, int cols, int m_col_stride, int o_stride, int m_row_stride,
                   int n_heads);

/* Transformer.MultiHeadAttention (src/Transformer.cs:150-156) as ONE launch:
 * scores over `seq_length` rows of `key`, softmax, weighted sum of `value`
 * rows, without the round trip through the `attention` scratch.  key / value
 * are the cache slices of the layer (caller adds layerOffset), rows of `dim`
 * halfs; head h uses columns h*head_size .. of q, key, value and output.
 * Scores are rounded to fp16 as the reference's attention buffer does.
 * head_size must be 128; other sizes: LLAMA2_ERR_UNSUPPORTED, use the three
 * modules above. */
int llama2_multi_head_attention(llama2_half* output, const llama2_half* query, const llama2_half* key,
                                const llama2_half* value, int head_size, int dim, int seq_length,
                                float scale, int n_heads);

/* RoPERotation.Forward (src/RoPERotation.cs:13-21, native/rope_kernel.cu:3-26)
 * at position `pos` followed by MultiHeadAttention (src/Transformer.cs:172-175)
 * in ONE launch: the query and row seq_length - 1 of `key` (the row the step's
 * QKVMatVec has just written) are rotated inside the attention kernel and
 * written back rotated, as llama2_rope leaves them, so the call equals
 * llama2_rope(query, key + (seq_length - 1) * dim, n_heads, 128, pos, theta,
 * n_heads) + llama2_multi_head_attention(...) bit for bit, without the second
 * launch.  No counterpart in the reference, which launches four kernels here.
 * Same limits as llama2_multi_head_attention (head_size 128). */
int llama2_rope_multi_head_attention(llama2_half* output, llama2_half* query, llama2_half* key,
                                     const llama2_half* value, int head_size, int dim,
                                     int seq_length, float scale, int n_heads, int pos,
                                     float theta);

/* ------------------------------------------------------- pointwise modules */

/* rmsnorm_kernel (native/rmsnorm_kernel.cuh:5), module RMSNorm.Forward
 * (src/RMSNorm.cs:13-14): output[i] = half(1/sqrtf(mean(x^2)+eps) * gamma[i] * x[i]).
 * output may be the same buffer as input (src/Transformer.cs:187). */
int llama2_rmsnorm(llama2_half* output, const llama2_half* input, const llama2_half* gamma,
                   int size, float eps);

/* rope_kernel (native/rope_kernel.cuh:6), module RoPERotation.Forward
 * (src/RoPERotation.cs:19-24); n_heads was gridDim.x.  Rotates the pairs
 * (i, i + head_size/2) of every head of q, and of k for heads < n_kv_heads;
 * k is the cache row, already offset by layerOffset + pos*kvDim. */
int llama2_rope(llama2_half* q, llama2_half* k, int n_kv_heads, int head_size, int pos,
                float theta, int n_heads);

/* softmax_kernel (native/softmax_kernel.cuh:5), module Softmax.Forward
 * (src/Softmax.cs:13-14); n_rows was gridDim.x: in-place softmax of
 * vector[r*size .. r*size+size) for r < n_rows; size <= LLAMA2_MAX_SOFTMAX_SIZE. */
int llama2_softmax(llama2_half* vector, int size, int n_rows);

/* argmax_kernel (native/argmax_kernel.cuh:5), module Argmax.Forward
 * (src/Argmax.cs:13-14): result[pos] = index of the largest input iff
 * write_token.  Ties resolve to the LOWEST index, deterministically (the
 * reference's CPU check, test/ArgmaxTests.cs:33-46; its kernel races). */
int llama2_argmax(const llama2_half* input, int size, int* result, int pos, int write_token);

/* embedding_kernel (native/embedding_kernel.cuh:5), module Embedding.Forward
 * (src/Embedding.cs:13-14): output[i] = table[tokens[pos]*size + i]; the token
 * id is read on the device. */
int llama2_embedding(llama2_half* output, const llama2_half* table, int size, const int* tokens,
                     int pos);

/* ------------------------------------------------ stochastic sampler modules
 * The four kernels of Sampler.Sample's temperature / top-p branch
 * (src/Sampler.cs:48-67).  1 <= size <= LLAMA2_MAX_SAMPLER_SIZE (the
 * reference's launch shapes fix size to a multiple of 125 resp. 32 up to
 * 32000; any size works here).  fp16 and int buffers 16-byte aligned. */

/* softmax_logits_kernel (native/softmax_logits_kernel.cuh:5), module
 * SoftmaxLogits.Forward (src/SoftmaxLogits.cs:14-15): indices[t] = t;
 * logits <- softmax(logits / temperature) in place with the reference's three
 * fp16 roundings (after the division, after expf, after the normalisation).
 * temperature > 0. */
int llama2_softmax_logits(llama2_half* logits, int size, float temperature, int* indices);

/* sort_kernel (native/sort_kernel.cuh:4), module Sort.Forward
 * (src/Sort.cs:14-15): sorts keys in DESCENDING order, in place, carrying
 * values along.  Stable (equal keys keep their order), like the reference's
 * cub::BlockRadixSort; keys are ordered as the radix sort orders fp16 bit
 * patterns (numeric order, +0 before -0, NaNs at the two ends). */
int llama2_sort(llama2_half* keys, int* values, int size);

/* cumulative_sum_kernel (native/cumulative_sum_kernel.cuh:5), module
 * CumulativeSum.Forward (src/CumulativeSum.cs:14-15): in-place inclusive
 * prefix sums, accumulated in fp32, each rounded to fp16. */
int llama2_cumulative_sum(llama2_half* values, int size);

/* sample_top_p_kernel (native/sample_top_p_kernel.cuh:5), module
 * SampleTopP.Forward (src/SampleTopP.cs:14-15): result[pos] = indices[m], m the
 * first position with float(logits[m]) >= threshold, or size-1 if none. */
int llama2_sample_top_p(const llama2_half* logits, const int* indices, int size, float threshold,
                        int* result, int pos);

/* The stochastic branch of Sampler.Sample (src/Sampler.cs:50-66) in one call (up to four launches):
 * softmax_logits; if 0 < top_p < 1: sort and threshold = coin * top_p, else
 * threshold = coin; cumulative_sum; sample_top_p into result[pos].  logits and
 * indices are overwritten exactly as by the four module calls (same device
 * code).  coin is the caller's uniform number in [0, 1). */
int llama2_sample(llama2_half* logits, int* indices, int size, float temperature, float top_p,
                  float coin, int* result, int pos);

/* ------------------------------------------- steps of several requests at once
 * The reference and the decoder below serve one sequence with a contiguous
 * cache; there is no counterpart for what follows.  Several requests keep
 * their cache rows in blocks of a shared pool and may start behind one prefix whose
 * rows they share (a system prompt, or the prompt whose continuations are
 * sampled in parallel).  A step is llama2_batch_tables once, then for every
 * layer llama2_batch_qk_norm_rope and llama2_batch_attention.  All three are
 * asynchronous on the library's stream and may be captured; everything that
 * changes from step to step is read on the device, so that one captured
 * step serves as long as n_requests, n_tokens and max_length stay large enough. */

/* Keys and values of one layer: row r of block b, head h, starts at
 * b * block_stride + (r * n_kv_heads + h) * head_size halfs.  A contiguous
 * cache is one whose blocks follow each other in order. */
typedef struct llama2_paged_cache {
    llama2_half* key;   /* 16-byte aligned */
    llama2_half* value; /* 16-byte aligned */
    long long block_stride; /* halfs between blocks, a multiple of 8; 0: block_size * n_kv_heads * head_size */
    int n_blocks;
    int block_size; /* rows per block: a power of two, 8 .. 1024 */
    int n_kv_heads;
    int head_size; /* 64 or 128 */
} llama2_paged_cache;

/* The requests of a step.  Arrays are device memory.  n_tokens is the number of
 * rows that the step's buffers have: rows behind the requests' own tokens (a
 * batch padded to a captured size) have position and slot -1, and every
 * operator leaves the rows of such tokens in its output as they were. */
typedef struct llama2_batch {
    int* block_tables;       /* [n_requests][table_stride]: the blocks of a request's own rows, in order */
    int* lengths;            /* [n_requests]: own rows of a request, the new tokens included */
    int* query_starts;       /* [n_requests + 1]: first token of every request, then the number of tokens */
    int* positions;          /* [n_tokens]: prefix_length + own row of the token, or -1 */
    int* slots;              /* [n_tokens]: block * block_size + row in the block, or -1 */
    const int* prefix_table; /* [ceil(prefix_length / block_size)]: the blocks of the shared rows; null if none */
    int n_requests;
    int n_tokens;
    int table_stride;
    int prefix_length; /* rows that all requests share, in front of their own */
    int max_length;    /* no request has more own rows than this (read by llama2_batch_attention) */
} llama2_batch;

/* Block tables and slots of a step, from the lengths.  Request b has cached[b] own
 * rows and brings counts[b] tokens (none is allowed).  It gets the blocks that its new rows
 * need from free_blocks[taken ..), in the order of the requests; batch->block_tables is
 * extended in place, lengths, query_starts, positions and slots are written, and
 * new_taken[0] is taken[0] plus the blocks that the requests up to the last one that is
 * not refused ask for.  lengths may be `cached` and new_taken may be `taken`; other arrays
 * must not overlap.
 * A request is refused -- its tokens get position and slot -1, its table and
 * length stay as they are, it takes no block -- if the free blocks left do not suffice for
 * it and all in front of it, if its rows would not fit into table_stride blocks, if its tokens
 * reach beyond n_tokens, or if its count or length is negative.  A request that needs no
 * block is not refused for want of blocks; where one goes on behind a request that was,
 * new_taken[0] is above n_free.  With taken[0] above n_free (or negative) the list counts as
 * empty and new_taken[0] is taken[0]: nobody gets a block until the caller, who has to find blocks
 * or pause requests then, gives a new list, or the number of blocks that really were handed out.  That
 * can be less than new_taken says (what refused requests asked for is in it where another, a resting
 * one too, goes on behind them), and is always the sum of ceil(lengths / block_size) over the requests
 * behind the step, less the same of `cached`.
 * Block ids are copied, not looked at; free_blocks and the tables must not hold an id twice.  An id whose
 * slots would be negative or pass 2^31 gives slot -1.
 * prefix_table and max_length are not read. */
int llama2_batch_tables(const llama2_batch* batch, const int* cached, const int* counts,
                        const int* free_blocks, int n_free, const int* taken, int* new_taken,
                        int block_size);

/* For every token with a position: q_output = rotated (normed) queries, and keys
 * and values to the token's slot of the cache, the keys rotated (normed).  Head x
 * of `head_size` elements: y = x / sqrt(mean(x^2) + eps) * gamma if gamma (q_gamma
 * for queries, k_gamma for keys; head_size halfs, null: no norm), then pairs (i, i +
 * head_size/2) rotated by position * theta^(-2 i / head_size) as llama2_rope does, one rounding at the
 * end.  The angle is good to 2^-25 of a turn at every position (llama2_rope's,
 * like the reference's, loses bits as positions grow: the two differ by roundings).
 * Rows of q, k, v and q_output are q_stride, kv_stride and q_output_stride halfs
 * apart (multiples of 8, pointers 16-byte aligned), so that they may be parts of one buffer.
 * q_output may be q with the same stride (rows of k and v between q's must have that stride
 * too); neither it nor the cache may overlap anything else.  Keys and values of the cache must not overlap.  No two tokens may
 * have the same slot.  A token whose slot is not one of the cache's is not stored.
 * Reads positions and slots of the batch.  1 <= theta. */
int llama2_batch_qk_norm_rope(llama2_half* q_output, const llama2_half* q, const llama2_half* k,
                              const llama2_half* v, const llama2_half* q_gamma,
                              const llama2_half* k_gamma, const llama2_batch* batch,
                              const llama2_paged_cache* cache, int n_heads, int q_output_stride,
                              int q_stride, int kv_stride, float eps, float theta);

/* Causal attention of all tokens: the token at position p of request b attends the
 * prefix_length rows of the prefix table and the own rows 0 .. p - prefix_length
 * of the request (row r: block_tables[b][r / block_size]); query head h
 * uses key/value head h / (n_heads / n_kv_heads).  Scores and softmax stay in fp32; on their
 * way into the products with the values, probabilities keep 22 bits where up to 16 query rows
 * are computed at a time (single tokens), and are rounded to fp16 where more are (prompts, a
 * prefix that many requests share)
 * (llama2_multi_head_attention rounds scores to fp16 instead, as the reference does).
 * Rows of a block id outside the cache are not attended; a token left without rows gives
 * zeros.  Rows behind a token's own, and the rest of the last block, have no influence
 * whatever they hold; an infinite value that a token does attend may reach its output as
 * NaN.  Where it saves reading, the shared rows are read once for up to 128 query rows
 * instead of once per request.  The same call gives the same bits every time.
 * positions of a request must not decrease; max_length bounds the launch, which costs time where it is far
 * above the lengths (one request of 777 rows of 32 heads 8.2 us, with 4096 9.9, with 131072 19.4), rows beyond it
 * are not attended; any scale is allowed, and scores as large as fp32 holds (a scaled score beyond that gives
 * NaN, or the row no weight).  `output` must not overlap the other buffers.
 * Reads query_starts, positions, block_tables and prefix_table of the batch, as
 * llama2_batch_tables leaves them.  At most 2^29 rows per token and 2^26 query rows.
 * Scratch: as llama2_multi_head_attention (call once before capturing), at most 512 MiB for a call. */
int llama2_batch_attention(llama2_half* output, const llama2_half* query, const llama2_batch* batch,
                           const llama2_paged_cache* cache, int n_heads, int output_stride,
                           int query_stride, float scale);

/* Low-rank adapters of one int4 tensor, a pool of which each token may use one: adapter a adds
 *   scales[a] * sum_{r < ranks[a]} up_a[n][r] * sum_k down_a[r][k] * input[k]
 * to output n.  Arrays are device memory; nothing beyond an adapter's rank has any influence. */
typedef struct llama2_adapters {
    const llama2_half* down; /* element k of rank r of adapter a at a * down_stride + r * rows + k; 16-byte aligned */
    const llama2_half* up;   /* rank r of output n of adapter a at a * up_stride + n * max_rank + r; 16-byte aligned */
    const float* scales;     /* [n_adapters] */
    const int* ranks;        /* [n_adapters]: 0 .. max_rank (values outside count as the nearer of the two) */
    long long down_stride;   /* halfs between adapters, a multiple of 8; 0: max_rank * rows */
    long long up_stride;     /* halfs between adapters, a multiple of 8; 0: cols * max_rank */
    int n_adapters;
    int max_rank; /* a multiple of 8, 8 .. 128 */
} llama2_adapters;

/* One int4 tensor of a product of many rows, and where its results go. */
typedef struct llama2_batch_matrix {
    llama2_qweight weight;
    llama2_half* output;             /* 16-byte aligned */
    const llama2_half* residual;     /* added to the product; null: none; may be output with the same stride */
    const llama2_adapters* adapters; /* host memory, read during the call; null: none */
    int cols;                        /* outputs, a multiple of 8 */
    int output_stride;               /* halfs between rows, a multiple of 8 */
    int residual_stride;
} llama2_batch_matrix;

#define LLAMA2_MAX_BATCH_MATRICES 4

/* Products of all tokens of a step with up to LLAMA2_MAX_BATCH_MATRICES int4 tensors that read the same input (q, k and
 * v; or one):
 *   output[t][n] = half(residual[t][n] + sum_k input[t][k] * (w - z) * s + adapter's part),
 * sums in fp32, one rounding at the end; what an adapter's ranks receive of the input is fp32 too, and above 64 tokens may keep
 * no more than 22 bits of the largest of 16 of them.  A step of one token may go through the decode step's kernels, which sum up input * w and
 * z * input apart for every 32 inputs: the error of its sums is then one of |input| (w + z) s, where that of more tokens is one of
 * |input| |w - z| s (it shows where all inputs have an offset in common that is large beside their differences).  Where an input, or a number of
 * the token's adapter, is infinite or NaN, the results that it contributes to are infinite or NaN; which of the two may differ with the number of tokens.
 * rows % 8 == 0, up to 65536; cols up to 2^20, input_stride up to 2^24; scales are finite; tensors are laid out as above
 * (ceil(rows/32)*4 words, ceil(rows/128) scales per output).
 * Token t uses adapter token_adapters[t] of every matrix that has adapters; a value that is not one of 0 .. n_adapters - 1:
 * none.  What one token or one adapter holds has no influence on the rows of other tokens.  token_adapters may be null where no
 * matrix has adapters.  Rows of tokens without a position are left as they were.  Reads n_tokens and positions of
 * the batch.  Outputs must not overlap each other, the input, or anything else that is read.  The same call gives the same bits every
 * time.  Scratch: as llama2_multi_head_attention (call once before capturing).  Asynchronous, may be captured. */
int llama2_batch_mat_mul_int4(const llama2_batch_matrix* matrices, int n_matrices, const llama2_half* input, int rows,
                              int input_stride, const int* token_adapters, const llama2_batch* batch);

/* The first half of the gated feed-forward block for all tokens of a step:
 *   output[t][n] = half( silu(g) * u ),  silu(v) = v / (1 + exp(-v)),
 * g and u the sums of llama2_batch_mat_mul_int4 with `gate` and `up` (and their adapters; null: none), in fp32.  rows up to
 * 32768, the rest as there. */
int llama2_batch_mat_mul_swiglu(llama2_half* output, const llama2_half* input, const llama2_qweight* gate,
                                const llama2_qweight* up, int rows, int cols, int output_stride, int input_stride,
                                const llama2_adapters* gate_adapters, const llama2_adapters* up_adapters,
                                const int* token_adapters, const llama2_batch* batch);

/* What stands between two blocks, for all tokens of a step:
 *   y = input, or norm(input) * input_gamma if input_gamma; y *= gate if gate
 *   r = residual + residual_scale * y   (r = residual if input is null)
 *   residual_output = half(r);  output = half(norm(r) * gamma)
 * with norm(v) = v / sqrt(mean(v^2) + eps), everything in fp32 (the squares too: from about 10^17 on a row's norm is 0), r not rounded in front of
 * its norm.  gammas and gate:
 * `size` halfs.  output (with gamma) or residual_output may be null; residual_output may be residual with the same stride,
 * output may be input with the same stride; otherwise outputs must not overlap anything.
 * size: a multiple of 8 up to 65536; strides are multiples of 8, pointers 16-byte aligned.  Rows of tokens without a position
 * are left as they were.  Reads n_tokens and positions of the batch.  Asynchronous, may be captured. */
int llama2_batch_residual_rmsnorm(llama2_half* output, llama2_half* residual_output, const llama2_half* residual,
                                  const llama2_half* input, const llama2_half* gamma, const llama2_half* input_gamma,
                                  const llama2_half* gate, const llama2_batch* batch, int size, int output_stride,
                                  int residual_output_stride, int residual_stride, int input_stride, float residual_scale,
                                  float eps);

/* Log probabilities, natural logarithms in fp32, of every row of logits under softmax(logits / temperature):
 *   log_probs[r][i]  of tokens[r][i] for i < n_tokens; of a token that is not one of 0 .. vocab_size - 1: -infinity
 *   entropies[r]     -sum p log p
 *   top_tokens[r][j], top_log_probs[r][j]  for j < n_top: the most likely tokens in order, equal ones by their index; behind the
 *                    last of a vocabulary smaller than n_top: -1 and -infinity
 * Any of the four may be null (n_tokens / n_top 0 where theirs are; top_log_probs needs top_tokens).  A logit of -infinity has
 * probability 0; of a row that holds nothing else all log probabilities are -infinity and the entropy is 0.  A row with NaN or +infinity has NaN for its log probabilities
 * and its entropy; its top tokens are in the order of the logits, NaN last.  Rows whose position is negative are left as they
 * were (positions null: none is).  n_tokens <= 1024, n_top <= LLAMA2_MAX_TOP_TOKENS, vocab_size <= 2^20, 1e-30 < temperature <= 1e30;
 * logits need no alignment beyond their 2 bytes.  Scratch: as llama2_multi_head_attention (call once before capturing).  Asynchronous,
 * may be captured. */
#define LLAMA2_MAX_TOP_TOKENS 64
int llama2_batch_log_probs(float* log_probs, float* entropies, int* top_tokens, float* top_log_probs,
                           const llama2_half* logits, const int* tokens, const int* positions, int n_rows, int vocab_size,
                           int logits_stride, int n_tokens, int n_top, float temperature);

/* ------------------------------------------------------- converter repack
 * The tensor transformations of ModelConverter.RepackQWeightByName
 * (src/ModelConverter.cs:196-275) on device buffers: what turns an AWQ
 * checkpoint's tensors into the layout every entry point above reads.  All
 * asynchronous on the library's stream; out and in must not overlap. */

/* RepackQData (src/ModelConverter.cs:277-317).  in: [height][width/8] words of
 * the AWQ "GEMM" format (nibble i of a word = column 8c + {0,2,4,6,1,3,5,7}[i]);
 * out: [width][ceil(height/8)] words, word y/8 of row x = rows y..y+7 of column
 * x.  Used for qweight (height = K) and qzeros (height = K/128).  When height
 * is not a multiple of 8 the unused nibbles of a row's last word are filled as
 * the reference fills them (first rows of the next column, zero behind the
 * last column), so converted files are byte-identical.  width % 8 == 0. */
int llama2_repack_qdata(uint32_t* out, const uint32_t* in, int height, int width);

/* RepackScales (src/ModelConverter.cs:319-328): [meta_height][width] halfs ->
 * [width][meta_height]. */
int llama2_repack_scales(llama2_half* out, const llama2_half* in, int meta_height, int width);

/* The Format.v1 branch (src/ModelConverter.cs:247-262): scale rows stored with
 * ceil(scales_size/8)*8 halfs each -> rows of scales_size halfs. */
int llama2_compact_scales_v1(llama2_half* out, const llama2_half* in, int scales_size, int width);

/* ------------------------------------------------------------ decode step */

/* src/Config.cs:6-19 -- the 32-byte model-file header, same field order. */
typedef struct llama2_config {
    int dim;
    int hidden_dim;
    int n_layers;
    int n_heads;
    int n_kv_heads;
    int vocab_size;
    int seq_len;
    float rope_theta;
} llama2_config;

/* src/PerLayerWeight.cs:5-16 */
typedef struct llama2_layer_weights {
    llama2_qweight query, key, value, output, gate, up, down;
    const llama2_half* rms_attention;
    const llama2_half* rms_feed_forward;
} llama2_layer_weights;

/* src/TransformerWeights.cs:8-14 */
typedef struct llama2_transformer_weights {
    const llama2_half* token_embedding_table;
    const llama2_half* classifier_weights;
    const llama2_half* rms_final_weight;
    const llama2_layer_weights* layers; /* host array of n_layers entries */
} llama2_transformer_weights;

/* src/RunState.cs:7-25.  attention holds n_heads*max(dim, seq_len) halfs,
 * key/value caches n_layers*seq_len*kv_dim halfs, tokens seq_len+1 ints,
 * indices vocab_size ints (only the stochastic sampler uses it: may be null
 * for greedy decoding). */
typedef struct llama2_run_state {
    llama2_half* x;
    llama2_half* xb;
    llama2_half* h;
    llama2_half* q;
    llama2_half* attention;
    llama2_half* logits;
    llama2_half* key_cache;
    llama2_half* value_cache;
    int* tokens;
    int* indices;
} llama2_run_state;

typedef struct llama2_decoder llama2_decoder;

/* How llama2_decode_forward issues the step. */
#define LLAMA2_DECODE_MODULES 0 /* the 10 module launches per layer of Transformer.Forward */
#define LLAMA2_DECODE_FUSED 1   /* fused kernels (norm+QKV+RoPE, attention, norm+SwiGLU, ...) */
#define LLAMA2_DECODE_GRAPH 2   /* OR-able: replay the step as a captured hipGraph (one per attention launch shape) */
/* OR-able with LLAMA2_DECODE_FUSED: the whole of Transformer.Forward
 * (src/Transformer.cs:158-190) as ONE persistent launch -- one workgroup per
 * compute unit walks through all layers, the vectors between the modules are
 * handed from workgroup to workgroup inside the launch, and the weight stream
 * never stops at a module boundary.  Same arithmetic as LLAMA2_DECODE_FUSED, and
 * the same results bit for bit up to 1536 attended rows (beyond, the launch
 * sequence merges attention blocks of 256 rows and this step blocks of 128).  Serves histories of up to 3072 rows (longer ones fall
 * back to the launch sequence, step by step) and the shapes it has kernels for
 * (Llama-2-7B: dim 4096, hidden_dim 11008, 32 heads on 256 compute units; and
 * small models of at most one row per wavefront and phase: on 256 compute units
 * dim <= 640 and hidden_dim <= 2048); otherwise llama2_decode_create
 * returns LLAMA2_ERR_UNSUPPORTED.  The launch needs the GPU to itself: all its
 * workgroups must be resident at once.  Every wait inside it is bounded; a step
 * that gives up raises a sticky flag: llama2_decode_sample and
 * llama2_decode_sample_top_p return LLAMA2_ERR_STEP_FAILED from then on, and
 * after the asynchronous llama2_decode_run / _run_sampled the caller asks
 * llama2_decode_check. */
#define LLAMA2_DECODE_PERSISTENT 4

/* Binds a config, a weight set and a run state (all borrowed, all must outlive
 * the decoder) to the per-step launch sequence of Transformer.Forward
 * (src/Transformer.cs:158-190).  GQA is rejected like the reference does
 * (src/Transformer.cs:53-56).  A fused decoder keeps a workspace for known
 * tokens in batches (llama2_decode_run): 78 MiB for Llama-2-7B, 145 MiB for 13B
 * with contexts of 1024 rows or more, at most half of the memory that is free
 * and at most LLAMA2_PREFILL_MIB (an environment variable); with less the
 * batches get smaller, with nothing all tokens go step by step. */
int llama2_decode_create(llama2_decoder** decoder, const llama2_config* config,
                         const llama2_transformer_weights* weights,
                         const llama2_run_state* state, int mode);
/* Transformer.Forward(position, nextPosition): leaves fp16 logits in
 * state->logits.  Asynchronous. */
int llama2_decode_forward(llama2_decoder* decoder, int position, int next_position);
/* Sampler.Sample greedy branch (src/Sampler.cs:44-47,69): argmax into
 * tokens[next_position] iff generate_token, then reads that token back
 * (the one host synchronisation per token).  The token after the last row of
 * the context (next_position == seq_len) has no slot in `tokens`
 * (src/RunState.cs:52): it is returned without being stored, and the
 * device-resident loops below do not store it either. */
int llama2_decode_sample(llama2_decoder* decoder, int next_position, int generate_token,
                         int* token);
/* Sampler.Sample with temperature and top-p (src/Sampler.cs:40-70): the greedy
 * branch when temperature == 0 or !generate_token, otherwise the token that
 * llama2_sample picks on state->logits / state->indices with the caller's
 * uniform `coin` in [0, 1); then reads tokens[next_position] back.  Only the
 * token is defined: the sort stops at the head of the distribution that holds
 * top_p of the mass, so logits / indices are left partly sorted. */
int llama2_decode_sample_top_p(llama2_decoder* decoder, int next_position, int generate_token,
                               float temperature, float top_p, float coin, int* token);
/* The uniform number the device-resident sampling loop draws for the token at
 * `position` from `seed` (splitmix64 of seed + position, top 24 bits); exported
 * so that a host loop can reproduce llama2_decode_run_sampled step by step. */
float llama2_sampler_coin(unsigned long long seed, int position);
/* `steps` iterations of forward + greedy sample starting at `position`
 * without any host synchronisation in between (tokens stay on the device;
 * positions below n_prompt keep their prompt token, as Transformer.Generate
 * does, src/Transformer.cs:96-104).  Does not stop on token < 3.  A fused
 * decoder sends all but the last of the known tokens through the layers in
 * batches when those are at least 8: the same cache rows up to the
 * order of the fp32 sums. */
int llama2_decode_run(llama2_decoder* decoder, int position, int steps, int n_prompt);
/* The same loop with the stochastic sampler: the token at next_position p is
 * drawn with coin = llama2_sampler_coin(seed, p).  temperature == 0 is
 * llama2_decode_run.  (The reference draws from an unseeded System.Random,
 * src/Sampler.cs:24,42, on the host; this keeps the loop on the device.)
 * The tokens are those of llama2_decode_sample_top_p with the same coins; what
 * state->logits and state->indices hold afterwards is not: when a short head of
 * the sorted distribution carries more than top_p of the mass, only that head
 * is sorted and summed. */
int llama2_decode_run_sampled(llama2_decoder* decoder, int position, int steps, int n_prompt,
                              float temperature, float top_p, unsigned long long seed);
/* Waits for the enqueued steps and reports LLAMA2_ERR_STEP_FAILED if a
 * persistent step (LLAMA2_DECODE_PERSISTENT) gave up a wait; LLAMA2_OK for the
 * other modes.  No counterpart in the reference (its kernels cannot fail this
 * way). */
int llama2_decode_check(llama2_decoder* decoder);
/* Number of unsuccessful polls (about a microsecond each) after which a wait
 * inside the persistent step gives up; default 2^21.  Clears the failure flag.
 * For tests of the failure path and for hosts that want a tighter bound. */
int llama2_decode_set_wait_limit(llama2_decoder* decoder, int polls);
/* The int4 mat-vec set of every layer of the decoder's model -- RMSNorm + fused
 * QKV (native/mat_vec_kernel.cu:166-203), o-proj + residual (:144-164), RMSNorm
 * + fused SwiGLU (:206-234), down-proj + residual -- chained through all layers
 * in one persistent launch, exactly as the persistent step runs them, but
 * without attention: the o-projection takes q as its input.  input: dim halfs
 * (the residual stream entering layer 0); output: dim halfs (the residual
 * stream after the last layer).  Needs LLAMA2_DECODE_PERSISTENT.  This is the
 * measurement and parity handle for the mat-vec family inside the persistent
 * step; the KV cache is not touched. */
int llama2_decode_matvec_chain(llama2_decoder* decoder, const llama2_half* input,
                               llama2_half* output);
int llama2_decode_destroy(llama2_decoder* decoder);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif
#endif /* LLAMA2_HIP_H */
