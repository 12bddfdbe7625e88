// C facade over the C++ host layer (llama2_host.hpp) so that the pytest suite
// can drive libLlama2::Transformer the way an application drives the
// reference's ITransformer.  Builds into libllama2_host.so.
#include "llama2_host.hpp"

#include <algorithm>
#include <string>

using namespace libLlama2;

namespace {
thread_local std::string g_error;

template <class F>
int guarded(F&& f)
{
    try {
        f();
        g_error.clear();
        return 0;
    } catch (const FileLoadException& e) {
        g_error = std::string("FileLoadException: ") + e.what();
        return 1;
    } catch (const NotImplementedException& e) {
        g_error = std::string("NotImplementedException: ") + e.what();
        return 2;
    } catch (const Llama2Exception& e) {
        g_error = std::string("Llama2Exception: ") + e.what();
        return 3;
    } catch (const std::exception& e) {
        g_error = std::string("exception: ") + e.what();
        return 4;
    }
}
} // namespace

extern "C" {

__attribute__((visibility("default"))) const char* l2h_last_error(void) { return g_error.c_str(); }

// The checks the Transformer constructor makes on a model file before it touches
// the GPU contents: header, GQA, size of the tensor stream.  No GPU needed.
__attribute__((visibility("default"))) int l2h_check_model_file(const char* path)
{
    return guarded([&] {
        MappedFile file(path);
        Config c = Config::LoadConfig(file.data(), file.size());
        if (c.kvDim() != c.dim)
            throw NotImplementedException("Differing kvDim dimention not currently supported.");
        const size_t remaining = file.size() - Config::Size;
        if (TransformerWeights::ExpectedBytes(c) != remaining)
            throw FileLoadException("Failed to read file. offset: " + std::to_string(TransformerWeights::ExpectedBytes(c)) +
                                    " != length: " + std::to_string(remaining));
    });
}

// ModelConverter::RepackQWeight on caller-provided host arrays; out_* sized as in the model file.
__attribute__((visibility("default"))) int l2h_repack_qweight(const uint32_t* qweight, const uint32_t* qzeros,
                                                              const uint16_t* scales, int height, int width, int format,
                                                              uint32_t* out_weight, uint32_t* out_zeros, uint16_t* out_scales)
{
    return guarded([&] {
        Check(llama2_init(0));
        auto r = ModelConverter::RepackQWeight(qweight, qzeros, scales, height, width,
                                               format == 0 ? ModelConverter::Format::v0 : ModelConverter::Format::v1);
        std::copy(r.Weight.begin(), r.Weight.end(), out_weight);
        std::copy(r.Zeros.begin(), r.Zeros.end(), out_zeros);
        std::copy(r.Scales.begin(), r.Scales.end(), out_scales);
    });
}

// A step of several requests through the three module classes; device pointers throughout, gammas may be null.
__attribute__((visibility("default"))) int l2h_batch_step(const llama2_batch* batch, const llama2_paged_cache* cache, int* counts,
                                                          int* free_blocks, int n_free, int* taken, Half* query, Half* key, Half* value,
                                                          Half* q_gamma, Half* k_gamma, Half* output, int n_heads, float theta, float scale)
{
    return guarded([&] {
        const size_t tokens = batch->n_tokens, row = static_cast<size_t>(n_heads) * cache->head_size,
                     kvRow = static_cast<size_t>(cache->n_kv_heads) * cache->head_size;
        auto halfs = [](Half* p, size_t n) { return DeviceVariable<Half>::Window(p, n); };
        auto q = halfs(query, tokens * row), k = halfs(key, tokens * kvRow), v = halfs(value, tokens * kvRow), out = halfs(output, tokens * row);
        auto gq = halfs(q_gamma, cache->head_size), gk = halfs(k_gamma, cache->head_size);
        auto c = DeviceVariable<int>::Window(counts, batch->n_requests), f = DeviceVariable<int>::Window(free_blocks, n_free),
             t = DeviceVariable<int>::Window(taken, 1);
        BatchTables().Forward(*batch, c, f, t, cache->block_size);
        BatchQKNormRoPE().Forward(q, q, k, v, q_gamma ? &gq : nullptr, k_gamma ? &gk : nullptr, *batch, *cache, n_heads, theta);
        BatchAttention().Forward(out, q, *batch, *cache, n_heads, scale);
    });
}

// The rest of a layer's step, from the attention's output on, and the answers from a row of logits per token, through the module
// classes: o = output projection onto x, norm, gated block, down projection, x += norm(that) * post_gamma, norm into xb; log
// probabilities of `given`.  Device pointers throughout, adapters may be null.
__attribute__((visibility("default"))) int l2h_batch_block(const llama2_batch* batch, const llama2_layer_weights* w, Half* attention, Half* x,
                                                           Half* xb, Half* h, Half* y, int dim, int hidden, const llama2_adapters* adapters,
                                                           int* token_adapters, Half* post_gamma, Half* next_gamma, Half* logits, int vocab,
                                                           int* given, float* log_probs, float* entropies, int* top_tokens, int n_top)
{
    return guarded([&] {
        const size_t tokens = batch->n_tokens;
        auto halfs = [](Half* p, size_t n) { return DeviceVariable<Half>::Window(p, n); };
        auto a = halfs(attention, tokens * dim), res = halfs(x, tokens * dim), normed = halfs(xb, tokens * dim), mid = halfs(h, tokens * hidden),
             out = halfs(y, tokens * dim), ff = halfs(const_cast<Half*>(w->rms_feed_forward), dim), post = halfs(post_gamma, dim),
             next = halfs(next_gamma, dim), l = halfs(logits, tokens * vocab);
        auto ids = DeviceVariable<int>::Window(token_adapters, tokens), g = DeviceVariable<int>::Window(given, tokens),
             top = DeviceVariable<int>::Window(top_tokens, tokens * n_top), pos = DeviceVariable<int>::Window(batch->positions, tokens);
        auto lp = DeviceVariable<float>::Window(log_probs, tokens), e = DeviceVariable<float>::Window(entropies, tokens);
        BatchMatMulInt4().Forward({{w->output, x, x, adapters, dim, dim, dim}}, a, dim, *batch, &ids);
        BatchResidualRMSNorm().Forward(normed, res, nullptr, ff, dim, *batch);
        BatchMatMulSwiGLU().Forward(mid, normed, w->gate, w->up, dim, hidden, *batch);
        BatchMatMulInt4().Forward({{w->down, y, nullptr, nullptr, dim, dim, 0}}, mid, hidden, *batch);
        BatchResidualRMSNorm().Forward(normed, res, &out, next, dim, *batch, &post);
        BatchLogProbs().Forward(&lp, &e, &top, nullptr, l, static_cast<int>(tokens), vocab, &g, 1, n_top, 1.0f, &pos);
    });
}

__attribute__((visibility("default"))) int l2h_transformer_open(const char* path, int mode, int stop_on_special, void** handle)
{
    *handle = nullptr;
    return guarded([&] { *handle = new Transformer(path, static_cast<Transformer::Mode>(mode), stop_on_special != 0); });
}

__attribute__((visibility("default"))) int l2h_transformer_open_sampled(const char* path, int mode, int stop_on_special,
                                                                        float temperature, float top_p,
                                                                        unsigned long long seed, void** handle)
{
    *handle = nullptr;
    return guarded([&] {
        *handle = new Transformer(path, static_cast<Transformer::Mode>(mode), stop_on_special != 0, temperature, top_p, seed);
    });
}

__attribute__((visibility("default"))) int l2h_transformer_generate(void* handle, const int* prompt, int n_prompt, int steps,
                                                                    int* out, int* n_out)
{
    return guarded([&] {
        auto* t = static_cast<Transformer*>(handle);
        std::vector<int> tokens = t->Generate(std::vector<int>(prompt, prompt + n_prompt), steps);
        for (size_t i = 0; i < tokens.size(); ++i)
            out[i] = tokens[i];
        *n_out = static_cast<int>(tokens.size());
    });
}

__attribute__((visibility("default"))) int l2h_transformer_logits(void* handle, uint16_t* out, int n)
{
    return guarded([&] {
        std::vector<Half> l = static_cast<Transformer*>(handle)->Logits();
        for (int i = 0; i < n && i < static_cast<int>(l.size()); ++i)
            out[i] = l[i];
    });
}

__attribute__((visibility("default"))) int l2h_transformer_seq_len(void* handle)
{
    return static_cast<Transformer*>(handle)->config.seq_len;
}

__attribute__((visibility("default"))) int l2h_transformer_close(void* handle)
{
    return guarded([&] { delete static_cast<Transformer*>(handle); });
}

} // extern "C"
