// Host-side helpers of tree-drafted decoding: mask rows and depths of a tree, rotary frequencies.
// See include/gqa_b200.h. No device memory is touched here.
#include "../../include/gqa_b200.h"

#include <cmath>
#include <cstring>

extern "C" {

int gqa_tree_masks(const int32_t* parents, const int32_t* sizes, int32_t batch, int32_t tokens,
                   uint32_t* mask, int32_t* depth) {
    if (parents == nullptr) return GQA_ERR_NULL;
    if (batch <= 0 || tokens <= 0 || tokens > GQA_TREE_MAX_TOKENS) return GQA_ERR_SHAPE;
    const int32_t words = (tokens + 31) / 32;
    // Everything is checked before anything is written.
    for (int32_t b = 0; b < batch; ++b) {
        const int32_t n = sizes != nullptr ? sizes[b] : tokens;
        if (n < 0 || n > tokens) return GQA_ERR_RANGE;
        const int32_t* par = parents + (size_t)b * tokens;
        for (int32_t t = 0; t < n; ++t) {
            if (t == 0 ? par[t] != -1 : (par[t] < 0 || par[t] >= t)) return GQA_ERR_RANGE;
        }
    }
    for (int32_t b = 0; b < batch; ++b) {
        const int32_t n = sizes != nullptr ? sizes[b] : tokens;
        const int32_t* par = parents + (size_t)b * tokens;
        uint32_t rows[GQA_TREE_MAX_TOKENS][GQA_TREE_MAX_TOKENS / 32] = {};
        int32_t deep[GQA_TREE_MAX_TOKENS] = {};
        for (int32_t t = 0; t < n; ++t) {
            if (t > 0) {
                std::memcpy(rows[t], rows[par[t]], sizeof(rows[t]));
                deep[t] = deep[par[t]] + 1;
            }
            rows[t][t / 32] |= 1u << (t % 32);
        }
        for (int32_t t = 0; t < tokens; ++t) {
            if (mask != nullptr) {
                std::memcpy(mask + ((size_t)b * tokens + t) * words, rows[t], words * sizeof(uint32_t));
            }
            if (depth != nullptr) depth[(size_t)b * tokens + t] = deep[t];
        }
    }
    return GQA_OK;
}

int gqa_rope_frequencies(int32_t rotary_dim, double base, int32_t scaling, double factor,
                         int32_t original_len, double beta_fast, double beta_slow, double* freq,
                         float* attn_factor) {
    if (freq == nullptr || attn_factor == nullptr) return GQA_ERR_NULL;
    if (rotary_dim < 8 || rotary_dim > 128 || rotary_dim % 8 != 0) return GQA_ERR_SHAPE;
    if (!(base > 0.0)) base = 1e6;
    if (!(beta_fast > 0.0)) beta_fast = 32.0;
    if (!(beta_slow > 0.0)) beta_slow = 1.0;
    if (scaling < GQA_ROPE_SCALE_NONE || scaling > GQA_ROPE_SCALE_YARN) return GQA_ERR_UNSUPPORTED;
    if (scaling != GQA_ROPE_SCALE_NONE && !(factor >= 1.0 && std::isfinite(factor))) return GQA_ERR_RANGE;
    if (scaling == GQA_ROPE_SCALE_YARN && (original_len <= 0 || !(beta_fast > beta_slow))) {
        return GQA_ERR_RANGE;
    }
    if (scaling == GQA_ROPE_SCALE_NTK) base *= std::pow(factor, rotary_dim / (rotary_dim - 2.0));
    for (int32_t i = 0; i < rotary_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rotary_dim);
        if (scaling == GQA_ROPE_SCALE_LINEAR) f /= factor;
        if (scaling == GQA_ROPE_SCALE_YARN) {
            // Turns of the pair over the trained context decide how much of it is stretched.
            const double turns = original_len * f / (2.0 * 3.14159265358979323846);
            double keep = (turns - beta_slow) / (beta_fast - beta_slow);
            keep = keep < 0.0 ? 0.0 : (keep > 1.0 ? 1.0 : keep);
            f = f * keep + f / factor * (1.0 - keep);
        }
        freq[i] = f;
    }
    *attn_factor = scaling == GQA_ROPE_SCALE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return GQA_OK;
}

}  // extern "C"
