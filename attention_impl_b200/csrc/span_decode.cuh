// Decode of one token per sequence over a SPAN of its cached tokens: the first few (sinks) and the last
// `window`, or all of them, optionally beside partial results for rows that the whole batch shares.
// Parameter block and launcher; the kernels are in span_decode.cu.
#pragma once

#include "common.cuh"

namespace attn {

struct SpanParams {
    const void *q, *k_new, *v_new, *k_cache, *v_cache;
    const int32_t *table, *offsets;     // slot per token, or a block table; inclusive cumulative lengths
    const int32_t* prefix;              // slots of rows that every sequence sees before its own
    int n_prefix;
    void* out;
    const float* parts;                 // to fold in, or null: o [n_parts, Hkv, B * G, D], then (m (log2), l) [n_parts, Hkv, B * G]
    int n_parts;
    int B, H, Hkv, D;
    int64_t n_tokens, n_slots;          // entries of a per-token table; pool rows
    int block_size, max_blocks;
    int window, sinks;                  // cached token t of ctx is seen iff t > ctx - window or t < sinks
    float scale_log2;
    const float *k_scale, *v_scale;
    int32_t* err_flag;
    int early;                          // inputs are complete when this kernel starts; only `parts` needs its wait
    // set by the launcher
    int hpc_log2, n_sets, splits;
};

// `span`: an estimate of the cached tokens that a sequence attends to; `ragged`: an average of very different numbers,
// not a bound that most sequences reach (both only for the split).
int span_decode_launch(SpanParams p, int64_t span, bool ragged, int q_dtype, int kv_dtype, cudaStream_t st);

}  // namespace attn
