// Tensor-core attention of 128-row query tiles over a list of pool rows (kernel in attend_tc.cu):
// chunks with a sliding window and sink tokens, and the shared prefix of a decode batch.
#pragma once

#include "common.cuh"

namespace attn {

struct AttendParams {
    const void *q, *k_cache, *v_cache;
    const int32_t* table;            // window: slot of every token, concatenated; prefix: slots of the shared rows
    int H, Hkv, B;
    int64_t n_slots;
    float scale_log2;
    int32_t* err_flag;
    // window
    const int32_t *kv_offsets, *q_offsets;
    void* out;
    int64_t n_q_tokens, n_kv_tokens;
    int window, sinks, head_pairs;
    int blocks, units;               // query blocks of the longest chunk, head units: set by the launcher
    // prefix
    float* parts;                    // o [n_parts, Hkv, B * G, D], then (m, l) [n_parts, Hkv, B * G]
    int n_prefix, splits, key_split;
    const float *k_scale, *v_scale;
};

bool attend_tc_supported(int D, int dtype, float scale);
// O of chunks; rows that no sequence covers are zeroed
int attend_window_launch(AttendParams p, int max_q_len, int D, int dtype, cudaStream_t st);
// partial rows of the shared prefix: sets p.splits and p.key_split from the sizes
void attend_prefix_plan(AttendParams& p);
__host__ __device__ inline int attend_prefix_parts(const AttendParams& p) { return p.splits * (p.key_split ? 2 : 1); }
int attend_prefix_launch(const AttendParams& p, int D, int dtype, bool e4m3, cudaStream_t st);

}  // namespace attn
