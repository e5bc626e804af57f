// Chunks of sequences with a sliding window and sink tokens: entry point and the generic kernel.  Not in the
// reference (its packed prefill: paged_attention_kernel.cu:15-98).  head_dim 64 and 128 in 16 bits run
// on the tensor cores (attend_tc.cu).
#include "attend_tc.cuh"

namespace attn {
namespace {

// Any type and any head_dim up to 32 * DPL: one warp per (query row, head), a lane per dim, online softmax over the
// visible keys (the sinks that precede the window, then the window).  Compatibility path.
template <typename T, int DPL>
__global__ void window_prefill_generic_kernel(const AttendParams p, int D, int max_q_len) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.z, h = blockIdx.y, hk = h / (p.H / p.Hkv);
    const int64_t q_beg = b ? p.q_offsets[b - 1] : 0, q_end = p.q_offsets[b];
    const int64_t kv_beg = b ? p.kv_offsets[b - 1] : 0, kv_end = p.kv_offsets[b];
    if (q_beg < 0 || q_end < q_beg || q_end > p.n_q_tokens || kv_beg < 0 || kv_end > p.n_kv_tokens || kv_end - kv_beg < q_end - q_beg ||
        q_end - q_beg > max_q_len) {
        if (p.err_flag && threadIdx.x == 0) atomicOr(p.err_flag, ATTN_B200_FLAG_BAD_OFFSETS);
        if (q_beg < 0 || q_end < q_beg || q_end > p.n_q_tokens || kv_beg < 0 || kv_end > p.n_kv_tokens || kv_end - kv_beg < q_end - q_beg)
            return;
    }
    const int64_t row = q_beg + (int64_t)blockIdx.x * (blockDim.x >> 5) + warp;
    if (row >= q_end) return;
    const int64_t pos = (kv_end - kv_beg) - (q_end - row);          // the query's position
    const int64_t first = pos - p.window + 1 > 0 ? pos - p.window + 1 : 0, sinks = p.sinks < first ? p.sinks : first;
    float q[DPL], o[DPL], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
        const int d = lane + 32 * i;
        o[i] = 0.f;
        q[i] = d < D ? to_f32<T>(((const T*)p.q)[(row * p.H + h) * D + d]) : 0.f;
    }
    const int64_t n = sinks + pos - first + 1;
    for (int64_t u = 0; u < n; ++u) {
        const int64_t slot = p.table[kv_beg + (u < sinks ? u : u - sinks + first)];
        if (slot < 0 || slot >= p.n_slots) {
            if (p.err_flag && lane == 0) atomicOr(p.err_flag, ATTN_B200_FLAG_BAD_SLOT);
            continue;
        }
        const T* kr = (const T*)p.k_cache + (slot * p.Hkv + hk) * D;
        const T* vr = (const T*)p.v_cache + (slot * p.Hkv + hk) * D;
        float s = 0.f, v[DPL];
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
            const int d = lane + 32 * i;
            v[i] = d < D ? to_f32<T>(vr[d]) : 0.f;
            if (d < D) s += q[i] * to_f32<T>(kr[d]);
        }
        s = group_sum<32>(s) * p.scale_log2;
        const float m_new = fmaxf(m, s), msub = m_new > -INFINITY ? m_new : 0.f;
        const float alpha = fast_exp2(m - msub), pr = fast_exp2(s - msub);
        l = l * alpha + pr;
        m = m_new;
#pragma unroll
        for (int i = 0; i < DPL; ++i) o[i] = o[i] * alpha + pr * v[i];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;                      // no key at all (bad slots): zeros
#pragma unroll
    for (int i = 0; i < DPL; ++i)
        if (lane + 32 * i < D) ((T*)p.out)[(row * p.H + h) * D + lane + 32 * i] = from_f32<T>(o[i] * inv);
}

template <typename T>
int launch_generic(const AttendParams& p, int D, int max_q_len, cudaStream_t st) {
    const cudaError_t e = cudaMemsetAsync(p.out, 0, (size_t)p.n_q_tokens * p.H * D * sizeof(T), st);    // rows that no sequence covers
    if (e != cudaSuccess) return (int)e;
    if (max_q_len == 0 || p.B == 0) return 0;
    const dim3 grid((unsigned)((max_q_len + 3) / 4), p.H, p.B);
    if (D <= 64) window_prefill_generic_kernel<T, 2><<<grid, 128, 0, st>>>(p, D, max_q_len);
    else if (D <= 128) window_prefill_generic_kernel<T, 4><<<grid, 128, 0, st>>>(p, D, max_q_len);
    else if (D <= 256) window_prefill_generic_kernel<T, 8><<<grid, 128, 0, st>>>(p, D, max_q_len);
    else window_prefill_generic_kernel<T, 16><<<grid, 128, 0, st>>>(p, D, max_q_len);
    return (int)cudaGetLastError();
}

}  // namespace
}  // namespace attn

extern "C" int attn_b200_paged_window_prefill(const void* q, const void* k_cache, const void* v_cache, const int32_t* slots,
                                              const int32_t* kv_offsets, const int32_t* q_offsets, void* out, int B,
                                              int64_t n_q_tokens, int64_t n_kv_tokens, int max_q_len, int H, int n_kv_heads,
                                              int D, int64_t n_slots, int window, int n_sinks, float scale, int dtype,
                                              int force_generic, int32_t* err_flag, void* stream) {
    using namespace attn;
    if (B < 0 || H <= 0 || n_kv_heads <= 0 || H % n_kv_heads || D <= 0 || n_q_tokens < 0 || n_kv_tokens < 0 || n_slots < 0 ||
        max_q_len < 0 || window <= 0 || n_sinks < 0)
        return ATTN_B200_EINVAL;
    if (dtype != ATTN_B200_F16 && dtype != ATTN_B200_BF16 && dtype != ATTN_B200_F32) return ATTN_B200_EDTYPE;
    if (D > 512) return ATTN_B200_ESHAPE;
    if (n_slots > 0x7fffffffLL || n_kv_tokens > 0x7fffffffLL || n_q_tokens > 0x7fffffffLL || B > 65535 || H > 65535)
        return ATTN_B200_ETOOLARGE;
    if (n_q_tokens == 0) return 0;
    if (!q || !out || (B && (!kv_offsets || !q_offsets)) || (n_kv_tokens && (!slots || !k_cache || !v_cache))) return ATTN_B200_EINVAL;
    AttendParams p{};
    p.q = q; p.k_cache = k_cache; p.v_cache = v_cache; p.table = slots;
    p.H = H; p.Hkv = n_kv_heads; p.B = B; p.n_slots = n_slots;
    p.scale_log2 = scale * kLog2e;
    p.err_flag = err_flag;
    p.kv_offsets = kv_offsets; p.q_offsets = q_offsets; p.out = out;
    p.n_q_tokens = n_q_tokens; p.n_kv_tokens = n_kv_tokens;
    p.window = window; p.sinks = n_sinks;
    cudaStream_t st = (cudaStream_t)stream;
    if (!force_generic && n_slots > 0 && attend_tc_supported(D, dtype, scale) &&
        (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15) == 0)
        return attend_window_launch(p, max_q_len, D, dtype, st);
    switch (dtype) {
        case ATTN_B200_F16: return launch_generic<__half>(p, D, max_q_len, st);
        case ATTN_B200_BF16: return launch_generic<__nv_bfloat16>(p, D, max_q_len, st);
        default: return launch_generic<float>(p, D, max_q_len, st);
    }
}
