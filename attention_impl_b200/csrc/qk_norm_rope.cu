// RMS norm of every query and key head, rotation and (optionally) the append to the KV pools, in one
// pass over the data.
//
//   x  <- x * rsqrt(mean_d x^2 + eps) * w[d]                                    per token and head
//   (x[d], x[d + r]) <- (x[d] c - x[d + r] s, x[d + r] c + x[d] s),  d < r,  c, s = cos/sin[pos, d]
//   k_cache[slot] = k, v_cache[slot] = v                                        optionally as e4m3(x / scale)
//
// The reference has neither the norm nor the append (its rotation: rotary_embedding.cu:10-36).  The
// sum of squares, the norm and the rotation are held in 32 bits and every stored value is rounded
// once, from the 32-bit result: the pool's e4m3 code comes from it too, not from the 16-bit k.
//
// Bound: HBM.  q, k (and v) are read once and written once (k and v once more into the pools); done as
// a norm followed by rope_write_kv_kernel, q and k would travel twice.
#include "common.cuh"

namespace attn {
namespace {

struct NormRopeParams {
    const void *q, *k, *v;
    void *q_out, *k_out;
    const void *wq, *wk;
    const int32_t* positions;
    const void *cos, *sin;
    const int32_t* slots;            // null: no append
    void *k_cache, *v_cache;
    const float *k_scale, *v_scale;  // null: the pools hold the input type
    int64_t n_tokens, q_stride, k_stride, v_stride, qo_stride, ko_stride;   // row strides in elements
    int64_t max_pos, n_slots;
    int hq, hk, d, rot;
    int w_f32, cs_f32;               // weights / tables are float instead of the input type
    float eps;
    int tpt_log2;                    // vector kernel: threads per token
    int32_t* err_flag;
};

// 16 bytes of T as floats and back
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <> struct Vec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
        unpack2(u.x, __half(), f[0], f[1]); unpack2(u.y, __half(), f[2], f[3]);
        unpack2(u.z, __half(), f[4], f[5]); unpack2(u.w, __half(), f[6], f[7]);
    }
    static __device__ __forceinline__ uint32_t p2(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        return make_uint4(p2(f[0], f[1]), p2(f[2], f[3]), p2(f[4], f[5]), p2(f[6], f[7]));
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
        unpack2(u.x, __nv_bfloat16(), f[0], f[1]); unpack2(u.y, __nv_bfloat16(), f[2], f[3]);
        unpack2(u.z, __nv_bfloat16(), f[4], f[5]); unpack2(u.w, __nv_bfloat16(), f[6], f[7]);
    }
    static __device__ __forceinline__ uint32_t p2(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        return make_uint4(p2(f[0], f[1]), p2(f[2], f[3]), p2(f[4], f[5]), p2(f[6], f[7]));
    }
};

// Vec<T>::N consecutive weights or table entries, stored as T or as float
template <typename T> __device__ __forceinline__ void load_aux(const void* base, int64_t at, int f32, float* f) {
    constexpr int N = Vec<T>::N;
    if (f32) {
#pragma unroll
        for (int i = 0; i < N; i += 4) Vec<float>::unpack(__ldg(reinterpret_cast<const uint4*>((const float*)base + at + i)), f + i);
    } else {
        Vec<T>::unpack(__ldg(reinterpret_cast<const uint4*>((const T*)base + at)), f);
    }
}

__device__ __forceinline__ uint32_t e4m3x4(const float* f) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
// Vec<T>::N values into a pool row (element index `at`); `scale` null: in the input type
template <typename T> __device__ __forceinline__ void store_pool(void* pool, int64_t at, const float* f, const float* scale, int head) {
    if (scale) {
        if constexpr (Vec<T>::N == 8) {
            const float s = scale[head];
            float g[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = f[i] / s;
            *reinterpret_cast<uint2*>((char*)pool + at) = make_uint2(e4m3x4(g), e4m3x4(g + 4));
        }
    } else {
        *reinterpret_cast<uint4*>((T*)pool + at) = Vec<T>::pack(f);
    }
}

__device__ __forceinline__ bool token_ok(const NormRopeParams& p, int64_t token, int lane0, int& pos, int64_t& slot) {
    pos = p.positions[token];
    const bool ok = pos >= 0 && pos < p.max_pos;
    slot = -1;
    if (p.slots) {
        const int s = p.slots[token];
        if (s >= 0 && s < p.n_slots) slot = s;
        else if (p.err_flag && lane0 == 0) atomicOr(p.err_flag, ATTN_B200_FLAG_BAD_SLOT);
    }
    if (!ok) {
        slot = -1;
        if (p.err_flag && lane0 == 0) atomicOr(p.err_flag, ATTN_B200_FLAG_BAD_POSITION);
    }
    return ok;
}

// Vector kernel.  A head is LPH lanes; a lane owns two 16-byte chunks of every head it visits: chunk s
// and its rotation partner s + r/N, or, beyond the rotated dims, two neighbours (the last one may be
// alone).  Both are in registers before anything is stored, so the output may be the input.  The sum
// of squares is log2(LPH) shuffles.  A lane keeps its place within the head, so its weights and its
// cos/sin entries are loaded once for all heads of the token.  A token's heads are dealt to 2^tpt_log2
// threads, kUnroll heads' loads in flight at a time.
constexpr int kThreads = 256, kUnroll = 2;

template <typename T, int LPH>
__global__ void __launch_bounds__(kThreads)
qk_norm_rope_kernel(const NormRopeParams p) {
    constexpr int N = Vec<T>::N;
    // a programmatic dependent (a decode kernel) may be scheduled from here on; it reads nothing this
    // kernel writes before its own wait
    asm volatile("griddepcontrol.launch_dependents;");
    const int tpt = 1 << p.tpt_log2;
    const int tid = threadIdx.x & (tpt - 1);
    const int64_t tok_raw = (int64_t)blockIdx.x * (kThreads >> p.tpt_log2) + (threadIdx.x >> p.tpt_log2);
    const bool live = tok_raw < p.n_tokens;               // whole LPH groups agree; shuffles run for all
    const int64_t token = live ? tok_raw : p.n_tokens - 1;
    int pos;
    int64_t slot;
    const bool pos_ok = token_ok(p, token, live ? tid : 1, pos, slot);

    const int hv = p.d / N, cph = p.rot / N;
    const int sub = tid & (LPH - 1), grp = tid / LPH, ngrp = tpt / LPH;
    // chunks of this lane (ca < 0: none; cb < 0: no second one)
    int ca, cb;
    const bool rotates = sub < cph;
    if (rotates) {
        ca = sub;
        cb = sub + cph;
    } else {
        ca = 2 * cph + 2 * (sub - cph);
        cb = ca + 1;
        if (ca >= hv) ca = -1;
        if (cb >= hv) cb = -1;
    }
    float c[N], s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) { c[i] = 1.f; s[i] = 0.f; }
    if (rotates && pos_ok) {
        load_aux<T>(p.cos, (int64_t)pos * p.rot + ca * N, p.cs_f32, c);
        load_aux<T>(p.sin, (int64_t)pos * p.rot + ca * N, p.cs_f32, s);
    }
    const int heads = p.hq + p.hk;
    const float inv_d = 1.f / (float)p.d;
    for (int h0 = grp; h0 - grp < heads; h0 += ngrp * kUnroll) {      // the same number of rounds for every thread
        uint4 ua[kUnroll], ub[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int h = h0 + u * ngrp;
            ua[u] = ub[u] = make_uint4(0, 0, 0, 0);
            if (h < heads) {
                const T* row = h < p.hq ? (const T*)p.q + token * p.q_stride + (int64_t)h * p.d
                                        : (const T*)p.k + token * p.k_stride + (int64_t)(h - p.hq) * p.d;
                if (ca >= 0) ua[u] = *reinterpret_cast<const uint4*>(row + ca * N);
                if (cb >= 0) ub[u] = *reinterpret_cast<const uint4*>(row + cb * N);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int h = h0 + u * ngrp;
            const bool is_q = h < p.hq;
            float a[N], b[N], w[N];
            Vec<T>::unpack(ua[u], a);
            Vec<T>::unpack(ub[u], b);
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) ss += a[i] * a[i] + b[i] * b[i];
            ss = group_sum<LPH>(ss);
            const float r = rsqrtf(ss * inv_d + p.eps);
            if (h >= heads || !live) continue;
            const void* wp = is_q ? p.wq : p.wk;
            if (ca >= 0) {
                load_aux<T>(wp, ca * N, p.w_f32, w);
#pragma unroll
                for (int i = 0; i < N; ++i) a[i] = a[i] * r * w[i];
            }
            if (cb >= 0) {
                load_aux<T>(wp, cb * N, p.w_f32, w);
#pragma unroll
                for (int i = 0; i < N; ++i) b[i] = b[i] * r * w[i];
            }
            if (rotates) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float x = a[i], y = b[i];
                    a[i] = x * c[i] - y * s[i];
                    b[i] = y * c[i] + x * s[i];
                }
            }
            if (!pos_ok) {              // no such table row: the token's outputs are zero and nothing is appended
#pragma unroll
                for (int i = 0; i < N; ++i) a[i] = b[i] = 0.f;
            }
            T* out = is_q ? (T*)p.q_out + token * p.qo_stride + (int64_t)h * p.d
                          : (T*)p.k_out + token * p.ko_stride + (int64_t)(h - p.hq) * p.d;
            if (ca >= 0) *reinterpret_cast<uint4*>(out + ca * N) = Vec<T>::pack(a);
            if (cb >= 0) *reinterpret_cast<uint4*>(out + cb * N) = Vec<T>::pack(b);
            if (!is_q && slot >= 0) {
                const int64_t at = (slot * p.hk + (h - p.hq)) * p.d;
                if (ca >= 0) store_pool<T>(p.k_cache, at + ca * N, a, p.k_scale, h - p.hq);
                if (cb >= 0) store_pool<T>(p.k_cache, at + cb * N, b, p.k_scale, h - p.hq);
            }
        }
    }
    if (slot < 0 || !live) return;
    const int v_items = p.hk * hv;
    for (int i0 = tid; i0 < v_items; i0 += tpt * 4) {
        uint4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * tpt;
            if (i < v_items) x[u] = ldg_stream128((const T*)p.v + token * p.v_stride + (int64_t)i * N);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * tpt;
            if (i >= v_items) break;
            if (p.v_scale) {
                float f[N];
                Vec<T>::unpack(x[u], f);
                store_pool<T>(p.v_cache, slot * p.hk * p.d + (int64_t)i * N, f, p.v_scale, i / hv);
            } else {
                *reinterpret_cast<uint4*>((T*)p.v_cache + slot * p.hk * p.d + (int64_t)i * N) = x[u];
            }
        }
    }
}

// Any head_dim, rotary width, stride and alignment: one warp per (token, head); a lane owns the pairs
// (d, d + r) and the dims beyond 2 r with d = lane (mod 32), so the output may be the input here too.
template <typename T>
__global__ void qk_norm_rope_generic_kernel(const NormRopeParams p, int64_t n_items, int heads) {
    const int64_t item = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (item >= n_items) return;
    const int lane = threadIdx.x & 31;
    const int64_t token = item / heads;
    const int h = (int)(item - token * heads);
    int pos;
    int64_t slot;
    const bool pos_ok = token_ok(p, token, lane, pos, slot);
    auto pool = [&](void* cache, const float* scale, int head, int d, float x) {
        const int64_t at = (slot * p.hk + head) * p.d + d;
        if (scale) ((uint8_t*)cache)[at] = __nv_cvt_float_to_fp8(x / scale[head], __NV_SATFINITE, __NV_E4M3);
        else ((T*)cache)[at] = from_f32<T>(x);
    };
    if (h >= p.hq + p.hk) {                        // a head of v: append only
        const int hv = h - p.hq - p.hk;
        const T* row = (const T*)p.v + token * p.v_stride + (int64_t)hv * p.d;
        if (slot >= 0)
            for (int d = lane; d < p.d; d += 32) pool(p.v_cache, p.v_scale, hv, d, to_f32<T>(row[d]));
        return;
    }
    const bool is_q = h < p.hq;
    const int hh = is_q ? h : h - p.hq;
    const T* row = is_q ? (const T*)p.q + token * p.q_stride + (int64_t)hh * p.d : (const T*)p.k + token * p.k_stride + (int64_t)hh * p.d;
    T* out = is_q ? (T*)p.q_out + token * p.qo_stride + (int64_t)hh * p.d : (T*)p.k_out + token * p.ko_stride + (int64_t)hh * p.d;
    float ss = 0.f;
    for (int d = lane; d < p.d; d += 32) {
        const float x = to_f32<T>(row[d]);
        ss += x * x;
    }
    ss = group_sum<32>(ss);                        // every lane has read the row before any lane writes it
    const float r = rsqrtf(ss / (float)p.d + p.eps);
    auto aux = [&](const void* base, int64_t at, int f32) { return f32 ? ((const float*)base)[at] : to_f32<T>(((const T*)base)[at]); };
    const void* w = is_q ? p.wq : p.wk;
    auto put = [&](int d, float x) {
        if (!pos_ok) x = 0.f;
        out[d] = from_f32<T>(x);
        if (!is_q && slot >= 0) pool(p.k_cache, p.k_scale, hh, d, x);
    };
    for (int d = lane; d < p.rot; d += 32) {
        const float a = to_f32<T>(row[d]) * r * aux(w, d, p.w_f32), b = to_f32<T>(row[d + p.rot]) * r * aux(w, d + p.rot, p.w_f32);
        const float c = pos_ok ? aux(p.cos, (int64_t)pos * p.rot + d, p.cs_f32) : 0.f;
        const float s = pos_ok ? aux(p.sin, (int64_t)pos * p.rot + d, p.cs_f32) : 0.f;
        put(d, a * c - b * s);
        put(d + p.rot, b * c + a * s);
    }
    for (int d = 2 * p.rot + lane; d < p.d; d += 32) put(d, to_f32<T>(row[d]) * r * aux(w, d, p.w_f32));
}

template <typename T> int launch(const NormRopeParams& p0, cudaStream_t st) {
    NormRopeParams p = p0;
    constexpr int N = Vec<T>::N;
    const int hv = p.d / N, slots = (hv + 1) / 2;
    uintptr_t bits = (uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.q_out | (uintptr_t)p.k_out | (uintptr_t)p.wq |
                     (uintptr_t)p.wk | (uintptr_t)p.cos | (uintptr_t)p.sin;
    int64_t strides = p.q_stride | p.k_stride | p.qo_stride | p.ko_stride;
    if (p.slots) {
        bits |= (uintptr_t)p.v | (uintptr_t)p.k_cache | (uintptr_t)p.v_cache;
        strides |= p.v_stride;
    }
    const int heads = p.hq + p.hk;
    if (p.d % N == 0 && p.rot % N == 0 && slots <= 32 && bits % 16 == 0 && strides % N == 0) {
        int lph = 1;
        while (lph < slots) lph <<= 1;
        // threads per token: two rounds of kUnroll heads each, at least one LPH group, at most the CTA
        int tl = 0;
        while ((1 << tl) < kThreads && ((1 << tl) < lph || (1 << tl) * 2 * kUnroll < heads * lph)) ++tl;
        p.tpt_log2 = tl;
        const int64_t per_cta = kThreads >> tl, ctas = (p.n_tokens + per_cta - 1) / per_cta;
        if (ctas > 0x7fffffff) return ATTN_B200_ETOOLARGE;
        switch (lph) {
            case 1: qk_norm_rope_kernel<T, 1><<<(unsigned)ctas, kThreads, 0, st>>>(p); break;
            case 2: qk_norm_rope_kernel<T, 2><<<(unsigned)ctas, kThreads, 0, st>>>(p); break;
            case 4: qk_norm_rope_kernel<T, 4><<<(unsigned)ctas, kThreads, 0, st>>>(p); break;
            case 8: qk_norm_rope_kernel<T, 8><<<(unsigned)ctas, kThreads, 0, st>>>(p); break;
            case 16: qk_norm_rope_kernel<T, 16><<<(unsigned)ctas, kThreads, 0, st>>>(p); break;
            default: qk_norm_rope_kernel<T, 32><<<(unsigned)ctas, kThreads, 0, st>>>(p); break;
        }
        return (int)cudaGetLastError();
    }
    const int per_token = heads + (p.slots ? p.hk : 0);
    const int64_t items = p.n_tokens * per_token, ctas = (items + 7) / 8;
    if (ctas > 0x7fffffff) return ATTN_B200_ETOOLARGE;
    qk_norm_rope_generic_kernel<T><<<(unsigned)ctas, 256, 0, st>>>(p, items, per_token);
    return (int)cudaGetLastError();
}

}  // namespace
}  // namespace attn

extern "C" int attn_b200_qk_norm_rope(const void* q, const void* k, const void* v, void* q_out, void* k_out,
                                      const void* q_weight, const void* k_weight, const int32_t* positions,
                                      const void* cos, const void* sin, const int32_t* slots, void* k_cache,
                                      void* v_cache, int64_t n_tokens, int n_heads_q, int n_heads_k, int head_dim,
                                      int rot_half, int64_t max_pos, int64_t n_slots, int64_t q_stride,
                                      int64_t k_stride, int64_t v_stride, int64_t q_out_stride, int64_t k_out_stride,
                                      float eps, int dtype, int weight_dtype, int table_dtype, int kv_dtype,
                                      const float* k_scale, const float* v_scale, int32_t* err_flag, void* stream) {
    using namespace attn;
    if (n_tokens < 0 || n_heads_q <= 0 || n_heads_k <= 0 || head_dim <= 0 || rot_half < 0 || max_pos < 0 || n_slots < 0)
        return ATTN_B200_EINVAL;
    if (2 * (int64_t)rot_half > head_dim) return ATTN_B200_ESHAPE;
    if (!(eps >= 0.f)) return ATTN_B200_EINVAL;
    if (dtype != ATTN_B200_F16 && dtype != ATTN_B200_BF16 && dtype != ATTN_B200_F32) return ATTN_B200_EDTYPE;
    if ((weight_dtype != dtype && weight_dtype != ATTN_B200_F32) || (table_dtype != dtype && table_dtype != ATTN_B200_F32))
        return ATTN_B200_EDTYPE;
    if (n_tokens == 0) return 0;
    if (!q || !k || !q_out || !k_out || !q_weight || !k_weight || !positions || (rot_half && (!cos || !sin))) return ATTN_B200_EINVAL;
    const bool quant = slots && kv_dtype == ATTN_B200_E4M3;
    if (slots) {
        if (!v || !k_cache || !v_cache) return ATTN_B200_EINVAL;
        if (kv_dtype != dtype && !quant) return ATTN_B200_EDTYPE;
        if (quant && dtype == ATTN_B200_F32) return ATTN_B200_EDTYPE;
        if (quant && (!k_scale || !v_scale)) return ATTN_B200_EINVAL;
    }
    NormRopeParams p{q, k, v, q_out, k_out, q_weight, k_weight, positions, cos, sin, slots, k_cache, v_cache,
                     quant ? k_scale : nullptr, quant ? v_scale : nullptr, n_tokens, q_stride, k_stride, v_stride,
                     q_out_stride, k_out_stride, max_pos, n_slots, n_heads_q, n_heads_k, head_dim, rot_half,
                     weight_dtype == ATTN_B200_F32 && dtype != ATTN_B200_F32, table_dtype == ATTN_B200_F32 && dtype != ATTN_B200_F32,
                     eps, 0, err_flag};
    cudaStream_t st = (cudaStream_t)stream;
    switch (dtype) {
        case ATTN_B200_F16: return launch<__half>(p, st);
        case ATTN_B200_BF16: return launch<__nv_bfloat16>(p, st);
        default: return launch<float>(p, st);
    }
}
