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
            const float r = fminf(1.f / scale[head], 3e38f);          // x / scale to 2 units in the last place, 0 stays 0
            float g[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = f[i] * r;
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
// of squares is log2(LPH) shuffles.  A token's heads are dealt to 2^tpt_log2 threads, kUnroll heads'
// loads in flight at a time, the first ones before the position is known.
//
// A lane keeps its place within the head, so weight and rotation become four coefficients per pair,
// formed once for the q heads and once for the k heads of the token:
//   a' = r (a Ac - b Bs),  b' = r (b Bc + a As)   with  Ac = w_a c, Bs = w_b s, Bc = w_b c, As = w_a s
// in packed pairs (fma.f32x2).  With the weights applied head by head the kernel was bound by instruction
// issue.  16384 tokens, 32 + 32 heads of 128, fp16 (537 MB): 160 us then, 102 with the coefficients, 95
// with the next round's loads ahead of the arithmetic and five CTAs per SM = 5.6 TB/s, 0.86 of the
// measured copy rate; with the append (940 MB) 222 -> 158 us = 5.9 TB/s.
constexpr int kThreads = 128, kUnroll = 2, kCtasPerSm = 5, kRounds = 4;

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmul.rn.f32x2 rd, ra, rb;\n\t"
        "mov.b64 {%0, %1}, rd;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
// read once; not ld.global.nc, because the output may be the input
__device__ __forceinline__ uint4 ld_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

template <typename T, int LPH>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
qk_norm_rope_kernel(NormRopeParams p) {
    constexpr int N = Vec<T>::N;
    // Launched as a programmatic dependent itself: nothing is read before the kernel ahead has completed.  A dependent
    // of this kernel (a decode kernel) may be scheduled from here on; it reads nothing written here before its own wait.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tpt = 1 << p.tpt_log2;
    const int tid = threadIdx.x & (tpt - 1);
    const int64_t tok_raw = (int64_t)blockIdx.x * (kThreads >> p.tpt_log2) + (threadIdx.x >> p.tpt_log2);
    const bool live = tok_raw < p.n_tokens;               // whole LPH groups agree; shuffles run for all
    const int64_t token = live ? tok_raw : p.n_tokens - 1;

    const int hv = p.d / N, cph = p.rot / N;
    const int sub = tid & (LPH - 1), grp = tid / LPH, ngrp = tpt / LPH;
    // chunks of this lane (without a second one, or without any, it works on zeros and stores nothing)
    const bool rotates = sub < cph;
    const int ca = rotates ? sub : 2 * cph + 2 * (sub - cph), cb = rotates ? sub + cph : ca + 1;
    const bool has_a = ca < hv, has_b = cb < hv;
    uint4 ua[kUnroll], ub[kUnroll];
    auto load = [&](const T* base, int heads, int h0) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int h = h0 + u * ngrp;
            const T* row = base + h * p.d;
            ua[u] = ub[u] = make_uint4(0, 0, 0, 0);
            if (h < heads && has_a) ua[u] = ld_once(row + ca * N);
            if (h < heads && has_b) ub[u] = ld_once(row + cb * N);
        }
    };
    const T* const q_row = (const T*)p.q + token * p.q_stride;
    const T* const k_row = (const T*)p.k + token * p.k_stride;
    load(q_row, p.hq, grp);
    // v is only copied; its first chunks are on their way with the first heads of q
    constexpr int kV = 2;
    const int v_items = p.slots ? p.hk * hv : 0;
    const T* const v_row = (const T*)p.v + token * p.v_stride;
    uint4 uv[kV];
    auto load_v = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kV; ++u)
            if (i0 + u * tpt < v_items) uv[u] = ldg_stream128(v_row + (int64_t)(i0 + u * tpt) * N);
    };
    load_v(tid);
    int pos;
    int64_t slot;
    const bool pos_ok = token_ok(p, token, live ? tid : 1, pos, slot);
    if (slot >= 0 && live) {
        for (int i0 = tid; i0 < v_items; i0 += tpt * kV) {
            if (i0 != tid) load_v(i0);
#pragma unroll
            for (int u = 0; u < kV; ++u) {
                const int i = i0 + u * tpt;
                if (i >= v_items) break;
                if (p.v_scale) {
                    float f[N];
                    Vec<T>::unpack(uv[u], f);
                    store_pool<T>(p.v_cache, slot * p.hk * p.d + (int64_t)i * N, f, p.v_scale, i / hv);
                } else {
                    *reinterpret_cast<uint4*>((T*)p.v_cache + slot * p.hk * p.d + (int64_t)i * N) = uv[u];
                }
            }
        }
    }
    float2 c[N / 2], s[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) { c[i] = make_float2(1.f, 1.f); s[i] = make_float2(0.f, 0.f); }
    if (rotates && pos_ok) {
        load_aux<T>(p.cos, (int64_t)pos * p.rot + ca * N, p.cs_f32, &c[0].x);
        load_aux<T>(p.sin, (int64_t)pos * p.rot + ca * N, p.cs_f32, &s[0].x);
    }
    const float inv_d = 1.f / (float)p.d;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int heads = which ? p.hk : p.hq;
        const T* const row = which ? k_row : q_row;
        T* const out = which ? (T*)p.k_out + token * p.ko_stride : (T*)p.q_out + token * p.qo_stride;
        const void* wp = which ? p.wk : p.wq;
        float2 ac[N / 2], bs[N / 2], bc[N / 2], as[N / 2];
        {
            float2 wa[N / 2], wb[N / 2];
#pragma unroll
            for (int i = 0; i < N / 2; ++i) wa[i] = wb[i] = make_float2(0.f, 0.f);
            if (has_a) load_aux<T>(wp, ca * N, p.w_f32, &wa[0].x);
            if (has_b) load_aux<T>(wp, cb * N, p.w_f32, &wb[0].x);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                ac[i] = mul2(wa[i], c[i]);
                as[i] = mul2(wa[i], s[i]);
                bc[i] = mul2(wb[i], c[i]);
                bs[i] = mul2(wb[i], make_float2(-s[i].x, -s[i].y));
            }
        }
        for (int h0 = grp; h0 - grp < heads; h0 += ngrp * kUnroll) {      // the same number of rounds for every thread
            uint4 va[kUnroll], vb[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                va[u] = ua[u];
                vb[u] = ub[u];
            }
            if (h0 + ngrp * kUnroll - grp < heads) load(row, heads, h0 + ngrp * kUnroll);
            else if (!which) load(k_row, p.hk, grp);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int h = h0 + u * ngrp;
                float2 a[N / 2], b[N / 2];
                Vec<T>::unpack(va[u], &a[0].x);
                Vec<T>::unpack(vb[u], &b[0].x);
                float2 s0 = mul2(a[0], a[0]), s1 = mul2(b[0], b[0]);
#pragma unroll
                for (int i = 1; i < N / 2; ++i) {
                    s0 = fma2(a[i], a[i], s0);
                    s1 = fma2(b[i], b[i], s1);
                }
                const float ss = group_sum<LPH>((s0.x + s0.y) + (s1.x + s1.y));
                if (h >= heads || !live) continue;
                const float r = rsqrtf(ss * inv_d + p.eps);
                const float2 r2 = make_float2(r, r);
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    const float2 x = a[i], y = b[i];
                    a[i] = mul2(x, ac[i]);
                    b[i] = mul2(y, bc[i]);
                    if (rotates) {
                        a[i] = fma2(y, bs[i], a[i]);
                        b[i] = fma2(x, as[i], b[i]);
                    }
                    a[i] = mul2(a[i], r2);
                    b[i] = mul2(b[i], r2);
                }
                if (!pos_ok) {              // no such table row: the token's outputs are zero and nothing is appended
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) a[i] = b[i] = make_float2(0.f, 0.f);
                }
                T* o = out + h * p.d;
                if (has_a) *reinterpret_cast<uint4*>(o + ca * N) = Vec<T>::pack(&a[0].x);
                if (has_b) *reinterpret_cast<uint4*>(o + cb * N) = Vec<T>::pack(&b[0].x);
                if (which && slot >= 0) {
                    const int64_t at = (slot * p.hk + h) * p.d;
                    if (has_a) store_pool<T>(p.k_cache, at + ca * N, &a[0].x, p.k_scale, h);
                    if (has_b) store_pool<T>(p.k_cache, at + cb * N, &b[0].x, p.k_scale, h);
                }
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
        // Threads per token: at least one LPH group, at most the CTA, and few enough that a thread makes
        // kRounds rounds over the q heads, which pays for its coefficients (16384 tokens, 32 + 32 heads of
        // 128, fp16: 102 us with four rounds, 109 with two, 110 with eight) - unless the tokens are too few to fill
        // the machine that way, when each gets as many threads as still make one wave (8 tokens: 3.7 us with one
        // round, 7 with four; 5000 tokens of 8 + 2 heads: 10.8 us, 14.8 with twice the threads in two waves).
        const int64_t fill = (int64_t)current_sm_count() * kCtasPerSm * kThreads;
        int tl = 0;
        while ((1 << tl) < kThreads && ((1 << tl) < lph || (1 << tl) * kRounds * kUnroll < p.hq * lph)) ++tl;
        while ((1 << tl) < kThreads && (1 << tl) * kUnroll < p.hq * lph && (p.n_tokens << (tl + 1)) <= fill) ++tl;
        p.tpt_log2 = tl;
        const int64_t per_cta = kThreads >> tl, ctas = (p.n_tokens + per_cta - 1) / per_cta;
        if (ctas > 0x7fffffff) return ATTN_B200_ETOOLARGE;
        void (*kernel)(NormRopeParams) = lph == 1 ? qk_norm_rope_kernel<T, 1> : lph == 2 ? qk_norm_rope_kernel<T, 2>
                                         : lph == 4 ? qk_norm_rope_kernel<T, 4> : lph == 8 ? qk_norm_rope_kernel<T, 8>
                                         : lph == 16 ? qk_norm_rope_kernel<T, 16> : qk_norm_rope_kernel<T, 32>;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)ctas);
        cfg.blockDim = dim3(kThreads);
        cfg.stream = st;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        return (int)cudaLaunchKernelEx(&cfg, kernel, (NormRopeParams)p);
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
