// Single-token attention over the visible span of a paged cache (sliding window with sink tokens), and
// over a sequence's own tokens beside a prefix that the batch shares.  Not in the reference; its
// unwindowed form is paged_attention_kernel.cu:100-187.
//
//   o = sum_t p_t v_t,  p = softmax over the visible cached tokens and the current one of scale <q, k_t>
//
// Bound: HBM, 2 D b bytes per visible token and KV head against 4 D G flops.  The visible tokens are
// renumbered u = 0 .. n-1 (sinks, then the window), so nothing outside the span is read, not even its
// table entries, and no tile is masked but the last.
//
// One launch, no workspace: a cluster of `splits` CTAs owns a sequence and a few KV heads, a warp walks
// every (splits * warps per head)-th tile of 16 tokens of one KV head, and the partial results meet in
// distributed shared memory.  Against a second kernel that folds partial rows from global memory this
// saves the rows' round trip and a launch.
//
// The tile arithmetic is that of decode_gqa.cuh: keys as M of mma.sync.m16n8k16, up to eight query heads
// of a KV head as N (tcgen05 would pad 1..8 rows to 128), K and V staged by cp.async in a ring private to
// the warp.  A KV head with more than eight query heads is walked once for every eight of them.
#include <atomic>

#include "span_decode.cuh"

namespace attn {
namespace {

constexpr int kWarps = 4, kTile = 16;

template <typename T> struct Mma16;
template <> struct Mma16<__half> {
    static __device__ __forceinline__ void run(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <> struct Mma16<__nv_bfloat16> {
    static __device__ __forceinline__ void run(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&w)[4]) {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int rank) {        // the same place in another CTA of the cluster
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The visible span of sequence b
struct Span {
    int64_t beg;        // first entry of a per-token table
    int b, first, sinks, n;      // n: with the shared rows, which come first
};
__device__ __forceinline__ Span span_of(const SpanParams& p, int b, bool report) {
    Span s;
    s.b = b;
    s.beg = b ? p.offsets[b - 1] : 0;
    const int64_t end = p.offsets[b];
    int64_t ctx = end - s.beg;
    bool bad = s.beg < 0 || ctx < 0;
    if (p.block_size > 1) bad |= ctx > (int64_t)p.max_blocks * p.block_size;
    else bad |= end > p.n_tokens;
    if (bad) {
        if (report && p.err_flag) atomicOr(p.err_flag, ATTN_B200_FLAG_BAD_OFFSETS);
        ctx = 0;
    }
    const int64_t first = ctx - p.window + 1;
    s.first = first > 0 ? (int)first : 0;
    s.sinks = p.sinks < s.first ? p.sinks : s.first;
    s.n = p.n_prefix + s.sinks + (int)ctx - s.first;
    return s;
}
// pool row of the u-th visible token, or -1
__device__ __forceinline__ int64_t slot_of(const SpanParams& p, const Span& s, int u) {
    const int v = u - p.n_prefix, t = v < s.sinks ? v : v - s.sinks + s.first;
    int64_t slot;
    if (v < 0) {
        slot = p.prefix[u];
    } else if (p.block_size > 1) {
        const int blk = p.table[(int64_t)s.b * p.max_blocks + t / p.block_size];
        slot = blk < 0 ? -1 : (int64_t)blk * p.block_size + t % p.block_size;
    } else {
        slot = p.table[s.beg + t];
    }
    if (slot < 0 || slot >= p.n_slots) {
        if (p.err_flag) atomicOr(p.err_flag, ATTN_B200_FLAG_BAD_SLOT);
        return -1;
    }
    return slot;
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void add4(float4& a, float w, const float4& x) {
    a.x += w * x.x;
    a.y += w * x.y;
    a.z += w * x.z;
    a.w += w * x.w;
}

constexpr int kMaxSplits = 16;
// Weights of the partial results a CTA folds: per head of the CTA, one per worker (CTA of the cluster x warp of the
// KV head), the current token's, and what turns a shared-row partial's 2^m into its weight
struct FoldWeights {
    float worker[kWarps * 8][kMaxSplits];   // heads of the CTA x workers: at most (4 x 8) x 16 or (1 x 8) x 64
    float fresh[kWarps * 8], top[kWarps * 8], inv[kWarps * 8];
};

// Folds the workers' partial results, the shared rows' partial results and the current token, and writes O.
// Every CTA of the cluster has, per warp, a partial row [heads][D] at `part` (warp stride `part_stride` bytes) and
// (m, l) pairs [heads of a warp] at `ml`; s_new [slot][heads] are the current token's scores.  A warp forms the weights
// of a head with a worker per lane, then the threads sum four output entries each, their loads from the other CTAs independent.
template <typename T, int D>
__device__ __forceinline__ void fold(const SpanParams& p, FoldWeights& fw, int b, int vh0, int rank, uint32_t part, uint32_t part_stride,
                                     uint32_t ml, const float* s_new, int heads) {
    const int hpc = 1 << p.hpc_log2, wph_log2 = 2 - p.hpc_log2, S = p.splits, workers = S << wph_log2;
    const int G = p.H / p.Hkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* const weight = &fw.worker[0][0];                  // [hpc * heads][workers]
    const int64_t set = (int64_t)p.B * p.H;
    const float2* const pml = reinterpret_cast<const float2*>(p.parts + p.n_parts * set * D);
    auto part_row = [&](int h) { return ((int64_t)(h / G) * p.B + b) * G + h % G; };      // of the first partial set
    auto head_of = [&](int gh) -> int {                      // query head of this CTA's gh-th, or -1
        const int slot = gh / heads, vh = vh0 + slot, hk = vh / p.n_sets, g = (vh - hk * p.n_sets) * 8 + gh - slot * heads;
        return hk < p.Hkv && g < G ? hk * G + g : -1;
    };
    for (int gh = warp; gh < hpc * heads; gh += kWarps) {
        const int h = head_of(gh), slot = gh / heads;
        if (h < 0) continue;
        const float sn = s_new[gh];
        float2 v[2];
        float M = sn;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int w = lane + 32 * i, warp_of = (slot << wph_log2) + (w & ((1 << wph_log2) - 1));
            v[i] = make_float2(-INFINITY, 0.f);
            if (w < workers) v[i] = ld_cluster2(in_cta(ml + (warp_of * heads + gh - slot * heads) * 8, w >> wph_log2));
            M = fmaxf(M, v[i].x);
        }
        const float2* const pm = pml + part_row(h);
        for (int k = lane; k < p.n_parts; k += 32) M = fmaxf(M, pm[k * set].x);
        M = group_max<32>(M);
        if (!(M > -INFINITY)) M = 0.f;                       // nothing but -inf: 0 / 0 below, as the formula has it
        float e[2], den = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            e[i] = fast_exp2(v[i].x - M);
            den += e[i] * v[i].y;
        }
        for (int k = lane; k < p.n_parts; k += 32) {
            const float2 x = pm[k * set];
            den += fast_exp2(x.x - M) * x.y;
        }
        const float fresh = fast_exp2(sn - M);
        const float inv = 1.f / (group_sum<32>(den) + fresh);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane + 32 * i < workers) weight[gh * workers + lane + 32 * i] = e[i] * inv;
        if (lane == 0) {
            fw.fresh[gh] = fresh * inv;
            fw.top[gh] = M;
            fw.inv[gh] = inv;
        }
    }
    __syncthreads();
    // Where there are more threads than output vectors, 2^k threads of a warp share one and split its partial results.
    const int items = hpc * heads * (D / 4), threads = S * kWarps * 32;
    int share = 1;
    while (share < 32 && items * share * 2 <= threads) share *= 2;
    const int first = rank * (kWarps * 32) + threadIdx.x, sub = first & (share - 1);
    for (int i = first / share; i - (lane / share) < items; i += threads / share) {       // whole warps together
        const int d = (i % (D / 4)) * 4, gh = i / (D / 4), slot = gh / heads, h = i < items ? head_of(gh) : -1;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (h >= 0) {
            const uint32_t part0 = part + (slot << wph_log2) * part_stride + ((gh - slot * heads) * D + d) * 4;
#pragma unroll 4
            for (int w = sub; w < workers; w += share)
                add4(o, weight[gh * workers + w], ld_cluster4(in_cta(part0 + (w & ((1 << wph_log2) - 1)) * part_stride, w >> wph_log2)));
            const int64_t row = part_row(h);
            const float4* po = reinterpret_cast<const float4*>(p.parts + row * D + d);
#pragma unroll 12
            for (int k = sub; k < p.n_parts; k += share) add4(o, fast_exp2(pml[k * set + row].x - fw.top[gh]) * fw.inv[gh], po[k * set * (D / 4)]);
        }
        for (int m = 1; m < share; m <<= 1) {
            o.x += __shfl_xor_sync(0xffffffffu, o.x, m);
            o.y += __shfl_xor_sync(0xffffffffu, o.y, m);
            o.z += __shfl_xor_sync(0xffffffffu, o.z, m);
            o.w += __shfl_xor_sync(0xffffffffu, o.w, m);
        }
        if (h < 0 || sub) continue;
        const T* vn = (const T*)p.v_new + ((int64_t)b * p.Hkv + h / G) * D + d;
        add4(o, fw.fresh[gh], make_float4(to_f32<T>(vn[0]), to_f32<T>(vn[1]), to_f32<T>(vn[2]), to_f32<T>(vn[3])));
        T* out = (T*)p.out + ((int64_t)b * p.H + h) * D + d;
        out[0] = from_f32<T>(o.x);
        out[1] = from_f32<T>(o.y);
        out[2] = from_f32<T>(o.z);
        out[3] = from_f32<T>(o.w);
    }
}

// A warp's ring of kStages tiles (kStages - 1 of them in flight).  Two stages and three CTAs per SM carry a full machine
// (D = 128, 16 bits, batch 64: 187 us against 207 with three stages and two CTAs); a launch of few CTAs is bound by
// the latency of its loads and takes as many stages as shared memory has for it.
template <int D, bool E4, int STAGES> struct Ring {
    static constexpr int kRow = E4 ? D : 2 * D;                  // bytes of a head's K (or V) row
    static constexpr int J = kRow / 64;                          // 16-byte chunks of a row per lane
    static constexpr int kStageBytes = kTile * 2 * kRow;
    static constexpr int kStages = STAGES;
    static constexpr int kWarpBytes = kStages * kStageBytes;
    static constexpr int kBytes = kWarps * kWarpBytes;
    static constexpr int kFit = 227 * 1024 / (kBytes + 4096);    // CTAs per SM by shared memory
    static constexpr int kCtasPerSm = kFit < 4 ? kFit : 4;       // and by registers
    static_assert(kFit >= 1, "shared memory");
    static_assert(kWarpBytes >= 8 * D * 4, "a warp's partial result reuses its ring");
};
template <int D, bool E4> constexpr int base_stages() { return kTile * 4 * D / (E4 ? 2 : 1) > 4096 ? 2 : 3; }

template <typename T, int D, bool E4, int STAGES>
__global__ void __launch_bounds__(kWarps * 32, (Ring<D, E4, STAGES>::kCtasPerSm))
span_decode_kernel(const SpanParams p) {
    using R = Ring<D, E4, STAGES>;
    using MT = typename std::conditional<E4, __half, T>::type;   // e4m3 rows are multiplied as fp16
    using M = Mma16<MT>;
    constexpr int J = R::J, E = E4 ? 4 : 2, CD = E4 ? 16 : 8;    // k-slices and dims per 16-byte chunk
    extern __shared__ __align__(16) unsigned char ring_raw[];
    __shared__ float2 s_ml[kWarps * 8];
    __shared__ float s_new[kWarps * 8];
    __shared__ FoldWeights s_fold;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = lane >> 2, c = lane & 3;
    const int hpc = 1 << p.hpc_log2, wph = kWarps >> p.hpc_log2;
    const int rank = blockIdx.x % p.splits;
    const int unit = blockIdx.x / p.splits;
    const int G = p.H / p.Hkv;
    const int groups = (p.Hkv * p.n_sets + hpc - 1) / hpc;
    const int b = unit / groups, vh0 = (unit - b * groups) * hpc;
    const int slot_in_cta = warp / wph, vh = vh0 + slot_in_cta;
    const int hk = vh / p.n_sets, g0 = (vh - hk * p.n_sets) * 8;
    const bool live = hk < p.Hkv;
    const int heads = G < 8 ? G : 8;                             // heads of a set that are kept
    const bool row_ok = live && g0 + n < G;

    if (!p.early) asm volatile("griddepcontrol.wait;" ::: "memory");

    const Span sp = span_of(p, b, threadIdx.x == 0);
    const int workers = p.splits * wph, me = rank * wph + (warp - slot_in_cta * wph);
    const int tiles = (sp.n + kTile - 1) / kTile;
    const int nt = live && tiles > me ? (tiles - me + workers - 1) / workers : 0;
    // pool row of token `lane` of this warp's t-th tile (lanes 0..15), or -1
    auto tile_slot = [&](int t) -> int {
        const int u = (me + t * workers) * kTile + lane;
        return (t < nt && lane < kTile && u < sp.n) ? (int)slot_of(p, sp, u) : -1;
    };
    const int64_t row_bytes = (int64_t)p.Hkv * R::kRow;
    const char* kbase = (const char*)p.k_cache + (int64_t)hk * R::kRow + c * 16;
    const char* vbase = (const char*)p.v_cache + (int64_t)hk * R::kRow + c * 16;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(ring_raw) + warp * R::kWarpBytes + lane * 16;
    // copies of tile t into its stage; returns the validity bits of its 16 tokens
    auto issue = [&](int t, int my_slot) -> unsigned {
        const uint32_t base = ring + (t % R::kStages) * R::kStageBytes;
#pragma unroll
        for (int grp = 0; grp < 2; ++grp) {
            const int sl = __shfl_sync(0xffffffffu, my_slot, grp * 8 + n);
            const int64_t off = (int64_t)(sl >= 0 ? sl : 0) * row_bytes;
            const int nb = sl >= 0 ? 16 : 0;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                copy16(base + ((grp * 2 + 0) * J + j) * 512, kbase + off + j * 64, nb);
                copy16(base + ((grp * 2 + 1) * J + j) * 512, vbase + off + j * 64, nb);
            }
        }
        return __ballot_sync(0xffffffffu, my_slot >= 0) & 0xffffu;
    };
    constexpr int kAhead = R::kStages - 1;
    unsigned valid[R::kStages];
    int next_slot = tile_slot(0);
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
        const int s0 = next_slot;
        next_slot = tile_slot(t + 1);
        valid[t] = 0;
        if (t < nt) valid[t] = issue(t, s0);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // Q^T as B fragments of head n (heads beyond G stay zero): slice E j + e holds the dims
    // (4 j + c) CD + 4 e + {0, 1} and + {2, 3}, the order in which the lanes hold K's dims.
    uint32_t bq[D / 16][2];
    float q_unit = 1.f;
    {
        const T* qrow = (const T*)p.q + ((int64_t)b * p.H + (row_ok ? hk * G + g0 + n : 0)) * D;
        float q_mul = 1.f;
        if constexpr (E4 && std::is_same<T, __nv_bfloat16>::value) {
            // bf16 queries are multiplied as fp16: brought to [1, 2) by a power of two first, so that
            // nothing overflows and what is lost is below 2^-24 of the head's largest entry
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < D / 4; ++i) top = fmaxf(top, row_ok ? fabsf(to_f32<T>(qrow[c * (D / 4) + i])) : 0.f);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (top > 1e-30f && top < 1e30f) {
                const int ex = ((__float_as_int(top) >> 23) & 255) - 127;
                q_unit = __int_as_float((127 + ex) << 23);
                q_mul = __int_as_float((127 - ex) << 23);
            }
        }
        // the current token's scores of the set's heads, kept until the end
        const T* krow = (const T*)p.k_new + ((int64_t)b * p.Hkv + (live ? hk : 0)) * D;
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int d0 = (4 * j + c) * CD + 4 * e;
                const uint2 w = row_ok ? *reinterpret_cast<const uint2*>(qrow + d0) : make_uint2(0, 0);
                const uint2 kw = *reinterpret_cast<const uint2*>(krow + d0);
                float x0, x1, x2, x3, y0, y1, y2, y3;
                unpack2(w.x, T(), x0, x1);
                unpack2(w.y, T(), x2, x3);
                unpack2(kw.x, T(), y0, y1);
                unpack2(kw.y, T(), y2, y3);
                dot += (x0 * y0 + x1 * y1) + (x2 * y2 + x3 * y3);
                if constexpr (std::is_same<T, MT>::value) {
                    bq[E * j + e][0] = w.x;
                    bq[E * j + e][1] = w.y;
                } else {
                    bq[E * j + e][0] = M::pack(x0 * q_mul, x1 * q_mul);
                    bq[E * j + e][1] = M::pack(x2 * q_mul, x3 * q_mul);
                }
            }
        dot += __shfl_xor_sync(0xffffffffu, dot, 1);
        dot += __shfl_xor_sync(0xffffffffu, dot, 2);
        if (warp == slot_in_cta * wph && c == 0 && n < heads) s_new[slot_in_cta * heads + n] = dot * p.scale_log2;
    }
    // heads 2c, 2c + 1 of this lane's score fragment
    const float ks = p.scale_log2 * (E4 && live ? p.k_scale[hk] : 1.f);
    const float qs[2] = {ks * __shfl_sync(0xffffffffu, q_unit, 8 * c), ks * __shfl_sync(0xffffffffu, q_unit, 8 * c + 4)};

    // O^T accumulators: block i = E j + e: {dim row n, head 2c | 2c+1 | dim row 8+n, head 2c | 2c+1}
    float oacc[D / 16][4];
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) oacc[i][k] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};      // l: this lane's keys only

    for (int t = 0; t < nt; ++t) {
        {
            const int s0 = next_slot;
            next_slot = tile_slot(t + kAhead + 1);
            valid[kAhead] = 0;
            if (t + kAhead < nt) valid[kAhead] = issue(t + kAhead, s0);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
        const uint32_t base = ring + (t % R::kStages) * R::kStageBytes;
        const unsigned vb = valid[0];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) valid[i] = valid[i + 1];

        auto fragment = [&](const uint32_t (&w0)[4], const uint32_t (&w1)[4], int e, uint32_t (&a)[4]) {
            if constexpr (E4) {
                __half2 lo0, hi0, lo1, hi1;
                e4m3x4_to_half2x2(w0[e], lo0, hi0);
                e4m3x4_to_half2x2(w1[e], lo1, hi1);
                a[0] = *reinterpret_cast<uint32_t*>(&lo0);
                a[1] = *reinterpret_cast<uint32_t*>(&lo1);
                a[2] = *reinterpret_cast<uint32_t*>(&hi0);
                a[3] = *reinterpret_cast<uint32_t*>(&hi1);
            } else {
                a[0] = w0[2 * e];
                a[1] = w1[2 * e];
                a[2] = w0[2 * e + 1];
                a[3] = w1[2 * e + 1];
            }
        };
        // S^T = K Q^T: rows = keys n, 8 + n; columns = heads 2c, 2c + 1
        float sacc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < J; ++j) {
            uint32_t w0[4], w1[4];
            lds128(base + j * 512, w0);
            lds128(base + (2 * J + j) * 512, w1);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                uint32_t a[4];
                fragment(w0, w1, e, a);
                M::run(sacc, a, bq[E * j + e][0], bq[E * j + e][1]);
            }
        }
        const bool ok0 = (vb >> n) & 1u, ok1 = (vb >> (8 + n)) & 1u;
        float pr[4], alpha[2];               // (key n, head 2c), (key n, 2c+1), (key 8+n, 2c), (key 8+n, 2c+1)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float s0 = ok0 ? sacc[i] * qs[i] : -INFINITY, s1 = ok1 ? sacc[2 + i] * qs[i] : -INFINITY;
            float tmax = fmaxf(s0, s1);
            tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, 4));
            tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, 8));
            tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, 16));
            const float m_new = fmaxf(m[i], tmax);
            const float msub = m_new > -INFINITY ? m_new : 0.f;
            alpha[i] = fast_exp2(m[i] - msub);
            pr[i] = fast_exp2(s0 - msub);
            pr[2 + i] = fast_exp2(s1 - msub);
            l[i] = l[i] * alpha[i] + (pr[i] + pr[2 + i]);
            m[i] = m_new;
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            oacc[i][0] *= alpha[0];
            oacc[i][1] *= alpha[1];
            oacc[i][2] *= alpha[0];
            oacc[i][3] *= alpha[1];
        }
        // P^T as the B operand, rounded to the MMA's type (the sums above keep 32 bits)
        const uint32_t pb0 = transpose8x8(M::pack(pr[0], pr[1]));      // head n; keys 2c, 2c + 1
        const uint32_t pb1 = transpose8x8(M::pack(pr[2], pr[3]));      // head n; keys 8 + 2c, 9 + 2c
#pragma unroll
        for (int j = 0; j < J; ++j) {
            uint32_t w0[4], w1[4];
            lds128(base + (J + j) * 512, w0);
            lds128(base + (3 * J + j) * 512, w1);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                uint32_t f[4];
                fragment(w0, w1, e, f);
                // V^T: rows 0..7 from the first pair of dims, rows 8..15 from the second; keys 0..7, then 8..15
                const uint32_t a[4] = {transpose8x8(f[0]), transpose8x8(f[2]), transpose8x8(f[1]), transpose8x8(f[3])};
                M::run(oacc[E * j + e], a, pb0, pb1);
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
    }
    // the warp's partial result, over its own ring: [heads][D], and (m, l)
    const float vs = E4 && live ? p.v_scale[hk] : 1.f;
    float* part = reinterpret_cast<float*>(ring_raw + warp * R::kWarpBytes);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int g = 2 * c + i;
        if (g >= heads) continue;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int d = (4 * j + (n >> 1)) * CD + 4 * e + (n & 1);
                part[g * D + d] = oacc[E * j + e][i] * vs;
                part[g * D + d + 2] = oacc[E * j + e][2 + i] * vs;
            }
        if (n == 0) s_ml[warp * heads + g] = make_float2(m[i], l[i]);
    }
    if (p.early) asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (p.splits > 1) cluster_sync();
    else __syncthreads();
    fold<T, D>(p, s_fold, b, vh0, rank, (uint32_t)__cvta_generic_to_shared(ring_raw), R::kWarpBytes, (uint32_t)__cvta_generic_to_shared(s_ml),
               s_new, heads);
    if (p.splits > 1) cluster_sync();              // nobody leaves while its shared memory is still read
}

// Any head_dim up to 32 * DPL, any type: one cluster per (sequence, query head), a warp per token, a lane
// per dim.  Compatibility path (fp32, odd head_dim).
template <typename T, typename KV, int DPL>
__global__ void __launch_bounds__(kWarps * 32)
span_decode_generic_kernel(const SpanParams p) {
    extern __shared__ __align__(16) unsigned char ring_raw[];
    __shared__ float2 s_ml[kWarps];
    __shared__ float s_new[1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.D;
    const int rank = blockIdx.x % p.splits, unit = blockIdx.x / p.splits;
    const int b = unit / p.H, h = unit - b * p.H, hk = h / (p.H / p.Hkv);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Span sp = span_of(p, b, threadIdx.x == 0);
    float q[DPL], o[DPL], dot = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
        const int d = lane + 32 * i;
        o[i] = 0.f;
        q[i] = d < D ? to_f32<T>(((const T*)p.q)[((int64_t)b * p.H + h) * D + d]) : 0.f;
        if (d < D) dot += q[i] * to_f32<T>(((const T*)p.k_new)[((int64_t)b * p.Hkv + hk) * D + d]);
    }
    dot = group_sum<32>(dot);
    if (threadIdx.x == 0) s_new[0] = dot * p.scale_log2;
    const float ks = p.scale_log2 * (p.k_scale ? p.k_scale[hk] : 1.f), vs = p.v_scale ? p.v_scale[hk] : 1.f;
    float m = -INFINITY, l = 0.f;
    for (int u = rank * kWarps + warp; u < sp.n; u += p.splits * kWarps) {
        const int64_t slot = slot_of(p, sp, u);
        if (slot < 0) continue;
        const KV* kr = (const KV*)p.k_cache + (slot * p.Hkv + hk) * D;
        const KV* vr = (const KV*)p.v_cache + (slot * p.Hkv + hk) * D;
        float s = 0.f, v[DPL];
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
            const int d = lane + 32 * i;
            v[i] = d < D ? to_f32<KV>(vr[d]) : 0.f;
            if (d < D) s += q[i] * to_f32<KV>(kr[d]);
        }
        s = group_sum<32>(s) * ks;
        const float m_new = fmaxf(m, s), msub = m_new > -INFINITY ? m_new : 0.f;
        const float alpha = fast_exp2(m - msub), pr = fast_exp2(s - msub);
        l = l * alpha + pr;
        m = m_new;
#pragma unroll
        for (int i = 0; i < DPL; ++i) o[i] = o[i] * alpha + pr * v[i];
    }
    float* part = reinterpret_cast<float*>(ring_raw) + warp * D;
#pragma unroll
    for (int i = 0; i < DPL; ++i)
        if (lane + 32 * i < D) part[lane + 32 * i] = o[i] * vs;
    if (lane == 0) s_ml[warp] = make_float2(m, l);
    cluster_sync();
    for (int d = rank * (kWarps * 32) + threadIdx.x; d < D; d += p.splits * kWarps * 32) {
        const uint32_t ml0 = (uint32_t)__cvta_generic_to_shared(s_ml), part0 = (uint32_t)__cvta_generic_to_shared(ring_raw) + d * 4;
        const float sn = s_new[0];
        float M = sn;
        for (int w = 0; w < p.splits * kWarps; ++w) M = fmaxf(M, ld_cluster2(in_cta(ml0 + (w % kWarps) * 8, w / kWarps)).x);
        if (!(M > -INFINITY)) M = 0.f;
        const float w_new = fast_exp2(sn - M);
        float den = w_new, num = w_new * to_f32<T>(((const T*)p.v_new)[((int64_t)b * p.Hkv + hk) * D + d]);
        for (int w = 0; w < p.splits * kWarps; ++w) {
            const float2 v = ld_cluster2(in_cta(ml0 + (w % kWarps) * 8, w / kWarps));
            const float e = fast_exp2(v.x - M);
            den += e * v.y;
            num += e * ld_cluster(in_cta(part0 + (w % kWarps) * D * 4, w / kWarps));
        }
        ((T*)p.out)[((int64_t)b * p.H + h) * D + d] = from_f32<T>(num / den);
    }
    cluster_sync();
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
template <typename K>
int launch(K kernel, const SpanParams& p, int64_t units, int smem, cudaStream_t st, std::atomic<uint64_t>& ready) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 64) return ATTN_B200_ETOOLARGE;
    if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {        // once per device and kernel
        if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess ||
            (e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess)
            return (int)e;
        ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (units * p.splits > 0x7fffffffLL) return ATTN_B200_ETOOLARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * p.splits));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    // the kernel waits (griddepcontrol.wait) before it reads what the kernel ahead of it may still write
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, int D, bool E4, int STAGES>
int launch_ring(const SpanParams& p, int64_t units, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    return launch(span_decode_kernel<T, D, E4, STAGES>, p, units, Ring<D, E4, STAGES>::kBytes, st, ready);
}

template <typename T, int D, bool E4>
int launch_mma(SpanParams p, int64_t span, bool ragged, cudaStream_t st) {
    constexpr int kBase = base_stages<D, E4>();
    using R = Ring<D, E4, kBase>;
    const int G = p.H / p.Hkv;
    p.n_sets = (G + 7) / 8;
    const int vheads = p.Hkv * p.n_sets;
    // Heads per CTA and CTAs per sequence: one wave of CTAs, as full as whole splits make it (a second wave costs a
    // CTA's whole start and end, ~6 us; a cluster of 16 about 4 more).  Few heads per CTA (several warps to a head)
    // start and end quickest: batch 8, 32 KV heads, 512 tokens 16.9 us with one head per CTA, 18 to 20 with four.  Four
    // adjacent heads read 4 times the contiguous bytes per token, which counts once DRAM is the bound: batch 64, 8 KV
    // heads, 4100 tokens 187 us with four heads and clusters of three, 258 with two, 349 with one.  Sequences of very
    // different lengths want many small CTAs: 64 with 16 to 1024 tokens, 36 us with one head per CTA, 52 with four.
    const int64_t slots = (int64_t)current_sm_count() * R::kCtasPerSm, tiles = (span + kTile - 1) / kTile;
    const int64_t bytes = (int64_t)p.B * span * 2 * p.Hkv * R::kRow;
    auto units_of = [&](int hl) { return (int64_t)p.B * ((vheads + (1 << hl) - 1) >> hl); };
    auto splits_of = [&](int hl) {
        const int64_t fit = slots / units_of(hl), most = (tiles + (kWarps >> hl) - 1) / (kWarps >> hl);
        const int64_t s = fit < most ? fit : most;
        return s >= 16 && tiles >= 64 * (kWarps >> hl) ? 16 : s > 8 ? 8 : s < 1 ? 1 : (int)s;     // 16: clusters beyond the portable size
    };
    int hl = 0;
    while (hl < 2 && (2 << hl) <= vheads &&
           (units_of(hl) > (ragged ? 2 * slots : slots) || (!ragged && bytes > (100 << 20) && slots / units_of(hl + 1) <= 8)))
        ++hl;
    const int64_t units = units_of(hl);
    const int s = splits_of(hl);
    p.hpc_log2 = hl;
    p.splits = s;
    // the deepest ring that leaves all CTAs resident, where a warp has tiles for it
    const bool deep = tiles >= 4 * s * (kWarps >> hl);
    const int64_t per_sm = (units * s + current_sm_count() - 1) / current_sm_count();
    if constexpr (4 * R::kStageBytes * 6 <= 200 * 1024) {
        if (deep && per_sm <= Ring<D, E4, 6>::kCtasPerSm) return launch_ring<T, D, E4, 6>(p, units, st);
    }
    if constexpr (kBase == 2) {
        if (deep && per_sm <= Ring<D, E4, 3>::kCtasPerSm) return launch_ring<T, D, E4, 3>(p, units, st);
    }
    return launch_ring<T, D, E4, kBase>(p, units, st);
}

template <typename T, typename KV, int DPL>
int launch_generic_d(SpanParams p, int64_t span, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    const int64_t units = (int64_t)p.B * p.H;
    int s = 1;
    while (s < 8 && units * s < current_sm_count() * 4 && span > (int64_t)s * kWarps * 8) s *= 2;
    p.splits = s;
    p.n_sets = 1;
    return launch(span_decode_generic_kernel<T, KV, DPL>, p, units, kWarps * 32 * DPL * 4, st, ready);
}
template <typename T, typename KV>
int launch_generic(const SpanParams& p, int64_t span, cudaStream_t st) {
    if (p.D <= 64) return launch_generic_d<T, KV, 2>(p, span, st);
    if (p.D <= 128) return launch_generic_d<T, KV, 4>(p, span, st);
    if (p.D <= 256) return launch_generic_d<T, KV, 8>(p, span, st);
    if (p.D <= 512) return launch_generic_d<T, KV, 16>(p, span, st);
    return ATTN_B200_ESHAPE;
}

template <typename T>
int dispatch16(const SpanParams& p, int64_t span, bool ragged, bool e4, cudaStream_t st) {
    const bool aligned = (((uintptr_t)p.q | (uintptr_t)p.k_new | (uintptr_t)p.k_cache | (uintptr_t)p.v_cache) & 15) == 0;
    if (aligned) {
        switch (p.D) {
            case 64: return e4 ? launch_mma<T, 64, true>(p, span, ragged, st) : launch_mma<T, 64, false>(p, span, ragged, st);
            case 128: return e4 ? launch_mma<T, 128, true>(p, span, ragged, st) : launch_mma<T, 128, false>(p, span, ragged, st);
            case 256: return e4 ? launch_mma<T, 256, true>(p, span, ragged, st) : launch_mma<T, 256, false>(p, span, ragged, st);
            default: break;
        }
    }
    if (p.n_parts) return ATTN_B200_ESHAPE;
    return e4 ? launch_generic<T, __nv_fp8_e4m3>(p, span, st) : launch_generic<T, T>(p, span, st);
}

}  // namespace

int span_decode_launch(SpanParams p, int64_t span, bool ragged, int q_dtype, int kv_dtype, cudaStream_t st) {
    const bool e4 = kv_dtype == ATTN_B200_E4M3;
    switch (q_dtype) {
        case ATTN_B200_F16: return dispatch16<__half>(p, span, ragged, e4, st);
        case ATTN_B200_BF16: return dispatch16<__nv_bfloat16>(p, span, ragged, e4, st);
        case ATTN_B200_F32: return p.n_parts ? ATTN_B200_ESHAPE : launch_generic<float, float>(p, span, st);
        default: return ATTN_B200_EDTYPE;
    }
}

}  // namespace attn

extern "C" int attn_b200_paged_window_decode(const void* q, const void* k_new, const void* v_new, const void* k_cache,
                                             const void* v_cache, const int32_t* slots, const int32_t* offsets, void* out,
                                             int B, int H, int n_kv_heads, int D, int64_t n_tokens, int64_t n_slots,
                                             int block_size, int max_blocks, int window, int n_sinks, float scale,
                                             const float* k_scale, const float* v_scale, int q_dtype, int kv_dtype,
                                             int32_t* err_flag, void* stream) {
    using namespace attn;
    if (B < 0 || H <= 0 || n_kv_heads <= 0 || H % n_kv_heads || D <= 0 || n_tokens < 0 || n_slots < 0 || block_size <= 0 ||
        max_blocks < 0 || window <= 0 || n_sinks < 0)
        return ATTN_B200_EINVAL;
    if (q_dtype != ATTN_B200_F16 && q_dtype != ATTN_B200_BF16 && q_dtype != ATTN_B200_F32) return ATTN_B200_EDTYPE;
    if (kv_dtype != q_dtype && !(kv_dtype == ATTN_B200_E4M3 && q_dtype != ATTN_B200_F32)) return ATTN_B200_EDTYPE;
    if (kv_dtype == ATTN_B200_E4M3 && (!k_scale || !v_scale)) return ATTN_B200_EINVAL;
    if (n_slots > 0x7fffffffLL) return ATTN_B200_ETOOLARGE;
    if (B == 0) return 0;
    if (!q || !k_new || !v_new || !offsets || !out || (n_tokens && (!slots || !k_cache || !v_cache))) return ATTN_B200_EINVAL;
    SpanParams p{};
    p.q = q; p.k_new = k_new; p.v_new = v_new; p.k_cache = k_cache; p.v_cache = v_cache;
    p.table = slots; p.offsets = offsets; p.out = out;
    p.B = B; p.H = H; p.Hkv = n_kv_heads; p.D = D;
    p.n_tokens = n_tokens; p.n_slots = n_slots;
    p.block_size = block_size; p.max_blocks = max_blocks;
    p.window = window; p.sinks = n_sinks;
    p.scale_log2 = scale * kLog2e;
    p.k_scale = kv_dtype == ATTN_B200_E4M3 ? k_scale : nullptr;
    p.v_scale = kv_dtype == ATTN_B200_E4M3 ? v_scale : nullptr;
    p.err_flag = err_flag;
    // sequences are taken to be alike: most fill the span, or the table shows that they cannot
    const int64_t seen = (int64_t)window - 1 + n_sinks, average = block_size > 1 ? (int64_t)max_blocks * block_size : n_tokens / B;
    return span_decode_launch(p, average < seen ? average + 1 : seen, false, q_dtype, kv_dtype, (cudaStream_t)stream);
}
