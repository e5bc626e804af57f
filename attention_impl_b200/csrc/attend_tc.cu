// Attention of 128-row query tiles over gathered pool rows on the 5th-generation tensor cores: tcgen05.mma
// with the scores, the probabilities and the output accumulator in tensor memory.  Two uses, neither in
// the reference (its packed prefill: paged_attention_kernel.cu:15-98):
//
//   window   chunks of sequences; the query at position i sees key j iff j <= i and (j > i - window or
//            j < sinks).  A CTA owns two tiles of 128 query rows: one tile for two heads of a KV head, or,
//            with an odd number of query heads per KV head, two neighbouring tiles of one head.
//   prefix   one query per sequence over rows that the whole batch shares: the B * G query rows of a KV
//            head are the tile, so a K or V row is read once for the batch instead of once a sequence.
//            The keys are split over CTAs; each writes partial rows [o, m, l] for a later fold.
//
// Keys come as a list u = 0 .. n-1 of pool rows (window: the sinks, then the stretch of the tile's windows),
// cut into tiles of 128 with the FIRST tile taking the remainder: a window of 1024 and 4 sinks is 9 whole
// tiles and one of 3 keys, which is multiplied and exponentiated 32 wide.  Because rows are gathered the
// list needs no alignment, and whatever lies outside it is never read.
//
// Bound: window - tensor pipe and the exponentials, as the packed prefill; prefix - up to 128 query rows
// HBM, from 256 rows on both about equally.  The pipeline (softmax warpgroups, MMA thread, gather
// warps, lazy rescaling of the accumulator) is that of paged_prefill_tc_kernel.  With up to 128 query rows the two
// softmax warpgroups take alternate key tiles of the same query tile (key_split), each with its own
// accumulator and partial rows, so that one's exponentials run under the other's products.
#include <atomic>
#include <climits>

#include "attend_tc.cuh"
#include "tcgen05_utils.cuh"

namespace attn {
namespace {

using namespace tc;

constexpr int BM = 128, BN = 128;
constexpr int kSub = 128 * 128;                 // bytes of a [128 rows x 64 elements] 128-byte-swizzled sub-tile
constexpr int kStages = 2;
constexpr int kThreads = 512;                   // softmax 0, softmax 1, {MMA thread, idle}, gather {K, K, V, V}
// Registers per thread.  setmaxnreg draws on the 512 * 128 the CTA was launched with.
template <bool E4> struct Regs {
    static constexpr int kSoftmax = E4 ? 192 : 208, kOther = E4 ? 48 : 56, kGather = E4 ? 80 : 40;
    static_assert(8 * 32 * kSoftmax + 4 * 32 * kOther + 4 * 32 * kGather <= kThreads * 128, "register pool");
};

template <int HD> struct Smem {
    static constexpr int kTile = HD / 64 * kSub;
    alignas(1024) unsigned char q[2][kTile];
    alignas(1024) unsigned char k[kStages][kTile];
    alignas(1024) unsigned char v[kStages][kTile];
    alignas(16) unsigned char bad[4][BN];       // rows of a tile without a pool row (ring of four tiles)
    alignas(8) unsigned long long q_full[2];
    unsigned long long s_full[2], p_half[2], p_full[2], o_full[2];
    unsigned long long k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    unsigned int tmem_base;
    int any_bad;
    int launch_abort;                           // a wait that runs out ends this CTA only (about a second)
    AbortBox box;
};

// What a CTA works on
struct Job {
    int n, w0, tiles;          // keys of the list, keys of the first tile, tiles
    int sinks, first;          // list entry u is token u < sinks ? u : u - sinks + first of the table at `beg`
    int64_t beg;
    int hk;
    int jb[2], je[2];          // tiles of each warpgroup (key_split: every second one from jb)
};
__device__ __forceinline__ int tile_base(const Job& job, int j) { return j ? job.w0 + (j - 1) * BN : 0; }
__device__ __forceinline__ int tile_keys(const Job& job, int j) { return j ? BN : job.w0; }
__device__ __forceinline__ int tile_of(const Job& job, int u) { return u < job.w0 ? 0 : (u - job.w0) / BN + 1; }
__device__ __forceinline__ void cut(Job& job, int n) {
    job.n = n;
    job.tiles = (n + BN - 1) / BN;
    job.w0 = n - (job.tiles - 1) * BN;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// One softmax thread = one query row: walks `count` tiles from `j0` in steps of `step`, leaves P in tensor memory
// over S, keeps the reference maximum m and the denominator l.  Visible entries u of the list: u <= hi and
// (u >= lo or u < ns).  Returns false when a wait ran out.
template <typename MT, int HD, int kPolyOf8>
__device__ __forceinline__ bool softmax_rows(Smem<HD>& sm, int w, uint32_t s_addr, uint32_t o_addr, const Job& job, int j0, int step,
                                             int count, int hi, int lo, int ns, float scale, float& m_ref, float& l) {
    AbortBox* const wc = &sm.box;
    constexpr float kLazy = 8.f;          // P <= 2^8: O is rescaled rarely
    m_ref = -INFINITY;
    l = 0.f;
    // brings O and l to a new reference maximum when some row of the warp outgrew the old one
    auto advance = [&](int i, float mx) -> bool {
        const float m_new = fmaxf(m_ref, mx * scale);
        if (__any_sync(0xffffffffu, m_new > m_ref + kLazy)) {
            if (i > 0) {
                // a row that has seen nothing yet keeps its zeros (-inf - -inf is not a number)
                const float alpha = m_ref == m_new ? 1.f : fast_exp2(m_ref - m_new);
                l *= alpha;
                if (!mbar_wait(&sm.o_full[w], (i - 1) & 1, wc)) return false;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) {
                    float ov[32];
                    tmem_ld32(o_addr + c * 32, ov);
#pragma unroll
                    for (int e = 0; e < 32; ++e) ov[e] *= alpha;
                    tmem_st32(o_addr + c * 32, reinterpret_cast<const uint32_t*>(ov));
                }
                tmem_st_wait();
            }
            m_ref = m_new;
        }
        return true;
    };
    for (int i = 0; i < count; ++i) {
        const int j = j0 + i * step, base = tile_base(job, j), keys = tile_keys(job, j);
        if (!mbar_wait(&sm.s_full[w], i & 1, wc)) return false;
        tc_fence_after();
        const bool any_bad = *(volatile int*)&sm.any_bad;
        const int h = min(hi - base, keys - 1), lw = lo - base, s = ns - base;     // in columns of this tile
        const bool masked = any_bad || h < BN - 1 || (lw > 0 && s < BN);
        auto hidden = [&](int c) { return c > h || (c < lw && c >= s) || (any_bad && sm.bad[j & 3][c & (BN - 1)]); };
        if (keys > 96) {
            float sv[BN];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32_nowait(s_addr + c * 32, sv + c * 32);
            tmem_ld_wait();
            if (masked) {
                if (any_bad) {
#pragma unroll
                    for (int c = 0; c < BN; ++c)
                        if (sm.bad[j & 3][c]) sv[c] = -INFINITY;
                }
#pragma unroll
                for (int c = 0; c < BN; ++c)
                    if (c > h || (c < lw && c >= s)) sv[c] = -INFINITY;
            }
            float mx8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) mx8[e] = fmaxf(sv[e], sv[8 + e]);
#pragma unroll
            for (int c = 16; c < BN; c += 16)
#pragma unroll
                for (int e = 0; e < 8; ++e) mx8[e] = max3(mx8[e], sv[c + e], sv[c + 8 + e]);
            const float mx = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])), fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
            if (!advance(i, mx)) return false;
            const float nm = m_ref > -INFINITY ? -m_ref : 0.f;
            float rs4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t pk[32];
#pragma unroll
                for (int e = 0; e < 64; e += 4) {
                    float x0, x1, x2, x3, p0, p1, p2, p3;
                    fma2(x0, x1, sv[c * 64 + e], sv[c * 64 + e + 1], scale, scale, nm, nm);
                    fma2(x2, x3, sv[c * 64 + e + 2], sv[c * 64 + e + 3], scale, scale, nm, nm);
                    p0 = fast_exp2(x0);
                    p1 = fast_exp2(x1);
                    if (kPolyOf8 == 2 && (e & 4)) {
                        exp2_poly2(p2, p3, x2, x3);
                    } else {
                        p2 = fast_exp2(x2);
                        p3 = fast_exp2(x3);
                    }
                    add2(rs4[0], rs4[1], rs4[0], rs4[1], p0, p1);
                    add2(rs4[2], rs4[3], rs4[2], rs4[3], p2, p3);
                    pk[e >> 1] = pack2<MT>(p0, p1);
                    pk[(e >> 1) + 1] = pack2<MT>(p2, p3);
                }
                tmem_st32(s_addr + c * 32, pk);
                if (c == 0) {
                    tmem_st_wait();
                    tc_fence_before();
                    mbar_arrive(&sm.p_half[w]);
                }
            }
            l += (rs4[0] + rs4[1]) + (rs4[2] + rs4[3]);
        } else {
            // a short first tile: 32 columns at a time, as many as it has
            const int chunks = (keys + 31) / 32;
            float mx = -INFINITY;
            for (int c = 0; c < chunks; ++c) {
                float sv[32];
                tmem_ld32(s_addr + c * 32, sv);
#pragma unroll
                for (int e = 0; e < 32; ++e) mx = fmaxf(mx, masked && hidden(c * 32 + e) ? -INFINITY : sv[e]);
            }
            if (!advance(i, mx)) return false;
            const float nm = m_ref > -INFINITY ? -m_ref : 0.f;
            for (int c = 0; c < chunks; ++c) {       // P of chunk c lands on columns 16 c .., already read
                float sv[32];
                uint32_t pk[16];
                tmem_ld32(s_addr + c * 32, sv);
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float p0 = masked && hidden(c * 32 + e) ? 0.f : fast_exp2(fmaf(sv[e], scale, nm));
                    const float p1 = masked && hidden(c * 32 + e + 1) ? 0.f : fast_exp2(fmaf(sv[e + 1], scale, nm));
                    l += p0 + p1;
                    pk[e >> 1] = pack2<MT>(p0, p1);
                }
                asm volatile(
                    "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                    ::"r"(s_addr + c * 16), "r"(pk[0]), "r"(pk[1]), "r"(pk[2]), "r"(pk[3]), "r"(pk[4]), "r"(pk[5]), "r"(pk[6]),
                      "r"(pk[7]), "r"(pk[8]), "r"(pk[9]), "r"(pk[10]), "r"(pk[11]), "r"(pk[12]), "r"(pk[13]), "r"(pk[14]),
                      "r"(pk[15]) : "memory");
                tmem_st_wait();
            }
            mbar_arrive(&sm.p_half[w]);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&sm.p_full[w]);
    }
    if (count > 0) {
        if (!mbar_wait(&sm.o_full[w], (count - 1) & 1, wc)) return false;
        tc_fence_after();
    }
    return true;
}

template <typename T, int HD, bool kPrefix, bool E4>
__global__ void __launch_bounds__(kThreads, 1)
attend_tc_kernel(const AttendParams p) {
    using MT = typename std::conditional<E4, __half, T>::type;       // e4m3 rows are multiplied as fp16
    constexpr int kTileBytes = Smem<HD>::kTile;
    constexpr int CPR = HD / 8, RPP = 64 / CPR, PASSES = BN / RPP;   // 16-byte chunks of a row; rows per pass of 64 threads
    extern __shared__ unsigned char smem_raw[];
    Smem<HD>& sm = *reinterpret_cast<Smem<HD>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    AbortBox* const wc = &sm.box;
    const int G = p.H / p.Hkv;

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    Job job;
    int head[2] = {0, 0}, row0[2] = {0, 0};      // window: head and first query row (in the chunk) of each tile
    int q_len = 0, shift = 0, t_first = 0;
    int64_t q_beg = 0;
    if (kPrefix) {
        job.hk = blockIdx.y;
        const int tiles = (p.n_prefix + BN - 1) / BN;
        // this CTA's share of the key tiles; the list's first tile is the short one
        const int a = (int)((int64_t)tiles * blockIdx.x / p.splits), e = (int)((int64_t)tiles * (blockIdx.x + 1) / p.splits);
        const int short_keys = p.n_prefix - (tiles - 1) * BN;
        const int u0 = a ? short_keys + (a - 1) * BN : 0, u1 = e ? short_keys + (e - 1) * BN : 0;
        job.beg = u0;
        job.sinks = job.first = 0;
        cut(job, u1 - u0);
        job.jb[0] = 0;
        job.jb[1] = p.key_split ? 1 : 0;
        job.je[0] = job.je[1] = job.tiles;
        row0[0] = blockIdx.z * (p.key_split ? BM : 2 * BM);
        row0[1] = row0[0] + (p.key_split ? 0 : BM);
        if (row0[1] >= p.B * G) job.je[1] = 0;
    } else {
        const int b = blockIdx.z;
        q_beg = b ? p.q_offsets[b - 1] : 0;
        const int64_t q_end = p.q_offsets[b], kv_beg = b ? p.kv_offsets[b - 1] : 0, kv_end = p.kv_offsets[b];
        if (q_beg < 0 || q_end < q_beg || q_end > p.n_q_tokens || kv_beg < 0 || kv_end > p.n_kv_tokens || kv_end - kv_beg < q_end - q_beg) {
            if (p.err_flag && threadIdx.x == 0) atomicOr(p.err_flag, ATTN_B200_FLAG_BAD_OFFSETS);
            return;
        }
        q_len = (int)(q_end - q_beg);
        const int kv_len = (int)(kv_end - kv_beg);
        shift = kv_len - q_len;
        const int q0 = blockIdx.x * (p.head_pairs ? BM : 2 * BM);
        if (q0 >= q_len) return;
        if (p.head_pairs) {
            const int per = G / 2;
            job.hk = blockIdx.y / per;
            head[0] = job.hk * G + (blockIdx.y - job.hk * per) * 2;
            head[1] = head[0] + 1;
            row0[0] = row0[1] = q0;
        } else {
            head[0] = head[1] = blockIdx.y;
            job.hk = blockIdx.y / G;
            row0[0] = q0;
            row0[1] = q0 + BM;
        }
        const int rows = p.head_pairs ? BM : 2 * BM;
        const int last = shift + min(q0 + rows, q_len) - 1;
        const int64_t lo = (int64_t)shift + q0 - p.window + 1;
        t_first = lo > 0 ? (int)lo : 0;
        job.beg = kv_beg;
        job.first = t_first;
        job.sinks = min(p.sinks, t_first);
        cut(job, job.sinks + last - t_first + 1);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            if (row0[w] >= q_len) {
                job.jb[w] = job.je[w] = 0;
                continue;
            }
            const int hi_w = shift + min(row0[w] + BM, q_len) - 1 - t_first + job.sinks;
            const int64_t lo_w = (int64_t)shift + row0[w] - p.window + 1 - t_first + job.sinks;
            job.je[w] = tile_of(job, hi_w) + 1;
            job.jb[w] = p.sinks > 0 || lo_w <= 0 ? 0 : tile_of(job, (int)lo_w);
        }
    }
    const bool key_split = kPrefix && p.key_split;

    if (threadIdx.x == 0) {
        for (int w = 0; w < 2; ++w) {
            mbar_init(&sm.q_full[w], 128);
            mbar_init(&sm.s_full[w], 1);
            mbar_init(&sm.p_half[w], 128);
            mbar_init(&sm.p_full[w], 128);
            mbar_init(&sm.o_full[w], 1);
        }
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sm.k_full[s], 64);
            mbar_init(&sm.k_empty[s], 1);
            mbar_init(&sm.v_full[s], 64);
            mbar_init(&sm.v_empty[s], 1);
        }
        sm.any_bad = 0;
        sm.box.abort = 0;
        sm.launch_abort = 0;
        sm.box.launch_abort = &sm.launch_abort;
        sm.box.err_flag = p.err_flag;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;

    if (warp >= 12) {
        // ------------------------------------------------------------------ gather: 64 threads K, 64 threads V
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<E4>::kGather));
        const int tid = threadIdx.x - 384, t64 = tid & 63;
        const bool v_stream = tid >= 64;
        const int c = t64 % CPR, rsub = t64 / CPR;
        unsigned long long* full = v_stream ? sm.v_full : sm.k_full;
        unsigned long long* empty = v_stream ? sm.v_empty : sm.k_empty;
        unsigned char (*stage)[kTileBytes] = v_stream ? sm.v : sm.k;
        // The CPR threads of a row group need the same PASSES slots: thread c fetches and checks those of
        // passes c and c + CPR, the copies take them by shuffle.
        // The slots of the next tile are fetched ahead of the wait for its stage.
        int ahead[2];
        auto fetch = [&](int j) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = (c + CPR * i) * RPP + rsub, u = tile_base(job, j) + r;
                const int t = u < job.sinks ? u : u - job.sinks + job.first;
                ahead[i] = j < job.tiles && r < tile_keys(job, j) ? __ldg(p.table + job.beg + t) : -1;
            }
        };
        fetch(0);
        bool ok = true;
        for (int j = 0; j < job.tiles; ++j) {
            const int s = j % kStages;
            int sl[2] = {ahead[0], ahead[1]};
            fetch(j + 1);
            if (j >= kStages) ok = mbar_wait(&empty[s], ((j - kStages) / kStages) & 1, wc);
            if (!__all_sync(0xffffffffu, ok)) break;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = (c + CPR * i) * RPP + rsub;
                if (sl[i] < 0 || sl[i] >= p.n_slots) {
                    bad |= r < tile_keys(job, j);
                    sl[i] = -1;
                }
                // bad[j & 3]: written before the tile is published and read until its P is there, which the
                // products of tile j + 2 wait for; those precede the release that lets tile j + 4 in
                if (!v_stream) sm.bad[j & 3][r] = sl[i] < 0;
            }
            if (bad) {
                if (!v_stream) sm.any_bad = 1;
                if (p.err_flag) atomicOr(p.err_flag, ATTN_B200_FLAG_BAD_SLOT);
            }
            if constexpr (!E4) {
                const uint32_t sbase = smem_u32(stage[s]) + (c >> 3) * kSub;
                const char* base = (const char*)(v_stream ? p.v_cache : p.k_cache) + ((int64_t)job.hk * HD + c * 8) * 2;
                const int64_t row_bytes = (int64_t)p.Hkv * HD * 2;
#pragma unroll
                for (int q = 0; q < PASSES; ++q) {
                    const int v = __shfl_sync(0xffffffffu, sl[q / CPR], q % CPR, CPR);
                    const int r = q * RPP + rsub;
                    cp16(sbase + r * 128 + (((c & 7) ^ (r & 7)) << 4), base + (int64_t)(v >= 0 ? v : 0) * row_bytes, v >= 0 ? 16 : 0);
                }
                asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
            } else {
                // 8-byte pieces (8 codes -> 16 bytes of fp16), kBatch rows in flight
                constexpr int kBatch = 16;
                const uint32_t sbase = smem_u32(stage[s]) + (c >> 3) * kSub;
                const char* base = (const char*)(v_stream ? p.v_cache : p.k_cache) + (int64_t)job.hk * HD + c * 8;
                const int64_t row_bytes = (int64_t)p.Hkv * HD;
#pragma unroll
                for (int q0 = 0; q0 < PASSES; q0 += kBatch) {
                    uint2 x[kBatch];
#pragma unroll
                    for (int q = 0; q < kBatch; ++q) {
                        const int v = __shfl_sync(0xffffffffu, sl[(q0 + q) / CPR], (q0 + q) % CPR, CPR);
                        x[q] = make_uint2(0, 0);
                        if (v >= 0) x[q] = __ldg(reinterpret_cast<const uint2*>(base + (int64_t)v * row_bytes));
                    }
#pragma unroll
                    for (int q = 0; q < kBatch; ++q) {
                        const int r = (q0 + q) * RPP + rsub;
                        __half2 h0, h1, h2, h3;
                        e4m3x4_to_half2x2(x[q].x, h0, h1);
                        e4m3x4_to_half2x2(x[q].y, h2, h3);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sbase + r * 128 + (((c & 7) ^ (r & 7)) << 4)),
                                     "r"(*reinterpret_cast<uint32_t*>(&h0)), "r"(*reinterpret_cast<uint32_t*>(&h1)),
                                     "r"(*reinterpret_cast<uint32_t*>(&h2)), "r"(*reinterpret_cast<uint32_t*>(&h3)) : "memory");
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&full[s]);
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<E4>::kOther));
        if (warp == 9) {
            // -------------------------------------------------------------- MMA issuer
            constexpr uint32_t fmt = std::is_same<MT, __nv_bfloat16>::value ? 1u : 0u;
            constexpr uint32_t idesc0 = (1u << 4) | (fmt << 7) | (fmt << 10) | ((BM >> 4) << 24);
            constexpr uint32_t idesc_pv = idesc0 | (1u << 16) | ((HD >> 3) << 17);
            if (elect_one()) {
                const uint64_t qd[2] = {smem_desc(smem_u32(sm.q[0]), 16, 1024), smem_desc(smem_u32(sm.q[key_split ? 0 : 1]), 16, 1024)};
                const uint64_t kd[2] = {smem_desc(smem_u32(sm.k[0]), 16, 1024), smem_desc(smem_u32(sm.k[1]), 16, 1024)};
                const uint64_t vd[2] = {smem_desc(smem_u32(sm.v[0]), kSub, 1024), smem_desc(smem_u32(sm.v[1]), kSub, 1024)};
                // columns that a tile is multiplied in: whole, or its keys rounded up to 32
                auto wide = [&](int j) { const int k = tile_keys(job, j); return k > 96 ? BN : (k + 31) / 32 * 32; };
                auto issue_qk = [&](int w, int j) {
                    const uint64_t a = qd[w], b2 = kd[j & 1];
                    const uint32_t idesc = idesc0 | ((uint32_t)(wide(j) >> 3) << 17);
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const uint32_t off16 = ((kk >> 2) * kSub + (kk & 3) * 32) >> 4;
                        umma_f16(tmem + w * 128, a + off16, b2 + off16, idesc, kk > 0);
                    }
                    umma_commit(&sm.s_full[w]);
                };
                auto pv_step = [&](int w, uint64_t v, int kk, bool first) {           // 16 keys
                    umma_f16_ts(tmem + 256 + w * 128, tmem + w * 128 + kk * 8, v + (uint64_t)(kk * (2048 >> 4)), idesc_pv, (!first || kk > 0) ? 1u : 0u);
                };
                int done[2] = {0, 0};            // tiles of each warpgroup whose P.V has been issued
                bool ok = true;
                auto finish_tile = [&](int w, int j) -> bool {        // P.V of tile j
                    const int i = done[w];
                    if (!mbar_wait_spin(&sm.p_half[w], i & 1, wc)) return false;
                    if (!mbar_wait_spin(&sm.v_full[j & 1], (j >> 1) & 1, wc)) return false;
                    tc_fence_after();
                    const bool whole = wide(j) == BN;
                    const uint64_t v = vd[j & 1];
                    if (whole) {
#pragma unroll
                        for (int kk = 0; kk < BN / 32; ++kk) pv_step(w, v, kk, i == 0);
                    }
                    if (!mbar_wait_spin(&sm.p_full[w], i & 1, wc)) return false;
                    tc_fence_after();
                    if (whole) {
#pragma unroll
                        for (int kk = BN / 32; kk < BN / 16; ++kk) pv_step(w, v, kk, false);
                    } else {
#pragma unroll 1
                        for (int kk = 0; kk < wide(j) / 16; ++kk) pv_step(w, v, kk, i == 0);
                    }
                    umma_commit(&sm.o_full[w]);
                    done[w] = i + 1;
                    return true;
                };
                auto start_tile = [&](int w, int j) -> bool {         // Q.K of tile j
                    if (!mbar_wait_spin(&sm.k_full[j & 1], (j >> 1) & 1, wc)) return false;
                    tc_fence_after();
                    issue_qk(w, j);
                    return true;
                };
                ok = mbar_wait_spin(&sm.q_full[0], 0, wc);
                if (ok && !key_split) ok = mbar_wait_spin(&sm.q_full[1], 0, wc);
                if (key_split) {
                    for (int j = 0; ok && j < 2 && j < job.tiles; ++j) {
                        ok = start_tile(j, j);
                        umma_commit(&sm.k_empty[j & 1]);
                    }
                    for (int j = 0; ok && j < job.tiles; ++j) {
                        if (!(ok = finish_tile(j & 1, j))) break;
                        umma_commit(&sm.v_empty[j & 1]);
                        if (j + 2 < job.tiles) {
                            if (!(ok = start_tile(j & 1, j + 2))) break;
                            umma_commit(&sm.k_empty[j & 1]);
                        }
                    }
                } else {
                    // every tile is some warpgroup's: the list is the union of two overlapping stretches
                    auto mine = [&](int w, int j) { return j >= job.jb[w] && j < job.je[w]; };
                    for (int w = 0; w < 2 && ok; ++w)
                        if (mine(w, 0)) ok = start_tile(w, 0);
                    if (ok) umma_commit(&sm.k_empty[0]);
                    for (int j = 0; ok && j < job.tiles; ++j) {
                        for (int w = 0; w < 2 && ok; ++w) {
                            if (mine(w, j)) ok = finish_tile(w, j);
                            if (ok && w == 1) umma_commit(&sm.v_empty[j & 1]);
                            if (ok && mine(w, j + 1)) ok = start_tile(w, j + 1);
                        }
                        if (ok && j + 1 < job.tiles) umma_commit(&sm.k_empty[(j + 1) & 1]);
                    }
                }
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------------ softmax warpgroups
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Regs<E4>::kSoftmax));
        const int w = warp >> 2, r = threadIdx.x & 127;
        const int n_rows = kPrefix ? p.B * G : q_len;
        // element offset of row `row` of this warpgroup's tile in q (and in the window's output), or -1
        auto row_at = [&](int row) -> int64_t {
            if (row >= n_rows) return -1;
            if (kPrefix) {
                const int b = row / G;
                return ((int64_t)b * p.H + job.hk * G + (row - b * G)) * HD;
            }
            return ((q_beg + row) * p.H + head[w]) * HD;
        };
        float scale = p.scale_log2;
        if (kPrefix && E4) scale *= p.k_scale[job.hk];
        if (!E4) {
            if (w == 0 || !key_split) {
                // a warp copies its own 32 rows, whole rows at a time, into the swizzled tile
                constexpr int rows_at_once = 32 / CPR;
                const int cc = lane % CPR, rr = lane / CPR;
#pragma unroll 4
                for (int i = 0; i < 32 / rows_at_once; ++i) {
                    const int lr = (warp & 3) * 32 + i * rows_at_once + rr;
                    const int64_t at = row_at(row0[w] + lr);
                    cp16(smem_u32(sm.q[w]) + (cc >> 3) * kSub + lr * 128 + (((cc & 7) ^ (lr & 7)) << 4),
                         (const T*)p.q + (at >= 0 ? at : 0) + cc * 8, at >= 0 ? 16 : 0);
                }
                asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
            }
        } else {
            // queries are multiplied as fp16: bf16 ones after a power of two that brings the row to [1, 2)
            const int64_t at = row_at(row0[w] + r);
            float mul = 1.f;
            if (std::is_same<T, __nv_bfloat16>::value) {
                float top = 0.f;
                for (int d = 0; d < HD; d += 8) {
                    const uint4 x = at >= 0 ? *reinterpret_cast<const uint4*>((const T*)p.q + at + d) : make_uint4(0, 0, 0, 0);
                    const uint32_t wd[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float a, b;
                        unpack2(wd[e], T(), a, b);
                        top = fmaxf(top, fmaxf(fabsf(a), fabsf(b)));
                    }
                }
                if (top > 1e-30f && top < 1e30f) {
                    const int ex = ((__float_as_int(top) >> 23) & 255) - 127;
                    mul = __int_as_float((127 - ex) << 23);
                    scale *= __int_as_float((127 + ex) << 23);
                }
            }
            if (w == 0 || !key_split) {
                for (int cc = 0; cc < CPR; ++cc) {
                    uint4 x = at >= 0 ? *reinterpret_cast<const uint4*>((const T*)p.q + at + cc * 8) : make_uint4(0, 0, 0, 0);
                    if (std::is_same<T, __nv_bfloat16>::value) {
                        uint32_t wd[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float a, b;
                            unpack2(wd[e], T(), a, b);
                            wd[e] = pack2<__half>(a * mul, b * mul);
                        }
                        x = make_uint4(wd[0], wd[1], wd[2], wd[3]);
                    }
                    *reinterpret_cast<uint4*>(sm.q[w] + (cc >> 3) * kSub + r * 128 + (((cc & 7) ^ (r & 7)) << 4)) = x;
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&sm.q_full[w]);

        const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_addr = lane_base + w * 128, o_addr = lane_base + 256 + w * 128;
        const int step = key_split ? 2 : 1;
        const int count = job.je[w] > job.jb[w] ? (job.je[w] - job.jb[w] + step - 1) / step : 0;
        const int row = row0[w] + r;
        int hi = INT_MAX, lo = 0, ns = 0;
        if (!kPrefix) {
            hi = shift + row - t_first + job.sinks;
            const int64_t lo64 = (int64_t)hi - p.window + 1;
            lo = lo64 > 0 ? (int)lo64 : 0;
            ns = p.sinks;
        }
        float m, l;
        // e4m3 and fp16: every exponential on the special-function unit; bf16: two of eight as a cubic on the FMA pipe
        const bool ok = softmax_rows<MT, HD, std::is_same<MT, __nv_bfloat16>::value ? 2 : 0>(sm, w, s_addr, o_addr, job, job.jb[w], step,
                                                                                             count, hi, lo, ns, scale, m, l);
        const int64_t at = row_at(row);
        if (ok && kPrefix) {
            const int b = row / G;
            float* dst = p.parts + (((int64_t)(blockIdx.x * step + (key_split ? w : 0)) * p.B + b) * p.H + job.hk * G + (row - b * G)) * (HD + 2);
            const float vs = E4 ? p.v_scale[job.hk] : 1.f;
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                float ov[32];
                __syncwarp();
                if (count > 0) tmem_ld32(o_addr + c * 32, ov);
#pragma unroll
                for (int e = 0; e < 32 && at >= 0; e += 2)
                    *reinterpret_cast<float2*>(dst + c * 32 + e) =
                        count > 0 ? make_float2(ov[e] * vs, ov[e + 1] * vs) : make_float2(0.f, 0.f);
            }
            if (at >= 0) *reinterpret_cast<float2*>(dst + HD) = make_float2(count > 0 ? m : -INFINITY, l);
        } else if (ok && count > 0) {
            // a row none of whose keys has a pool row is zero
            const float inv = m > -INFINITY || l != l ? 1.f / l : 0.f;
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                float ov[32];
                __syncwarp();
                tmem_ld32(o_addr + c * 32, ov);
                uint4* dst = reinterpret_cast<uint4*>((T*)p.out + (at >= 0 ? at : 0) + c * 32);
#pragma unroll
                for (int e = 0; e < 4 && at >= 0; ++e)
                    dst[e] = make_uint4(pack2<T>(ov[8 * e] * inv, ov[8 * e + 1] * inv), pack2<T>(ov[8 * e + 2] * inv, ov[8 * e + 3] * inv),
                                        pack2<T>(ov[8 * e + 4] * inv, ov[8 * e + 5] * inv), pack2<T>(ov[8 * e + 6] * inv, ov[8 * e + 7] * inv));
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Rows that no query tile writes: past the last sequence, beyond max_q_len, or of a sequence whose offsets are bad.
__global__ void zero_rows_kernel(void* out, const int32_t* q_offsets, const int32_t* kv_offsets, int B, int64_t n_q, int64_t n_kv, int covered,
                                 int64_t row_bytes, int32_t* err_flag) {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t vecs = row_bytes / 16;
    auto clamped = [&](int64_t v) { return v < 0 ? (int64_t)0 : (v > n_q ? n_q : v); };
    for (int b = blockIdx.x; b <= B; b += gridDim.x) {
        const int64_t beg = b ? q_offsets[b - 1] : 0, end = b < B ? q_offsets[b] : n_q;
        int64_t from = clamped(beg);
        const int64_t to = clamped(end);
        if (b < B) {
            const int64_t kb = b ? kv_offsets[b - 1] : 0, ke = kv_offsets[b];
            const bool good = beg >= 0 && end >= beg && end <= n_q && kb >= 0 && ke <= n_kv && ke - kb >= end - beg;
            if (good) {
                if (end - beg <= covered) continue;
                if (err_flag && threadIdx.x == 0) atomicOr(err_flag, ATTN_B200_FLAG_BAD_OFFSETS);
                from = beg + covered;
            }
        }
        uint4* base = reinterpret_cast<uint4*>((char*)out + from * row_bytes);
        for (int64_t i = threadIdx.x; i < (to - from) * vecs; i += blockDim.x) base[i] = make_uint4(0, 0, 0, 0);
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// Launch as a programmatic dependent: the kernels wait (griddepcontrol.wait) before they read anything.
template <typename... A>
int launch_dependent(void (*kernel)(A...), dim3 grid, int threads, int smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, int HD, bool kPrefix, bool E4>
int launch(const AttendParams& p, dim3 grid, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    const int smem = (int)sizeof(Smem<HD>) + 1024;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 64) return ATTN_B200_ETOOLARGE;
    if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
        if ((e = cudaFuncSetAttribute(attend_tc_kernel<T, HD, kPrefix, E4>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess)
            return (int)e;
        ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    return launch_dependent(attend_tc_kernel<T, HD, kPrefix, E4>, grid, kThreads, smem, st, p);
}

}  // namespace

bool attend_tc_supported(int D, int dtype, float scale) {
    return (D == 64 || D == 128) && (dtype == ATTN_B200_F16 || dtype == ATTN_B200_BF16) && scale > 0.f && scale < 1e30f;
}

int attend_window_launch(AttendParams p, int max_q_len, int D, int dtype, cudaStream_t st) {
    const int G = p.H / p.Hkv;
    p.head_pairs = G % 2 == 0;
    const int rows = p.head_pairs ? BM : 2 * BM, blocks = (int)(((int64_t)max_q_len + rows - 1) / rows);
    const int units = p.head_pairs ? p.H / 2 : p.H;
    if (p.B > 65535 || units > 65535) return ATTN_B200_ETOOLARGE;
    if (p.n_q_tokens > 0) {
        const int rc = launch_dependent(zero_rows_kernel, dim3(p.B < 63 ? p.B + 1 : 64), 256, 0, st, p.out, p.q_offsets, p.kv_offsets, p.B,
                                        p.n_q_tokens, p.n_kv_tokens, blocks * rows, (int64_t)p.H * D * 2, p.err_flag);
        if (rc) return rc;
    }
    if (blocks == 0 || p.B == 0) return 0;
    const dim3 grid(blocks, units, p.B);
    const bool bf = dtype == ATTN_B200_BF16;
    if (D == 64) return bf ? launch<__nv_bfloat16, 64, false, false>(p, grid, st) : launch<__half, 64, false, false>(p, grid, st);
    return bf ? launch<__nv_bfloat16, 128, false, false>(p, grid, st) : launch<__half, 128, false, false>(p, grid, st);
}

void attend_prefix_plan(AttendParams& p) {
    const int64_t rows = (int64_t)p.B * (p.H / p.Hkv);
    p.key_split = rows <= BM;
    const int64_t groups = p.key_split ? 1 : (rows + 2 * BM - 1) / (2 * BM), items = groups * p.Hkv;
    const int tiles = (p.n_prefix + BN - 1) / BN;
    // one CTA per SM: the number of splits with the fewest tile steps in the longest chain; a wave costs
    // about three steps besides (set-up, first rows, partial rows)
    int64_t best = -1;
    p.splits = 1;
    for (int s = 1; s <= 148 && s <= tiles; ++s) {
        const int64_t cost = (items * s + 147) / 148 * ((tiles + s - 1) / s + 3);
        if (best < 0 || cost < best) {
            best = cost;
            p.splits = s;
        }
    }
}

int attend_prefix_launch(const AttendParams& p, int D, int dtype, bool e4, cudaStream_t st) {
    const int64_t rows = (int64_t)p.B * (p.H / p.Hkv);
    const int64_t groups = p.key_split ? 1 : (rows + 2 * BM - 1) / (2 * BM);
    if (groups > 65535 || p.Hkv > 65535) return ATTN_B200_ETOOLARGE;
    const dim3 grid(p.splits, p.Hkv, (unsigned)groups);
    const bool bf = dtype == ATTN_B200_BF16;
    if (D == 64) {
        if (e4) return bf ? launch<__nv_bfloat16, 64, true, true>(p, grid, st) : launch<__half, 64, true, true>(p, grid, st);
        return bf ? launch<__nv_bfloat16, 64, true, false>(p, grid, st) : launch<__half, 64, true, false>(p, grid, st);
    }
    if (e4) return bf ? launch<__nv_bfloat16, 128, true, true>(p, grid, st) : launch<__half, 128, true, true>(p, grid, st);
    return bf ? launch<__nv_bfloat16, 128, true, false>(p, grid, st) : launch<__half, 128, true, false>(p, grid, st);
}

}  // namespace attn
