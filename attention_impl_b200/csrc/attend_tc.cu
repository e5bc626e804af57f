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
constexpr int kItems = 4;                       // items published ahead
// Warps 0-3 and 4-7 softmax, 8 item list, 9 MMA thread, 10 query tiles; 12-15 K and V, 32 rows of a tile each.  With
// e4m3 rows 12-13 and 14-15 turn the raw K and V rows into fp16.
// Registers per thread: setmaxnreg draws on the 512 * 128 that the CTA was launched with.  The softmax warps fit their row of
// 128 scores in 184; what the MMA thread and the gather warps spill counts more, for all others wait for them (four prompts: 303
// us with 184 / 88 / 56, 317 with 184 / 72 / 72, 332 with 208 / 56 / 40).
constexpr int kThreads = 512;
template <bool E4> struct Cfg {
    static constexpr int kSoftmax = 184, kOther = E4 ? 72 : 88, kGather = E4 ? 72 : 56;
    static_assert(8 * 32 * kSoftmax + 4 * 32 * kOther + 4 * 32 * kGather <= kThreads * 128, "register pool");
};

// What the CTA works on next: a pair of query tiles and their list of keys
struct Item {
    int tiles, w0, n;          // key tiles (0: no more work), keys of the first tile, keys
    int sinks, first;          // list entry u is token u < sinks ? u : u - sinks + first of the table at `beg`
    int64_t beg;
    int hk;
    int jb[2], je[2];          // key tiles of each warpgroup (key_split: every second one from jb)
    int row0[2], head[2];      // first query row (window: in the chunk) and head (window) of each query tile
    int n_rows, shift;         // query rows of the sequence (prefix: of the KV head); window: position of row 0
    int64_t q_beg;
    int part;                  // prefix: first of this CTA's partial sets
};

enum Mode { kWindow, kPrefixPair, kPrefixSplit };      // kPrefixSplit: AttendParams::key_split

template <int HD, int kMode, bool E4> struct Smem {
    static constexpr int kTile = HD / 64 * kSub;
    // Two stages each of K and V, three where one query tile leaves room: a batch that fits one tile waits for DRAM
    static constexpr int kStages = kMode == kPrefixSplit && !E4 ? 3 : 2;
    static constexpr int kExtra = kMode == kWindow || E4 ? kSub : 16;
    alignas(1024) unsigned char q[kMode == kPrefixSplit ? 1 : 2][kTile];
    alignas(1024) unsigned char k[kStages][kTile];
    alignas(1024) unsigned char v[kStages][kTile];
    alignas(1024) unsigned char extra[2][kExtra];       // window: output staging; e4m3: raw K tile, raw V tile
    uint32_t bad[8][4];                                 // bit r: row r of a tile has no pool row (ring of eight tiles)
    signed char row_exp[2][BM];                         // bf16 queries over e4m3 rows: the power of two taken out of q
    Item item[kItems];
    alignas(8) unsigned long long item_full[kItems], item_empty[kItems];
    unsigned long long q_full[2], q_empty[2], o_free[2], raw_full[2], raw_empty[2];
    unsigned long long s_full[2], p_half[2], p_full[2], o_full[2];
    unsigned long long k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    unsigned int tmem_base;
    int any_bad;
    int launch_abort;                                   // a wait that runs out ends this CTA only (about a second)
    AbortBox box;
};
__device__ __forceinline__ int tile_base(int w0, int j) { return j ? w0 + (j - 1) * BN : 0; }
__device__ __forceinline__ int tile_keys(int w0, int j) { return j ? BN : w0; }
__device__ __forceinline__ int tile_of(const Item& it, int u) { return u < it.w0 ? 0 : (u - it.w0) / BN + 1; }
__device__ __forceinline__ void cut(Item& it, int n) {
    it.n = n;
    it.tiles = (n + BN - 1) / BN;
    it.w0 = n - (it.tiles - 1) * BN;
}
__device__ __forceinline__ bool active(const Item& it, int w) { return it.je[w] > it.jb[w]; }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Four rows of a two-dimensional tensor, one box (a row piece) each, to consecutive rows in shared memory; a row outside
// the tensor arrives as zeros.  The tensor map's box is one row high.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, int x, const int (&row)[4], void* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row[0]), "r"(row[1]), "r"(row[2]), "r"(row[3]), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t src) {
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(src) : "memory");
    return x;
}

// Blocks of query rows of sequence b (window), -1 if its offsets make no sense
__device__ __forceinline__ int window_blocks(const AttendParams& p, int b) {
    if (b >= p.B) return 0;
    const int64_t q_beg = b ? p.q_offsets[b - 1] : 0, q_end = p.q_offsets[b];
    const int64_t kv_beg = b ? p.kv_offsets[b - 1] : 0, kv_end = p.kv_offsets[b];
    if (q_beg < 0 || q_end < q_beg || q_end > p.n_q_tokens || kv_beg < 0 || kv_end > p.n_kv_tokens || kv_end - kv_beg < q_end - q_beg) {
        if (p.err_flag) atomicOr(p.err_flag, ATTN_B200_FLAG_BAD_OFFSETS);
        return -1;
    }
    const int rows = p.head_pairs ? BM : 2 * BM;
    const int64_t n = (q_end - q_beg + rows - 1) / rows;
    return (int)(n < p.blocks ? n : p.blocks);
}

// Block `blk` of sequence b for head unit `unit` (the sequence's offsets are good and it has that block)
__device__ __forceinline__ void window_item(const AttendParams& p, int b, int blk, int unit, Item& it) {
    const int G = p.H / p.Hkv;
    const int64_t q_beg = b ? p.q_offsets[b - 1] : 0, q_end = p.q_offsets[b];
    const int64_t kv_beg = b ? p.kv_offsets[b - 1] : 0, kv_end = p.kv_offsets[b];
    const int q_len = (int)(q_end - q_beg), kv_len = (int)(kv_end - kv_beg), shift = kv_len - q_len;
    const int rows = p.head_pairs ? BM : 2 * BM, q0 = blk * rows;
    if (p.head_pairs) {
        it.hk = unit / (G / 2);
        it.head[0] = unit * 2;
        it.head[1] = unit * 2 + 1;
        it.row0[0] = it.row0[1] = q0;
    } else {
        it.hk = unit / G;
        it.head[0] = it.head[1] = unit;
        it.row0[0] = q0;
        it.row0[1] = q0 + BM;
    }
    const int last = shift + min(q0 + rows, q_len) - 1;
    const int64_t lo = (int64_t)shift + q0 - p.window + 1;
    it.first = lo > 0 ? (int)lo : 0;
    it.sinks = min(p.sinks, it.first);
    it.beg = kv_beg;
    cut(it, it.sinks + last - it.first + 1);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        it.jb[w] = it.je[w] = 0;
        if (it.row0[w] >= q_len) continue;
        const int hi_w = shift + min(it.row0[w] + BM, q_len) - 1 - it.first + it.sinks;
        const int64_t lo_w = (int64_t)shift + it.row0[w] - p.window + 1 - it.first + it.sinks;
        it.je[w] = tile_of(it, hi_w) + 1;
        it.jb[w] = p.sinks > 0 || lo_w <= 0 ? 0 : tile_of(it, (int)lo_w);
    }
    it.n_rows = q_len;
    it.shift = shift;
    it.q_beg = q_beg;
}

// The one item of a prefix CTA: its share of the key tiles (the list's first tile is the short one) for a pair
// of query tiles of a KV head
__device__ __forceinline__ void prefix_item(const AttendParams& p, Item& it) {
    const int G = p.H / p.Hkv, per = p.splits * p.Hkv;
    const int group = blockIdx.x / per, rest = blockIdx.x - group * per;
    it.hk = rest / p.splits;
    const int split = rest - it.hk * p.splits;
    const int tiles = (p.n_prefix + BN - 1) / BN, short_keys = p.n_prefix - (tiles - 1) * BN;
    const int a = (int)((int64_t)tiles * split / p.splits), e = (int)((int64_t)tiles * (split + 1) / p.splits);
    const int u0 = a ? short_keys + (a - 1) * BN : 0, u1 = e ? short_keys + (e - 1) * BN : 0;
    it.beg = u0;
    it.sinks = it.first = 0;
    cut(it, u1 - u0);
    it.n_rows = p.B * G;
    it.row0[0] = group * (p.key_split ? BM : 2 * BM);
    it.row0[1] = it.row0[0] + (p.key_split ? 0 : BM);
    it.head[0] = it.head[1] = 0;
    it.jb[0] = 0;
    it.jb[1] = p.key_split ? 1 : 0;
    it.je[0] = it.tiles;
    it.je[1] = it.row0[1] < it.n_rows ? it.tiles : 0;
    it.shift = 0;
    it.q_beg = 0;
    it.part = split * (p.key_split ? 2 : 1);
}

// One softmax thread = one query row: walks `count` tiles from `j0` in steps of `step`, leaves P in tensor memory
// over S, keeps the reference maximum m and the denominator l.  Visible entries u of the list: u <= hi and
// (u >= lo or u < ns).  `c0`: tiles this warpgroup has seen before (barrier phases), `g0`: tiles of the CTA
// before this item.  Returns false when a wait ran out.
template <typename MT, int HD, typename SM>
__device__ __forceinline__ bool softmax_rows(SM& sm, int w, uint32_t s_addr, uint32_t o_addr, int w0, int j0, int step,
                                             int count, int c0, int g0, int hi, int lo, int ns, float scale, float& m_ref, float& l) {
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
                if (!mbar_wait(&sm.o_full[w], (c0 + i - 1) & 1, wc)) return false;
                tc_fence_after();
#pragma unroll 1
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
        const int j = j0 + i * step, base = tile_base(w0, j), keys = tile_keys(w0, j);
        if (!mbar_wait(&sm.s_full[w], (c0 + i) & 1, wc)) return false;
        tc_fence_after();
        const bool any_bad = *(volatile int*)&sm.any_bad;
        const uint32_t* const bad = sm.bad[(g0 + j) & 7];
        const int h = min(hi - base, keys - 1), lw = lo - base, s = ns - base;     // in columns of this tile
        // Chunks of 32 columns: `dead` ones no row of the warp sees, `whole` ones all rows see, of the others `bits` are
        // the columns that this row sees.
        int h_max = BN - 1, h_min = BN - 1, lw_max = 0, lw_min = 0;
        const bool masked = __any_sync(0xffffffffu, any_bad || h < BN - 1 || (lw > 0 && s < BN));
        if (masked) {
            h_max = __reduce_max_sync(0xffffffffu, h);
            h_min = __reduce_min_sync(0xffffffffu, h);
            lw_max = __reduce_max_sync(0xffffffffu, lw);
            lw_min = __reduce_min_sync(0xffffffffu, lw);
        }
        auto dead = [&](int c) { return c > h_max || (c + 31 < lw_min && c >= s); };
        auto whole = [&](int c) { return !any_bad && c + 31 <= h_min && (c >= lw_max || c + 31 < s); };
        auto bits = [&](int c) -> uint32_t {
            auto below = [&](int x) { return x <= c ? 0u : x >= c + 32 ? 0xffffffffu : (1u << (x - c)) - 1u; };     // columns < x
            uint32_t m = below(h + 1) & (~below(lw) | below(s));
            if (any_bad) m &= ~bad[c >> 5];
            return m;
        };
        if (keys > 96) {
            if (masked) {
                // -inf into the columns that are not seen, in tensor memory, before the whole row is read as any other.
                // (Reading a masked row in chunks, twice, with the dead chunks' exponentials left out took 3 us against
                // the 1.3 of a row without a mask; this way the main path keeps its registers.)
#pragma unroll 1
                for (int c = 0; c < BN; c += 32) {
                    if (whole(c)) continue;
                    uint32_t x[32];
                    if (dead(c)) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[e] = 0xff800000u;
                    } else {
                        tmem_ld32(s_addr + c, reinterpret_cast<float*>(x));
                        const uint32_t m = bits(c);
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[e] = m >> e & 1u ? x[e] : 0xff800000u;
                    }
                    tmem_st32(s_addr + c, x);
                }
                tmem_st_wait();
            }
            float sv[BN];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32_nowait(s_addr + c * 32, sv + c * 32);
            tmem_ld_wait();
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
                    // all on the special-function unit: with two of sixteen as a cubic on the FMA pipe, which the packed
                    // prefill gains from, four prompts took 312 us instead of 306 (issue slots, not the unit, are short here)
                    p0 = fast_exp2(x0);
                    p1 = fast_exp2(x1);
                    p2 = fast_exp2(x2);
                    p3 = fast_exp2(x3);
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
            // a short first tile: as many chunks of 32 columns as it has, read from tensor memory for the maximum and
            // again for P
            const int chunks = (keys + 31) / 32;
            float mx = -INFINITY;
            for (int c = 0; c < chunks * 32; c += 32) {
                if (dead(c)) continue;
                float sv[32];
                tmem_ld32(s_addr + c, sv);
                if (!whole(c)) {
                    const uint32_t m = bits(c);
#pragma unroll
                    for (int e = 0; e < 32; ++e) sv[e] = m >> e & 1u ? sv[e] : -INFINITY;
                }
                float a = fmaxf(sv[0], sv[1]), b = fmaxf(sv[2], sv[3]);
#pragma unroll
                for (int e = 4; e < 32; e += 4) {
                    a = max3(a, sv[e], sv[e + 1]);
                    b = max3(b, sv[e + 2], sv[e + 3]);
                }
                mx = max3(mx, a, b);
            }
            if (!advance(i, mx)) return false;
            const float nm = m_ref > -INFINITY ? -m_ref : 0.f;
            float l4[4] = {0.f, 0.f, 0.f, 0.f};
            for (int c = 0; c < chunks * 32; c += 32) {       // P of a chunk lands on columns c / 2 .., already read
                uint32_t pk[16];
                if (dead(c)) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) pk[e] = 0u;
                } else {
                    float sv[32];
                    tmem_ld32(s_addr + c, sv);
                    const uint32_t m = whole(c) ? 0xffffffffu : bits(c);
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        float x[4];
                        fma2(x[0], x[1], sv[e], sv[e + 1], scale, scale, nm, nm);
                        fma2(x[2], x[3], sv[e + 2], sv[e + 3], scale, scale, nm, nm);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            x[k] = m >> (e + k) & 1u ? fast_exp2(x[k]) : 0.f;
                            l4[k] += x[k];
                        }
                        pk[e >> 1] = pack2<MT>(x[0], x[1]);
                        pk[(e >> 1) + 1] = pack2<MT>(x[2], x[3]);
                    }
                }
                asm volatile(
                    "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                    ::"r"(s_addr + (c >> 1)), "r"(pk[0]), "r"(pk[1]), "r"(pk[2]), "r"(pk[3]), "r"(pk[4]), "r"(pk[5]), "r"(pk[6]),
                      "r"(pk[7]), "r"(pk[8]), "r"(pk[9]), "r"(pk[10]), "r"(pk[11]), "r"(pk[12]), "r"(pk[13]), "r"(pk[14]),
                      "r"(pk[15]) : "memory");
                if (c == 32 || (chunks == 1 && c == 0)) {      // the first 64 keys (of a short tile the MMA thread wants all)
                    tmem_st_wait();
                    tc_fence_before();
                    mbar_arrive(&sm.p_half[w]);
                }
            }
            l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&sm.p_full[w]);
    }
    if (!mbar_wait(&sm.o_full[w], (c0 + count - 1) & 1, wc)) return false;
    tc_fence_after();
    return true;
}

// One query row of a window item over again, by a warp, key by key and only the keys it sees.  A tile's V rows are
// multiplied with P = 0 for the rows that do not see them, and 0 times an infinity or a NaN is a NaN: a row whose
// result is not finite goes through here, where such a value reaches only the rows that see it.
template <typename T, int HD>
__device__ __noinline__ void row_by_itself(const AttendParams& p, const Item& it, int head, int row) {
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 31;
    const int pos = it.shift + row;
    const int64_t lo = (int64_t)pos - p.window + 1;
    const int first = lo > 0 ? (int)lo : 0, sinks = min(p.sinks, first);
    const int64_t at = ((it.q_beg + row) * p.H + head) * HD;
    float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        q[i] = to_f32<T>(((const T*)p.q)[at + lane + 32 * i]);
        o[i] = 0.f;
    }
    for (int u = 0; u < sinks + pos - first + 1; ++u) {
        const int slot = p.table[it.beg + (u < sinks ? u : u - sinks + first)];
        if (slot < 0 || slot >= p.n_slots) continue;
        const int64_t kv = ((int64_t)slot * p.Hkv + it.hk) * HD + lane;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s += q[i] * to_f32<T>(((const T*)p.k_cache)[kv + 32 * i]);
        s = group_sum<32>(s) * p.scale_log2;
        const float m_new = fmaxf(m, s), sub = m_new > -INFINITY ? m_new : 0.f;
        const float alpha = fast_exp2(m - sub), pr = fast_exp2(s - sub);
        l = l * alpha + pr;
        m = m_new;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = o[i] * alpha + pr * to_f32<T>(((const T*)p.v_cache)[kv + 32 * i]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < E; ++i) ((T*)p.out)[at + lane + 32 * i] = from_f32<T>(o[i] * inv);
}

// A window launch is persistent: one CTA per SM takes every gridDim.x-th item, and the item list, the query tiles and
// the K/V rings run ahead of the softmax, so that the set-up of an item hides under the one before it.  A prefix
// CTA has one item.
//
// K and V rows are gathered by TMA (tile::gather4): a lane owns four rows of a tile, fetches and checks their slots one
// tile ahead and issues one copy per 128 bytes of row; a slot outside the pool becomes the row behind its last one, which
// arrives as zeros.  Issuing is the bound (about 45 ns per copy of a warp, whatever other warps do): one warp per stream
// took 3 us for a tile, so four warps share both.  (Copied by 128 threads with cp.async, 16 bytes at a time, a tile took
// 2 to 4 us beside the softmax warps, whose issue slots those copies also take.)
template <typename T, int HD, int kMode, bool E4>
__global__ void __launch_bounds__(kThreads, 1)
attend_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o, const AttendParams p) {
    constexpr bool kPrefix = kMode != kWindow, key_split = kMode == kPrefixSplit;
    using MT = typename std::conditional<E4, __half, T>::type;       // e4m3 rows are multiplied as fp16
    using R = Cfg<E4>;
    using SM = Smem<HD, kMode, E4>;
    constexpr int kTileBytes = SM::kTile, kStages = SM::kStages;
    constexpr int QC = HD / 8;                                       // 16-byte chunks of a query row
    extern __shared__ unsigned char smem_raw[];
    SM& sm = *reinterpret_cast<SM*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    AbortBox* const wc = &sm.box;
    const int G = p.H / p.Hkv;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kItems; ++i) {
            mbar_init(&sm.item_full[i], 1);
            mbar_init(&sm.item_empty[i], E4 ? 13 : 14);       // one lane of every warp that reads the list
        }
        for (int w = 0; w < 2; ++w) {
            mbar_init(&sm.q_full[w], kPrefix ? 128 : 1);
            mbar_init(&sm.raw_full[w], 1);
            mbar_init(&sm.raw_empty[w], 64);
            mbar_init(&sm.q_empty[w], 1);
            mbar_init(&sm.o_free[w], 128);
            mbar_init(&sm.s_full[w], 1);
            mbar_init(&sm.p_half[w], 128);
            mbar_init(&sm.p_full[w], 128);
            mbar_init(&sm.o_full[w], 1);
        }
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sm.k_full[s], E4 ? 64 : 4);
            mbar_init(&sm.k_empty[s], 1);
            mbar_init(&sm.v_full[s], E4 ? 64 : 4);
            mbar_init(&sm.v_empty[s], 1);
        }
        sm.any_bad = 0;
        sm.launch_abort = 0;
        sm.box.abort = 0;
        sm.box.launch_abort = &sm.launch_abort;
        sm.box.err_flag = p.err_flag;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (kPrefix && warp == 8 && lane == 0) prefix_item(p, sm.item[0]);
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;
    // everything above is the CTA's own; from here on it reads what earlier kernels wrote
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // n-th item of this CTA: null when there are no more (or a wait ran out)
    auto next_item = [&](int n) -> const Item* {
        if (!mbar_wait(&sm.item_full[n % kItems], (n / kItems) & 1, wc)) return nullptr;
        const Item* it = &sm.item[n % kItems];
        return it->tiles ? it : nullptr;
    };
    auto done_with = [&](int n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.item_empty[n % kItems]);
    };
    // Query rows row, row + step, ... of warpgroup w's tile: `at` is the row's element offset in q (and in the
    // window's output), -1 past the end
    struct Rows {
        int64_t at0;
        int left, g, G, stride;
        __device__ __forceinline__ int64_t at() const { return left > 0 ? at0 : -1; }
        __device__ __forceinline__ void next(int step) {
            left -= step;
            if (kPrefix) {              // row b G + g: head g of sequence b
                at0 += step * HD;
                for (g += step; g >= G; g -= G) at0 += stride;
            } else {
                at0 += (int64_t)step * stride;
            }
        }
    };
    auto rows_from = [&](const Item& it, int w, int row) -> Rows {
        if (kPrefix) {
            const int b = row / G, g = row - b * G;
            return Rows{((int64_t)b * p.H + it.hk * G + g) * HD, it.n_rows - row, g, G, (p.H - G) * HD};
        }
        return Rows{((it.q_beg + row) * p.H + it.head[w]) * HD, it.n_rows - row, 0, 1, p.H * HD};
    };
    // prefix: a warp copies query rows r0 .. r0 + n - 1 of a tile into its swizzled place, whole rows at a time
    auto load_q = [&](const Item& it, int w, int r0, int n) {
        constexpr int kAtOnce = 32 / QC;
        const int cc = lane % QC, rr = lane / QC;
        const uint32_t dst = smem_u32(sm.q[w]) + (cc >> 3) * kSub;
        Rows rows = rows_from(it, w, it.row0[w] + r0 + rr);
        if constexpr (!(E4 && std::is_same<T, __nv_bfloat16>::value)) {
#pragma unroll 8
            for (int i = 0; i < n; i += kAtOnce) {
                const int r = r0 + i + rr;
                const int64_t at = rows.at();
                cp16(dst + r * 128 + (((cc & 7) ^ (r & 7)) << 4), (const T*)p.q + (at >= 0 ? at : 0) + cc * 8, at >= 0 ? 16 : 0);
                rows.next(kAtOnce);
            }
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
        } else {
            // bf16 queries over e4m3 rows are multiplied as fp16, after a power of two that brings the row to [1, 2):
            // nothing overflows, and what is lost is below 2^-24 of its largest entry
#pragma unroll 4
            for (int i = 0; i < n; i += kAtOnce) {
                const int r = r0 + i + rr;
                const int64_t at = rows.at();
                const uint4 x = at >= 0 ? *reinterpret_cast<const uint4*>((const T*)p.q + at + cc * 8) : make_uint4(0, 0, 0, 0);
                rows.next(kAtOnce);
                const uint32_t wd[4] = {x.x, x.y, x.z, x.w};
                float f[8], top = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    unpack2(wd[e], T(), f[2 * e], f[2 * e + 1]);
                    top = fmaxf(top, fmaxf(fabsf(f[2 * e]), fabsf(f[2 * e + 1])));
                }
                top = group_max<QC>(top);
                int ex = 0;
                if (top > 1e-30f && top < 1e30f) ex = ((__float_as_int(top) >> 23) & 255) - 127;
                const float mul = __int_as_float((127 - ex) << 23);
                if (cc == 0) sm.row_exp[w][r] = (signed char)ex;
                st_shared16(dst + r * 128 + (((cc & 7) ^ (r & 7)) << 4), pack2<__half>(f[0] * mul, f[1] * mul), pack2<__half>(f[2] * mul, f[3] * mul),
                            pack2<__half>(f[4] * mul, f[5] * mul), pack2<__half>(f[6] * mul, f[7] * mul));
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&sm.q_full[w]);
    };

    // Slots of an item's tiles, four rows from `r0` of a tile per lane, fetched ahead of their use
    struct Slots {
        const int32_t* table;
        int w0, tiles, sinks, skip, n_slots;
        __device__ __forceinline__ Slots(const AttendParams& p, const Item& it)
            : table(p.table + it.beg), w0(it.w0), tiles(it.tiles), sinks(it.sinks), skip(it.first - it.sinks), n_slots((int)p.n_slots) {}
        __device__ __forceinline__ void fetch(int j, int r0, int (&x)[4]) const {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = r0 + i, u = tile_base(w0, j) + r;
                x[i] = j < tiles && r < BN && r < tile_keys(w0, j) ? __ldg(table + (u < sinks ? u : u + skip)) : -1;
            }
        }
    };
    // Slots -> rows to gather; `mark`: notes which rows of the tile (the CTA's t-th) there are none for, a word per eight
    // lanes.  bad[t & 7] is read until the tile's P is there; the MMA thread waits for that before it issues anything of
    // four tiles later, and so before the release that lets a tile into this place again.
    auto to_rows = [&](const Slots& sl, int j, int t, int r0, const int (&x)[4], int (&row)[4], bool mark) {
        uint32_t none = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = x[i] >= 0 && x[i] < sl.n_slots;
            none |= in ? 0u : 1u << i;
            row[i] = in ? x[i] : sl.n_slots;
        }
        if (mark) {
            const int keys = tile_keys(sl.w0, j) - r0;                    // those of the four that are keys at all
            const bool bad = none & (keys >= 4 ? 15u : keys <= 0 ? 0u : (1u << keys) - 1u);
            none <<= (r0 & 31);
            none |= __shfl_xor_sync(0xffffffffu, none, 1);
            none |= __shfl_xor_sync(0xffffffffu, none, 2);
            none |= __shfl_xor_sync(0xffffffffu, none, 4);
            if ((lane & 7) == 0 && (E4 || lane == 0)) sm.bad[t & 7][r0 >> 5] = none;
            if (bad) {
                sm.any_bad = 1;
                if (p.err_flag) atomicOr(p.err_flag, ATTN_B200_FLAG_BAD_SLOT);
            }
        }
    };

    if (E4 && warp >= 12) {
        // ------------------------------------------------------------------ e4m3 rows: 64 threads K, 64 threads V
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::kGather));
        constexpr int CPR = HD / 16, RPP = 64 / CPR, PASSES = BN / RPP;     // 16-byte chunks of a raw row; rows per pass of 64 threads
        const int v = warp >= 14, t64 = threadIdx.x & 63;
        const bool fetches = (warp & 1) == 0;                               // the stream's first warp gathers
        const int c = t64 % CPR, rsub = t64 / CPR;
        unsigned long long* full = v ? sm.v_full : sm.k_full;
        unsigned long long* empty = v ? sm.v_empty : sm.k_empty;
        const CUtensorMap* const map = v ? &map_v : &map_k;
        const uint32_t raw = smem_u32(sm.extra[v]);
        int issued = 0;
        if (const Item* const ip = next_item(0)) {                          // prefix only: one item
            const Slots sl(p, *ip);
            const int tiles = sl.tiles, x0 = ip->hk * HD;
            int ahead[4], cur[4];
            auto gather = [&](int j) {                                      // raw rows of tile j, whose slots are in `ahead`
                to_rows(sl, j, j, lane * 4, ahead, cur, false);
                if (lane == 0) mbar_expect_tx(&sm.raw_full[v], BN * HD);
                __syncwarp();
                tma_gather4(raw + lane * 4 * HD, map, x0, cur, &sm.raw_full[v]);
                ++issued;
            };
            if (fetches) {
                sl.fetch(0, lane * 4, ahead);
                gather(0);
            }
            for (int j = 0; j < tiles; ++j) {
                const int s = j % kStages;
                int mine[4] = {ahead[0], ahead[1], ahead[2], ahead[3]};
                if (fetches) sl.fetch(j + 1, lane * 4, ahead);
                bool ok = mbar_wait(&sm.raw_full[v], j & 1, wc);
                if (ok && j >= kStages) ok = mbar_wait(&empty[s], ((j - kStages) / kStages) & 1, wc);
                if (!__all_sync(0xffffffffu, ok)) break;
                if (fetches) to_rows(sl, j, j, lane * 4, mine, cur, !v);
                // 16 codes -> chunks 2 c and 2 c + 1 of the row in fp16
                const uint32_t dst = smem_u32(v ? sm.v[s] : sm.k[s]) + (c >> 2) * kSub;
#pragma unroll 4
                for (int q = 0; q < PASSES; ++q) {
                    const int r = q * RPP + rsub;
                    const uint4 x = ld_shared16(raw + r * HD + c * 16);
                    __half2 h[8];
                    e4m3x4_to_half2x2(x.x, h[0], h[1]);
                    e4m3x4_to_half2x2(x.y, h[2], h[3]);
                    e4m3x4_to_half2x2(x.z, h[4], h[5]);
                    e4m3x4_to_half2x2(x.w, h[6], h[7]);
                    const uint32_t* u = reinterpret_cast<const uint32_t*>(h);
                    const uint32_t at = dst + r * 128;
                    st_shared16(at + ((((2 * c) & 7) ^ (r & 7)) << 4), u[0], u[1], u[2], u[3]);
                    st_shared16(at + ((((2 * c + 1) & 7) ^ (r & 7)) << 4), u[4], u[5], u[6], u[7]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&full[s]);
                mbar_arrive(&sm.raw_empty[v]);
                if (fetches && j + 1 < tiles) {            // the next raw rows travel while this tile is in use
                    if (!__all_sync(0xffffffffu, mbar_wait(&sm.raw_empty[v], j & 1, wc))) break;
                    gather(j + 1);
                }
            }
            done_with(0);
        }
        if (fetches && lane == 0 && sm.box.abort && issued > 0) {      // a copy still in flight gets a bounded time to land
            const long long t0 = clock64();
            while (!mbar_try(&sm.raw_full[v], (issued - 1) & 1) && clock64() - t0 < WAIT_CYCLES) {}
        }
    } else if (!E4 && warp >= 12) {
        // ------------------------------------------------------------------ K and V rows 32 (warp - 12) .. + 31 of every tile
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::kGather));
        const int r0 = (warp - 12) * 32 + (lane & 7) * 4;                   // lanes 0-7 gather, four rows each
        const uint32_t at = r0 * 128;
        int g = 0, issued_k = 0, issued_v = 0;
        bool ok = true;
        for (int n = 0; ok; ++n) {
            const Item* const ip = next_item(n);
            if (__any_sync(0xffffffffu, !ip)) break;
            const Slots sl(p, *ip);
            const int x0 = ip->hk * HD, tiles = sl.tiles;
            int ahead[4];
            sl.fetch(0, r0, ahead);
            for (int j = 0; j < tiles; ++j) {
                const int t = g + j, s = t % kStages;
                const uint32_t ph = ((t - kStages) / kStages) & 1;
                int row[4], cur[4] = {ahead[0], ahead[1], ahead[2], ahead[3]};
                sl.fetch(j + 1, r0, ahead);
                if (t >= kStages) ok = mbar_wait(&sm.k_empty[s], ph, wc);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                to_rows(sl, j, t, r0, cur, row, true);
                __syncwarp();                           // the notes of all lanes stand before lane 0 arrives
                if (lane == 0) mbar_expect_tx(&sm.k_full[s], kTileBytes / 4);
                __syncwarp();
                if (lane < 8) {
#pragma unroll
                    for (int c = 0; c < HD / 64; ++c) tma_gather4(smem_u32(sm.k[s]) + at + c * kSub, &map_k, x0 + c * 64, row, &sm.k_full[s]);
                }
                ++issued_k;
                __syncwarp();
                if (t >= kStages) ok = mbar_wait(&sm.v_empty[s], ph, wc);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                if (lane == 0) mbar_expect_tx(&sm.v_full[s], kTileBytes / 4);
                __syncwarp();
                if (lane < 8) {
#pragma unroll
                    for (int c = 0; c < HD / 64; ++c) tma_gather4(smem_u32(sm.v[s]) + at + c * kSub, &map_v, x0 + c * 64, row, &sm.v_full[s]);
                }
                ++issued_v;
                __syncwarp();
            }
            if (!ok) break;
            g += tiles;
            done_with(n);
        }
        if (lane == 0 && sm.box.abort) {                 // copies still in flight get a bounded time to land
            const long long t0 = clock64();
            for (int t = issued_k > kStages ? issued_k - kStages : 0; t < issued_k; ++t)
                while (!mbar_try(&sm.k_full[t % kStages], (t / kStages) & 1) && clock64() - t0 < WAIT_CYCLES) {}
            for (int t = issued_v > kStages ? issued_v - kStages : 0; t < issued_v; ++t)
                while (!mbar_try(&sm.v_full[t % kStages], (t / kStages) & 1) && clock64() - t0 < WAIT_CYCLES) {}
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::kOther));
        if (warp == 8) {
            // -------------------------------------------------------------- item list
            // The items of a window launch are the existing blocks of all sequences times the head units, the unit changing
            // fastest (its CTAs share K and V); this CTA takes every gridDim.x-th.  The warp looks at 32 sequences at a
            // time, once each, so empty and short chunks cost next to nothing.
            int base = 0, mine = 0, upto = 0, before = 0;       // sequences base .. base + 31: blocks of lane's, scan of them, blocks ahead of base
            auto look = [&] {
                mine = max(window_blocks(p, base + lane), 0);
                upto = mine;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= d) upto += x;
                }
            };
            if (!kPrefix) look();
            for (int n = 0;; ++n) {
                bool end = kPrefix && n > 0;
                int b = 0, blk = 0, unit = 0;
                if (!kPrefix) {
                    const int64_t id = blockIdx.x + (int64_t)n * gridDim.x, block = id / p.units;
                    unit = (int)(id - block * p.units);
                    while (!end && block >= before + (int64_t)__shfl_sync(0xffffffffu, upto, 31)) {
                        before += __shfl_sync(0xffffffffu, upto, 31);
                        base += 32;
                        if (base >= p.B) end = true;
                        else look();
                    }
                    if (!end) {
                        const int in = (int)(block - before);
                        const int src = __ffs(__ballot_sync(0xffffffffu, upto > in)) - 1;
                        b = base + src;
                        blk = in - __shfl_sync(0xffffffffu, upto - mine, src);
                    }
                }
                bool ok = n < kItems || mbar_wait(&sm.item_empty[n % kItems], (n / kItems - 1) & 1, wc);
                if (!__all_sync(0xffffffffu, ok)) break;
                if (lane == 0) {
                    Item& it = sm.item[n % kItems];
                    if (end) it.tiles = 0;
                    else if (!kPrefix) window_item(p, b, blk, unit, it);       // (a prefix CTA's is there)
                    mbar_arrive(&sm.item_full[n % kItems]);
                }
                if (end) break;
            }
        } else if (warp == 9) {
            // -------------------------------------------------------------- MMA issuer
            constexpr uint32_t fmt = std::is_same<MT, __nv_bfloat16>::value ? 1u : 0u;
            constexpr uint32_t idesc0 = (1u << 4) | (fmt << 7) | (fmt << 10) | ((BM >> 4) << 24);
            constexpr uint32_t idesc_pv = idesc0 | (1u << 16) | ((HD >> 3) << 17);
            if (elect_one()) {
                const uint64_t qd = smem_desc(smem_u32(sm.q[0]), 16, 1024), kd = smem_desc(smem_u32(sm.k[0]), 16, 1024);
                const uint64_t vd = smem_desc(smem_u32(sm.v[0]), kSub, 1024);
                constexpr uint64_t kTile16 = kTileBytes >> 4;
                int g = 0;                       // tiles of earlier items
                int done0 = 0, done1 = 0;        // tiles of each warpgroup whose P.V has been issued
                int uses0 = 0, uses1 = 0;        // items in which it had work
                // W: the warpgroup, a compile-time 0 or 1, so that all of this stays in registers
                auto start_tile = [&](auto W, int t, int wide) -> bool {                  // Q.K of tile t (of the CTA)
                    constexpr int w = decltype(W)::value;
                    if (!mbar_wait(&sm.k_full[t % kStages], (t / kStages) & 1, wc)) return false;
                    tc_fence_after();
                    const uint64_t a = qd + (w ? (key_split ? 0 : kTile16) : 0), b2 = kd + (t % kStages) * kTile16;
                    const uint32_t idesc = idesc0 | ((uint32_t)(wide >> 3) << 17);
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const uint32_t off16 = ((kk >> 2) * kSub + (kk & 3) * 32) >> 4;
                        umma_f16(tmem + w * 128, a + off16, b2 + off16, idesc, kk > 0);
                    }
                    umma_commit(&sm.s_full[w]);
                    return true;
                };
                auto finish_tile = [&](auto W, int t, int wide, bool first) -> bool {     // P.V of tile t
                    constexpr int w = decltype(W)::value;
                    int& done = w ? done1 : done0;
                    const uint32_t ph = done & 1;
                    ++done;
                    const uint64_t v = vd + (t % kStages) * kTile16;
                    const uint32_t d = tmem + 256 + w * 128, a = tmem + w * 128;
                    if (first && (w ? uses1 : uses0) > 0 && !mbar_wait(&sm.o_free[w], ((w ? uses1 : uses0) - 1) & 1, wc)) return false;
                    if (!mbar_wait(&sm.p_half[w], ph, wc)) return false;
                    if (!mbar_wait(&sm.v_full[t % kStages], (t / kStages) & 1, wc)) return false;
                    tc_fence_after();
                    if (wide == BN) {
#pragma unroll
                        for (int kk = 0; kk < BN / 32; ++kk) umma_f16_ts(d, a + kk * 8, v + ((kk * 2048) >> 4), idesc_pv, (!first || kk > 0) ? 1u : 0u);
                        if (!mbar_wait(&sm.p_full[w], ph, wc)) return false;
                        tc_fence_after();
#pragma unroll
                        for (int kk = BN / 32; kk < BN / 16; ++kk) umma_f16_ts(d, a + kk * 8, v + ((kk * 2048) >> 4), idesc_pv, 1u);
                    } else {
                        if (!mbar_wait(&sm.p_full[w], ph, wc)) return false;
                        tc_fence_after();
#pragma unroll 1
                        for (int kk = 0; kk < wide / 16; ++kk)
                            umma_f16_ts(d, a + kk * 8, v + (uint64_t)(kk * (2048 >> 4)), idesc_pv, (!first || kk > 0) ? 1u : 0u);
                    }
                    umma_commit(&sm.o_full[w]);
                    return true;
                };
                const std::integral_constant<int, 0> W0{};
                const std::integral_constant<int, 1> W1{};
                for (int n = 0;; ++n) {
                    const Item* const ip = next_item(n);
                    if (!ip) break;
                    const int tiles = ip->tiles, jb0 = ip->jb[0], jb1 = ip->jb[1], je0 = ip->je[0], je1 = ip->je[1];
                    // columns that a tile is multiplied in: whole, or its keys rounded up to 32
                    const int wide0 = ip->w0 > 96 ? BN : (ip->w0 + 31) / 32 * 32;
                    auto wide = [&](int j) { return j ? BN : wide0; };
                    bool ok = mbar_wait(&sm.q_full[0], uses0 & 1, wc);        // the first query tile always has rows
                    if (key_split) {
                        if (ok) ok = start_tile(W0, 0, wide0);
                        umma_commit(&sm.k_empty[0]);
                        if (ok && tiles > 1) {
                            ok = start_tile(W1, 1, BN);
                            umma_commit(&sm.k_empty[1]);
                        }
                        for (int j = 0; ok && j < tiles; j += 2) {
                            if (!(ok = finish_tile(W0, j, wide(j), j == 0))) break;
                            umma_commit(&sm.v_empty[j % kStages]);
                            if (j + 2 < tiles) {
                                if (!(ok = start_tile(W0, j + 2, BN))) break;
                                umma_commit(&sm.k_empty[(j + 2) % kStages]);
                            }
                            if (j + 1 == tiles) break;
                            if (!(ok = finish_tile(W1, j + 1, BN, j == 0))) break;
                            umma_commit(&sm.v_empty[(j + 1) % kStages]);
                            if (j + 3 < tiles) {
                                if (!(ok = start_tile(W1, j + 3, BN))) break;
                                umma_commit(&sm.k_empty[(j + 3) % kStages]);
                            }
                        }
                    } else {
                        if (ok && je1 > jb1) ok = mbar_wait(&sm.q_full[1], uses1 & 1, wc);
                        // every tile is some warpgroup's: the list is the union of two overlapping stretches
                        if (ok && jb0 == 0) ok = start_tile(W0, g, wide0);
                        if (ok && je0 == 1) umma_commit(&sm.q_empty[0]);
                        if (ok && jb1 == 0 && je1 > 0) {
                            ok = start_tile(W1, g, wide0);
                            if (je1 == 1) umma_commit(&sm.q_empty[1]);
                        }
                        umma_commit(&sm.k_empty[g % kStages]);
                        for (int j = 0; ok && j < tiles; ++j) {
                            const int t = g + j;
                            if (j >= jb0 && j < je0 && !(ok = finish_tile(W0, t, wide(j), j == jb0))) break;
                            if (j + 1 >= jb0 && j + 1 < je0) {
                                if (!(ok = start_tile(W0, t + 1, BN))) break;
                                if (j + 2 == je0) umma_commit(&sm.q_empty[0]);
                            }
                            if (j >= jb1 && j < je1 && !(ok = finish_tile(W1, t, wide(j), j == jb1))) break;
                            umma_commit(&sm.v_empty[t % kStages]);
                            if (j + 1 >= jb1 && j + 1 < je1) {
                                if (!(ok = start_tile(W1, t + 1, BN))) break;
                                if (j + 2 == je1) umma_commit(&sm.q_empty[1]);
                            }
                            if (j + 1 < tiles) umma_commit(&sm.k_empty[(t + 1) % kStages]);
                        }
                    }
                    if (!ok) break;
                    uses0 += je0 > jb0;
                    uses1 += je1 > jb1;
                    g += tiles;
                    mbar_arrive(&sm.item_empty[n % kItems]);
                }
            }
            __syncwarp();
        } else if (!kPrefix && warp == 11) {
            // -------------------------------------------------------------- rows that no query tile writes: zeros
            // past the last sequence, beyond max_q_len, or of a sequence whose offsets are bad; every CTA takes a share
            const int64_t vecs = (int64_t)p.H * HD / 8;
            auto zero = [&](int64_t from, int64_t to) {
                from = from < 0 ? 0 : from;
                to = to > p.n_q_tokens ? p.n_q_tokens : to;
                for (int64_t row = from + blockIdx.x; row < to; row += gridDim.x) {
                    uint4* const dst = reinterpret_cast<uint4*>((T*)p.out + row * p.H * HD);
                    for (int64_t i = lane; i < vecs; i += 32) dst[i] = make_uint4(0, 0, 0, 0);
                }
            };
            const int64_t covered = (int64_t)p.blocks * (p.head_pairs ? BM : 2 * BM);
            for (int base = 0; base < p.B; base += 32) {
                const int b = base + lane;
                int64_t from = 0, to = 0;
                if (b < p.B) {
                    from = b ? p.q_offsets[b - 1] : 0;
                    to = p.q_offsets[b];
                    if (window_blocks(p, b) >= 0) {
                        if (to - from > covered && p.err_flag) atomicOr(p.err_flag, ATTN_B200_FLAG_BAD_OFFSETS);
                        from += covered;
                    }
                }
                for (unsigned todo = __ballot_sync(0xffffffffu, to > from); todo; todo &= todo - 1) {
                    const int src = __ffs(todo) - 1;
                    zero(__shfl_sync(0xffffffffu, from, src), __shfl_sync(0xffffffffu, to, src));
                }
            }
            const int64_t end = p.B ? p.q_offsets[p.B - 1] : 0;
            zero(end, p.n_q_tokens);
        } else if (!kPrefix && warp == 10) {
            // -------------------------------------------------------------- query tiles
            int uses[2] = {0, 0};
            bool ok = true;
            for (int n = 0; ok; ++n) {
                const Item* const ip = next_item(n);
                if (__any_sync(0xffffffffu, !ip)) break;
                const Item& it = *ip;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (!ok || !active(it, w)) continue;
                    ok = uses[w] == 0 || mbar_wait(&sm.q_empty[w], (uses[w] - 1) & 1, wc);
                    if (!(ok = __all_sync(0xffffffffu, ok))) continue;
                    ++uses[w];
                    if (lane == 0) {
                        // rows past the chunk's end are another sequence's (or zeros past the tensor): computed, not stored
                        mbar_expect_tx(&sm.q_full[w], kTileBytes);
#pragma unroll
                        for (int c = 0; c < HD / 64; ++c)
                            tma_load_2d(sm.q[w] + c * kSub, &map_q, it.head[w] * HD + c * 64, (int)(it.q_beg + it.row0[w]), &sm.q_full[w]);
                    }
                    __syncwarp();
                }
                if (ok) done_with(n);
            }
            if (lane == 0 && sm.box.abort) {
                const long long t0 = clock64();
                for (int w = 0; w < 2; ++w)
                    if (uses[w] > 0) while (!mbar_try(&sm.q_full[w], (uses[w] - 1) & 1) && clock64() - t0 < WAIT_CYCLES) {}
            }
        }
    } else {
        // ------------------------------------------------------------------ softmax warpgroups
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R::kSoftmax));
        const int w = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_addr = lane_base + w * 128, o_addr = lane_base + 256 + w * 128;
        constexpr int step = key_split ? 2 : 1;
        int c0 = 0, g = 0;
        for (int n = 0;; ++n) {
            const Item* const ip = next_item(n);
            if (__any_sync(0xffffffffu, !ip)) break;
            const Item& it = *ip;
            const int count = active(it, w) ? (it.je[w] - it.jb[w] + step - 1) / step : 0;
            const int row = it.row0[w] + r;
            int hi = INT_MAX, lo = 0, ns = 0;
            if (!kPrefix) {
                hi = it.shift + row - it.first + it.sinks;
                const int64_t lo64 = (int64_t)hi - p.window + 1;
                lo = lo64 > 0 ? (int)lo64 : 0;
                ns = p.sinks;
            }
            // a prefix CTA has one item, whose queries the softmax warps fetch themselves
            if (kPrefix && count > 0 && !(key_split && w == 1)) load_q(it, w, (warp & 3) * 32, 32);
            float scale = p.scale_log2, m = -INFINITY, l = 0.f;
            if (kPrefix && E4) {
                scale *= p.k_scale[it.hk];
                if (std::is_same<T, __nv_bfloat16>::value && count > 0) {
                    // the row's power of two is there when its first scores are
                    if (!__all_sync(0xffffffffu, mbar_wait(&sm.s_full[w], c0 & 1, wc))) break;
                    scale *= __int_as_float((127 + sm.row_exp[key_split ? 0 : w][r]) << 23);
                }
            }
            if (count > 0 && !__all_sync(0xffffffffu, softmax_rows<MT, HD>(
                                                          sm, w, s_addr, o_addr, it.w0, it.jb[w], step, count, c0, g, hi, lo, ns, scale, m, l)))
                break;
            c0 += count;
            g += it.tiles;
            // The accumulator goes to registers, from there through shared memory (a warp its own rows, 16-byte
            // chunks swizzled by the row) and leaves in whole rows: written straight from registers every
            // store instruction touches 32 rows.
            const int lr = lane, row_w = it.row0[w] + (warp & 3) * 32;       // this warp's first row
            if (kPrefix) {
                // Partial rows lie by KV head, [n_parts, Hkv, B * G, HD], so that a warp's 32 rows are one box of a TMA
                // store per 32 columns.  Staged where this warpgroup's last K tile (its query tile) was.
                const float vs = E4 ? p.v_scale[it.hk] : 1.f;
                const int64_t rows_all = (int64_t)p.B * p.H, part = it.part + (key_split ? w : 0);
                const int64_t row0 = part * rows_all + (int64_t)it.hk * it.n_rows;        // first row of the KV head's block
                const int last = it.tiles - 1 - ((it.tiles - 1 + w) & 1);                 // key_split: this warpgroup's last tile, or -1
                unsigned char* const stage = (key_split ? sm.k[(last + kStages) % kStages] : sm.q[key_split ? 0 : w]) + (warp & 3) * (kTileBytes / 4);
                constexpr int kBoxes = kTileBytes / 4 / 4096;                             // boxes that fit the warp's share
                const bool box = row_w + 32 <= it.n_rows;
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    const uint32_t buf = smem_u32(stage) + (c / 32 % kBoxes) * 4096;
                    if (c >= 32 * kBoxes) {
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kBoxes - 1) : "memory");
                        __syncwarp();
                    }
                    float ov[32];
                    if (count > 0) {
                        tmem_ld32(o_addr + c, ov);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) ov[e] = 0.f;
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        st_shared16(buf + lr * 128 + ((e ^ (lr & 7)) << 4), __float_as_uint(ov[4 * e] * vs), __float_as_uint(ov[4 * e + 1] * vs),
                                    __float_as_uint(ov[4 * e + 2] * vs), __float_as_uint(ov[4 * e + 3] * vs));
                    if (box) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (box) {
                        if (lane == 0) {
                            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                                         ::"l"(reinterpret_cast<uint64_t>(&map_o)), "r"(c), "r"((int)(row0 + row_w)), "r"(buf) : "memory");
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                    } else {
#pragma unroll 1
                        for (int i = lane / 8; i < 32 && row_w + i < it.n_rows; i += 4)
                            *reinterpret_cast<uint4*>(p.parts + (row0 + row_w + i) * HD + c + lane % 8 * 4) =
                                ld_shared16(buf + i * 128 + ((lane % 8 ^ (i & 7)) << 4));
                        __syncwarp();
                    }
                }
                float2* const ml = reinterpret_cast<float2*>(p.parts + (int64_t)attend_prefix_parts(p) * rows_all * HD);
                if (row < it.n_rows) ml[row0 + row] = make_float2(count > 0 ? m : -INFINITY, l);
            } else if (count > 0) {
                // a row none of whose keys has a pool row is zero
                const float inv = m > -INFINITY || l != l ? 1.f / l : 0.f;
                // A warp's 4 KB of staging hold 64 columns of its 32 rows in the 128-byte-swizzled layout of a TMA box; one
                // lane stores the box, or, where the chunk ends inside it, the lanes copy the rows that exist.
                unsigned char* const stage = sm.extra[w] + (warp & 3) * 4096;
                const uint32_t mine = smem_u32(stage) + lr * 128;
                const bool box = row_w + 32 <= it.n_rows;
                float probe = 0.f, probe2 = 0.f;    // turn into a NaN where an entry is not finite
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    float ov[32];
                    tmem_ld32(o_addr + c, ov);
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        fma2(probe, probe2, ov[e], ov[e + 1], 0.f, 0.f, probe, probe2);
                        fma2(ov[e], ov[e + 1], ov[e], ov[e + 1], inv, inv, -0.f, -0.f);
                    }
                    if (c + 32 == HD) {             // the next item may overwrite the accumulator
                        tc_fence_before();
                        mbar_arrive(&sm.o_free[w]);
                    }
                    if (c % 64 == 0) {              // the store before has read the buffer
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        __syncwarp();
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        st_shared16(mine + (((e + c / 8 % 8) ^ (lr & 7)) << 4), pack2<T>(ov[8 * e], ov[8 * e + 1]),
                                    pack2<T>(ov[8 * e + 2], ov[8 * e + 3]), pack2<T>(ov[8 * e + 4], ov[8 * e + 5]),
                                    pack2<T>(ov[8 * e + 6], ov[8 * e + 7]));
                    if (c % 64 == 0) continue;
                    if (box) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) {
                            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                                         ::"l"(reinterpret_cast<uint64_t>(&map_o)), "r"(it.head[w] * HD + c - 32), "r"((int)(it.q_beg + row_w)),
                                           "r"(smem_u32(stage)) : "memory");
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                    } else {
                        __syncwarp();
                        Rows rows = rows_from(it, w, row_w + lane / 8);
                        T* const dst = (T*)p.out + c - 32 + lane % 8 * 8;
#pragma unroll 1
                        for (int i = 0; i < 32; i += 4) {
                            const int rr = i + lane / 8, cc = lane % 8;
                            const uint4 x = ld_shared16(smem_u32(stage) + rr * 128 + ((cc ^ (rr & 7)) << 4));
                            const int64_t at = rows.at();
                            if (at >= 0) *reinterpret_cast<uint4*>(dst + at) = x;
                            rows.next(4);
                        }
                        __syncwarp();
                    }
                }
                unsigned odd = __ballot_sync(0xffffffffu, probe + probe2 != 0.f && row < it.n_rows);
                if (odd) {
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");       // the box is written first
                    __syncwarp();
                    for (; odd; odd &= odd - 1) row_by_itself<T, HD>(p, it, it.head[w], row_w + __ffs(odd) - 1);
                }
            }
            done_with(n);
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");           // the stores are done before the CTA is
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// Launch as a programmatic dependent: the kernels wait (griddepcontrol.wait) before they read anything.
template <typename... K, typename... A>
int launch_dependent(void (*kernel)(K...), dim3 grid, int threads, int smem, cudaStream_t st, const A&... args) {
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


typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<EncodeTiled>(f) : nullptr;
    }();
    return fn;
}
// [rows, cols] row-major; boxes of `width` elements x `height` rows
int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int elem_bytes, int width, int height, bool swizzle) {
    const EncodeTiled fn = encoder();
    if (!fn) return (int)cudaErrorNotSupported;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(cols * elem_bytes)};
    const cuuint32_t box[2] = {(cuuint32_t)width, (cuuint32_t)height}, step[2] = {1, 1};
    // the copies move bits: every 16-bit type is taken as fp16
    const CUtensorMapDataType type = elem_bytes == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : elem_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    const CUresult r = fn(map, type, 2, const_cast<void*>(base), dims,
                          strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

template <typename T, int HD, int kMode, bool E4>
int launch(const AttendParams& p, dim3 grid, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    constexpr int smem = (int)sizeof(Smem<HD, kMode, E4>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory");
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 64) return ATTN_B200_ETOOLARGE;
    if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
        if ((e = cudaFuncSetAttribute(attend_tc_kernel<T, HD, kMode, E4>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess)
            return (int)e;
        ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    CUtensorMap mq, mk, mv, mo;
    const int64_t cols = (int64_t)p.Hkv * HD;
    int rc;
    if ((rc = make_map(&mk, p.k_cache, p.n_slots, cols, E4 ? 1 : 2, E4 ? HD : 64, 1, !E4)) ||
        (rc = make_map(&mv, p.v_cache, p.n_slots, cols, E4 ? 1 : 2, E4 ? HD : 64, 1, !E4)))
        return rc;
    if (kMode == kWindow) {
        if ((rc = make_map(&mq, p.q, p.n_q_tokens, (int64_t)p.H * HD, 2, 64, BM, true)) ||
            (rc = make_map(&mo, p.out, p.n_q_tokens, (int64_t)p.H * HD, 2, 64, 32, true)))
            return rc;
    } else {
        mq = mk;               // not used
        const int64_t rows = (int64_t)attend_prefix_parts(p) * p.B * p.H;
        if (rows > 0x7fffffffLL) return ATTN_B200_ETOOLARGE;
        if ((rc = make_map(&mo, p.parts, rows, HD, 4, 32, 32, true))) return rc;
    }
    return launch_dependent(attend_tc_kernel<T, HD, kMode, E4>, grid, kThreads, smem, st, mq, mk, mv, mo, p);
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
    p.blocks = blocks;
    p.units = units;
    // one CTA per SM, no more than there can be items
    const int64_t most = (p.n_q_tokens / rows + p.B) * units, sms = current_sm_count();
    const dim3 grid((unsigned)(most < 1 ? 1 : most < sms ? most : sms));
    const bool bf = dtype == ATTN_B200_BF16;
    if (D == 64) return bf ? launch<__nv_bfloat16, 64, kWindow, false>(p, grid, st) : launch<__half, 64, kWindow, false>(p, grid, st);
    return bf ? launch<__nv_bfloat16, 128, kWindow, false>(p, grid, st) : launch<__half, 128, kWindow, false>(p, grid, st);
}

void attend_prefix_plan(AttendParams& p) {
    const int64_t rows = (int64_t)p.B * (p.H / p.Hkv);
    p.key_split = rows <= BM;
    const int64_t groups = p.key_split ? 1 : (rows + 2 * BM - 1) / (2 * BM), items = groups * p.Hkv;
    const int tiles = (p.n_prefix + BN - 1) / BN;
    // one CTA per SM: the number of splits with the fewest tile steps in the longest chain; a wave costs
    // about three steps besides (set-up, first rows, partial rows)
    const int sms = current_sm_count();
    int64_t best = -1;
    p.splits = 1;
    for (int s = 1; s <= sms && s <= tiles; ++s) {
        const int64_t cost = (items * s + sms - 1) / sms * ((tiles + s - 1) / s + 3);
        if (best < 0 || cost < best) {
            best = cost;
            p.splits = s;
        }
    }
}

int attend_prefix_launch(const AttendParams& p, int D, int dtype, bool e4, cudaStream_t st) {
    const int64_t rows = (int64_t)p.B * (p.H / p.Hkv);
    const int64_t groups = p.key_split ? 1 : (rows + 2 * BM - 1) / (2 * BM);
    if (p.splits * p.Hkv * groups > 0x7fffffffLL) return ATTN_B200_ETOOLARGE;
    const dim3 grid((unsigned)(p.splits * p.Hkv * groups));
    auto go = [&](auto hd, auto mode, auto e) -> int {
        constexpr int HD = decltype(hd)::value, M = decltype(mode)::value;
        constexpr bool E = decltype(e)::value;
        return dtype == ATTN_B200_BF16 ? launch<__nv_bfloat16, HD, M, E>(p, grid, st) : launch<__half, HD, M, E>(p, grid, st);
    };
    auto with_mode = [&](auto hd, auto mode) { return e4 ? go(hd, mode, std::true_type{}) : go(hd, mode, std::false_type{}); };
    auto with_dim = [&](auto hd) {
        return p.key_split ? with_mode(hd, std::integral_constant<int, kPrefixSplit>{}) : with_mode(hd, std::integral_constant<int, kPrefixPair>{});
    };
    return D == 64 ? with_dim(std::integral_constant<int, 64>{}) : with_dim(std::integral_constant<int, 128>{});
}

}  // namespace attn
