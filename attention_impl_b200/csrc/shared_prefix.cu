// Decode of a batch whose sequences share one long prefix.  Not in the reference; without sharing it is
// paged_attention_kernel.cu:100-187.
//
//   o_b = softmax over (prefix rows, own rows of b, the current token) of scale <q_b, k>, applied to v
//
// Two ways.  Together, two launches: attend_tc.cu multiplies the whole batch's query rows of a KV head with the prefix, so its rows
// travel once instead of B times, and leaves partial rows [o, m, l] per split of the keys.
// span_decode.cu walks every sequence's own rows and folds the prefix's partials and the current token in.
// The second kernel is a programmatic dependent of the first and needs only its partial rows from it: it walks
// the own rows as soon as the first kernel's CTAs leave room.  Per sequence, one launch: span_decode.cu visits the
// prefix's rows before the own ones, for every sequence again (out of L2 mostly).
//
// Measured (D = 128, 1 to 64 sequences, 32 KV heads / 8 / 1, 96 to 8192 rows, 16-bit and e4m3 pools): the second launch and
// the fold of partial rows cost 6 to 8 us, so one launch wins while the prefix's bytes times the batch stay below
// about 48 MB (4 x 2048 rows of 8 heads in fp16, 34 MB: 13.8 us against 16.5; 4 x 768 of 32 heads, 50 MB: 14.0 and 13.8;
// 16 x 256 of 32 heads, 67 MB: 19.3 and 18.7; 64 x 2048 of 8 heads, 537 MB: 81 and 24), and always for one sequence
// (8192 rows of 32 heads: 36.8 against 42.9).
#include "attend_tc.cuh"
#include "span_decode.cuh"

namespace attn {
namespace {

constexpr int64_t kTogetherBytes = 48 << 20;

// `how`: 0 chooses, 1 per sequence, 2 together.  Whether the prefix is multiplied once for all.
bool together(int how, int B, int Hkv, int D, int q_dtype, int kv_dtype, float scale, int64_t n_prefix) {
    if (how == 1 || n_prefix == 0 || !attend_tc_supported(D, q_dtype, scale)) return false;
    return how == 2 || (B > 1 && n_prefix * B * Hkv * D * (kv_dtype == ATTN_B200_E4M3 ? 2 : 4) > kTogetherBytes);
}
AttendParams plan(int B, int H, int Hkv, int64_t n_prefix) {
    AttendParams a{};
    a.B = B;
    a.H = H;
    a.Hkv = Hkv;
    a.n_prefix = (int)n_prefix;
    attend_prefix_plan(a);
    return a;
}

}  // namespace
}  // namespace attn

extern "C" size_t attn_b200_shared_prefix_workspace_bytes(int B, int H, int n_kv_heads, int D, int64_t n_prefix, float scale,
                                                          int q_dtype, int kv_dtype, int how) {
    using namespace attn;
    if (B <= 0 || H <= 0 || n_kv_heads <= 0 || H % n_kv_heads || D <= 0 || n_prefix <= 0 || n_prefix > 0x7fffffffLL) return 0;
    if (!together(how, B, n_kv_heads, D, q_dtype, kv_dtype, scale, n_prefix)) return 0;
    return (size_t)attend_prefix_parts(plan(B, H, n_kv_heads, n_prefix)) * B * H * (D + 2) * sizeof(float);
}

extern "C" int attn_b200_shared_prefix_decode(const void* q, const void* k_new, const void* v_new, const void* k_cache,
                                              const void* v_cache, const int32_t* prefix_slots, const int32_t* slots,
                                              const int32_t* offsets, void* out, void* workspace, size_t workspace_bytes, int B,
                                              int H, int n_kv_heads, int D, int64_t n_prefix, int64_t n_tokens, int64_t n_slots,
                                              float scale, const float* k_scale, const float* v_scale, int q_dtype, int kv_dtype,
                                              int how, int32_t* err_flag, void* stream) {
    using namespace attn;
    if (B < 0 || H <= 0 || n_kv_heads <= 0 || H % n_kv_heads || D <= 0 || n_prefix < 0 || n_tokens < 0 || n_slots < 0 ||
        how < 0 || how > 2)
        return ATTN_B200_EINVAL;
    if (q_dtype != ATTN_B200_F16 && q_dtype != ATTN_B200_BF16 && q_dtype != ATTN_B200_F32) return ATTN_B200_EDTYPE;
    const bool e4 = kv_dtype == ATTN_B200_E4M3;
    if (kv_dtype != q_dtype && !(e4 && q_dtype != ATTN_B200_F32)) return ATTN_B200_EDTYPE;
    if (e4 && (!k_scale || !v_scale)) return ATTN_B200_EINVAL;
    if (n_slots > 0x7fffffffLL || n_prefix + n_tokens > 0x7fffffffLL) return ATTN_B200_ETOOLARGE;
    if (B == 0) return 0;
    if (!q || !k_new || !v_new || !offsets || !out || (n_prefix && !prefix_slots) || (n_tokens && !slots) ||
        (n_prefix + n_tokens && (!k_cache || !v_cache)))
        return ATTN_B200_EINVAL;
    cudaStream_t st = (cudaStream_t)stream;
    SpanParams p{};
    p.q = q; p.k_new = k_new; p.v_new = v_new; p.k_cache = k_cache; p.v_cache = v_cache;
    p.table = slots; p.offsets = offsets; p.out = out;
    p.B = B; p.H = H; p.Hkv = n_kv_heads; p.D = D;
    p.n_tokens = n_tokens; p.n_slots = n_slots;
    p.block_size = 1;
    p.window = 0x7fffffff;
    p.scale_log2 = scale * kLog2e;
    p.k_scale = e4 ? k_scale : nullptr;
    p.v_scale = e4 ? v_scale : nullptr;
    p.err_flag = err_flag;
    const bool aligned = (((uintptr_t)q | (uintptr_t)k_new | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0;
    const bool can = aligned && n_slots > 0 && n_prefix > 0 && attend_tc_supported(D, q_dtype, scale);
    if (how == 2 && !can) return ATTN_B200_ESHAPE;
    if (can && together(how, B, n_kv_heads, D, q_dtype, kv_dtype, scale, n_prefix)) {
        AttendParams a = plan(B, H, n_kv_heads, n_prefix);
        const int parts = attend_prefix_parts(a);
        if ((uintptr_t)workspace % 16 || !workspace || workspace_bytes < (size_t)parts * B * H * (D + 2) * sizeof(float))
            return ATTN_B200_EWORKSPACE;
        a.q = q; a.k_cache = k_cache; a.v_cache = v_cache; a.table = prefix_slots;
        a.n_slots = n_slots;
        a.scale_log2 = p.scale_log2;
        a.err_flag = err_flag;
        a.parts = (float*)workspace;
        a.k_scale = p.k_scale; a.v_scale = p.v_scale;
        if (const int rc = attend_prefix_launch(a, D, q_dtype, e4, st)) return rc;
        p.parts = a.parts;
        p.n_parts = parts;
        p.early = 1;
        return span_decode_launch(p, n_tokens / B + 1, B > 1, q_dtype, kv_dtype, st);
    }
    p.prefix = prefix_slots;
    p.n_prefix = (int)n_prefix;
    return span_decode_launch(p, n_prefix + n_tokens / B + 1, B > 1 && n_tokens > B * n_prefix, q_dtype, kv_dtype, st);
}
