"""CPU: the serving operators' C entry points check their arguments before they touch the GPU, the Python
operators refuse host tensors, and the 64-bit reference they are tested against agrees with the oracle
where the two overlap."""
import pytest
import torch

from oracle import attention_oracle as orc
from oracle import serving_oracle as so

EINVAL, EDTYPE, ESHAPE, EWORKSPACE, ETOOLARGE = -1, -2, -3, -4, -5
F16, BF16, F32, E4M3 = 0, 1, 2, 3
X = 4096            # stands for a device pointer: none of these calls gets as far as using it


def _norm(n=4, hq=2, hk=1, d=64, rot=32, ptr=X, slots=None, eps=1e-6, dt=F16, w=F16, t=F16, kv=F16, ks=None, cache=None):
    from attention_impl_b200._lib import lib
    return lib.attn_b200_qk_norm_rope(ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, slots, cache, cache, n, hq, hk, d, rot, 8, 8,
                                      hq * d, hk * d, hk * d, hq * d, hk * d, eps, dt, w, t, kv, ks, ks, None, None)


def test_norm_rope_arguments():
    assert _norm(n=0) == 0
    for kw, want in ((dict(n=-1), EINVAL), (dict(hq=0), EINVAL), (dict(hk=0), EINVAL), (dict(d=0), EINVAL), (dict(rot=-1), EINVAL),
                     (dict(rot=33), ESHAPE), (dict(eps=-1.0), EINVAL), (dict(eps=float("nan")), EINVAL), (dict(dt=E4M3), EDTYPE),
                     (dict(w=BF16), EDTYPE), (dict(t=BF16), EDTYPE), (dict(ptr=None), EINVAL), (dict(slots=X), EINVAL),
                     (dict(slots=X, cache=X, kv=BF16), EDTYPE), (dict(slots=X, cache=X, kv=E4M3), EINVAL),
                     (dict(slots=X, cache=X, kv=E4M3, ks=X, dt=F32, w=F32, t=F32), EDTYPE)):
        assert _norm(**kw) == want, kw


def _window(B=2, H=4, hkv=2, D=64, n=10, slots=16, bs=1, mb=0, window=4, sinks=0, ks=None, q=F16, kv=F16, ptr=X):
    from attention_impl_b200._lib import lib
    return lib.attn_b200_paged_window_decode(ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, B, H, hkv, D, n, slots, bs, mb, window, sinks, 1.0, ks,
                                             ks, q, kv, None, None)


def test_window_decode_arguments():
    assert _window(B=0) == 0
    for kw, want in ((dict(B=-1), EINVAL), (dict(H=0), EINVAL), (dict(hkv=3), EINVAL), (dict(D=0), EINVAL), (dict(window=0), EINVAL),
                     (dict(sinks=-1), EINVAL), (dict(bs=0), EINVAL), (dict(mb=-1), EINVAL), (dict(n=-1), EINVAL), (dict(q=E4M3), EDTYPE),
                     (dict(kv=BF16), EDTYPE), (dict(q=F32, kv=E4M3), EDTYPE), (dict(kv=E4M3), EINVAL), (dict(slots=1 << 31), ETOOLARGE),
                     (dict(ptr=None), EINVAL)):
        assert _window(**kw) == want, kw


def _prefill(B=2, nq=8, nkv=20, mq=8, H=4, hkv=2, D=64, slots=32, window=4, sinks=0, dt=F16, ptr=X):
    from attention_impl_b200._lib import lib
    return lib.attn_b200_paged_window_prefill(ptr, ptr, ptr, ptr, ptr, ptr, ptr, B, nq, nkv, mq, H, hkv, D, slots, window, sinks, 1.0, dt, 0,
                                              None, None)


def test_window_prefill_arguments():
    assert _prefill(nq=0) == 0
    for kw, want in ((dict(B=-1), EINVAL), (dict(H=0), EINVAL), (dict(hkv=3), EINVAL), (dict(mq=-1), EINVAL), (dict(window=0), EINVAL),
                     (dict(sinks=-1), EINVAL), (dict(dt=E4M3), EDTYPE), (dict(D=513), ESHAPE), (dict(slots=1 << 31), ETOOLARGE),
                     (dict(B=65536), ETOOLARGE), (dict(ptr=None), EINVAL)):
        assert _prefill(**kw) == want, kw


def _shared(B=2, H=4, hkv=2, D=64, P=100, n=10, slots=256, ws=X, ws_bytes=0, ks=None, q=F16, kv=F16, ptr=X, scale=1.0,
            how=2):
    from attention_impl_b200._lib import lib
    return lib.attn_b200_shared_prefix_decode(ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ws, ws_bytes, B, H, hkv, D, P, n, slots, scale, ks, ks,
                                              q, kv, how, None, None)


def test_shared_prefix_arguments():
    from attention_impl_b200._lib import lib
    assert _shared(B=0) == 0
    for kw, want in ((dict(B=-1), EINVAL), (dict(hkv=3), EINVAL), (dict(P=-1), EINVAL), (dict(n=-1), EINVAL), (dict(q=E4M3), EDTYPE),
                     (dict(kv=BF16), EDTYPE), (dict(kv=E4M3), EINVAL), (dict(P=1 << 31), ETOOLARGE), (dict(slots=1 << 31), ETOOLARGE),
                     (dict(ptr=None), EINVAL), (dict(ws=None), EWORKSPACE), (dict(), EWORKSPACE), (dict(ws=X + 4, ws_bytes=1 << 30), EWORKSPACE),
                     (dict(how=3), EINVAL), (dict(D=80), ESHAPE), (dict(P=0), ESHAPE), (dict(scale=-1.0), ESHAPE), (dict(ptr=X + 2), ESHAPE),
                     (dict(q=F32, kv=F32), ESHAPE)):
        assert _shared(**kw) == want, kw
    need = lib.attn_b200_shared_prefix_workspace_bytes
    assert need(2, 4, 2, 64, 100, 1.0, F16, F16, 1) == 0            # read per sequence
    for bad in ((2, 4, 2, 64, 100, 1.0, F32, F32), (2, 4, 2, 80, 100, 1.0, F16, F16), (2, 4, 2, 64, 100, -1.0, F16, F16),
                (0, 4, 2, 64, 100, 1.0, F16, F16), (2, 4, 2, 64, 0, 1.0, F16, F16)):
        assert need(*bad, 2) == 0
    # at least one partial set of rows [o[D], m, l], at most two for every key tile
    for B, H, hkv, P in ((2, 4, 2, 100), (64, 32, 8, 32768), (300, 8, 1, 5000)):
        n = need(B, H, hkv, 128, P, 1.0, F16, E4M3, 2)
        assert n % (B * H * 130 * 4) == 0 and 1 <= n // (B * H * 130 * 4) <= 2 * -(-P // 128)
    # the choice: bytes of the prefix times the batch above 48 MB, more than one sequence
    assert need(4, 32, 8, 128, 2048, 1.0, F16, F16, 0) == 0 and need(4, 32, 8, 128, 4096, 1.0, F16, F16, 0) > 0
    assert need(4, 32, 8, 128, 4096, 1.0, F16, E4M3, 0) == 0 and need(1, 32, 8, 128, 1 << 20, 1.0, F16, F16, 0) == 0


def test_host_tensors_are_refused():
    import attention_impl_b200 as A
    q = torch.zeros(2, 256, dtype=torch.float16)
    i = torch.zeros(4, dtype=torch.int32)
    w = torch.ones(128, dtype=torch.float16)
    t = torch.ones(8, 64, dtype=torch.float16)
    for call in (lambda: A.qk_norm_rope(q, q, w, w, i[:2], t, t, 128),
                 lambda: A.qk_norm_rope_and_cache_write(q, q, q, w, w, i[:2], t, t, i[:2], q, q, 128),
                 lambda: A.paged_window_attention_forward(q, q, q, q, q, i, i[:2], 2, 4),
                 lambda: A.paged_window_prefill_attention(q, q, q, i, i[:2], i[:2], 2, 4),
                 lambda: A.shared_prefix_attention_forward(q, q, q, q, q, i, i, i[:2], 2)):
        with pytest.raises(RuntimeError, match="Q must be a CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="Q must be a CUDA tensor"):
        A.qk_norm_rope(None, q, w, w, i[:2], t, t, 128)


def test_reference_agrees_with_the_oracle():
    g = torch.Generator().manual_seed(0)
    H, D, lens = 2, 16, [5, 0, 9]
    Q, K, V = (torch.randn(3, H * D, generator=g) for _ in range(3))
    Kc, Vc = (torch.randn(20, H * D, generator=g) for _ in range(2))
    table = torch.randperm(20, generator=g)[:14]
    rows = [table[:5], table[5:5], table[5:]]
    ref, _ = so.decode(Q, K, V, [Kc[r] for r in rows], [Vc[r] for r in rows], H, D ** -0.5)
    off = torch.tensor(lens).cumsum(0).int()
    got = orc.paged_decode(Q, K, V, Kc, Vc, table.int(), off, H, scale=D ** -0.5)
    got = got[-1] if isinstance(got, (list, tuple)) else got
    assert (got.double().view(ref.shape) - ref).abs().max() < 1e-5
    # a window that covers everything, and a prefill row against the single-token form
    assert torch.equal(so.decode(Q, K, V, [Kc[r] for r in rows], [Vc[r] for r in rows], H, 0.25, 10, 0)[0],
                       so.decode(Q, K, V, [Kc[r] for r in rows], [Vc[r] for r in rows], H, 0.25)[0])
    k, v, q = Kc[:9], Vc[:9], torch.randn(9, H * D, generator=g)
    full, _ = so.prefill(q, [k], [v], [9], H, 0.25, 4, 1)
    for i in range(9):
        one, _ = so.decode(q[i:i + 1], k[i:i + 1], v[i:i + 1], [k[:i]], [v[:i]], H, 0.25, 4, 1)
        assert (one[0] - full[i]).abs().max() < 1e-12
