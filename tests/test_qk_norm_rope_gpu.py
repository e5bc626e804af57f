"""GPU: per-head norm with rotation, and with the cache append, against the 64-bit formula.

Tolerance per entry: half a step of the output type relative to the value, plus the 32-bit arithmetic's
share.  That is a sum of head_dim squares (a lane adds at most 64, then 5 shuffles), a reciprocal
square root of 2 ulp, two products and a two-term combination: below 80 * 2^-24 of |a| + |b|."""
import pytest
import torch

from oracle import attention_oracle as orc
from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu
F16, BF16, F32, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn
TINY = {F16: 2.0 ** -25, BF16: 1e-40, F32: 1e-45}          # half a step below the smallest normal number


def _close(got, ref, size, dtype):
    got = got.detach().cpu().double().reshape(ref.shape)
    tol = (torch.finfo(dtype).eps / 2) * ref.abs() + 80 * 2.0 ** -24 * size * (1 + torch.finfo(dtype).eps) + TINY[dtype]
    bad = (got - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} entries off, worst {float(((got - ref).abs() - tol).max())}"


def _make(N, Hq, Hk, D, rot, dtype, seed, w_dtype=None, t_dtype=None, packed=False, max_pos=512, std=1.0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(N, (Hq + 2 * Hk) * D, generator=g) * std).to(dtype)
    dev = qkv.cuda()
    cut = [Hq * D, Hk * D, Hk * D]
    Q, K, V = dev.split(cut, 1) if packed else (x.contiguous() for x in dev.split(cut, 1))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(w_dtype or dtype) for _ in range(2))
    pos = torch.randint(0, max_pos, (N,), generator=g).int()
    ang = torch.rand(max_pos, rot, generator=g, dtype=torch.float64) * 6.28
    cos, sin = ang.cos().to(t_dtype or dtype), ang.sin().to(t_dtype or dtype)
    return qkv.split(cut, 1), (Q, K, V), wq, wk, pos, cos, sin


CASES = [  # N, Hq, Hk, D, rot
    (1, 1, 1, 128, 64), (3, 32, 8, 128, 64), (37, 32, 32, 128, 32), (130, 7, 1, 64, 32), (65, 5, 5, 96, 24),
    (19, 4, 2, 256, 128), (9, 3, 1, 256, 8), (8, 2, 1, 512, 64), (5, 2, 2, 16, 8), (4, 3, 3, 8, 0),
    (11, 4, 2, 80, 40), (6, 2, 1, 20, 6), (7, 3, 2, 33, 16), (2, 2, 1, 2, 1), (3, 1, 1, 1024, 100),
    (1030, 2, 1, 128, 64)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("N,Hq,Hk,D,rot", CASES)
def test_norm_rope_against_64_bits(dtype, N, Hq, Hk, D, rot):
    import attention_impl_b200 as A
    (q, k, _), (Q, K, _), wq, wk, pos, cos, sin = _make(N, Hq, Hk, D, rot, dtype, N + D)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    keep = Q.clone(), K.clone()
    Qo, Ko = A.qk_norm_rope(Q, K, wq.cuda(), wk.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), D, eps=1e-5, err_flag=flag)
    for x, o, w in ((q, Qo, wq), (k, Ko, wk)):
        _close(o, *so.qk_norm_rope(x, w, pos, cos, sin, D, 1e-5), dtype)
    assert torch.equal(Q, keep[0]) and torch.equal(K, keep[1]) and int(flag) == 0
    # in place: the same bits
    A.qk_norm_rope(Q, K, wq.cuda(), wk.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), D, eps=1e-5, out=(Q, K))
    assert torch.equal(Q, Qo) and torch.equal(K, Ko)


@pytest.mark.parametrize("dtype,w_dtype,t_dtype", [(F16, F32, F16), (BF16, BF16, F32), (BF16, F32, F32)])
@pytest.mark.parametrize("D,rot", [(128, 64), (64, 8), (33, 16)])
def test_packed_projection_and_float_tables(dtype, w_dtype, t_dtype, D, rot):
    """q, k, v as column slices of one projection, float32 weights and tables, the append in the same pass."""
    import attention_impl_b200 as A
    N, Hq, Hk, rows = 45, 6, 2, 101
    (q, k, v), (Q, K, V), wq, wk, pos, cos, sin = _make(N, Hq, Hk, D, rot, dtype, 5, w_dtype, t_dtype, packed=True)
    sl = torch.randperm(rows, generator=torch.Generator().manual_seed(1))[:N].int()
    Kc = torch.full((rows, Hk * D), 3.0, dtype=dtype, device="cuda")
    Vc = Kc.clone()
    Qo, Ko = A.qk_norm_rope_and_cache_write(Q, K, V, wq.cuda(), wk.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), sl.cuda(),
                                            Kc, Vc, D)
    assert Qo.is_contiguous() and Ko.is_contiguous()
    for x, o, w in ((q, Qo, wq), (k, Ko, wk)):
        _close(o, *so.qk_norm_rope(x, w, pos, cos, sin, D, 1e-6), dtype)
    ref_k, ref_v = torch.full_like(Kc, 3.0), torch.full_like(Vc, 3.0)
    ref_k[sl.long().cuda()] = Ko
    ref_v[sl.long().cuda()] = V
    assert torch.equal(Kc, ref_k) and torch.equal(Vc, ref_v)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,rot", [(128, 64), (64, 16), (20, 6)])
def test_append_in_8_bits(dtype, D, rot):
    import attention_impl_b200 as A
    N, Hq, Hk, rows = 77, 4, 2, 90
    (q, k, v), (Q, K, V), wq, wk, pos, cos, sin = _make(N, Hq, Hk, D, rot, dtype, 6)
    sl = torch.randperm(rows, generator=torch.Generator().manual_seed(2))[:N].int()
    ks, vs = torch.tensor([0.01, 0.002]), torch.tensor([0.008, 0.02])        # 0.002: saturates
    Kc = torch.zeros(rows, Hk * D, device="cuda").to(E4M3)
    Vc = torch.zeros(rows, Hk * D, device="cuda").to(E4M3)
    A.qk_norm_rope_and_cache_write(Q, K, V, wq.cuda(), wk.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), sl.cuda(), Kc, Vc, D,
                                   k_scale=ks.cuda(), v_scale=vs.cuda())
    k64, size = so.qk_norm_rope(k, wk, pos, cos, sin, D, 1e-6)
    for pool, x, s, wide in ((Kc, k64, ks, size), (Vc, v.double().view(N, Hk, D), vs, v.double().view(N, Hk, D).abs())):
        ref = (x / s.double()[:, None]).clamp(-448, 448)
        got = pool.cpu().to(torch.float64)[sl.long()].view(N, Hk, D)
        tol = 2.0 ** -4 * ref.abs() + 2.0 ** -10 + 80 * 2.0 ** -24 * wide / s.double()[:, None]
        assert ((got - ref).abs() <= tol).all()
        rest = torch.ones(rows, dtype=torch.bool)
        rest[sl.long()] = False
        assert (pool.cpu().view(torch.uint8)[rest] == 0).all()


def test_extreme_rows():
    """A zero row, a row of the type's largest values, subnormals, infinity and NaN."""
    import attention_impl_b200 as A
    for D, rot in ((128, 64), (33, 16)):
        (q, _, _), (Q, K, _), wq, wk, pos, cos, sin = _make(6, 1, 1, D, rot, F16, 7)
        Q[0], Q[1], Q[2] = 0, 65504, 2.0 ** -24
        Q[3, 5], Q[4, 5] = float("inf"), float("nan")
        Qo, _ = A.qk_norm_rope(Q, K, wq.cuda(), wk.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), D)
        ref, size = so.qk_norm_rope(Q.cpu(), wq, pos, cos, sin, D, 1e-6)
        _close(Qo[[0, 1, 2, 5]], ref[[0, 1, 2, 5]], size[[0, 1, 2, 5]], F16)
        assert (Qo[0] == 0).all()
        assert torch.equal(torch.isnan(Qo[3:5]).cpu(), torch.isnan(ref[3:5]).view(2, -1))


def test_bad_positions_and_slots():
    import attention_impl_b200 as A
    for D, rot in ((128, 64), (33, 16)):
        (q, k, v), (Q, K, V), wq, wk, pos, cos, sin = _make(8, 4, 2, D, rot, BF16, 8)
        pos[1], pos[2] = -1, 512
        sl = torch.arange(8).int()
        sl[3], sl[4] = -1, 20
        Kc = torch.full((20, 2 * D), 9.0, dtype=BF16, device="cuda")
        Vc = Kc.clone()
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        Qo, Ko = A.qk_norm_rope_and_cache_write(Q, K, V, wq.cuda(), wk.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), sl.cuda(),
                                                Kc, Vc, D, err_flag=flag)
        assert int(flag) == 3
        good = [0, 3, 4, 5, 6, 7]
        pos[1] = pos[2] = 0
        for x, o, w in ((q, Qo, wq), (k, Ko, wk)):
            ref, size = so.qk_norm_rope(x, w, pos, cos, sin, D, 1e-6)
            _close(o[good], ref[good], size[good], BF16)
            assert (o[1:3] == 0).all()
        assert torch.equal(Kc[[0, 5, 6, 7]], Ko[[0, 5, 6, 7]]) and torch.equal(Vc[[0, 5, 6, 7]], V[[0, 5, 6, 7]])
        assert (Kc[[1, 2, 3, 4]] == 9).all() and (Kc[8:] == 9).all() and (Vc[[1, 2, 3, 4]] == 9).all() and (Vc[8:] == 9).all()


def test_pool_rows_beyond_32_bit_offsets():
    """Slots whose element offset passes 2^31 (a pool of 8.6 GB)."""
    import attention_impl_b200 as A
    D, Hk, rows = 128, 32, (1 << 31) // 4096 + 64
    (q, k, v), (Q, K, V), wq, wk, pos, cos, sin = _make(2, 32, Hk, D, 64, F16, 9)
    pool = torch.zeros(rows, Hk * D, dtype=F16, device="cuda")
    sl = torch.tensor([rows - 1, 3]).int()
    Vc = pool.view(torch.float16)
    _, Ko = A.qk_norm_rope_and_cache_write(Q, K, V, wq.cuda(), wk.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), sl.cuda(), pool,
                                           torch.zeros_like(pool), D)
    assert torch.equal(pool[rows - 1], Ko[0]) and torch.equal(pool[3], Ko[1])
    del pool, Vc


def test_no_tokens_other_stream_and_graph():
    import attention_impl_b200 as A
    (q, k, _), (Q, K, _), wq, wk, pos, cos, sin = (_make(33, 4, 2, 128, 64, F16, 10))
    w = wq.cuda(), wk.cuda()
    t = pos.cuda(), cos.cuda(), sin.cuda()
    Qo, Ko = A.qk_norm_rope(Q[:0], K[:0], *w, t[0][:0], *t[1:], 128)
    assert Qo.shape == (0, 512) and Ko.shape == (0, 256)
    Qo, Ko = A.qk_norm_rope(Q, K, *w, *t, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        Q2, K2 = A.qk_norm_rope(Q, K, *w, *t, 128)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(Q2, Qo) and torch.equal(K2, Ko)
    out = torch.empty_like(Q), torch.empty_like(K)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.qk_norm_rope(Q, K, *w, *t, 128, out=out)
    Q.mul_(2.0)          # exact, and the norm takes it out again but for eps
    graph.replay()
    ref, size = so.qk_norm_rope(Q.cpu(), wq, pos, cos, sin, 128, 1e-6)
    _close(out[0], ref, size, F16)
    assert torch.equal(out[1], Ko)


def test_refusals():
    import attention_impl_b200 as A
    _, (Q, K, V), wq, wk, pos, cos, sin = _make(4, 4, 2, 64, 32, F16, 11)
    w = wq.cuda(), wk.cuda()
    t = pos.cuda(), cos.cuda(), sin.cuda()
    call = lambda q=Q, k=K, ww=w, tt=t, d=64, **kw: A.qk_norm_rope(q, k, *ww, *tt, d, **kw)  # noqa: E731
    call()
    for bad in (dict(q=Q.double()), dict(k=K.float()), dict(q=Q[:3]), dict(d=48), dict(q=Q.t()), dict(eps=-1.0),
                dict(eps=float("nan")), dict(ww=(w[0][:32].contiguous(), w[1])), dict(ww=(w[0].float(), w[1])),
                dict(ww=(w[0].bfloat16(), w[1].bfloat16())), dict(tt=(t[0].long(), *t[1:])), dict(tt=(t[0][:3], *t[1:])),
                dict(tt=(t[0], t[1], t[2].float())), dict(tt=(t[0], t[1], t[2][:5])), dict(d=32), dict(q=Q.cpu()),
                dict(tt=(t[0].cpu(), *t[1:])), dict(q=Q[0].expand(4, 256)), dict(err_flag=torch.zeros(1, device="cuda")),
                dict(out=(torch.empty_like(Q), K[:, :64])), dict(out=(K, Q)), dict(out=(Q, Q[:, :128])),
                dict(out=(torch.empty_like(Q).float(), torch.empty_like(K)))):
        with pytest.raises(RuntimeError):
            call(**bad)
    both = torch.zeros(4, 512, dtype=F16, device="cuda")
    with pytest.raises(RuntimeError):       # K's columns would be overwritten while other heads still read them
        A.qk_norm_rope(both[:, :256], both[:, 256:384], *w, *t, 64, out=(both[:, 64:320], torch.empty_like(K)))
    A.qk_norm_rope(both[:, :256], both[:, 256:384], *w, *t, 64, out=(both[:, :256], both[:, 384:]))
    sl = torch.arange(4).int().cuda()
    Kc = torch.zeros(8, 128, dtype=F16, device="cuda")
    write = lambda s=sl, kc=Kc, vc=Kc.clone(), v=V, **kw: A.qk_norm_rope_and_cache_write(Q, K, v, *w, *t, s, kc, vc, 64, **kw)  # noqa: E731
    write()
    for bad in (dict(s=sl[:3]), dict(s=sl.long()), dict(s=None), dict(kc=Kc[:, :64].contiguous()), dict(kc=Kc.float()),
                dict(vc=Kc[:4]), dict(v=V[:, :64]), dict(v=None), dict(kc=Kc.to(E4M3), vc=Kc.to(E4M3)),
                dict(kc=Kc.to(E4M3), vc=Kc.to(E4M3), k_scale=torch.ones(2, device="cuda"), v_scale=torch.ones(1, device="cuda")),
                dict(kc=Kc.to(E4M3), vc=Kc, k_scale=torch.ones(2, device="cuda"), v_scale=torch.ones(2, device="cuda"))):
        with pytest.raises(RuntimeError):
            write(**bad)


def test_rotation_alone_matches_the_existing_operator():
    """With unit weights on rows that are already normalised the rotation is rotary_embedding_inplace's, to
    the roundings of that operator (three per entry instead of one)."""
    import attention_impl_b200 as A
    N, H, D = 16, 4, 128
    g = torch.Generator().manual_seed(12)
    x = torch.sign(torch.randn(N, H * D, generator=g)).half()             # mean square exactly 1
    pos = torch.randint(0, 4096, (N,), generator=g).int()
    cos, sin = orc.rope_tables(D, 4096, dtype=F16)
    one = torch.ones(D, dtype=F16, device="cuda")
    Qo, _ = A.qk_norm_rope(x.cuda(), x.cuda(), one, one, pos.cuda(), cos.cuda(), sin.cuda(), D, eps=0.0)
    old = x.cuda()
    A.rotary_embedding_inplace(old, x.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), D)
    # |c|, |s| <= 1: two product roundings of at most 2^-12 each, the sum's rounding of at most 2^-11 (values
    # up to sqrt(2)), and this operator's own of at most 2^-11
    assert (Qo.float() - old.float()).abs().max() <= 2 * 2.0 ** -12 + 2 * 2.0 ** -11
