"""GPU: decoding behind a shared prefix against the 64-bit formula."""
import pytest
import torch

from oracle import serving_oracle as so
from serving_helpers import BF16, E4M3, F16, F32, close, offsets, pool

pytestmark = pytest.mark.gpu


def _case(P, lens, H, Hkv, D, dtype, kv="same", seed=0):
    g = torch.Generator().manual_seed(seed + P + D + len(lens))
    B, total = len(lens), sum(lens)
    rows = P + total + 4
    Q, K, V = (torch.randn(B, n * D, generator=g).to(dtype) for n in (H, Hkv, Hkv))
    Kc, k64, ks = pool(g, rows, Hkv, D, dtype, kv)
    Vc, v64, vs = pool(g, rows, Hkv, D, dtype, kv)
    perm = torch.randperm(rows, generator=g)[:P + total]
    prefix, table = perm[:P], perm[P:]
    ends = torch.tensor(list(lens)).cumsum(0).tolist()
    seqs = [torch.cat([prefix, table[e - n:e]]) for n, e in zip(lens, ends)]
    ref, size = so.decode(Q, K, V, [k64[s] for s in seqs], [v64[s] for s in seqs], H, D ** -0.5)
    args = [Q.cuda(), K.cuda(), V.cuda(), Kc, Vc, prefix.int().cuda(), table.int().cuda(), offsets(lens).cuda(), H]
    tc = dtype != F32 and D in (64, 128)
    return args, dict(k_scale=ks, v_scale=vs), ref, size, F32 if not tc and D != 256 or dtype == F32 else F16 if kv == "e4m3" else dtype, (
        P + max(lens) + 1)


def _run(*a, **kw):
    import attention_impl_b200 as A
    args, more, ref, size, pt, n = _case(*a, **kw)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    D, dtype = args[0].size(1) // args[8], args[0].dtype
    # every way that the case has: read per sequence, multiplied together, and the choice
    for together in ([True] if args[5].numel() and D in (64, 128) and dtype != F32 else []) + [False, None]:
        out = A.shared_prefix_attention_forward(*args, **more, err_flag=flag, together=together)
        assert int(flag) == 0
        close(out, ref, size, dtype, pt, n)
    return args, more, out


@pytest.mark.parametrize("P", [0, 1, 63, 64, 65, 100, 127, 128, 129, 200, 256, 384, 385, 1000])
@pytest.mark.parametrize("dtype,kv", [(F16, "same"), (BF16, "same"), (F16, "e4m3"), (BF16, "e4m3")])
def test_prefix_lengths(P, dtype, kv):
    _run(P, [0, 5, 70], 4, 2, 128, dtype, kv)


@pytest.mark.parametrize("B,H,Hkv", [(1, 1, 1), (1, 8, 8), (2, 6, 2), (16, 8, 1), (17, 8, 1), (32, 8, 1), (33, 8, 1), (128, 2, 2), (129, 1, 1),
                                     (40, 20, 4), (70, 9, 1), (300, 2, 1)])
@pytest.mark.parametrize("D,kv", [(64, "same"), (128, "same"), (128, "e4m3"), (64, "e4m3")])
def test_batches_and_head_layouts(B, H, Hkv, D, kv):
    """Rows of a KV head from one to several pairs of 128-row tiles."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 20, (B,), generator=g).tolist()
    _run(300, lens, H, Hkv, D, BF16 if B % 2 else F16, kv)


@pytest.mark.parametrize("dtype,D,kv", [(F32, 128, "same"), (F16, 80, "same"), (BF16, 256, "same"), (F16, 256, "e4m3"), (F32, 33, "same"),
                                        (F16, 512, "same"), (BF16, 48, "e4m3")])
def test_other_types_and_head_dims(dtype, D, kv):
    _run(150, [0, 40, 3], 4, 2, D, dtype, kv)


def test_long_prefix():
    _run(20000, [0, 100, 3, 999], 8, 2, 128, BF16)
    _run(9001, [10] * 20, 16, 2, 128, F16, "e4m3")
    _run(5000, [0] * 3, 4, 4, 64, F16)


def test_agrees_with_the_operator_without_sharing():
    import attention_impl_b200 as A
    args, more, out = _run(500, [0, 30, 100, 7], 8, 8, 128, F16)
    Q, K, V, Kc, Vc, prefix, table, off, H = args
    ends = [0] + off.tolist()
    full = torch.cat([torch.cat([prefix, table[a:b]]) for a, b in zip(ends, ends[1:])])
    lens = torch.tensor([500 + b - a for a, b in zip(ends, ends[1:])])
    _, _, plain = A.paged_kv_attention_forward(Q, K, V, Kc, Vc, full, lens.cumsum(0).int().cuda(), H, return_sp=False)
    assert (out.float() - plain.float()).abs().max() <= 4 * 2.0 ** -11 * float(args[4].abs().max())


def test_prefix_far_below_and_far_above():
    """A prefix that the softmax drops beside the own tokens, and the other way round."""
    import attention_impl_b200 as A
    D, P, n = 128, 300, 40
    g = torch.Generator().manual_seed(4)
    for sign, way in ((1, True), (-1, True), (1, False), (-1, False)):
        q = torch.ones(2, D).half()
        kc = torch.cat([torch.full((P, D), 6.0 * sign), torch.full((n, D), -6.0 * sign)]).half()
        vc = torch.randn(P + n, D, generator=g).half()
        k, v = torch.full((2, D), -6.0 * sign).half(), torch.randn(2, D, generator=g).half()
        out = A.shared_prefix_attention_forward(q.cuda(), k.cuda(), v.cuda(), kc.cuda(), vc.cuda(), torch.arange(P).int().cuda(),
                                                torch.arange(P, P + n).int().cuda(), torch.tensor([0, n]).int().cuda(), 1, together=way)
        rows = [torch.arange(P), torch.arange(P + n)]
        ref, size = so.decode(q, k, v, [kc[r] for r in rows], [vc[r] for r in rows], 1, D ** -0.5)
        close(out, ref, size, F16, F16, P + n)


def test_bf16_queries_of_any_size_over_8_bit_pools():
    import attention_impl_b200 as A
    args, more, *_ = _case(200, [10, 3], 4, 2, 128, BF16, "e4m3")
    args[1] = args[1] * 0
    for way in (True, False):
        a = A.shared_prefix_attention_forward(*args, **more, scale=0.1, together=way)
        for e in (2.0 ** 90, 2.0 ** -90):
            b = A.shared_prefix_attention_forward(args[0] * e, *args[1:], **more, scale=0.1 / e, together=way)
            assert (a.float() - b.float()).abs().max() <= 2 * 2.0 ** -8 * float(a.abs().max())


@pytest.mark.parametrize("D,way", [(128, True), (128, False), (80, False)])
def test_bad_slots_and_offsets(D, way):
    import attention_impl_b200 as A
    args, more, *_ = _case(300, [20, 30], 4, 2, D, F16)
    Q, K, V, Kc, Vc, prefix, table, off, H = args
    prefix, table = prefix.clone(), table.clone()
    prefix[[0, 50, 299]] = torch.tensor([-1, Kc.size(0), 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    table[[5, 22]] = -3
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = A.shared_prefix_attention_forward(Q, K, V, Kc, Vc, prefix, table, off, H, err_flag=flag, together=way)
    assert int(flag) == 1
    ok = lambda t: t[(t >= 0) & (t < Kc.size(0))].cpu().long()  # noqa: E731
    rows = [torch.cat([ok(prefix), ok(table[:20])]), torch.cat([ok(prefix), ok(table[20:])])]
    k64, v64 = Kc.cpu().double(), Vc.cpu().double()
    ref, size = so.decode(Q.cpu(), K.cpu(), V.cpu(), [k64[r] for r in rows], [v64[r] for r in rows], H, D ** -0.5)
    close(got, ref, size, F16, F16 if D == 128 else F32, 331)
    # every prefix row missing: the own rows alone
    flag.zero_()
    got = A.shared_prefix_attention_forward(Q, K, V, Kc, Vc, prefix * 0 - 1, args[6], off, H, err_flag=flag, together=way)
    rows = [args[6][:20].cpu().long(), args[6][20:].cpu().long()]
    ref, size = so.decode(Q.cpu(), K.cpu(), V.cpu(), [k64[r] for r in rows], [v64[r] for r in rows], H, D ** -0.5)
    close(got, ref, size, F16, F16 if D == 128 else F32, 31)
    assert int(flag) == 1
    flag.zero_()
    got = A.shared_prefix_attention_forward(*args[:7], torch.tensor([20, 51], dtype=torch.int32, device="cuda"), H, err_flag=flag, together=way)
    assert int(flag) == 4 and torch.isfinite(got).all()


def test_nothing_to_do():
    import attention_impl_b200 as A
    z = lambda *s, dt=F16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    e = z(0, dt=torch.int32)
    assert A.shared_prefix_attention_forward(z(0, 256), z(0, 256), z(0, 256), z(4, 256), z(4, 256), e, e, e, 2).shape == (0, 256)
    v = torch.randn(3, 256, device="cuda").half()
    out = A.shared_prefix_attention_forward(v, v, v, z(0, 256), z(0, 256), e, e, z(3, dt=torch.int32), 2)
    assert torch.equal(out, v)


def test_streams_graphs_and_repeats_give_the_same_bits():
    import attention_impl_b200 as A
    args, more, *_ = _case(700, [20, 0, 300, 5], 8, 2, 128, BF16)
    first = A.shared_prefix_attention_forward(*args, together=True)
    for _ in range(5):
        assert torch.equal(A.shared_prefix_attention_forward(*args, together=True), first)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.empty_like(first) for _ in streams]
    torch.cuda.synchronize()
    for s, o in zip(streams, outs):
        with torch.cuda.stream(s):
            A.shared_prefix_attention_forward(*args, out=o, together=True)
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    from attention_impl_b200.ops import shared_prefix_workspace_bytes
    need = shared_prefix_workspace_bytes(4, 8, 2, 128, 700, 128 ** -0.5, 1, 1, True)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.shared_prefix_attention_forward(*args, out=out, workspace=ws, together=True)
    for _ in range(3):
        out.zero_()
        ws.fill_(255)
        graph.replay()
        assert torch.equal(out, first)


def test_inputs_written_by_the_kernel_ahead():
    """The call is a programmatic dependent of what precedes it: queries and pools written just before."""
    import attention_impl_b200 as A
    args, more, *_ = _case(2000, [64] * 8, 8, 2, 128, F16)
    want = A.shared_prefix_attention_forward(*args, together=True)
    Q, K, V, Kc, Vc = (x.clone() for x in args[:5])
    for _ in range(20):
        for x, y in zip((Kc, Vc, Q, K, V), (args[3], args[4], args[0], args[1], args[2])):
            x.zero_()
            x.copy_(y)
        assert torch.equal(A.shared_prefix_attention_forward(Q, K, V, Kc, Vc, *args[5:], together=True), want)


def test_refusals():
    import attention_impl_b200 as A
    args, more, *_ = _case(100, [5, 9], 4, 2, 64, F16)
    call = lambda i=None, x=None, **kw: A.shared_prefix_attention_forward(*[x if j == i else a for j, a in enumerate(args)], **kw)  # noqa: E731
    call()
    for i, x in ((0, args[0].cpu()), (0, args[0].double()), (1, args[1][:1]), (3, args[3].bfloat16()), (4, args[4][:3]),
                 (5, args[5].long()), (5, args[5].cpu()), (6, args[6][::2]), (7, args[7][:1]), (8, 3), (3, args[3].to(E4M3))):
        with pytest.raises(RuntimeError):
            call(i, x)
    need = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    for kw in (dict(workspace=need[:64], together=True), dict(workspace=need[4:], together=True), dict(out=args[0][:1]), dict(workspace=need.cpu()),
               dict(err_flag=torch.zeros(1, device="cuda"))):
        with pytest.raises(RuntimeError):
            call(**kw)
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(i=5, x=args[5][:0])):
        call(**bad)
        with pytest.raises(RuntimeError, match="head_dim"):
            call(**bad, together=True)


@pytest.mark.parametrize("kv", ["same", "e4m3"])
def test_tensors_off_the_16_byte_grid(kv):
    import attention_impl_b200 as A
    args, more, ref, size, pt, n = _case(200, [20, 0, 30], 4, 2, 128, BF16, kv)

    def shifted(x):
        buf = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
        y = buf[1:].view(x.shape)
        y.copy_(x)
        return y
    for i in range(5):
        moved = list(args)
        moved[i] = shifted(args[i])
        close(A.shared_prefix_attention_forward(*moved, **more), ref, size, BF16, pt, n)
    out = shifted(args[0])
    A.shared_prefix_attention_forward(*args, **more, out=out)
    close(out, ref, size, BF16, pt, n)
