"""GPU: chunks of sequences with a sliding window and sink tokens against the 64-bit formula.  Keys that no
query of the call sees have stale table entries and NaN in their pool rows."""
import pytest
import torch

from oracle import serving_oracle as so
from serving_helpers import BF16, F16, F32, close, offsets, pool

pytestmark = pytest.mark.gpu


def _case(q_lens, past, H, Hkv, D, dtype, window, sinks, seed=0):
    g = torch.Generator().manual_seed(seed + D + 7 * len(q_lens))
    kv_lens = [a + b for a, b in zip(q_lens, past)]
    total = sum(kv_lens)
    rows = total + 3
    Q = torch.randn(sum(q_lens), H * D, generator=g).to(dtype)
    Kc, k64, _ = pool(g, rows, Hkv, D, dtype, "same")
    Vc, v64, _ = pool(g, rows, Hkv, D, dtype, "same")
    table = torch.randperm(rows, generator=g)[:total].int()
    live, slots, at = torch.zeros(total, dtype=torch.bool), [], 0
    for q, n in zip(q_lens, kv_lens):
        slots.append(table[at:at + n].long())
        if q:
            live[at + max(0, n - q - window + 1):at + n] = True
            live[at:at + min(sinks, n)] = True
        at += n
    dead = torch.ones(rows, dtype=torch.bool)
    dead[table[live].long()] = False
    Kc[dead.cuda()] = float("nan")
    Vc[dead.cuda()] = float("nan")
    stale = table.clone()
    stale[~live] = -7
    ref, size = so.prefill(Q, [k64[s] for s in slots], [v64[s] for s in slots], q_lens, H, D ** -0.5, window, sinks)
    return [Q.cuda(), Kc, Vc, stale.cuda(), offsets(kv_lens).cuda(), offsets(q_lens).cuda(), H, window, sinks], ref, size, max(
        min(n, window + sinks) for n in kv_lens)


def _run(*a, generic=False, **kw):
    import attention_impl_b200 as A
    args, ref, size, n = _case(*a, **kw)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = A.paged_window_prefill_attention(*args, err_flag=flag, force_generic=generic)
    assert int(flag) == 0
    D, dtype = a[4], a[5]
    close(out, ref, size, dtype, F32 if generic or D not in (64, 128) or dtype == F32 else dtype, n)
    return args, out


CHUNKS = ([1, 5, 130, 300, 0, 128], [0, 40, 17, 0, 90, 500])


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (2, 0), (31, 3), (64, 4), (127, 0), (128, 0), (129, 1), (125, 4), (200, 150),
                                          (256, 4), (1000, 0), (3, 700)])
@pytest.mark.parametrize("dtype,H,Hkv,D", [(F16, 4, 2, 128), (BF16, 3, 1, 128), (BF16, 4, 4, 64)])
def test_windows_and_chunks(dtype, H, Hkv, D, window, sinks):
    _run(*CHUNKS, H, Hkv, D, dtype, window, sinks)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (2, 1), (5, 5), (8, 1), (6, 2), (10, 5), (14, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_head_layouts(H, Hkv, D):
    _run([200, 33], [60, 0], H, Hkv, D, F16, 90, 5)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [1, 33, 80, 256, 512])
def test_other_head_dims(dtype, D):
    _run([40, 1, 0, 70], [10, 33, 5, 0], 4, 2, D, dtype, 25, 3)


@pytest.mark.parametrize("D", [64, 128])
def test_generic_kernel_on_the_same_cases(D):
    _run(*CHUNKS, 4, 2, D, F16, 129, 4, generic=True)
    _run(*CHUNKS, 4, 2, D, F32, 129, 4)


@pytest.mark.parametrize("n", [1, 95, 96, 97, 127, 128, 129, 160, 161, 192, 224, 255, 256, 257, 384, 385])
def test_every_width_of_the_first_tile(n):
    """Single queries over n keys (window wider than all): lists of n entries."""
    _run([1], [n - 1], 2, 1, 128, F16, 10 ** 6, 0)
    _run([n], [0], 2, 1, 64, BF16, 10 ** 6, 0)


def test_long_prompt():
    _run([2100], [0], 4, 2, 128, BF16, 513, 4)
    _run([700], [5000], 3, 3, 128, F16, 1024, 64)


def test_window_covering_everything_is_the_plain_operator():
    import attention_impl_b200 as A
    args, out = _run([150, 33], [20, 100], 4, 4, 128, F16, 10 ** 12, 0)
    plain = A.paged_prefill_attention(*args[:6], 4)
    # both are within the roundings of P and O (half a step of fp16 each) of the exact result, whose entries and
    # sums of p |v| are below 5
    assert (out.float() - plain.float()).abs().max() <= 4 * 2.0 ** -11 * 5


def test_agrees_with_the_single_token_form():
    import attention_impl_b200 as A
    for D, dtype in ((128, F16), (64, BF16)):
        args, ref, size, n = _case([1, 1, 1], [0, 70, 400], 4, 2, D, dtype, 100, 4)
        Q, Kc, Vc, table, kv, qo, H, w, s = args
        last = kv.long() - 1
        rows = table[last].long()
        lens = torch.tensor([0, 70, 400])
        keep = torch.ones(table.numel(), dtype=torch.bool, device="cuda")
        keep[last] = False
        got = A.paged_window_attention_forward(Q, Kc[rows], Vc[rows], Kc, Vc, table[keep], lens.cumsum(0).int().cuda(), H, w, s)
        close(got, ref, size, dtype, dtype, n)
        close(A.paged_window_prefill_attention(*args), ref, size, dtype, dtype, n)


@pytest.mark.parametrize("D", [128, 64, 80])
def test_bad_slots(D):
    """Missing rows are skipped, in whole tiles, short ones and for a query that is left without any key."""
    import attention_impl_b200 as A
    args, *_ = _case([40, 200], [0, 100], 4, 2, D, F16, 150, 4)
    table = args[3].clone()
    gone = [0, 3, 41, 100, 101, 250, 339]
    table[gone] = torch.tensor([-1, 2 ** 31 - 1] * 3 + [-5], dtype=torch.int32, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = A.paged_window_prefill_attention(*args[:3], table, *args[4:], err_flag=flag)
    assert int(flag) == 1 and (got[0] == 0).all()
    Q, k, v, t = args[0].cpu().double(), args[1].cpu().double(), args[2].cpu().double(), table.cpu().long()
    for b, (q0, n, kv0, kvn) in enumerate(((0, 40, 0, 40), (40, 200, 40, 300))):
        for r in range(1 if b == 0 else 0, n, 13):
            i = kvn - n + r
            see = [kv0 + j for j in so.visible(i, 150, 4) if 0 <= int(t[kv0 + j]) < k.size(0)]
            rows = t[see]
            ref, p = so.attend(Q[q0 + r].view(4, D), k[rows].view(-1, 2, D), v[rows].view(-1, 2, D), D ** -0.5)
            size = torch.einsum("hn,nhd->hd", p, v[rows].view(-1, 2, D).abs().repeat_interleave(2, 1))
            close(got[q0 + r].view(4, D), ref, size, F16, F16, len(see))


@pytest.mark.parametrize("D", [128, 80])
def test_uncovered_rows_and_bad_offsets(D):
    import attention_impl_b200 as A
    args, ref, size, n = _case([30, 50], [0, 20], 2, 2, D, F16, 25, 2)
    Q = torch.cat([args[0], torch.ones(7, 2 * D, dtype=F16, device="cuda")])
    out = torch.full_like(Q, 5.0)
    A.paged_window_prefill_attention(Q, *args[1:], out=out)
    close(out[:80], ref, size, F16, F16, n)
    assert (out[80:] == 0).all()
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    for kv, qo in (([30, 100], [30, 500]), ([30, 20], [30, 80]), ([30, 500], [30, 80]), ([30, 100], [30, 20]), ([-3, 100], [-3, 80]),
                   ([10, 100], [30, 80])):
        flag.zero_()
        off = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (kv, qo)]
        got = A.paged_window_prefill_attention(Q, *args[1:4], *off, *args[6:], max_q_len=87, err_flag=flag)
        assert int(flag) & 4 and torch.isfinite(got).all()
    # a max_q_len that is too small: the rows within it are right, the rest is not garbage
    flag.zero_()
    got = A.paged_window_prefill_attention(*args, max_q_len=20, err_flag=flag)
    rows = torch.isfinite(got).all(1)
    assert rows.all()
    close(got[:20], ref[:20], size[:20], F16, F16, n)


def test_nothing_to_do():
    import attention_impl_b200 as A
    z = lambda *s, dt=F16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    assert A.paged_window_prefill_attention(z(0, 256), z(4, 256), z(4, 256), i(), i(), i(), 2, 8).shape == (0, 256)
    for D in (128, 80):
        out = A.paged_window_prefill_attention(torch.ones(3, 2 * D, dtype=F16, device="cuda"), z(4, 2 * D), z(4, 2 * D), i(), i(0, 0), i(0, 0), 2, 8)
        assert (out == 0).all()
        out = A.paged_window_prefill_attention(torch.ones(3, 2 * D, dtype=F16, device="cuda"), z(4, 2 * D), z(4, 2 * D), i(), i(), i(), 2, 8)
        assert (out == 0).all()


def test_streams_graphs_and_repeats_give_the_same_bits():
    import attention_impl_b200 as A
    args, ref, size, n = _case([300, 77, 129], [100, 0, 300], 4, 2, 128, BF16, 200, 4)
    first = A.paged_window_prefill_attention(*args)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.empty_like(first) for _ in streams]
    torch.cuda.synchronize()
    for s, o in zip(streams, outs):
        with torch.cuda.stream(s):
            A.paged_window_prefill_attention(*args, max_q_len=300, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    out = torch.zeros_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.paged_window_prefill_attention(*args, max_q_len=300, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, first)


def test_scales():
    import attention_impl_b200 as A
    args, *_ = _case([60], [30], 2, 1, 128, F16, 50, 2)
    Q, k, v, t = args[0].cpu(), args[1].cpu(), args[2].cpu(), args[3].cpu().long()
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    for scale in (0.5, 1e-3, 0.0, -0.1):
        got = A.paged_window_prefill_attention(*args, scale=scale)
        ref, size = so.prefill(Q, [k[t.clamp(min=0)]], [v[t.clamp(min=0)]], [60], 2, scale, 50, 2)
        # scores up to 0.5 * 60: the 32-bit share of the bound grows with them
        close(got, ref, size * (1 + 3 * (scale == 0.5)), F16, F16, 52)


def test_refusals():
    import attention_impl_b200 as A
    args, *_ = _case([9, 20], [3, 0], 4, 2, 64, F16, 8, 1)
    call = lambda i=None, x=None, **kw: A.paged_window_prefill_attention(*[x if j == i else a for j, a in enumerate(args)], **kw)  # noqa: E731
    call()
    for i, x in ((0, args[0].cpu()), (0, args[0].double()), (0, args[0].t()), (1, args[1].float()), (1, args[1][:, :100].contiguous()),
                 (2, args[2][:2]), (3, args[3].long()), (4, args[4][:1]), (5, args[5].long()), (6, 3), (6, 0), (7, 0), (7, -3), (8, -1),
                 (1, args[1].to(torch.float8_e4m3fn)), (5, args[5].cpu())):
        with pytest.raises(RuntimeError):
            call(i, x)
    for kw in (dict(out=args[0][:3]), dict(out=args[0].float()), dict(max_q_len=-1), dict(err_flag=torch.zeros(1, device="cuda"))):
        with pytest.raises(RuntimeError):
            call(**kw)
    big = torch.zeros(2, 4 * 520, dtype=F16, device="cuda")
    with pytest.raises(RuntimeError, match="head_dim"):
        A.paged_window_prefill_attention(big, big, big, args[3], args[4] * 0, args[5] * 0, 4, 4, max_q_len=2)


def test_many_sequences():
    """More sequences than the item list looks at at a time, empty ones and one-token chunks among them, a long tail of
    rows that belong to nobody."""
    import attention_impl_b200 as A
    g = torch.Generator().manual_seed(8)
    q = [int(x) for x in torch.randint(0, 4, (150,), generator=g)]
    q[3], q[40], q[149] = 300, 129, 140
    past = torch.randint(0, 60, (150,), generator=g).tolist()
    args, ref, size, n = _case(q, past, 2, 1, 64, F16, 40, 3)
    Q = torch.cat([args[0], torch.full((3000, 128), 7.0, dtype=F16, device="cuda")])
    out = A.paged_window_prefill_attention(Q, *args[1:], out=torch.full_like(Q, float("nan")))
    close(out[:sum(q)], ref, size, F16, F16, n)
    assert (out[sum(q):] == 0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_tensors_off_the_16_byte_grid(D):
    import attention_impl_b200 as A
    args, ref, size, n = _case([50, 200], [30, 0], 4, 2, D, BF16, 70, 4)

    def shifted(x):
        buf = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
        y = buf[1:].view(x.shape)
        y.copy_(x)
        return y
    for i in range(3):
        moved = list(args)
        moved[i] = shifted(args[i])
        close(A.paged_window_prefill_attention(*moved), ref, size, BF16, BF16, n)
    out = shifted(args[0])
    A.paged_window_prefill_attention(*args, out=out)
    close(out, ref, size, BF16, BF16, n)


@pytest.mark.parametrize("D,dtype", [(128, F16), (64, BF16), (80, F16)])
def test_not_a_number_reaches_only_who_sees_it(D, dtype):
    """Infinities and NaN in K and V of tokens that later queries, earlier queries (left behind by the window), or only
    some heads see."""
    import attention_impl_b200 as A
    q, past, H, Hkv, w, s = [200, 90], [40, 10], 4, 2, 50, 3
    args, *_ = _case(q, past, H, Hkv, D, dtype, w, s)
    Q, Kc, Vc, table = args[:4]
    clean = A.paged_window_prefill_attention(*args)
    t = table.long()
    for kv_at, pool, value in ((120, Vc, float("inf")), (200, Vc, float("nan")), (130, Kc, float("nan")), (1, Vc, -float("inf"))):
        row = int(t[kv_at])
        old = pool[row].clone()
        pool[row, :D] = value                                  # KV head 0: query heads 0 and 1, sequence 0
        got = A.paged_window_prefill_attention(*args)
        pool[row] = old
        pos = torch.arange(40, 240, device="cuda")
        sees = (pos >= kv_at) & ((kv_at > pos - w) | (kv_at < s))
        hit = torch.zeros(290, H * D, dtype=torch.bool, device="cuda")
        hit[:200][sees, :2 * D] = True
        assert not torch.isfinite(got[hit]).any() and hit.any()
        # the others: the same values, to the roundings of P (a row of the tile may have been computed by itself)
        size = float(Vc[torch.isfinite(Vc).all(1)].abs().max())
        assert (got[~hit].float() - clean[~hit].float()).abs().max() <= 4 * torch.finfo(dtype).eps / 2 * size
