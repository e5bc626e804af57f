"""GPU: single-token attention with a sliding window and sink tokens against the 64-bit formula.

Everything outside a sequence's span is poisoned: its table entries point outside the pools and its pool
rows hold NaN, so any read of them shows."""
import math

import pytest
import torch

from oracle import serving_oracle as so
from serving_helpers import BF16, E4M3, F16, F32, close, offsets, pool

pytestmark = pytest.mark.gpu


def _case(lens, H, Hkv, D, dtype, kv, window, sinks, block=1, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * len(lens) + D)
    B = len(lens)
    Q, K, V = (torch.randn(B, n * D, generator=g).to(dtype) for n in (H, Hkv, Hkv))
    seen = [torch.tensor([t < sinks or t > n - window for t in range(n)], dtype=torch.bool) for n in lens]
    if block == 1:
        total = sum(lens)
        rows = total + 5
        table = torch.randperm(rows, generator=g)[:total].int()
        slots, at = [], 0
        for n in lens:
            slots.append(table[at:at + n].long())
            at += n
    else:
        most = max(1, -(-max(lens) // block)) + 1
        rows = B * most * block
        table = torch.randperm(B * most, generator=g).int().view(B, most)
        slots = [table[b].long()[torch.arange(n) // block] * block + torch.arange(n) % block for b, n in enumerate(lens)]
    Kc, k64, ks = pool(g, rows, Hkv, D, dtype, kv)
    Vc, v64, vs = pool(g, rows, Hkv, D, dtype, kv)
    # poison
    dead = torch.ones(rows, dtype=torch.bool)
    for s, m in zip(slots, seen):
        dead[s[m]] = False
    for p in (Kc, Vc):
        p.view(torch.uint8 if kv == "e4m3" else p.dtype)[dead.cuda()] = 0x7f if kv == "e4m3" else float("nan")
    table = table.clone()
    if block == 1:
        table[~torch.cat(seen)] = 2 ** 31 - 1
    else:
        for b, (n, m) in enumerate(zip(lens, seen)):
            for i in range(table.size(1)):
                if not m[i * block:(i + 1) * block].any():
                    table[b, i] = -7
    ref, size = so.decode(Q, K, V, [k64[s] for s in slots], [v64[s] for s in slots], H, D ** -0.5, window, sinks)
    args = [Q.cuda(), K.cuda(), V.cuda(), Kc, Vc, table.cuda(), offsets(lens).cuda(), H, window, sinks]
    return args, dict(k_scale=ks, v_scale=vs, block_size=block), ref, size, F32 if dtype == F32 or D not in (64, 128, 256) else (
        F16 if kv == "e4m3" else dtype), max(min(n, window + sinks) for n in lens) + 1


def _run(*a, **kw):
    import attention_impl_b200 as A
    args, more, ref, size, pt, n = _case(*a, **kw)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = A.paged_window_attention_forward(*args, **more, err_flag=flag)
    assert int(flag) == 0
    close(out, ref, size, args[0].dtype, pt, n)
    return args, more, out


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 200, 333]


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (2, 1), (16, 0), (17, 4), (64, 4), (100, 33), (333, 0), (334, 4),
                                          (1000, 7), (5, 400)])
@pytest.mark.parametrize("dtype,kv", [(F16, "same"), (BF16, "same"), (F16, "e4m3"), (BF16, "e4m3")])
def test_windows_and_lengths(dtype, kv, window, sinks):
    _run(LENS, 8, 2, 128, dtype, kv, window, sinks)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 4), (5, 5), (3, 1), (7, 1), (8, 1), (9, 1), (16, 1), (20, 4), (34, 2), (6, 6), (12, 3)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kv", ["same", "e4m3"])
def test_head_layouts(H, Hkv, D, kv):
    _run([40, 7, 150], H, Hkv, D, F16, kv, 70, 4)


@pytest.mark.parametrize("dtype,kv", [(F32, "same"), (F16, "same"), (BF16, "e4m3")])
@pytest.mark.parametrize("D", [1, 2, 33, 80, 96, 160, 512])
def test_other_head_dims(dtype, kv, D):
    _run([0, 3, 90, 41], 4, 2, D, dtype, kv, 50, 2)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_fp32(D):
    _run([0, 3, 90, 300], 4, 4, D, F32, "same", 130, 4)


@pytest.mark.parametrize("block", [2, 7, 16, 64])
@pytest.mark.parametrize("kv,D", [("same", 128), ("e4m3", 64), ("same", 96)])
def test_block_tables(block, kv, D):
    _run(LENS, 4, 2, D, F16, kv, 77, 5, block=block)


@pytest.mark.parametrize("B", [1, 2, 40, 130])
def test_batches(B):
    """Every split of the launcher: few sequences (clusters of many CTAs) to many."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 260 if B > 2 else 3000, (B,), generator=g).tolist()
    _run(lens, 8, 4, 64, BF16, "same", 200 if B > 2 else 2500, 4, seed=B)


def test_long_context_one_sequence():
    _run([40000], 8, 1, 128, F16, "same", 8192, 4)


def test_window_covering_everything_is_the_plain_operator():
    import attention_impl_b200 as A
    args, more, out = _run([0, 5, 100, 250], 8, 8, 128, F16, "same", 10 ** 12, 0)
    S, P, O = A.paged_kv_attention_forward(*args[:7], 8, return_sp=False)
    # each is within the bound of its own roundings of the exact result: two halves of fp16 for O, P on one side
    assert (out.float() - O.float()).abs().max() <= 4 * 2.0 ** -11 * float(args[2].abs().max())


def test_every_cached_score_far_below_and_far_above_the_current_one():
    """Keys that the softmax drops, and a current token that it drops."""
    import attention_impl_b200 as A
    for sign in (1.0, -1.0):
        D, n = 128, 50
        q = torch.ones(1, D, dtype=F16)
        kc = (torch.ones(n, D) * 8 * sign).half()
        vc = torch.randn(n, D, generator=torch.Generator().manual_seed(1)).half()
        k, v = (-q * 8 * sign), torch.full((1, D), 2.0, dtype=F16)
        out = A.paged_window_attention_forward(q.cuda(), k.cuda(), v.cuda(), kc.cuda(), vc.cuda(),
                                               torch.arange(n).int().cuda(), torch.tensor([n]).int().cuda(), 1, n + 1)
        ref, size = so.decode(q, k, v, [kc], [vc], 1, D ** -0.5)
        close(out, ref, size, F16, F16, n)


def test_nan_and_infinity_in_the_span_only():
    """A NaN inside the span reaches its own sequence and KV head; +inf V is inf, and nothing else changes."""
    import attention_impl_b200 as A
    args, more, ref, size, pt, n = _case([60, 60, 60], 4, 2, 128, F16, "same", 30, 2)
    clean = A.paged_window_attention_forward(*args, **more)
    row = int(args[5][60 + 45])                        # sequence 1, inside its window
    args[3][row, :128] = float("nan")                  # KV head 0
    got = A.paged_window_attention_forward(*args, **more)
    assert torch.isnan(got[1, :256]).all() and torch.equal(got[1, 256:], clean[1, 256:])
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    args[3][row, :128] = 0
    args[4][row, 3] = float("inf")
    got = A.paged_window_attention_forward(*args, **more)
    assert torch.isinf(got[1, [3, 131]]).all()
    rest = torch.ones(512, dtype=torch.bool)
    rest[[3, 131]] = False
    assert torch.isfinite(got[1, rest.cuda()]).all()


def test_bf16_queries_of_any_size_over_8_bit_pools():
    """q up to 1e30 and down to 1e-30 (keys scaled the other way): the products run in fp16 after a power of two."""
    import attention_impl_b200 as A
    args, more, ref, size, pt, n = _case([70, 20], 4, 2, 64, BF16, "e4m3", 50, 2)
    for e in (2.0 ** 90, 2.0 ** -90):
        big = [args[0] * e, args[1] * 0, *args[2:]]
        base = [args[0], args[1] * 0, *args[2:]]
        a = A.paged_window_attention_forward(*base, **more, scale=0.1)
        b = A.paged_window_attention_forward(*big, **more, scale=0.1 / e)
        # the same roundings; scale / e is the same number but for its 24 bits, and scores are at most about 30
        assert (a.float() - b.float()).abs().max() <= 2 * 2.0 ** -8 * float(a.abs().max())


def test_bad_slots_and_offsets():
    import attention_impl_b200 as A
    for D in (128, 96):
        args, more, ref, size, pt, n = _case([40, 30, 20], 4, 2, D, F16, "same", 100, 0)
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        table, rows = args[5].clone(), args[3].size(0)
        table[[3, 50]] = torch.tensor([-1, rows], dtype=torch.int32, device="cuda")
        got = A.paged_window_attention_forward(*args[:5], table, *args[6:], err_flag=flag)
        assert int(flag) == 1
        k64, v64 = args[3].cpu().double(), args[4].cpu().double()
        t = args[5].cpu().long()
        keep = [[i for i in range(0, 40) if i != 3], [i for i in range(40, 70) if i != 50], list(range(70, 90))]
        ref, size = so.decode(args[0].cpu(), args[1].cpu(), args[2].cpu(), [k64[t[i]] for i in keep], [v64[t[i]] for i in keep], 4,
                              D ** -0.5)
        close(got, ref, size, F16, pt, 41)
        # decreasing offsets, offsets past the table: those sequences count as empty
        flag.zero_()
        off = torch.tensor([40, 30, 91], dtype=torch.int32, device="cuda")
        got = A.paged_window_attention_forward(*args[:6], off, *args[7:], err_flag=flag)
        assert int(flag) == 4
        V = args[2].view(3, 2, 1, D).expand(3, 2, 2, D).reshape(3, 4 * D)
        assert torch.equal(got[1:], V[1:])


def test_no_sequences_and_empty_pools():
    import attention_impl_b200 as A
    z = lambda *s, dt=F16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    out = A.paged_window_attention_forward(z(0, 256), z(0, 256), z(0, 256), z(4, 256), z(4, 256), z(0, dt=torch.int32),
                                           z(0, dt=torch.int32), 2, 8)
    assert out.shape == (0, 256)
    for D in (128, 96):
        v = torch.randn(3, 2 * D, device="cuda").half()
        out = A.paged_window_attention_forward(v, v, v, z(0, 2 * D), z(0, 2 * D), z(0, dt=torch.int32), z(3, dt=torch.int32), 2, 8)
        assert torch.equal(out, v)


def test_pool_offsets_beyond_32_bits():
    import attention_impl_b200 as A
    rows = (1 << 31) // 2048 + 100
    g = torch.Generator().manual_seed(3)
    Kc, Vc = (torch.zeros(rows, 2048, dtype=F16, device="cuda") for _ in range(2))
    k, v = (torch.randn(40, 2048, generator=g).half() for _ in range(2))
    Kc[-40:], Vc[-40:] = k.cuda(), v.cuda()
    Q, K, V = (torch.randn(1, 2048, generator=g).half() for _ in range(3))
    table = torch.arange(rows - 40, rows).int()
    out = A.paged_window_attention_forward(Q.cuda(), K.cuda(), V.cuda(), Kc, Vc, table.cuda(), torch.tensor([40]).int().cuda(), 16, 31, 2)
    ref, size = so.decode(Q, K, V, [k], [v], 16, 128 ** -0.5, 31, 2)
    close(out, ref, size, F16, F16, 41)


def test_streams_graphs_and_repeats_give_the_same_bits():
    import attention_impl_b200 as A
    args, more, ref, size, pt, n = _case([500, 3, 90, 250], 8, 2, 128, BF16, "same", 300, 4)
    first = A.paged_window_attention_forward(*args, **more)
    for _ in range(5):
        assert torch.equal(A.paged_window_attention_forward(*args, **more), first)
    outs, streams = [torch.empty_like(first) for _ in range(3)], [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for o, s in zip(outs, streams):
        with torch.cuda.stream(s):
            A.paged_window_attention_forward(*args, **more, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    out = torch.zeros_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.paged_window_attention_forward(*args, **more, out=out)
    # lengths come from the device: shorter sequences in the same tables' capacity
    lens = [400, 3, 100, 250]
    args2, more2, ref2, size2, _, _ = _case(lens, 8, 2, 128, BF16, "same", 300, 4, seed=9)
    graph.replay()
    assert torch.equal(out, first)
    args[0].copy_(args2[0]); args[1].copy_(args2[1]); args[2].copy_(args2[2])
    args[5][:sum(lens)].copy_(args2[5]); args[6].copy_(args2[6])
    args[3][:args2[3].size(0)].copy_(args2[3]); args[4][:args2[4].size(0)].copy_(args2[4])
    graph.replay()
    close(out, ref2, size2, BF16, BF16, n)


def test_refusals():
    import attention_impl_b200 as A
    args, more, *_ = _case([5, 9], 4, 2, 64, F16, "same", 4, 1)
    call = lambda i=None, x=None, **kw: A.paged_window_attention_forward(*[x if j == i else a for j, a in enumerate(args)], **kw)  # noqa: E731
    call()
    for i, x in ((0, args[0].cpu()), (0, args[0].double()), (0, args[0].t()), (1, args[1][:1]),
                 (1, args[1].bfloat16()), (3, args[3].bfloat16()), (3, args[3][:, :96].contiguous()), (4, args[4][:3]),
                 (5, args[5].long()), (5, args[5][::2]), (6, args[6][:1]), (6, args[6].long()), (7, 3), (7, 0), (8, 0), (8, -1),
                 (8, 2.5), (9, -1), (3, args[3].to(E4M3)), (6, args[6].cpu())):
        with pytest.raises(RuntimeError):
            call(i, x)
    for kw in (dict(block_size=0), dict(block_size=16), dict(out=torch.empty(2, 128, dtype=F16, device="cuda")),
               dict(out=args[0].float()), dict(err_flag=torch.zeros(1, device="cuda")), dict(err_flag=torch.zeros(1).int())):
        with pytest.raises(RuntimeError):
            call(**kw)
    big = torch.zeros(2, 4 * 520, dtype=F16, device="cuda")
    with pytest.raises(RuntimeError, match="head_dim"):
        A.paged_window_attention_forward(big, big, big, big, big, args[5], args[6] * 0, 4, 4)


@pytest.mark.parametrize("kv", ["same", "e4m3"])
def test_tensors_off_the_16_byte_grid(kv):
    import attention_impl_b200 as A
    args, more, ref, size, pt, n = _case([70, 200], 4, 2, 128, F16, kv, 90, 4)

    def shifted(x):
        buf = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
        y = buf[1:].view(x.shape)
        y.copy_(x)
        return y
    for i in range(5):
        moved = list(args)
        moved[i] = shifted(args[i])
        close(A.paged_window_attention_forward(*moved, **more), ref, size, F16, pt, n)
    out = shifted(args[0])
    A.paged_window_attention_forward(*args, **more, out=out)
    close(out, ref, size, F16, pt, n)


FIRST_CALLS = """
import torch
import attention_impl_b200 as A
D, H = 128, 4
t = lambda *s: torch.randn(*s, device="cuda").half()
i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
q, k, kc = t(4, H * D), t(4, 2 * D), t(300, 2 * D)
w, c = torch.ones(D, device="cuda").half(), torch.ones(64, 64, device="cuda").half()
table, prefix, off, pos = torch.arange(40, device="cuda").int(), torch.arange(100, 300, device="cuda").int(), i(10, 20, 30, 40), i(0, 1, 2, 3)
calls = [lambda: A.qk_norm_rope(q, k, w, w, pos, c, c, D)[0],
         lambda: A.paged_window_attention_forward(q, k, k, kc, kc, table, off, H, 8, 2),
         None,
         lambda: A.shared_prefix_attention_forward(q, k, k, kc, kc, prefix, table, off, H)]
pos1 = pos + 1
calls[2] = lambda: A.paged_window_prefill_attention(q, kc, kc, table, off, pos1, H, 8, 2, max_q_len=1)
torch.cuda.synchronize()
got = []
for call in calls:                       # the very first call of each is the captured one
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    graph.replay()
    torch.cuda.synchronize()
    got.append(out.clone())
for call, x in zip(calls, got):
    assert torch.equal(call(), x)
print("captured first calls agree")
"""


def test_first_call_of_a_process_may_be_a_captured_one():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "agree" in r.stdout, r.stderr[-2000:]
