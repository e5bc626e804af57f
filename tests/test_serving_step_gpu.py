"""GPU: the serving operators together, as a serving loop runs them over one pair of pools: prompts in chunks and then
captured decode steps of a model with normalised queries and keys and windowed attention; and decode steps of a
batch behind one shared prefix.  Every attention output is held against the 64-bit formula on what the pools hold,
every appended row against the 64-bit norm and rotation."""
import pytest
import torch

from oracle import serving_oracle as so
from serving_helpers import BF16, E4M3, F16, close

pytestmark = pytest.mark.gpu
H, HKV, D, ROT = 4, 2, 128, 64


class _Model:
    """Random projections' outputs, norm weights and rotation tables."""

    def __init__(self, dtype, seed, max_pos=1024):
        self.g = torch.Generator().manual_seed(seed)
        self.dtype = dtype
        self.wq, self.wk = ((1 + 0.2 * torch.randn(D, generator=self.g)).to(dtype) for _ in range(2))
        ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(ROT, dtype=torch.float64) / ROT)
        self.cos, self.sin = ang.cos().to(dtype), ang.sin().to(dtype)
        self.aux = [x.cuda() for x in (self.wq, self.wk)], [x.cuda() for x in (self.cos, self.sin)]

    def qkv(self, n):
        return torch.randn(n, (H + 2 * HKV) * D, generator=self.g).to(self.dtype)

    def split(self, x):
        return x.split([H * D, HKV * D, HKV * D], 1)

    def check_rows(self, x, pos, q_out, k_rows, v_rows, scales):
        """Rotated queries and appended rows against the formula: half a step of the type, and the 32-bit share."""
        q, k, v = self.split(x)
        eps = torch.finfo(self.dtype).eps / 2
        for got, src, w, s in ((q_out, q, self.wq, None), (k_rows, k, self.wk, scales and scales[0])):
            ref, size = so.qk_norm_rope(src, w, pos, self.cos, self.sin, D, 1e-6)
            half = eps if s is None else 2.0 ** -4
            floor = 0 if s is None else 2.0 ** -10 * s.double()[:, None]
            got = got.cpu().double().view(ref.shape)
            assert ((got - ref).abs() <= half * ref.abs() + 80 * 2.0 ** -24 * size + floor + 2.0 ** -25).all()
        if scales is None:
            assert torch.equal(v_rows.cpu().double(), v.double())


def _wide(pool, scale):
    x = pool.cpu().double()
    return x if scale is None else (x.view(x.size(0), HKV, D) * scale.double()[:, None]).view(x.shape)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sinks", [(96, 4), (1, 2), (4096, 0)])
def test_windowed_model_prompts_and_decode_steps(dtype, window, sinks):
    import attention_impl_b200 as A
    m = _Model(dtype, 1)
    (wq, wk), (cos, sin) = m.aux
    B, rows = 3, 1500
    Kc, Vc = (torch.zeros(rows, HKV * D, dtype=dtype, device="cuda") for _ in range(2))
    free = torch.randperm(rows - 1, generator=m.g) + 1                   # row 0 stays free for the graph's warm-up
    slots = [torch.empty(0, dtype=torch.long) for _ in range(B)]
    used = 0
    i32 = lambda x: torch.as_tensor(x).to(torch.int32).cuda()  # noqa: E731
    for chunk in ([130, 1, 40], [70, 260, 0]):                            # prompts in two chunks
        n, past = sum(chunk), [s.numel() for s in slots]
        x = m.qkv(n)
        new = free[used:used + n].split(chunk)
        used += n
        pos = torch.cat([torch.arange(p, p + c) for p, c in zip(past, chunk)])
        slots = [torch.cat([s, t]) for s, t in zip(slots, new)]
        q, k, v = m.split(x.cuda())
        qo, ko = A.qk_norm_rope_and_cache_write(q, k, v, wq, wk, i32(pos), cos, sin, i32(torch.cat(new)), Kc, Vc, D)
        m.check_rows(x, pos, qo, Kc[torch.cat(new)], Vc[torch.cat(new)], None)
        kv_off, q_off = i32(torch.tensor([s.numel() for s in slots]).cumsum(0)), i32(torch.tensor(chunk).cumsum(0))
        o = A.paged_window_prefill_attention(qo, Kc, Vc, i32(torch.cat(slots)), kv_off, q_off, H, window, sinks, max_q_len=max(chunk))
        k64, v64 = _wide(Kc, None), _wide(Vc, None)
        ref, size = so.prefill(qo.cpu(), [k64[s] for s in slots], [v64[s] for s in slots], chunk, H, D ** -0.5, window, sinks)
        close(o, ref, size, dtype, dtype, 400)
    step = A.DecodeStepGraph(Kc, Vc, cos, sin, B, H, D, 1200, dtype=dtype, q_weight=wq, k_weight=wk, window=window, n_sinks=sinks)
    for _ in range(3):
        x = m.qkv(B)
        q, k, v = m.split(x)
        new, pos = free[used:used + B], torch.tensor([s.numel() for s in slots])
        used += B
        h = step.host
        h["q"].copy_(q), h["k"].copy_(k), h["v"].copy_(v)
        h["positions"].copy_(pos), h["new_slots"].copy_(new), h["offsets"].copy_(pos.cumsum(0))
        table = torch.cat(slots).int()
        keep = torch.cat([(torch.arange(n) < sinks) | (torch.arange(n) > n - window) for n in pos.tolist()])
        table[~keep] = -1                                                # given back
        h["cache_indices"][:table.numel()].copy_(table)
        step.upload(table.numel())
        o = step.replay()
        torch.cuda.synchronize()
        assert int(step.err_flag) == 0
        m.check_rows(x, pos, step.q, Kc[new], Vc[new], None)
        assert torch.equal(step.k, Kc[new])
        k64, v64 = _wide(Kc, None), _wide(Vc, None)
        ref, size = so.decode(step.q.cpu(), step.k.cpu(), v, [k64[s] for s in slots], [v64[s] for s in slots], H, D ** -0.5, window, sinks)
        close(o, ref, size, dtype, dtype, 400)
        slots = [torch.cat([s, t[None]]) for s, t in zip(slots, new)]


@pytest.mark.parametrize("together", [True, False])
@pytest.mark.parametrize("dtype,kv", [(F16, "same"), (BF16, "e4m3")])
def test_batch_behind_a_shared_prefix(dtype, kv, together):
    import attention_impl_b200 as A
    m = _Model(dtype, 2)
    (wq, wk), (cos, sin) = m.aux
    B, P, rows = 5, 333, 600
    scales = (torch.tensor([0.011, 0.013]), torch.tensor([0.012, 0.01])) if kv == "e4m3" else None
    pdt = E4M3 if kv == "e4m3" else dtype
    Kc, Vc = (torch.zeros(rows, HKV * D, dtype=dtype, device="cuda").to(pdt) for _ in range(2))
    sc = dict(zip(("k_scale", "v_scale"), (s.cuda() for s in scales))) if scales else {}
    free = torch.randperm(rows, generator=m.g)
    prefix, used = free[:P], P
    i32 = lambda x: torch.as_tensor(x).to(torch.int32).cuda()  # noqa: E731
    x = m.qkv(P)
    q, k, v = m.split(x.cuda())
    A.qk_norm_rope_and_cache_write(q, k, v, wq, wk, i32(torch.arange(P)), cos, sin, i32(prefix), Kc, Vc, D, **sc)
    own = [torch.empty(0, dtype=torch.long) for _ in range(B)]
    for _ in range(4):
        x = m.qkv(B)
        pos = torch.tensor([P + s.numel() for s in own])
        new = free[used:used + B]
        used += B
        q, k, v = m.split(x.cuda())
        qo, ko = A.qk_norm_rope_and_cache_write(q, k, v, wq, wk, i32(pos), cos, sin, i32(new), Kc, Vc, D, **sc)
        rows_k = _wide(Kc.view(torch.uint8)[new].view(pdt) if scales else Kc[new], scales and scales[0])
        m.check_rows(x, pos, qo, rows_k, Vc.view(torch.uint8)[new].view(pdt) if scales else Vc[new], scales)
        table, off = torch.cat(own), torch.tensor([s.numel() for s in own]).cumsum(0)
        o = A.shared_prefix_attention_forward(qo, ko, v.contiguous(), Kc, Vc, i32(prefix), i32(table), i32(off), H, together=together, **sc)
        k64, v64 = _wide(Kc, scales and scales[0]), _wide(Vc, scales and scales[1])
        seqs = [torch.cat([prefix, s]) for s in own]
        ref, size = so.decode(qo.cpu(), ko.cpu(), v.cpu(), [k64[s] for s in seqs], [v64[s] for s in seqs], H, D ** -0.5)
        close(o, ref, size, dtype, F16 if scales else dtype, 340)
        own = [torch.cat([s, t[None]]) for s, t in zip(own, new)]


def test_step_graph_arguments():
    import attention_impl_b200 as A
    m = _Model(F16, 3)
    (wq, wk), (cos, sin) = m.aux
    Kc, Vc = (torch.zeros(16, HKV * D, dtype=F16, device="cuda") for _ in range(2))
    for kw in (dict(q_weight=wq), dict(k_weight=wk), dict(n_sinks=2), dict(window=0)):
        with pytest.raises(RuntimeError):
            A.DecodeStepGraph(Kc, Vc, cos, sin, 2, H, D, 32, **kw)


def test_outputs_apart_from_what_is_read():
    """An output that shares memory with the queries, the new token's rows or a pool is refused; a neighbour is not."""
    import attention_impl_b200 as A
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    buf = torch.randn(12, HKV * D, device="cuda").to(F16)
    Q, K, V, out, Kc, Vc = buf[:2], buf[2:4], buf[4:6], buf[6:8], buf[8:10], buf[10:12]
    calls = (lambda o: A.paged_window_attention_forward(Q, K, V, Kc, Vc, i32([0, 1]), i32([1, 2]), HKV, 4, out=o),
             lambda o: A.shared_prefix_attention_forward(Q, K, V, Kc, Vc, i32([0]), i32([1]), i32([0, 1]), HKV, out=o),
             lambda o: A.paged_window_prefill_attention(Q, Kc, Vc, i32([0, 1]), i32([1, 2]), i32([1, 2]), HKV, 4, out=o, max_q_len=1))
    for n, call in enumerate(calls):
        want = call(None)
        assert torch.equal(call(out), want)
        for o in (Q, buf[1:3], Kc, Vc, buf[7:9]) + (() if n == 2 else (K, V, buf[5:7])):
            with pytest.raises(RuntimeError, match="share memory"):
                call(o)
    pos, tab, w = i32([0, 1]), torch.ones(2, D // 2, device="cuda", dtype=F16), torch.ones(D, device="cuda", dtype=F16)
    norm = lambda o: A.qk_norm_rope_and_cache_write(Q, K, V, w, w, pos, tab, tab, pos, Kc, Vc, D, out=o)  # noqa: E731
    for o in ((out, Kc), (Vc, K), (buf[9:11], K)):
        with pytest.raises(RuntimeError, match="share no memory"):
            norm(o)
    norm((out, K))
