"""What is measured of the serving operators: per-head query/key norm with rotation and cache append,
attention with a sliding window and sink tokens (one token and whole chunks), and decoding of a batch
that shares one long prefix.

Where ``own`` is false ``run`` computes the operators in elementary torch operations in 32 bits;
where it is true it makes the calls a serving loop makes of ``attention_impl_b200``.
"""
import math
import random

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn


# ----------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of eight sequences, multi-head: nothing but latency
        dict(name="norm_rope step of 8", op="norm_rope", tokens=8, hq=32, hk=32, d=128, rot=64, dtype="fp16", write="same",
             packed=False),
        # a prefill chunk out of one packed q|k|v projection, half of each head rotated, 8-bit pools
        dict(name="norm_rope chunk e4m3", op="norm_rope", tokens=1801, hq=32, hk=8, d=128, rot=32, dtype="bf16",
             write="e4m3", packed=True),
        # the rotation workload's shape: a whole packed prompt batch, no cache behind it
        dict(name="norm_rope 16384 tokens", op="norm_rope", tokens=16384, hq=32, hk=32, d=128, rot=64, dtype="fp16",
             write="none", packed=False),
        # a small batch of short sequences: every call is latency
        dict(name="window step of 8", op="window_decode", b=8, h=32, hkv=32, d=128, dtype="fp16", kv="same", ctx_lo=1,
             ctx_hi=1000, window=512, sinks=4, block=1),
        # one long conversation, narrow heads
        dict(name="window step of 1 long", op="window_decode", b=1, h=32, hkv=8, d=64, dtype="bf16", kv="same",
             ctx_lo=40000, ctx_hi=40000, window=8192, sinks=4, block=1),
        # a full batch of long contexts, grouped-query heads
        dict(name="window step of 64", op="window_decode", b=64, h=32, hkv=8, d=128, dtype="bf16", kv="same", ctx_lo=1024,
             ctx_hi=32768, window=4096, sinks=4, block=1),
        # 8-bit pools behind a block table, an odd window
        dict(name="window step of 33 e4m3", op="window_decode", b=33, h=32, hkv=8, d=128, dtype="fp16", kv="e4m3", ctx_lo=1,
             ctx_hi=40000, window=1023, sinks=1, block=16),
        # short chunks of three requests behind cached prefixes of different lengths
        dict(name="window chunks of 3", op="window_prefill", b=3, h=32, hkv=8, d=128, dtype="fp16", q_lo=1, q_hi=500,
             past_lo=0, past_hi=3000, window=256, sinks=4),
        # whole prompts
        dict(name="window prompts of 4", op="window_prefill", b=4, h=32, hkv=8, d=128, dtype="bf16", q_lo=3500, q_hi=4500,
             past_lo=0, past_hi=0, window=1024, sinks=4),
        # a small batch behind one system prompt, multi-head
        dict(name="prefix 1025 batch 8", op="shared_prefix", b=8, h=32, hkv=32, d=128, dtype="fp16", kv="same", prefix=1025,
             own_lo=0, own_hi=64),
        # a full batch of questions on one long document
        dict(name="prefix 32768 batch 64", op="shared_prefix", b=64, h=32, hkv=8, d=128, dtype="bf16", kv="same",
             prefix=32768, own_lo=16, own_hi=1024),
        # the same with 8-bit pools
        dict(name="prefix 8191 batch 48 e4m3", op="shared_prefix", b=48, h=32, hkv=8, d=128, dtype="fp16", kv="e4m3",
             prefix=8191, own_lo=0, own_hi=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "window_decode", "window_prefill", "shared_prefix"])
    if op == "norm_rope":
        d = rng.choice([64, 96, 128, 256])
        hk = rng.choice([1, 2, 4, 5, 8, 16])
        hq = hk * rng.choice([1, 2, 3, 4, 7, 8])
        dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        most = 16384 * 64 * 128 // ((hq + 2 * hk) * d)
        return dict(op=op, tokens=_log(rng, 1, min(most, 20000)), hq=hq, hk=hk, d=d, rot=rng.choice([d // 2, d // 2, d // 4, 8]),
                    dtype=dtype, write=rng.choice(["none", "same", "same", "e4m3"] if dtype != "fp32" else ["none", "same"]),
                    packed=rng.random() < 0.5)
    if op == "window_decode":
        d = rng.choice([64, 128, 128, 256])
        hkv = rng.choice([1, 2, 4, 5, 8, 16, 32])
        h = hkv * rng.choice([1, 2, 3, 4, 7, 8] if hkv <= 8 else [1, 2])
        lo = _log(rng, 1, 30000)
        window = _log(rng, 1, 8192)
        b = _log(rng, 1, 128)
        while b > 1 and b * min(lo + 20000, window + 64) * hkv * d > 64 * 4100 * 1024 or b * (lo + 20000) * hkv * d > 4e9:
            b = b // 2
        return dict(op=op, b=max(b, 1), h=h, hkv=hkv, d=d, dtype=rng.choice(["fp16", "bf16"]),
                    kv=rng.choice(["same", "same", "e4m3"]), ctx_lo=rng.choice([0, 1, lo]), ctx_hi=lo + _log(rng, 1, 20000),
                    window=window, sinks=rng.choice([0, 1, 4, 4, 16, 64]), block=rng.choice([1, 1, 16, 64]))
    if op == "window_prefill":
        hkv = rng.choice([1, 2, 4, 8])
        h = hkv * rng.choice([1, 2, 3, 4])
        hi = _log(rng, 1, 4500)
        return dict(op=op, b=rng.randint(1, 4), h=h, hkv=hkv, d=rng.choice([64, 128, 128]), dtype=rng.choice(["fp16", "bf16"]),
                    q_lo=rng.choice([0, 1, hi // 2 + 1]), q_hi=hi, past_lo=0, past_hi=rng.choice([0, _log(rng, 1, 5000)]),
                    window=_log(rng, 1, 2048), sinks=rng.choice([0, 1, 4, 4, 33, 130]))
    hkv = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 3, 4, 8])
    return dict(op=op, b=_log(rng, 1, 64), h=hkv * g if hkv * g <= 32 else 32, hkv=hkv, d=rng.choice([64, 128, 128]),
                dtype=rng.choice(["fp16", "bf16"]), kv=rng.choice(["same", "same", "e4m3"]), prefix=_log(rng, 1, 32768),
                own_lo=0, own_hi=_log(rng, 1, 1024))


def _lengths(count, lo, hi, salt):
    """Ragged lengths of a case: the same for every seed, both ends among them, so that ``work`` knows them."""
    r = random.Random(1000 * salt + 17 * lo + hi)
    got = [r.randint(lo, hi) for _ in range(count)]
    got[-1] = hi
    if count > 1:
        got[0] = lo
    return got


# ----------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------
def _normal(gen, rows, cols, dtype):
    out = torch.empty(rows, cols, dtype=dtype, device="cuda")
    return out.normal_(generator=gen)


def _pool(gen, rows, hkv, d, dtype, kv):
    """(K or V pool, per-head scales or None): N(0, 1) rows, in 8 bits as codes of x / (absmax / 448)."""
    if kv == "same":
        return _normal(gen, rows, hkv * d, dtype), None
    scale = torch.full((hkv,), 5.5 / 448, device="cuda") * torch.linspace(0.9, 1.1, hkv, device="cuda")
    x = _normal(gen, rows, hkv * d, torch.float16).view(rows, hkv, d)
    return (x / scale.to(torch.float16)[:, None]).clamp_(-448, 448).to(E4M3).view(rows, hkv * d), scale


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _running(values):
    total, out = 0, []
    for v in values:
        total += v
        out.append(total)
    return out


def _angles(d_rot, length, dtype):
    freq = 10000.0 ** (-torch.arange(d_rot, dtype=torch.float64, device="cuda") / d_rot)
    ang = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * freq
    return ang.cos().to(dtype), ang.sin().to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    perm = lambda n: torch.randperm(n, generator=gen, device="cuda").to(torch.int32)  # noqa: E731
    s = dict(case)
    dt = TYPES[case["dtype"]]
    if case["op"] == "norm_rope":
        n, hq, hk, d = case["tokens"], case["hq"], case["hk"], case["d"]
        if case["packed"]:
            qkv = _normal(gen, n, (hq + 2 * hk) * d, dt)
            s["q"], s["k"], s["v"] = qkv[:, :hq * d], qkv[:, hq * d:(hq + hk) * d], qkv[:, (hq + hk) * d:]
        else:
            s["q"], s["k"], s["v"] = (_normal(gen, n, h * d, dt) for h in (hq, hk, hk))
        s["wq"], s["wk"] = ((1 + 0.2 * _normal(gen, 1, d, torch.float32)[0]).to(dt) for _ in range(2))
        s["cos"], s["sin"] = _angles(case["rot"], 8192, dt)
        s["positions"] = torch.randint(0, 8192, (n,), generator=gen, device="cuda").to(torch.int32)
        if case["write"] != "none":
            rows = n + n // 4 + 1
            s["slots"] = perm(rows)[:n].contiguous()
            pdt = E4M3 if case["write"] == "e4m3" else dt
            s["kc"], s["vc"] = (torch.zeros(rows, hk * d, dtype=dt, device="cuda").to(pdt) for _ in range(2))
            s["ks"] = s["vs"] = None
            if case["write"] == "e4m3":
                s["ks"], s["vs"] = (torch.full((hk,), 6.0 / 448, device="cuda") for _ in range(2))
        return s
    h, hkv, d, b = case["h"], case["hkv"], case["d"], case["b"]
    if case["op"] == "window_decode":
        lens = _lengths(b, case["ctx_lo"], case["ctx_hi"], 1)
        s["longest"] = max(lens)
        bs = case["block"]
        if bs == 1:
            rows = sum(lens) + 1
            s["table"] = perm(rows)[:sum(lens)].contiguous()
        else:
            most = -(-max(max(lens), 1) // bs)
            rows = b * most * bs
            s["table"] = perm(b * most).view(b, most)
        s["offsets"] = _int(_running(lens))
    elif case["op"] == "window_prefill":
        q_lens, past = _lengths(b, case["q_lo"], case["q_hi"], 2), _lengths(b, case["past_lo"], case["past_hi"], 3)
        kv_lens = [x + y for x, y in zip(q_lens, past)]
        s["q_lens"], s["kv_lens"], s["max_q"] = q_lens, kv_lens, max(q_lens)
        s["q_offsets"], s["kv_offsets"] = _int(_running(q_lens)), _int(_running(kv_lens))
        rows = sum(kv_lens) + 1
        s["table"] = perm(rows)[:sum(kv_lens)].contiguous()
        s["q"] = _normal(gen, sum(q_lens), h * d, dt)
        s["kc"], s["vc"] = (_pool(gen, rows, hkv, d, dt, "same")[0] for _ in range(2))
        return s
    else:
        lens = _lengths(b, case["own_lo"], case["own_hi"], 4)
        s["longest"] = max(lens)
        rows = case["prefix"] + sum(lens) + 1
        p = perm(rows)
        s["prefix_table"] = p[:case["prefix"]].contiguous()
        s["table"] = p[case["prefix"]:case["prefix"] + sum(lens)].contiguous()
        s["offsets"] = _int(_running(lens))
    s["q"], s["k"], s["v"] = (_normal(gen, b, n * d, dt) for n in (h, hkv, hkv))
    (s["kc"], s["ks"]), (s["vc"], s["vs"]) = (_pool(gen, rows, hkv, d, dt, case["kv"]) for _ in range(2))
    return s


# ----------------------------------------------------------------------------------------------
# the calls, and the plain forms
# ----------------------------------------------------------------------------------------------
def run(s):
    if s["op"] == "norm_rope":
        q, k = _own_norm_rope(s) if own else _norm_rope(s)
        return [q, k] if s["write"] == "none" else [q, k, s["kc"], s["vc"]]
    if s["op"] == "window_decode":
        return _own_window_decode(s) if own else _window_decode(s)
    if s["op"] == "window_prefill":
        return _own_window_prefill(s) if own else _window_prefill(s)
    return _own_shared_prefix(s) if own else _shared_prefix(s)


def _own_norm_rope(s):
    import attention_impl_b200 as A
    if s["write"] == "none":
        return A.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["positions"], s["cos"], s["sin"], s["d"])
    return A.qk_norm_rope_and_cache_write(s["q"], s["k"], s["v"], s["wq"], s["wk"], s["positions"], s["cos"], s["sin"],
                                          s["slots"], s["kc"], s["vc"], s["d"], k_scale=s["ks"], v_scale=s["vs"])


def _own_window_decode(s):
    import attention_impl_b200 as A
    return A.paged_window_attention_forward(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["table"], s["offsets"], s["h"],
                                            s["window"], s["sinks"], k_scale=s["ks"], v_scale=s["vs"], block_size=s["block"])


def _own_window_prefill(s):
    import attention_impl_b200 as A
    return A.paged_window_prefill_attention(s["q"], s["kc"], s["vc"], s["table"], s["kv_offsets"], s["q_offsets"], s["h"],
                                            s["window"], s["sinks"], max_q_len=s["max_q"])


def _own_shared_prefix(s):
    import attention_impl_b200 as A
    return A.shared_prefix_attention_forward(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["prefix_table"], s["table"],
                                             s["offsets"], s["h"], k_scale=s["ks"], v_scale=s["vs"])


def _rotate(x, w, cos, sin, d):
    """RMS norm of every head, times w, then the rotation of its first 2 * rot dims; 32 bits."""
    x = x.reshape(x.size(0), -1, d).float()
    x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.float()
    r = cos.size(-1)
    a, b = x[..., :r], x[..., r:2 * r]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * r:]], -1)


def _norm_rope(s):
    pos = s["positions"].long()
    cos, sin = s["cos"][pos].float()[:, None], s["sin"][pos].float()[:, None]
    dt, d = s["q"].dtype, s["d"]
    q, k = _rotate(s["q"], s["wq"], cos, sin, d), _rotate(s["k"], s["wk"], cos, sin, d)
    if s["write"] != "none":
        _append(s["kc"], k, s["slots"].long(), s["ks"])
        _append(s["vc"], s["v"].reshape(k.shape), s["slots"].long(), s["vs"])
    return q.flatten(1).to(dt), k.flatten(1).to(dt)


def _append(pool, x, slots, scale):
    if scale is None:
        pool[slots] = x.flatten(1).to(pool.dtype)
    else:
        codes = (x.float() / scale[:, None]).clamp(-448, 448).to(pool.dtype)
        pool.view(torch.uint8)[slots] = codes.flatten(1).view(torch.uint8)


def _rows(pool, slots, scale, hkv, d):
    """Pool rows in 32 bits, [*slots.shape, hkv, d]."""
    x = (pool if scale is None else pool.view(torch.uint8))[slots]
    x = (x if scale is None else x.view(E4M3)).float().view(*slots.shape, hkv, d)
    return x if scale is None else x * scale[:, None]


def _begins(offsets):
    ends = offsets.long()
    return torch.cat([ends.new_zeros(1), ends[:-1]]), ends


def _window_decode(s):
    b, h, hkv, d = s["b"], s["h"], s["hkv"], s["d"]
    begin, end = _begins(s["offsets"])
    ctx = (end - begin)[:, None]
    # the visible cached tokens of a sequence, packed: its sinks, then its window without the current token
    first = (ctx - s["window"] + 1).clamp(min=0)
    sinks = first.clamp(max=s["sinks"])
    n = sinks + ctx - first
    u = torch.arange(min(s["longest"], s["sinks"] + s["window"] - 1), device="cuda")[None]
    seen = u < n
    token = torch.where(seen, torch.where(u < sinks, u, u - sinks + first), 0)
    if s["block"] == 1:
        slots = s["table"][(begin[:, None] + token).clamp(max=max(s["table"].numel() - 1, 0))].long() if s["table"].numel() else token
    else:
        slots = s["table"].long().gather(1, token // s["block"]) * s["block"] + token % s["block"]
    return _attend(s, slots, seen, None)


def _attend(s, slots, seen, prefix):
    """One query per sequence over its own rows, the current token and, if given, rows that all share."""
    b, h, hkv, d = s["b"], s["h"], s["hkv"], s["d"]
    q = s["q"].float().view(b, hkv, h // hkv, d) / math.sqrt(d)
    k, v = _rows(s["kc"], slots, s["ks"], hkv, d), _rows(s["vc"], slots, s["vs"], hkv, d)
    kn, vn = s["k"].float().view(b, hkv, 1, d), s["v"].float().view(b, hkv, 1, d)
    scores = [(q @ k.permute(0, 2, 3, 1)).masked_fill_(~seen[:, None, None], -math.inf), q @ kn.transpose(-1, -2)]
    if prefix is not None:
        kp, vp = _rows(s["kc"], prefix, s["ks"], hkv, d), _rows(s["vc"], prefix, s["vs"], hkv, d)
        qp = q.transpose(0, 1).reshape(hkv, -1, d)
        scores.append((qp @ kp.permute(1, 2, 0)).view(hkv, b, h // hkv, -1).transpose(0, 1))
    top = torch.stack([x.amax(-1) for x in scores if x.size(-1)]).amax(0)[..., None]
    p = [(x - top).exp() for x in scores]
    total = sum(x.sum(-1, keepdim=True) for x in p)
    o = p[0] @ v.transpose(1, 2) + p[1] * vn
    if prefix is not None:
        o = o + (p[2].transpose(0, 1).reshape(hkv, -1, p[2].size(-1)) @ vp.transpose(0, 1)).view(hkv, b, h // hkv, d).transpose(0, 1)
    return (o / total).reshape(b, h * d).to(s["q"].dtype)


def _shared_prefix(s):
    begin, end = _begins(s["offsets"])
    token = torch.arange(s["longest"], device="cuda")[None] + begin[:, None]
    seen = token < end[:, None]
    slots = s["table"][torch.where(seen, token, 0)].long() if s["table"].numel() else torch.zeros_like(token)
    return _attend(s, slots, seen, s["prefix_table"].long())


def _window_prefill(s):
    """Blocks of 256 consecutive queries of one sequence, each against the sinks and its stretch of keys."""
    h, hkv, d, w, n = s["h"], s["hkv"], s["d"], s["window"], s["sinks"]
    size = 256
    out = torch.zeros_like(s["q"])
    q_begin, q_end = _begins(s["q_offsets"])
    kv_begin, kv_end = _begins(s["kv_offsets"])
    blocks = -(-max(s["max_q"], 1) // size)
    # block i of sequence b: query rows [b, i, r]; those past the sequence's end go to a spare row
    r = torch.arange(blocks * size, device="cuda").view(1, blocks, size)
    row = q_begin[:, None, None] + r
    real = row < q_end[:, None, None]
    past = (kv_end - kv_begin) - (q_end - q_begin)
    at = past[:, None, None] + r                                                      # position of the query
    key = torch.cat([torch.arange(n, device="cuda").expand(at.size(0), blocks, n),
                     at[..., :1] - w + 1 + torch.arange(w + size - 1, device="cuda")], -1)
    usable = torch.cat([key[..., :n] >= 0, key[..., n:] >= n], -1) & (key < (kv_end - kv_begin)[:, None, None])
    slots = s["table"].long()[(kv_begin[:, None, None] + key).clamp(0, s["table"].numel() - 1)]
    keep = real[..., 0]                                                               # blocks with a real query
    slots, usable, key, at, row, real = (x[keep] for x in (slots, usable, key, at, row, real))
    if slots.size(0) == 0:
        return out
    k, v = _rows(s["kc"], slots, None, hkv, d), _rows(s["vc"], slots, None, hkv, d)
    spare = torch.cat([s["q"], s["q"].new_zeros(1, h * d)])
    row = torch.where(real, row, s["q"].size(0))
    q = spare[row].float().view(-1, size, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).flatten(2, 3) / math.sqrt(d)
    seen = usable[:, None] & (key[:, None] <= at[..., None]) & ((key[:, None] > at[..., None] - w) | (key[:, None] < n))
    x = (q @ k.permute(0, 2, 3, 1)).view(-1, hkv, h // hkv, size, key.size(-1))
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(top.masked_fill_(top == -math.inf, 0)).exp_()
    total = x.sum(-1, keepdim=True)
    o = x.flatten(2, 3) @ v.transpose(1, 2)
    o = (o.view(-1, hkv, h // hkv, size, d) / total).permute(0, 3, 1, 2, 4).reshape(-1, h * d).to(s["q"].dtype)
    out[row[real]] = o[real.flatten()]
    return out


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm_rope":
        n, hq, hk, d = case["tokens"], case["hq"], case["hk"], case["d"]
        b = 2 * n * (hq + hk) * d * size + 2 * min(n, 8192) * case["rot"] * size + 4 * n
        if case["write"] != "none":
            b += n * hk * d * (size + 2 * (1 if case["write"] == "e4m3" else size)) + 4 * n
        return {"bytes": b, "flops": 7 * n * (hq + hk) * d}
    h, hkv, d, b = case["h"], case["hkv"], case["d"], case["b"]
    if case["op"] == "window_prefill":
        q_lens, past = _lengths(b, case["q_lo"], case["q_hi"], 2), _lengths(b, case["past_lo"], case["past_hi"], 3)
        w, n = case["window"], case["sinks"]
        seen = keys = 0
        for q, p in zip(q_lens, past):
            for i in range(p, p + q):
                seen += min(i + 1, w + min(n, max(0, i - w + 1)))
            low = max(0, p - w + 1)
            keys += (p + q - low + min(n, low)) if q else 0
        return {"bytes": 2 * sum(q_lens) * h * d * size + keys * (2 * hkv * d * size + 4), "flops": 4 * seen * h * d}
    if case["op"] == "window_decode":
        lens = _lengths(b, case["ctx_lo"], case["ctx_hi"], 1)
        seen = sum(min(c, case["window"] - 1 + min(case["sinks"], max(0, c - case["window"] + 1))) for c in lens)
        read = seen
    else:
        lens = _lengths(b, case["own_lo"], case["own_hi"], 4)
        seen, read = sum(lens) + b * case["prefix"], sum(lens) + case["prefix"]
    kv = 1 if case["kv"] == "e4m3" else size
    return {"bytes": read * (2 * hkv * d * kv + 4) + 2 * b * (h + hkv) * d * size, "flops": 4 * (seen + b) * h * d}


# ----------------------------------------------------------------------------------------------
# the definitions in 64 bits, one sequence and head after the other
# ----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        return _exact_norm_rope(s)
    d, g = s["d"], s["h"] // s["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    wide = lambda x, scale: x.double() if scale is None else (x.double().unflatten(-1, (-1, d)) * scale.double()[:, None]).flatten(-2)  # noqa: E731
    table = s["table"].long()
    stop = 0
    for b in range(s["b"]):
        start = stop
        if case["op"] == "window_prefill":
            start = sum(s["kv_lens"][:b])
            rows = table[start:start + s["kv_lens"][b]]
            q0 = sum(s["q_lens"][:b])
            n_q = s["q_lens"][b]
            if n_q == 0:
                continue
            i = torch.arange(rows.numel() - n_q, rows.numel(), device="cuda")[:, None]
            j = torch.arange(rows.numel(), device="cuda")[None]
            hidden = (j > i) | ((j <= i - s["window"]) & (j >= s["sinks"]))
            q, into = s["q"][q0:q0 + n_q].double(), out[q0:q0 + n_q]
            k, v = s["kc"][rows].double(), s["vc"][rows].double()
        else:
            stop = int(s["offsets"][b])
            ctx = torch.arange(stop - start, device="cuda")
            if case["op"] == "window_decode":
                ctx = ctx[(ctx < s["sinks"]) | (ctx > ctx.numel() - s["window"])]
                rows = table[start + ctx] if s["block"] == 1 else table[b][ctx // s["block"]] * s["block"] + ctx % s["block"]
            else:
                rows = torch.cat([s["prefix_table"].long(), table[start:stop]])
            hidden = None
            q, into = s["q"][b:b + 1].double(), out[b:b + 1]
            pick = lambda pool, scale: wide(pool.view(torch.uint8)[rows].view(E4M3) if scale is not None else pool[rows], scale)  # noqa: E731
            k = torch.cat([pick(s["kc"], s["ks"]), s["k"][b:b + 1].double()])
            v = torch.cat([pick(s["vc"], s["vs"]), s["v"][b:b + 1].double()])
        for head in range(s["h"]):
            a, c = slice(head * d, head * d + d), slice(head // g * d, head // g * d + d)
            x = q[:, a] @ k[:, c].T * d ** -0.5
            if hidden is not None:
                x[hidden] = -math.inf
            into[:, a] = torch.softmax(x, -1) @ v[:, c]
    return out


def _exact_norm_rope(s):
    d, r, n = s["d"], s["rot"], s["tokens"]
    pos = s["positions"].long()
    turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
    got = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.double().reshape(n, -1, d)
        x = x / torch.linalg.vector_norm(x, dim=-1, keepdim=True).square().div(d).add(1e-6).sqrt() * w.double()
        z = torch.complex(x[..., :r].contiguous(), x[..., r:2 * r].contiguous()) * turn
        got.append(torch.cat([z.real, z.imag, x[..., 2 * r:]], -1))
    out = [x.flatten(1) for x in got]
    if s["write"] != "none":
        for pool, x, scale in ((s["kc"], got[1], s["ks"]), (s["vc"], s["v"].double().reshape(n, -1, d), s["vs"])):
            full = pool.double()
            full[s["slots"].long()] = (x if scale is None else x / scale.double()[:, None]).flatten(1)
            out.append(full)
    return out
