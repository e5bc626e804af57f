"""Plain implementations in 64 bits of the serving operators that the reference does not have: the
per-head norm with rotation and cache append, attention with a sliding window and sink tokens, and
decoding behind a shared prefix.  CPU tensors, one sequence and one head after the other."""
import torch


def qk_norm_rope(x, weight, positions, cos, sin, head_dim, eps):
    """``x`` [N, H*head_dim] -> (result [N, H, head_dim], the sum of the magnitudes each entry is a
    combination of, for error bounds)."""
    n, r = x.size(0), cos.size(1)
    x = x.double().reshape(n, -1, head_dim)
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    c, s = cos.double()[positions.long()][:, None], sin.double()[positions.long()][:, None]
    a, b, rest = y[..., :r], y[..., r:2 * r], y[..., 2 * r:]
    out = torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    size = torch.cat([a.abs() + b.abs(), a.abs() + b.abs(), rest.abs()], -1)
    return out, size


def visible(i, window, n_sinks):
    """Keys that the query at position ``i`` of its sequence sees (window=None: all up to itself)."""
    if window is None:
        return list(range(i + 1))
    return [j for j in range(i + 1) if j < n_sinks or j > i - window]


def attend(q, k, v, scale):
    """q [H, D], k, v [n, Hkv, D] (64 bits) -> (o [H, D], probabilities [H, n])."""
    g = q.size(0) // k.size(1)
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    p = torch.softmax(torch.einsum("hd,nhd->hn", q, kk) * scale, -1)
    return torch.einsum("hn,nhd->hd", p, vv), p


def decode(Q, K, V, k_rows, v_rows, num_heads, scale, window=None, n_sinks=0):
    """One token per sequence.  ``k_rows``/``v_rows``: per sequence its cached rows [ctx, Hkv*D] in 64 bits
    (dequantised).  Returns O [B, H*D] and sum_j p_j |v_j| per output entry, for error bounds."""
    B, H, D = Q.size(0), num_heads, Q.size(1) // num_heads
    out, size = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    for b in range(B):
        k = torch.cat([k_rows[b].double(), K[b:b + 1].double()]).view(-1, K.size(1) // D, D)
        v = torch.cat([v_rows[b].double(), V[b:b + 1].double()]).view(-1, V.size(1) // D, D)
        see = visible(k.size(0) - 1, window, n_sinks)
        out[b], p = attend(Q[b].double().view(H, D), k[see], v[see], scale)
        size[b] = torch.einsum("hn,nhd->hd", p, v[see].abs().repeat_interleave(H // v.size(1), 1))
    return out.view(B, H * D), size.view(B, H * D)


def prefill(Q, k_rows, v_rows, q_lens, num_heads, scale, window, n_sinks):
    """Chunks: sequence b's queries are its last ``q_lens[b]`` tokens, its keys ``k_rows[b]`` [kv_len, Hkv*D].
    Returns O and sum_j p_j |v_j| per entry."""
    H, D = num_heads, Q.size(1) // num_heads
    out, size, at = torch.zeros(Q.shape, dtype=torch.float64), torch.zeros(Q.shape, dtype=torch.float64), 0
    for k, v, n in zip(k_rows, v_rows, q_lens):
        k, v = k.double().view(k.size(0), -1, D), v.double().view(v.size(0), -1, D)
        g = H // k.size(1)
        past = k.size(0) - n
        i = torch.arange(past, past + n)[:, None]
        j = torch.arange(k.size(0))[None]
        hidden = (j > i) | ((j <= i - window) & (j >= n_sinks))
        for h in range(H):
            x = Q[at:at + n, h * D:(h + 1) * D].double() @ k[:, h // g].T * scale
            p = torch.softmax(x.masked_fill(hidden, -float("inf")), -1)
            out[at:at + n, h * D:(h + 1) * D] = p @ v[:, h // g]
            size[at:at + n, h * D:(h + 1) * D] = p @ v[:, h // g].abs()
        at += n
    return out, size
