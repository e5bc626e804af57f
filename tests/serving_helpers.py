"""Inputs and error bounds shared by the tests of the windowed and the shared-prefix attention."""
import torch

F16, BF16, F32, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn


def pool(gen, rows, hkv, d, dtype, kv):
    """(pool on the GPU, its rows in 64 bits, scales on the GPU or None)."""
    x = torch.randn(rows, hkv * d, generator=gen)
    if kv == "same":
        x = x.to(dtype)
        return x.cuda(), x.double(), None
    scale = 0.01 + 0.002 * torch.arange(hkv, dtype=torch.float32)
    codes = (x.view(rows, hkv, d) / scale[:, None]).clamp(-448, 448).to(E4M3)
    wide = codes.to(torch.float64) * scale.double()[:, None]
    return codes.view(rows, hkv * d).cuda(), wide.view(rows, hkv * d), scale.cuda()


def offsets(lens):
    return torch.tensor(list(lens), dtype=torch.int64).cumsum(0).to(torch.int32)


def close(got, ref, size, dtype, p_dtype, n_keys):
    """Bound per output entry, ref = sum p v, size = sum p |v|:
      half a step of the output type relative to the value;
      half a step of the type P is rounded to for the second product, relative to size (fp32: none), and for
      fp16 P its subnormal half step 2^-25 for each of the keys (N(0,1) values: mean |v| below 1);
      2^-13 of size for the 32-bit part: scores of at most 13 * log2 e accumulated over head_dim / 16 MMA steps
      that may each truncate at 2^-23 of that, the exponential's 2^-22 and the sums."""
    got = got.detach().cpu().double()
    half = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
    tol = half[dtype] * ref.abs() * (1 + 2.0 ** -7) + (half[p_dtype] + 2.0 ** -13) * size
    if p_dtype == F16:
        tol = tol + n_keys * 2.0 ** -25
    if dtype == F16:
        tol = tol + 2.0 ** -25
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst excess {float(((got - ref).abs() - tol).max()):.3g}"
