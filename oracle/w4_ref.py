"""CPU restatement in 64 bits of the 4-bit group-scaled weights. TEST INFRASTRUCTURE ONLY.

The reference has no 4-bit weights: the definitions are those of include/bfp8.h (bfp8_gemm_group_w4,
bfp8_quant_group_w4_f32), parity unpinned.

`product` also returns how far a correct fp32 implementation may be from it.  u = 2^-23 bounds the relative error of an fp32
addition, truncating or not.  q - z is exact, a product with x has at most 11 + 4 bits and is exact in fp32; a group's sum
is at most group / 16 additions of the tensor core deep (its inner additions keep more bits), then one multiply-add per
group, a tree over warps and CTAs of at most 15 + 8 sums, and the bias: (group / 16 + groups + 24) u of sum |terms| in all.
Storing 16 bits adds half a step: 2^-8 of the value in bf16, 2^-11 in fp16 (and half its smallest number, 2^-25).
"""

import torch

U = 2.0 ** -23


def unpack(codes):
    return torch.stack((codes & 15, codes >> 4), dim=-1).flatten(1).double()


def weight(codes, scales, zeros, group):
    q = unpack(codes)
    k = q.shape[1]
    rep = lambda v: v.double().repeat_interleave(group, dim=1)[:, :k]      # noqa: E731
    return (q - (8.0 if zeros is None else rep(zeros))) * rep(scales)


def product(x, codes, scales, zeros, group, bias, out_dtype):
    w, xd = weight(codes, scales, zeros, group), x.double()
    y = xd @ w.t()
    depth = (group // 16 + scales.shape[1] + 24) * U
    bound = xd.abs() @ w.abs().t() * depth
    if bias is not None:
        y = y + bias.double()
        bound = bound + U * y.abs()
    half_step, least = {torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25),
                        torch.float32: (2.0 ** -24, 2.0 ** -150)}[out_dtype]
    return y, bound + half_step * (y.abs() + bound) + least


def quantize(w, group, zeros, scale_dtype):
    n, k = w.shape
    codes = torch.empty((n, k), dtype=torch.uint8)
    g = (k + group - 1) // group
    scales, z = torch.empty((n, g), dtype=scale_dtype), torch.empty((n, g), dtype=torch.uint8)
    for j in range(g):
        part = w[:, j * group:(j + 1) * group]
        lo, hi = part.amin(dim=1).clamp_max(0), part.amax(dim=1).clamp_min(0)
        s = ((hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7).to(scale_dtype)
        s = torch.where(s == 0, torch.ones_like(s), s)
        zz = torch.round(-lo / s.float()).clamp(0, 15) if zeros else torch.full_like(lo, 8)
        codes[:, j * group:(j + 1) * group] = (torch.round(part / s.float()[:, None]) + zz[:, None]).clamp(0, 15).to(torch.uint8)
        scales[:, j], z[:, j] = s, zz.to(torch.uint8)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), scales, z if zeros else None
