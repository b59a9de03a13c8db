"""CPU restatement in 64 bits of the routed block-FP8 experts and their router. TEST INFRASTRUCTURE ONLY.

The reference has no mixture-of-experts kernels, so parity is unpinned: the definitions are those of include/bfp8.h
(bfp8_moe_route, bfp8_moe_block128); the quantization rule is the one the other oracles pin
(python/gaudi_kernels/block_fp8_oracle.py:25-28,31-35 of tracycam/gaudi-kernels).

`experts` also returns how far a correct fp32 implementation may be from it, element by element.  u = 2^-23 bounds the
relative error of an fp32 addition, truncating or not:
  * a product of E4M3 numbers is exact; a sum over K is at most (K / 32) + (K / 128) + 8 additions deep - one per 32-wide
    step of the tensor core, whose inner additions keep more bits than the result, one per promoted block - so it is off by
    that many u of sum |terms|;
  * h = silu(g) u follows g and u with |silu'| <= 1.1 and is itself off by a few roundings (8 u);
  * a code of h / scale can be any code between those of the ratio moved down and up by the ratio's error;
  * the weighted sum adds top_k + 2 roundings, and storing bf16 half a step, 2^-8 of the value.
"""

import numpy as np
import torch

U = 2.0 ** -23
BLOCK = 128


def grid_value(r, half):
    """Value of the E4M3 code nearest to r (64-bit, ties to even, clamped to 448); with half the code is halved again."""
    def nearest(v):
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
        return torch.round(v / step) * step
    q = nearest(r).clamp(-448.0, 448.0)
    return nearest(q / 2) if half else q


def quantize(v, half, err=None):
    """64-bit values of the codes of v [rows, cols] in groups of 128 columns; with err (absolute, same shape) also a bound
    on how far the quantized values of any v +- err may be from them."""
    rows, cols = v.shape
    out, slack = torch.empty_like(v), torch.zeros_like(v)
    for a in range(0, cols, BLOCK):
        part = v[:, a:a + BLOCK]
        amax = part.abs().amax(dim=1, keepdim=True)
        scale = (amax.float().clamp_min(1e-10) * torch.tensor(np.float32(1.0 / 448.0))).double()
        ratio = part / scale
        stored = scale * (2 if half else 1)
        q = grid_value(ratio, half)
        out[:, a:a + BLOCK] = q * stored
        if err is not None:
            e = err[:, a:a + BLOCK]
            # amax moves by at most the largest error of the group, and two roundings form the scale
            rel = e.amax(dim=1, keepdim=True) / amax.clamp_min(1e-10) + 4 * U
            d = e / scale + ratio.abs() * rel
            spread = torch.maximum(grid_value(ratio + d, half) - q, q - grid_value(ratio - d, half))
            slack[:, a:a + BLOCK] = (spread + q.abs() * rel) * stored
    return (out, slack) if err is not None else out


def weight_values(codes, scales):
    """64-bit values of E4M3 codes [rows, cols] with 128 x 128 block scales."""
    rows, cols = codes.shape
    full = scales.double().repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    return codes.view(torch.float8_e4m3fn).float().double() * full


def _depth(k):
    return (k // 32 + k // 128 + 8) * U


def experts(x, ids, weights, w13, s13, w2, s2, half):
    """(y [T, H], bound [T, H]) in 64 bits, y before the bf16 rounding (which bound includes)."""
    t, h = x.shape
    e, _, inter, _ = w13.shape
    xq = quantize(x.double(), half)
    y, bound = torch.zeros((t, h), dtype=torch.float64), torch.zeros((t, h), dtype=torch.float64)
    for r in range(e):
        tok, choice = torch.nonzero(ids == r, as_tuple=True)
        if not tok.numel():
            continue
        wg, wu, wd = weight_values(w13[r, 0], s13[r, 0]), weight_values(w13[r, 1], s13[r, 1]), weight_values(w2[r], s2[r])
        v = xq[tok]
        g, u = v @ wg.t(), v @ wu.t()
        eg, eu = v.abs() @ wg.abs().t() * _depth(h), v.abs() @ wu.abs().t() * _depth(h)
        act = g * torch.sigmoid(g)
        hv = act * u
        eh = 1.1 * eg * (u.abs() + eu) + act.abs() * eu + 8 * U * hv.abs()
        hq, slack = quantize(hv, half, eh)
        w = weights[tok, choice].double()[:, None]
        part = hq @ wd.t()
        off = slack @ wd.abs().t() + (hq.abs() + slack) @ wd.abs().t() * _depth(inter)
        y.index_add_(0, tok, w * part)
        bound.index_add_(0, tok, w.abs() * (off + (ids.shape[1] + 2) * U * (part.abs() + off)))
    return y, bound + 2.0 ** -8 * (y.abs() + bound) + 2.0 ** -133


def route(x, router, top_k, scoring="softmax", renormalize=True, bias=None, scale=1.0):
    """(ids, weights in 64 bits, smallest gap between a chosen key and the next)."""
    logits = (x.double() @ router.double().t()).float()
    score = logits if scoring == "softmax" else torch.sigmoid(logits.double()).float()
    key = score if bias is None else score + bias
    t, e = key.shape
    ids = torch.empty((t, top_k), dtype=torch.int32)
    w = torch.empty((t, top_k), dtype=torch.float64)
    gap = float("inf")
    for r in range(t):
        row = [float("-inf") if np.isnan(v) else v for v in key[r].tolist()]
        nan = [np.isnan(v) for v in key[r].tolist()]
        order = sorted(range(e), key=lambda c: (nan[c], -row[c], c))
        for a, b in zip(order[:top_k], order[1:]):
            if row[a] != row[b]:
                gap = min(gap, row[a] - row[b])
        chosen = score[r, order[:top_k]].double()
        if scoring == "softmax":
            p = torch.exp(chosen - chosen[0])
            p = p / (p.sum() if renormalize else torch.exp(score[r].double() - chosen[0]).sum())
        else:
            p = chosen / (chosen.sum() + 1e-20) if renormalize else chosen
        ids[r] = torch.tensor(order[:top_k], dtype=torch.int32)
        w[r] = p * scale
    return ids, w, gap
