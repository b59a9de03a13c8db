"""Operators of a decode step beside the dense block-FP8 products: routed experts and 4-bit weights, and their plain forms.

`listed()` names the cases, `draw(rng)` makes one more of the same ranges, `prepare` builds what a serving process holds
before the call, `run` is one call - the package's own where `own` is set, else elementary torch operations in 32 bits -
`exact` the same from the definition in 64 bits, `work` the bytes and operations such a call cannot do without.

The definitions:

route   l[t, e] = fp32(sum_h x[t, h] r[e, h]).  softmax: the top_k largest l of a token (ties: lowest index), weights
        softmax(l) at them, with `renorm` softmax over the chosen ones alone.  sigmoid: s = fp32(sigmoid(l)), chosen by
        fp32(s + bias), weights s at them, with `renorm` divided by their sum; all weights times `scale`.
moe     x is quantized to E4M3 in groups of 128 columns (scale = max(amax, 1e-10) fp32(1/448), `half`: codes halved,
        scale doubled), h[s] = silu(gate) up of slot s = (token, choice) in its expert, quantized the same way, and
        y[t] = sum_s w[s] down(h[s]); weights are E4M3 with a scale per 128 x 128 block.  A slot of expert -1 adds nothing.
layer   route, then moe on its choice.
w4      y = x W^T + bias, W[n, k] = (q[n, k] - z[n, k / group]) s[n, k / group], q of 4 bits, two in a byte (low: even k).
"""

import math

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}

# A drawn case reads and multiplies no more than the largest listed one
MAX_BYTES = 6.6e9
MAX_FLOPS = 6.6e10


def listed():
    return [
        # the router alone, as a program with its own expert kernels calls it: one token, and a full decode batch
        {"name": "route_t1", "kind": "route", "t": 1, "e": 64, "k": 8, "h": 2048, "scoring": "softmax", "renorm": True, "scale": 1.0},
        {"name": "route_t128_sigmoid", "kind": "route", "t": 128, "e": 256, "k": 8, "h": 4096, "scoring": "sigmoid", "renorm": True, "scale": 2.5},
        # few large experts, one token: two experts of the dense FFN's size
        {"name": "moe_t1_e8", "kind": "moe", "t": 1, "e": 8, "eg": 8, "k": 2, "h": 4096, "i": 14336, "half": True},
        # sizes that are no multiple of the scale block; five tokens in flight
        {"name": "moe_t5_ragged", "kind": "moe", "t": 5, "e": 60, "eg": 60, "k": 4, "h": 2000, "i": 1360, "half": False},
        # one GPU of eight in an expert-parallel group: most choices of the 128 tokens are another GPU's
        {"name": "moe_t128_local", "kind": "moe", "t": 128, "e": 32, "eg": 256, "k": 8, "h": 4096, "i": 2048, "half": False},
        # a whole layer for one token: many small experts, latency counts
        {"name": "layer_t1", "kind": "layer", "t": 1, "e": 128, "k": 8, "h": 2048, "i": 768, "half": False, "scoring": "softmax", "renorm": True, "scale": 1.0},
        # a whole layer for a decode batch that reaches nearly every expert: the largest case
        {"name": "layer_t64", "kind": "layer", "t": 64, "e": 256, "k": 8, "h": 4096, "i": 2048, "half": True, "scoring": "sigmoid", "renorm": True, "scale": 2.5},
        # 4-bit projections: the smallest call, the dense FFN's up and down projections, a large one for a small batch, odd sizes
        {"name": "w4_m1_small", "kind": "w4", "m": 1, "k": 1024, "n": 1024, "group": 32, "dtype": "bf16", "zeros": False, "bias": False},
        {"name": "w4_m1_up", "kind": "w4", "m": 1, "k": 4096, "n": 14336, "group": 128, "dtype": "bf16", "zeros": False, "bias": False},
        {"name": "w4_m8_large", "kind": "w4", "m": 8, "k": 8192, "n": 28672, "group": 64, "dtype": "f16", "zeros": True, "bias": False},
        {"name": "w4_m3_ragged", "kind": "w4", "m": 3, "k": 4000, "n": 1003, "group": 128, "dtype": "bf16", "zeros": True, "bias": True},
        {"name": "w4_m32_down", "kind": "w4", "m": 32, "k": 14336, "n": 4096, "group": 128, "dtype": "bf16", "zeros": True, "bias": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, least):
    """A width: mostly a multiple of the scale block, sometimes only of `least`."""
    v = _log_int(rng, lo, hi)
    step = rng.choice((BLOCK, BLOCK, BLOCK, least))
    return max(step, v // step * step)


def _router(rng):
    return {"scoring": rng.choice(("softmax", "sigmoid")), "renorm": rng.random() < 0.7, "scale": rng.choice((1.0, 2.5))}


def draw(rng):
    while True:
        kind = rng.choice(("route", "moe", "moe", "layer", "layer", "w4", "w4", "w4"))
        if kind == "w4":
            c = {"kind": kind, "m": _log_int(rng, 1, 32), "k": _size(rng, 256, 28672, 32), "n": _size(rng, 64, 28672, 1),
                 "group": rng.choice((32, 64, 128)), "dtype": rng.choice(("bf16", "f16")), "zeros": rng.random() < 0.5,
                 "bias": rng.random() < 0.3}
        else:
            e = _log_int(rng, 4, 256)
            c = {"kind": kind, "t": _log_int(rng, 1, 128), "e": e, "k": min(e, _log_int(rng, 1, 10)), "h": _size(rng, 512, 8192, 16)}
            if kind != "route":
                c["i"], c["half"] = _size(rng, 256, 14336, 16), rng.random() < 0.5
            if kind == "moe":
                c["eg"] = e * rng.choice((1, 1, 1, 2, 8))
            else:
                c.update(_router(rng))
        w = work(c)
        held = c["e"] * 3 * c["h"] * c["i"] if kind in ("moe", "layer") else 0
        if max(w["bytes"], held) <= MAX_BYTES and w["flops"] <= MAX_FLOPS:
            return c


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _expert_weight(gen, lead, rows, cols):
    """OCP E4M3 codes [*lead, rows, cols] of an N(0, 0.02) weight and their 128 x 128 block scales, as a checkpoint holds them."""
    count = math.prod(lead)
    codes = torch.empty((count, rows, cols), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((count, _blocks(rows), _blocks(cols)), device="cuda")
    step = max(1, (1 << 28) // (rows * cols))
    for a in range(0, count, step):
        b = min(count, a + step)
        w = torch.randn((b - a, rows, cols), generator=gen, device="cuda") * 0.02
        pad = torch.nn.functional.pad(w, (0, -cols % BLOCK, 0, -rows % BLOCK))
        tiles = pad.view(b - a, _blocks(rows), BLOCK, _blocks(cols), BLOCK)
        s = tiles.abs().amax(dim=(2, 4)).clamp_min(1e-10) / 448.0
        q = (tiles / s[:, :, None, :, None]).clamp(-448, 448).view_as(pad)[:, :rows, :cols]
        codes[a:b], scales[a:b] = q.to(torch.float8_e4m3fn), s
    return codes.view(*lead, rows, cols), scales.view(*lead, _blocks(rows), _blocks(cols))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["kind"] == "w4":
        m, k, n, dt = case["m"], case["k"], case["n"], DTYPES[case["dtype"]]
        g = -(-k // case["group"])
        s["x"] = torch.randn((m, k), generator=gen, device="cuda").to(dt)
        s["codes"] = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        s["scales"] = (torch.rand((n, g), generator=gen, device="cuda") * 0.006 + 0.004).to(dt)
        s["zeros_"] = torch.randint(4, 12, (n, g), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        s["bias_"] = torch.randn((n,), generator=gen, device="cuda") * 0.1 if case["bias"] else None
        return s
    t, e, k, h = case["t"], case["e"], case["k"], case["h"]
    s["x"] = torch.randn((t, h), generator=gen, device="cuda").to(torch.bfloat16)
    if case["kind"] != "moe":
        s["router"] = (torch.randn((e, h), generator=gen, device="cuda") / math.sqrt(h)).to(torch.bfloat16)
        s["bias_"] = torch.randn((e,), generator=gen, device="cuda") * 0.05 if case["scoring"] == "sigmoid" else None
    else:
        # the choice of a router over all `eg` experts of the group, of which the first `e` are here: -1 for the others
        choice = torch.rand((t, case["eg"]), generator=gen, device="cuda").topk(k, dim=1).indices
        s["ids"] = torch.where(choice < e, choice, -1).to(torch.int32)
        s["weights"] = torch.softmax(torch.randn((t, k), generator=gen, device="cuda"), dim=1)
    if case["kind"] != "route":
        s["w13"], s["s13"] = _expert_weight(gen, (e, 2), case["i"], h)
        s["w2"], s["s2"] = _expert_weight(gen, (e,), h, case["i"])
    return s


# ---- plain forms ------------------------------------------------------------------------------

def _plain_route(s):
    logits = (s["x"].double() @ s["router"].double().t()).float()
    if s["scoring"] == "softmax":
        ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :s["k"]]
        w = torch.softmax(logits.gather(1, ids), dim=1) if s["renorm"] else torch.softmax(logits, dim=1).gather(1, ids)
    else:
        score = (1.0 / (1.0 + torch.exp(-logits.double()))).float()
        ids = torch.sort(score + s["bias_"], dim=1, descending=True, stable=True).indices[:, :s["k"]]
        w = score.gather(1, ids)
        if s["renorm"]:
            w = w / (w.sum(dim=1, keepdim=True) + 1e-20)
    return ids.to(torch.int32), w * s["scale"]


def _plain_quant(v, half):
    """The values that the E4M3 codes of v stand for, groups of 128 along the last dimension."""
    n = v.shape[-1]
    groups = torch.nn.functional.pad(v, (0, -n % BLOCK)).unflatten(-1, (-1, BLOCK))
    scale = groups.abs().amax(dim=-1, keepdim=True).clamp_min(1e-10) * torch.tensor(1.0 / 448.0, dtype=torch.float32, device=v.device)
    q = (groups / scale).clamp(-448, 448).to(torch.float8_e4m3fn)
    if half:
        q, scale = (q.to(torch.float16) * 0.5).to(torch.float8_e4m3fn), scale * 2
    return (q.float() * scale).flatten(-2)[..., :n]


def _plain_weight(codes, scales):
    rows, cols = codes.shape[-2:]
    full = scales.repeat_interleave(BLOCK, dim=-2)[..., :rows, :].repeat_interleave(BLOCK, dim=-1)[..., :cols]
    return codes.float() * full


def _plain_moe(s, ids, weights):
    active = torch.unique(ids)
    active = active[active >= 0].long()
    if active.numel() == 0:
        return torch.zeros_like(s["x"])
    xq = _plain_quant(s["x"].float(), s["half"])
    w13 = _plain_weight(s["w13"][active], s["s13"][active])                     # [A, 2, I, H]
    gate = torch.matmul(xq, w13[:, 0].transpose(1, 2))                          # [A, T, I]
    up = torch.matmul(xq, w13[:, 1].transpose(1, 2))
    hq = _plain_quant(gate / (1.0 + torch.exp(-gate)) * up, s["half"])
    down = torch.matmul(hq, _plain_weight(s["w2"][active], s["s2"][active]).transpose(1, 2))      # [A, T, H]
    share = ((ids[:, :, None] == active) * weights[:, :, None]).sum(dim=1)      # [T, A]
    return (share.t()[:, :, None] * down).sum(dim=0).to(s["x"].dtype)


def _plain_w4(s):
    codes = s["codes"]
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(1).float()
    n, k = q.shape
    q = torch.nn.functional.pad(q, (0, -k % s["group"])).unflatten(1, (-1, s["group"]))
    z = 8.0 if s["zeros_"] is None else s["zeros_"].float()[:, :, None]
    w = ((q - z) * s["scales"].float()[:, :, None]).flatten(1)[:, :k]
    y = s["x"].float() @ w.t()
    return (y if s["bias_"] is None else y + s["bias_"]).to(s["x"].dtype)


def run(state):
    s, kind = state, state["kind"]
    if own:
        import gaudi_kernels_b200 as gk
        if kind == "w4":
            return gk.gemm_group_w4(s["x"], s["codes"], s["scales"], s["zeros_"], group=s["group"], bias=s["bias_"])
        if kind == "moe":
            return gk.moe_block_fp8(s["x"], s["ids"], s["weights"], s["w13"], s["s13"], s["w2"], s["s2"],
                                    native_half=s["half"], check=False)
        route = {"scoring": s["scoring"], "renormalize": s["renorm"], "bias": s["bias_"], "scale": s["scale"]}
        if kind == "route":
            return gk.route_topk(s["x"], s["router"], s["k"], **route)
        return gk.moe_layer_block_fp8(s["x"], s["router"], s["k"], s["w13"], s["s13"], s["w2"], s["s2"],
                                      native_half=s["half"], check=False, **route)
    if kind == "w4":
        return _plain_w4(s)
    ids, weights = (s["ids"], s["weights"]) if kind == "moe" else _plain_route(s)
    if kind == "route":
        return ids, weights
    y = _plain_moe(s, ids, weights)
    return y if kind == "moe" else (y, ids, weights)


def work(case):
    if case["kind"] == "w4":
        m, k, n, g = case["m"], case["k"], case["n"], -(-case["k"] // case["group"])
        return {"bytes": n * k / 2 + n * g * (3 if case["zeros"] else 2) + 2 * m * (k + n) + (4 * n if case["bias"] else 0),
                "flops": 2.0 * m * n * k}
    t, e, k, h = case["t"], case["e"], case["k"], case["h"]
    if case["kind"] == "route":
        return {"bytes": 2 * (t + e) * h + 8 * t * k, "flops": 2.0 * t * e * h}
    i, eg = case["i"], case.get("eg", e)
    hit = e * (1 - (1 - k / eg) ** t)                      # experts that some token chose, on average
    slots = t * k * e / eg
    both = {"bytes": hit * 3 * h * i + 4 * t * h + 8 * t * k, "flops": 6.0 * slots * h * i}
    if case["kind"] == "layer":
        both["bytes"] += 2 * e * h
        both["flops"] += 2.0 * t * e * h
    return both


# ---- the definition in 64 bits ----------------------------------------------------------------

def _exact_route(s):
    x, r = s["x"].double(), s["router"].double()
    logit = torch.einsum("th,eh->te", x, r).float().double()
    score = logit if s["scoring"] == "softmax" else torch.sigmoid(logit).float().double()
    key = score if s["scoring"] == "softmax" else (score.float() + s["bias_"]).double()
    rows_i, rows_w = [], []
    for t in range(x.shape[0]):
        order = sorted(range(key.shape[1]), key=lambda e, row=key[t].tolist(): (-row[e], e))[:s["k"]]
        chosen = score[t, order]
        if s["scoring"] == "softmax":
            w = torch.exp(chosen - score[t].max())
            w = w / (w.sum() if s["renorm"] else torch.exp(score[t] - score[t].max()).sum())
        else:
            w = chosen / (chosen.sum() + 1e-20) if s["renorm"] else chosen
        rows_i.append(order)
        rows_w.append(w * s["scale"])
    return torch.tensor(rows_i, dtype=torch.int32, device=x.device), torch.stack(rows_w)


def _exact_codes(v, half):
    """64-bit values of the codes of one matrix; the scale is the fp32 number that the definition stores."""
    rows, cols = v.shape
    got = torch.empty_like(v)
    for a in range(0, cols, BLOCK):
        part = v[:, a:a + BLOCK]
        scale = torch.maximum(part.abs().amax(dim=1).float(), torch.tensor(1e-10, device=v.device)) * torch.tensor(1.0 / 448.0, dtype=torch.float32, device=v.device)
        u = part / scale.double()[:, None]
        # nearest E4M3 value, ties to even: the grid step of u is 2^(floor(log2 |u|) - 3), at least 2^-9
        step = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3)
        c = (torch.round(u / step) * step).clamp(-448, 448)
        if half:
            c = c / 2
            step = torch.exp2(torch.floor(torch.log2(c.abs().clamp_min(2.0 ** -6))) - 3)
            c = torch.round(c / step) * step
            scale = scale * 2
        got[:, a:a + BLOCK] = c * scale.double()[:, None]
    return got


def _exact_weight(codes, scales):
    w = codes.double()
    for a in range(scales.shape[0]):
        for b in range(scales.shape[1]):
            w[a * BLOCK:(a + 1) * BLOCK, b * BLOCK:(b + 1) * BLOCK] *= scales[a, b]
    return w


def _exact_moe(s, ids, weights):
    xq = _exact_codes(s["x"].double(), s["half"])
    y = torch.zeros_like(xq)
    for e in sorted(set(ids.flatten().tolist()) - {-1}):
        token, choice = torch.nonzero(ids == e, as_tuple=True)
        gate = xq[token] @ _exact_weight(s["w13"][e, 0], s["s13"][e, 0]).t()
        up = xq[token] @ _exact_weight(s["w13"][e, 1], s["s13"][e, 1]).t()
        hq = _exact_codes(gate * torch.sigmoid(gate) * up, s["half"])
        part = hq @ _exact_weight(s["w2"][e], s["s2"][e]).t()
        y.index_add_(0, token, part * weights[token, choice].double()[:, None])
    return y


def exact(case, seed):
    if case["kind"] in ("moe", "layer") and case["e"] * _blocks(case["h"]) * _blocks(case["i"]) > 160000:
        return None                                        # a loop over every scale block would take minutes
    s = prepare(case, seed)
    if case["kind"] == "w4":
        q = torch.empty((case["n"], case["k"]), dtype=torch.float64, device="cuda")
        q[:, 0::2], q[:, 1::2] = (s["codes"] % 16).double(), (s["codes"] // 16).double()
        y = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for j in range(s["scales"].shape[1]):
            a, b = j * case["group"], min(case["k"], (j + 1) * case["group"])
            z = 8.0 if s["zeros_"] is None else s["zeros_"][:, j].double()[:, None]
            y += s["x"][:, a:b].double() @ ((q[:, a:b] - z) * s["scales"][:, j].double()[:, None]).t()
        return y if s["bias_"] is None else y + s["bias_"].double()
    if case["kind"] == "moe":
        return _exact_moe(s, s["ids"], s["weights"])
    ids, weights = _exact_route(s)
    if case["kind"] == "route":
        return ids, weights
    return _exact_moe(s, ids, weights.float()), ids, weights
