"""GPU parity of the 4-bit group-scaled products and their quantizer against the 64-bit restatement (oracle/w4_ref.py)."""

import pytest
import torch

from oracle import w4_ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def gk():
    import gaudi_kernels_b200 as g
    from gaudi_kernels_b200 import _lib
    _lib.load()
    return g


def _problem(m, n, k, group, dtype, zeros, seed=0):
    gen = torch.Generator().manual_seed(m + 10 * n + 100 * k + group + seed)
    x = (torch.randn((m, k), generator=gen) * 1.5).to(dtype)
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, dtype=torch.uint8)
    g = (k + group - 1) // group
    scales = (torch.rand((n, g), generator=gen) * 0.02 + 0.001).to(dtype)
    z = torch.randint(0, 16, (n, g), generator=gen, dtype=torch.uint8) if zeros else None
    return x, codes, scales, z


def _dev(t):
    return None if t is None else t.to(DEV)


def _check(got, x, codes, scales, z, group, bias=None):
    y, bound = w4_ref.product(x, codes, scales, z, group, bias, got.dtype)
    off = (got.double().cpu() - y).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), "worst %.3g of the bound" % float((off / bound).max())
    assert float(bound.norm()) <= 0.01 * float(y.norm())


SHAPES = [
    # m, n, k
    (1, 1, 32), (1, 16, 64), (1, 17, 96), (2, 1003, 4000), (3, 33, 288), (4, 64, 256), (5, 100, 544), (7, 2064, 512),
    (8, 300, 1056), (9, 48, 320), (13, 257, 2048), (16, 129, 768), (17, 65, 352), (25, 400, 640), (32, 130, 1312),
    (33, 48, 256), (70, 96, 416), (1, 4096, 8192), (6, 6000, 1024), (12, 9600, 512), (31, 9500, 288), (2, 40000, 64),
]


@pytest.mark.parametrize("dtype,zeros", [(torch.bfloat16, True), (torch.float16, False), (torch.float16, True), (torch.bfloat16, False)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_matches_the_definition(gk, m, n, k, group, dtype, zeros):
    if n * k > 1 << 22 and (group, dtype, zeros) not in ((64, torch.bfloat16, True), (128, torch.float16, False)):
        pytest.skip("the large ones in two of the twelve forms")
    x, codes, scales, z = _problem(m, n, k, group, dtype, zeros)
    got = gk.gemm_group_w4(_dev(x), _dev(codes), _dev(scales), _dev(z), group=group, check=True)
    assert got.dtype == dtype
    _check(got, x, codes, scales, z, group)


# On 148 SMs these leave groups of 16 rows over that four warps share: 5, 7, 9, 10, 13, 14 or 15 groups per CTA, with and
# without clusters, the last CTA's rows and the last k ragged
REST = [
    (13, 9584, 1568), (9, 14213, 256), (13, 3184, 1568), (13, 19632, 544), (9, 21567, 544), (9, 4743, 3680), (9, 28585, 544),
    (9, 30918, 256), (16, 3171, 3616), (1, 33201, 256), (13, 33345, 256), (16, 3374, 3776), (3, 7416, 3104), (8, 28719, 1056),
]


@pytest.mark.parametrize("group,dtype,zeros", [(32, torch.bfloat16, True), (64, torch.float16, True), (128, torch.bfloat16, False)])
@pytest.mark.parametrize("m,n,k", REST)
def test_rows_left_over(gk, m, n, k, group, dtype, zeros):
    x, codes, scales, z = _problem(m, n, k, group, dtype, zeros)
    x, codes, scales, z = _dev(x), _dev(codes), _dev(scales), _dev(z)
    got = gk.gemm_group_w4(x, codes, scales, z, group=group, check=True)
    _check(got.cpu(), x.cpu(), codes.cpu(), scales.cpu(), None if z is None else z.cpu(), group)
    assert torch.equal(got, gk.gemm_group_w4(x, codes, scales, z, group=group))


# Passes of 32 rows, full and short, of one and of two warps per 16 weight rows, with and without clusters
MANY = [(32, 4100, 4096), (20, 9001, 1056), (31, 2065, 2080), (64, 4096, 1024), (57, 11003, 544), (17, 26001, 1056), (29, 5003, 3104),
        (33, 30777, 544), (47, 14336, 2048)]


@pytest.mark.parametrize("group,dtype,zeros", [(32, torch.float16, True), (64, torch.bfloat16, False), (128, torch.float16, True)])
@pytest.mark.parametrize("m,n,k", MANY)
def test_passes_of_32_rows(gk, m, n, k, group, dtype, zeros):
    x, codes, scales, z = _problem(m, n, k, group, dtype, zeros)
    x[m // 2, 3] = float("nan")                            # one row of a pass: the others do not see it
    got = gk.gemm_group_w4(_dev(x), _dev(codes), _dev(scales), _dev(z), group=group, check=True).cpu()
    assert torch.isnan(got[m // 2]).all()
    keep = [r for r in range(m) if r != m // 2]
    _check(got[keep], x[keep], codes, scales, z, group)


@pytest.mark.parametrize("m,n,k", [(1, 77, 416), (11, 1000, 512), (40, 50, 288)])
def test_fp32_output_and_bias(gk, m, n, k):
    x, codes, scales, z = _problem(m, n, k, 64, torch.bfloat16, True)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)) * 3
    got = gk.gemm_group_w4(_dev(x), _dev(codes), _dev(scales), _dev(z), group=64, bias=_dev(bias), out_dtype=torch.float32)
    _check(got, x, codes, scales, z, 64, bias)
    low = gk.gemm_group_w4(_dev(x), _dev(codes), _dev(scales), _dev(z), group=64, bias=_dev(bias))
    assert torch.equal(low, got.to(torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_code_and_zero_point_is_exact(gk, dtype):
    # x picks single columns, so the output is one weight: 16 codes x 16 zero points with a scale of 2
    n, k = 256, 128
    q = (torch.arange(n) // 16)[:, None].expand(n, k) + torch.arange(k)[None, :]
    q = (q % 16).to(torch.uint8)
    codes = q[:, 0::2] | (q[:, 1::2] << 4)
    z = (torch.arange(n) % 16).to(torch.uint8)[:, None].expand(n, 4).contiguous()
    scales = torch.full((n, 4), 2.0, dtype=dtype)
    for first in (0, 32, 64, 96):
        x = torch.zeros((32, k), dtype=dtype)
        x[torch.arange(32), first + torch.arange(32)] = 1.0
        got = gk.gemm_group_w4(_dev(x), _dev(codes), _dev(scales), _dev(z), group=32)
        want = 2.0 * (q[:, first:first + 32].float() - z[:, :1].float()).t()
        assert torch.equal(got.float().cpu(), want)


def test_strided_rows_and_a_given_output(gk):
    x, codes, scales, z = _problem(5, 130, 256, 64, torch.bfloat16, True)
    want = gk.gemm_group_w4(_dev(x), _dev(codes), _dev(scales), _dev(z), group=64)
    big = torch.full((7, 140), 3.0, dtype=torch.bfloat16, device=DEV)
    for pitch, first in ((264, 8), (261, 3)):              # rows TMA can read, rows that are copied first
        wide = torch.full((5, pitch), 9.0, dtype=torch.bfloat16, device=DEV)
        wide[:, first:first + 256] = _dev(x)
        out = gk.gemm_group_w4(wide[:, first:first + 256], _dev(codes), _dev(scales), _dev(z), group=64, out=big[1:6, 7:137])
        assert torch.equal(out, want)
    assert (big[0] == 3).all() and (big[6] == 3).all() and (big[:, :7] == 3).all() and (big[:, 137:] == 3).all()


@pytest.mark.parametrize("m", [1, 5, 40])
def test_an_output_over_the_rows_it_is_made_of(gk, m):
    x, codes, scales, z = [_dev(v) for v in _problem(m, 4096, 4096, 128, torch.bfloat16, True)]
    scales = scales * 0.01
    want = gk.gemm_group_w4(x, codes, scales, z, group=128)
    for _ in range(3):
        y = x.clone()
        assert gk.gemm_group_w4(y, codes, scales, z, group=128, out=y) is y and torch.equal(y, want)
    wide = torch.zeros((m, 6144), dtype=torch.bfloat16, device=DEV)
    wide[:, :4096] = x                                     # half of the output on x's columns, half beside them
    gk.gemm_group_w4(wide[:, :4096], codes, scales, z, group=128, out=wide[:, 2048:])
    assert torch.equal(wide[:, 2048:], want) and torch.equal(wide[:, :2048], x[:, :2048])


def test_broadcast_rows(gk):
    x, codes, scales, z = _problem(5, 130, 256, 64, torch.bfloat16, True)
    same = _dev(x)[2:3].expand(5, 256)
    want = gk.gemm_group_w4(same.contiguous(), _dev(codes), _dev(scales), _dev(z), group=64)
    assert torch.equal(gk.gemm_group_w4(same, _dev(codes), _dev(scales), _dev(z), group=64), want)


def test_nonfinite_rows_stay_alone(gk):
    x, codes, scales, z = _problem(6, 200, 512, 128, torch.bfloat16, True)
    x[2, 17], x[4, 300] = float("nan"), float("inf")
    got = gk.gemm_group_w4(_dev(x), _dev(codes), _dev(scales), _dev(z), group=128).cpu()
    assert torch.isnan(got[2]).all() and not torch.isfinite(got[4]).any()
    keep = [0, 1, 3, 5]
    _check(got[keep], x[keep], codes, scales, z, 128)
    # an infinite x times a positive (negative) weight is plus (minus) infinity, as in the formula
    w = w4_ref.weight(codes, scales, z, 128)[:, 300]
    assert torch.equal(got[4][w > 0], torch.full_like(got[4][w > 0], float("inf")))
    assert torch.equal(got[4][w < 0], torch.full_like(got[4][w < 0], float("-inf")))


def test_no_rows(gk):
    x, codes, scales, z = _problem(1, 40, 64, 32, torch.float16, False)
    assert gk.gemm_group_w4(_dev(x)[:0], _dev(codes), _dev(scales), group=32).shape == (0, 40)


def test_calls_overlap_and_replay(gk):
    x, codes, scales, z = [_dev(v) for v in _problem(4, 2000, 1024, 64, torch.float16, True)]
    want = gk.gemm_group_w4(x, codes, scales, z, group=64)
    side = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for n in range(24):
        with torch.cuda.stream(side[n % 3]):
            outs.append(gk.gemm_group_w4(x, codes, scales, z, group=64))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    xs = x.clone()
    with torch.cuda.graph(graph):
        y = gk.gemm_group_w4(xs, codes, scales, z, group=64)
    for f in (1.0, -2.0):
        xs.copy_(x * f)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want * f)                    # a power of two and a sign scale every rounding alike


def test_weights_at_rest_change_nothing(gk):
    # every product reads what the one before it wrote, with the codes asked for early
    _, codes, scales, z = [_dev(v) for v in _problem(1, 1024, 1024, 32, torch.bfloat16, True)]
    x = torch.randn((4, 1024), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)

    def chain():
        y = x
        for _ in range(8):
            y = gk.gemm_group_w4(y, codes, scales * 0.05, z, group=32)
        return y

    want = chain()
    prev = gk.set_weights_at_rest(True)
    try:
        torch.cuda.synchronize()
        for _ in range(5):
            assert torch.equal(chain(), want)
    finally:
        gk.set_weights_at_rest(prev)


@pytest.mark.parametrize("group,dtype,zeros", [(32, torch.bfloat16, True), (128, torch.float16, False)])
@pytest.mark.parametrize("m,n", [(4, 1024), (4, 4096), (4, 33216), (13, 19648), (13, 33216), (32, 4096), (32, 28672), (40, 9600)])
def test_products_at_rest_behind_products(gk, m, n, group, dtype, zeros):
    # nothing but products in the stream, each launched over the end of the one whose result it reads: from 1024 columns to n and
    # back, alone and in clusters, with rows left over and in passes of 32 rows; also replayed from a graph
    up = [_dev(v) for v in _problem(m, n, 1024, group, dtype, zeros)]
    down = [_dev(v) for v in _problem(m, 1024, n, group, dtype, zeros)]
    up[2], down[2] = up[2] * 0.25, down[2] * 0.0625         # outputs stay in fp16's range
    x = up[0]

    def chain(wait):
        y = x
        for _ in range(4):
            y = gk.gemm_group_w4(y, *up[1:], group=group)
            if wait:
                torch.cuda.synchronize()
            y = gk.gemm_group_w4(y, *down[1:], group=group)
            if wait:
                torch.cuda.synchronize()
        return y

    want = chain(True)
    assert torch.isfinite(want).all() and (want != 0).any()
    prev = gk.set_weights_at_rest(True)
    try:
        torch.cuda.synchronize()
        for _ in range(5):
            assert torch.equal(chain(False), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = chain(False)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    finally:
        gk.set_weights_at_rest(prev)


@pytest.mark.parametrize("group,dtype,zeros", [(32, torch.float16, True), (64, torch.bfloat16, False), (128, torch.bfloat16, True)])
@pytest.mark.parametrize("m,n,k", [(1, 40, 28672), (5, 300, 20000), (8, 129, 65536), (12, 1003, 14336), (16, 90, 28672), (30, 500, 28672)])
def test_long_rows(gk, m, n, k, group, dtype, zeros):
    x, codes, scales, z = _problem(m, n, k, group, dtype, zeros)
    scales = scales * 0.25                                 # fp16 outputs stay in range
    got = gk.gemm_group_w4(_dev(x), _dev(codes), _dev(scales), _dev(z), group=group, check=True)
    y, bound = w4_ref.product(x, codes, scales, z, group, None, dtype)
    assert torch.isfinite(got).all() and ((got.double().cpu() - y).abs() <= bound).all()
    # how small that bound is: 2048 + 26 additions at most, 2^-23 each of sum |terms|, and for terms of random signs
    # sum |terms| is about sqrt(k) = 256 at most times |y|: 6.4 % beside the rounding of the output
    assert float(bound.norm()) <= 0.07 * float(y.norm())


def test_codes_written_just_before_the_product(gk):
    # with weights at rest declared, codes that a kernel of the same stream has just written: one that lets its successor start
    # early (the activation quantizer's bytes taken as codes) and the quantizer of the format
    gen = torch.Generator().manual_seed(11)
    x = _dev(torch.randn((4, 1024), generator=gen).to(torch.bfloat16))
    rows = [_dev(torch.randn((4096, 512), generator=gen).to(torch.bfloat16)) for _ in range(3)]
    scales = torch.ones((4096, 16), dtype=torch.bfloat16, device=DEV)
    w = [_dev(torch.randn((4096, 1024), generator=gen)) for _ in range(3)]

    def both(i):
        codes = gk.quantize_act_1x128(rows[i])[0].view(torch.uint8)
        y = gk.gemm_group_w4(x, codes, scales, group=64, fresh_codes=True)
        codes, s, z = gk.quantize_group_w4(w[i], 64)
        return y, gk.gemm_group_w4(x, codes, s, z, group=64, fresh_codes=True)

    want = [both(i) for i in range(3)]
    prev = gk.set_weights_at_rest(True)
    try:
        for n in range(12):
            assert all(torch.equal(a, b) for a, b in zip(both(n % 3), want[n % 3]))
    finally:
        gk.set_weights_at_rest(prev)


@pytest.mark.parametrize("m,n", [(3, 1024), (20, 1024)])
def test_the_previous_kernels_time_is_not_a_products_own_wait(gk, m, n):
    # One row of 2^24 by 16 weight rows keeps at most eight SMs busy for milliseconds and lets its successor start at once on
    # the others.  The product behind it may wait 100,000 cycles (about 50 us) for its own copies, which take a few.
    long_k = 1 << 24
    long_x = torch.zeros((1, long_k), dtype=torch.bfloat16, device=DEV)
    long_codes = torch.zeros((16, long_k // 2), dtype=torch.uint8, device=DEV)
    long_scales = torch.ones((16, long_k // 128), dtype=torch.bfloat16, device=DEV)
    x, codes, scales, z = [_dev(v) for v in _problem(m, n, 1024, 64, torch.bfloat16, True)]
    want = gk.gemm_group_w4(x, codes, scales, z, group=64, check=True)
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        gk.gemm_group_w4(long_x, long_codes, long_scales, group=128)
        got = gk.gemm_group_w4(x, codes, scales, z, group=64, check=True, wait_limit_cycles=100000)
        b.record()
        b.synchronize()
        assert torch.equal(got, want) and a.elapsed_time(b) > 0.3      # well beyond the limit: 100,000 cycles are 0.05 ms


@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (5, 96, 64), (33, 416, 128), (64, 1024, 32), (7, 160, 64)])
def test_quantizer_bits(gk, n, k, group, zeros, scale_dtype):
    w = torch.randn((n, k), generator=torch.Generator().manual_seed(n + k)) * 0.05
    w[0, :32] = 0.0
    if n > 4:
        w[3] = w[3].abs()                                  # one-sided groups
        w[4] = 1e-30                                       # a scale that rounds to zero in fp16
    want = w4_ref.quantize(w, group, zeros, scale_dtype)
    got = gk.quantize_group_w4(w.to(DEV), group, zeros, scale_dtype)
    host = gk.quantize_group_w4(w, group, zeros, scale_dtype)
    for a, b, c in zip(got, want, host):
        assert (a is None and b is None and c is None) or (torch.equal(a.cpu(), b) and torch.equal(c, b))


@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float16])
def test_quantizer_groups_that_are_not_finite_stay_alone(gk, scale_dtype, zeros):
    w = torch.randn((4, 128), generator=torch.Generator().manual_seed(1))
    want = [v if v is None else v.cpu() for v in gk.quantize_group_w4(w.to(DEV), 32, zeros, scale_dtype)]
    bad = w.clone()
    bad[0, 5], bad[1, 40], bad[2, 70], bad[3, 127] = float("nan"), float("inf"), float("-inf"), 3e38 if zeros else float("nan")
    bad[3, 126] = -3e38                                    # with zero points the range itself overflows
    codes, scales, z = [v if v is None else v.cpu() for v in gk.quantize_group_w4(bad.to(DEV), 32, zeros, scale_dtype)]
    for r in range(4):                                     # row r's group r
        assert not torch.isfinite(scales[r, r]) and (torch.isnan(scales[r, r]) == (r == 0 or r == 3 and not zeros))
        assert not torch.isfinite(w4_ref.weight(codes, scales, z, 32)[r, 32 * r:32 * r + 32]).any()
        keep = [g for g in range(4) if g != r]
        assert torch.equal(scales[r, keep], want[1][r, keep]) and (z is None or torch.equal(z[r, keep], want[2][r, keep]))
        assert torch.equal(codes.view(4, 4, 16)[r, keep], want[0].view(4, 4, 16)[r, keep])


def test_quantized_weight_is_near_the_weight(gk):
    w = torch.randn((40, 512), generator=torch.Generator().manual_seed(4)) * 0.05
    codes, scales, z = gk.quantize_group_w4(w.to(DEV), 64)
    back = w4_ref.weight(codes.cpu(), scales.cpu(), z.cpu(), 64)
    step = scales.cpu().double().repeat_interleave(64, dim=1)
    # half a step; where the rounded scale or zero point cuts the range's ends off, up to half a step more and the scale's
    # rounding, 15 * 2^-8 of a step
    assert ((back - w.double()).abs() <= step * 1.06).all()


def test_a_decode_ffn_of_routed_and_shared_experts(gk):
    # the operators together: routed block-FP8 experts plus a shared expert in 4 bits, against 64 bits
    from oracle import moe_ref
    import test_gpu_moe
    t, k, e, h, i = 3, 2, 6, 256, 128
    x, _, _, *w = test_gpu_moe._problem(t, k, e, h, i)
    x = (x.float() * 0.5).to(torch.bfloat16)
    gen = torch.Generator().manual_seed(9)
    router = (torch.randn((e, h), generator=gen) / 16).to(torch.bfloat16)
    gu, dn = torch.randn((2 * i, h), generator=gen) * 0.06, torch.randn((h, i), generator=gen) * 0.06
    q13, q2 = gk.quantize_group_w4(gu.to(DEV), 64), gk.quantize_group_w4(dn.to(DEV), 32)
    routed, ids, weights = gk.moe_layer_block_fp8(x.to(DEV), router.to(DEV), k, *[v.to(DEV) for v in w])
    gate_up = gk.gemm_group_w4(x.to(DEV), *q13, group=64)
    shared = gk.gemm_group_w4(gk.silu_and_mul(gate_up), *q2, group=32, out_dtype=torch.float32)
    got = (routed.float() + shared).double().cpu()
    want_ids, want_w, gap = moe_ref.route(x, router, k)
    assert gap > 1e-7 and torch.equal(ids.cpu(), want_ids)
    y, bound = moe_ref.experts(x, want_ids, want_w.float(), *w, False)
    w13, w2 = [w4_ref.weight(*[v.cpu() for v in q], g) for q, g in ((q13, 64), (q2, 32))]
    both = x.double() @ w13.t()
    gate, up = both[:, :i], both[:, i:]
    mid = gate * torch.sigmoid(gate) * up
    z = mid @ w2.t()
    # gate, up and their product are rounded to bf16 (2^-8 each, the gate's through |silu'| <= 1.1 and |g silu' / silu| <= 2
    # near its size): at most 2^-8 (1.1 |g u| + |mid| + |mid|) per value; the routing weights are fp32 (2^-18, see the router)
    off = (2.0 ** -8 * (1.1 * (gate * up).abs() + 2.05 * mid.abs())) @ w2.abs().t() * 1.02 + 2.0 ** -18 * y.abs()
    assert ((got - y - z).abs() <= bound + off).all()
