"""GPU parity of the router and of the routed block-FP8 experts against their 64-bit restatement (oracle/moe_ref.py)."""

import pytest
import torch

from oracle import fp8_codec_ref, moe_ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def gk():
    import gaudi_kernels_b200 as g
    from gaudi_kernels_b200 import _lib
    _lib.load()
    return g


def _codes(gen, *shape):
    """Every E4M3 code but NaN, both signs."""
    c = torch.randint(0, 0x7f, shape, generator=gen, dtype=torch.uint8)
    return c | (torch.randint(0, 2, shape, generator=gen, dtype=torch.uint8) << 7)


def _blocks(n):
    return (n + 127) // 128


def _problem(t, k, e, h, i, seed=0):
    gen = torch.Generator().manual_seed(1000 * t + 100 * k + e + h + i + seed)
    x = (torch.randn((t, h), generator=gen) * 1.5).to(torch.bfloat16)
    w13, w2 = _codes(gen, e, 2, i, h), _codes(gen, e, h, i)
    s13 = torch.rand((e, 2, _blocks(i), _blocks(h)), generator=gen) * 1e-3 + 1e-4
    s2 = torch.rand((e, _blocks(h), _blocks(i)), generator=gen) * 1e-3 + 1e-4
    ids = torch.stack([torch.randperm(max(e, k), generator=gen)[:k] % e for _ in range(t)]).to(torch.int32)
    weights = torch.rand((t, k), generator=gen) + 0.05
    return x, ids, weights, w13, s13, w2, s2


def _run(gk, args, **kw):
    return gk.moe_block_fp8(*[a.to(DEV) for a in args], **kw)


def _check(got, args, half):
    y, bound = moe_ref.experts(*args, half)
    off = (got.double().cpu() - y).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), "worst %.3g of the bound" % float((off / bound).max())
    # the bound itself is tight: most of it is the bf16 step
    assert float(bound.norm()) <= 0.05 * float(y.norm()) + 1e-30


SHAPES = [
    # t, k, e, h, i
    (1, 1, 1, 16, 16),                 # the smallest sizes
    (1, 2, 4, 128, 128),               # one block everywhere, fewer units than CTAs
    (1, 8, 128, 512, 256),             # one token, many experts
    (2, 1, 3, 2048, 128),              # long K of gate / up, one item each: split over many CTAs
    (3, 2, 5, 144, 272),               # ragged in both widths
    (5, 4, 9, 400, 208),
    (7, 3, 16, 1040, 1360),
    (16, 8, 16, 256, 384),
    (17, 3, 6, 512, 256),              # beyond 16 tokens
    (33, 2, 3, 272, 144),              # chunks of more than 16 slots
    (64, 4, 4, 384, 128),              # an expert with exactly 64 slots
    (65, 2, 2, 128, 640),              # ... with 65: a second chunk of one
    (128, 2, 1, 256, 128),             # one expert takes 256 slots
    (128, 16, 64, 128, 128),           # the most slots
    (100, 6, 512, 160, 144),           # the most experts
]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("t,k,e,h,i", SHAPES)
def test_experts_match_the_definition(gk, t, k, e, h, i, half):
    args = _problem(t, k, e, h, i)
    _check(_run(gk, args, native_half=half), args, half)


# widths of real layers in one dimension at a time, and the widest allowed
WIDE = [(1, 1, 2, 7168, 256), (3, 2, 4, 256, 14336), (20, 2, 3, 8192, 272), (20, 2, 3, 272, 8208), (1, 1, 1, 65536, 16), (18, 1, 2, 16, 65536)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("t,k,e,h,i", WIDE)
def test_wide_experts_match_the_definition(gk, t, k, e, h, i, half):
    args = _problem(t, k, e, h, i)
    got = _run(gk, args, native_half=half)
    if max(h, i) < 65536:
        _check(got, args, half)
    else:                                                  # the bound of so long a sum is no longer small beside the result
        y, bound = moe_ref.experts(*args, half)
        assert ((got.double().cpu() - y).abs() <= bound).all()


@pytest.mark.parametrize("t,k", [(9, 3), (40, 2)])
@pytest.mark.parametrize("ctas", [1, 2, 5, 31, 147])
def test_any_number_of_ctas(gk, t, k, ctas):
    # the parts of an item that several CTAs share, for every way the list can be cut
    args = _problem(t, k, 4, 640, 528)
    _check(_run(gk, args, max_ctas=ctas), args, False)


@pytest.mark.parametrize("t", [6, 70])
def test_masked_repeated_and_missing_choices(gk, t):
    x, ids, weights, *w = _problem(t, 4, 6, 272, 144)
    ids[0] = -1                                        # a token whose experts are all elsewhere
    ids[1] = 3                                         # the same expert four times
    ids[2, 1:] = -1
    ids[3:, 2] = 5
    weights[4, 0] = 0.0
    weights[5] = -weights[5]
    ids[ids == 4] = -7                                 # any negative number; expert 4 gets no slot
    args = (x, ids, weights, *w)
    got = _run(gk, args)
    _check(got, args, False)
    assert (got[0] == 0).all()


def test_no_choice_at_all(gk):
    x, ids, *rest = _problem(3, 2, 4, 128, 128)
    got = _run(gk, (x, torch.full_like(ids, -1), *rest))
    assert got.shape == (3, 128) and (got == 0).all()


def test_no_tokens(gk):
    x, ids, weights, *w = _problem(1, 2, 4, 128, 128)
    assert _run(gk, (x[:0], ids[:0], weights[:0], *w)).shape == (0, 128)
    r = torch.zeros((4, 128), dtype=torch.bfloat16, device=DEV)
    out, i2, w2 = gk.moe_layer_block_fp8(x[:0].to(DEV), r, 2, *[a.to(DEV) for a in w])
    assert out.shape == (0, 128) and i2.shape == (0, 2) and w2.shape == (0, 2)


def test_an_index_beyond_the_last_expert_is_reported_and_adds_nothing(gk):
    args = _problem(4, 2, 5, 128, 256)
    ids = args[1]
    kept = ids.clone()
    ids[1, 0], kept[1, 0] = 5, -1
    ids[3, 1], kept[3, 1] = 2 ** 31 - 1, -1
    with pytest.raises(ValueError, match="beyond the last expert"):
        _run(gk, args)
    _check(_run(gk, args, check=False), (args[0], kept, *args[2:]), False)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("t", [5, 20])
def test_nonfinite_tokens_stay_alone(gk, t, value):
    x, ids, weights, *w = _problem(t, 2, 3, 256, 144)
    x[2, 200] = value
    got = _run(gk, (x, ids, weights, *w)).cpu()
    assert not torch.isfinite(got[2]).any()
    keep = [r for r in range(t) if r != 2]
    _check(got[keep], (x[keep], ids[keep], weights[keep], *w), False)


def test_zero_rows_and_tiny_values(gk):
    x, ids, weights, *w = _problem(4, 2, 3, 256, 128)
    x[0] = 0.0
    x[1, 128:] = 0.0
    x[2] *= 1e-30                                      # below the floor of the scale
    args = (x, ids, weights, *w)
    got = _run(gk, args)
    assert (got[0] == 0).all()
    _check(got, args, False)


def test_strided_rows_and_a_given_output(gk):
    x, ids, weights, *w = _problem(5, 2, 4, 272, 128)
    want = _run(gk, (x, ids, weights, *w))
    wide = torch.full((5, 301), 7.0, dtype=torch.bfloat16, device=DEV)
    wide[:, 1:273] = x.to(DEV)                         # rows that start anywhere: the unaligned loads
    big = torch.full((7, 280), 3.0, dtype=torch.bfloat16, device=DEV)
    out = gk.moe_block_fp8(wide[:, 1:273], ids.to(DEV), weights.to(DEV), *[a.to(DEV) for a in w], out=big[1:6, 4:276])
    assert torch.equal(out, want) and out.data_ptr() == big[1:6, 4:276].data_ptr()
    assert (big[0] == 3).all() and (big[6] == 3).all() and (big[:, :4] == 3).all() and (big[:, 276:] == 3).all()


def test_broadcast_rows_and_an_output_in_place(gk):
    x, ids, weights, *w = [a.to(DEV) for a in _problem(6, 2, 4, 272, 128)]
    same = x[2:3].expand(6, 272)
    want = gk.moe_block_fp8(same.contiguous(), ids, weights, *w)
    assert torch.equal(gk.moe_block_fp8(same, ids, weights, *w), want)
    r = torch.randn((4, 272), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    for a, b in zip(gk.route_topk(same, r, 2), gk.route_topk(same.contiguous(), r, 2)):
        assert torch.equal(a, b)
    want, keep = gk.moe_block_fp8(x, ids, weights, *w), x.clone()
    assert gk.moe_block_fp8(x, ids, weights, *w, out=x) is x and torch.equal(x, want)
    x.copy_(keep)
    want = gk.moe_layer_block_fp8(x, r, 2, *w)
    got = gk.moe_layer_block_fp8(x, r, 2, *w, out=x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_weights_prepared_in_the_half_range(gk):
    x, ids, weights, w13, s13, w2, s2 = _problem(6, 2, 4, 272, 144)
    p13, q13 = gk.prepare_weight(w13.view(torch.float8_e4m3fn).to(DEV), s13.to(DEV))
    p2, q2 = gk.prepare_weight(w2.view(torch.float8_e4m3fn).to(DEV), s2.to(DEV))
    assert p13.shape == w13.shape and torch.equal(q13.cpu(), 2 * s13)
    got = gk.moe_block_fp8(x.to(DEV), ids.to(DEV), weights.to(DEV), p13, q13, p2, q2, native_half=True)
    _check(got, (x, ids, weights, p13.cpu().view(torch.uint8), q13.cpu(), p2.cpu().view(torch.uint8), q2.cpu()), True)


def test_many_calls_of_several_shapes_at_once(gk):
    # cooperative launches of four streams beside a library product: every wait ends, every result is the lone call's
    from gaudi_kernels_b200.block_fp8_gemm import new_status
    shapes = ((1, 8, 32, 512, 384), (12, 4, 16, 1040, 656), (40, 4, 32, 512, 256), (128, 8, 32, 256, 128))
    args = [[a.to(DEV) for a in _problem(*s)] for s in shapes]
    want = [gk.moe_block_fp8(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in range(5)]
    status = [new_status(torch.device(DEV)) for _ in args]
    big = torch.ones((4096, 4096), dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    outs = [[] for _ in args]
    for n in range(40):
        for i, a in enumerate(args):
            with torch.cuda.stream(streams[i]):
                outs[i].append(gk.moe_block_fp8(*a, check=False, status=status[i]))
        if n % 8 == 0:
            with torch.cuda.stream(streams[4]):
                big @ big
    torch.cuda.synchronize()
    assert all(s.tolist()[2] == 0 for s in status)
    assert all(torch.equal(o, w) for got, w in zip(outs, want) for o in got)


def test_results_repeat_and_calls_overlap(gk):
    args = [a.to(DEV) for a in _problem(12, 4, 8, 640, 400)]
    want = gk.moe_block_fp8(*args)
    side = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for n in range(24):
        with torch.cuda.stream(side[n % 3]):
            outs.append(gk.moe_block_fp8(*args, check=False))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_captured_calls_replay_on_new_inputs(gk):
    x, ids, weights, *w = [a.to(DEV) for a in _problem(9, 3, 8, 384, 256)]
    gen = torch.Generator().manual_seed(5)
    router = torch.randn((8, 384), generator=gen).to(torch.bfloat16).to(DEV)
    other = torch.randn((9, 384), generator=gen).to(torch.bfloat16).to(DEV)
    gk.moe_layer_block_fp8(x, router, 3, *w)
    xs = x.clone()
    graphs = []
    for _ in range(2):                                  # two graphs of the same leaves, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, i, g = gk.moe_layer_block_fp8(xs, router, 3, *w, check=False)
            z = gk.moe_block_fp8(y, i, g, *w, check=False)
        graphs.append((graph, y, z))
    for v in (x, other, x):
        want_y, want_i, want_g = gk.moe_layer_block_fp8(v, router, 3, *w)
        want_z = gk.moe_block_fp8(want_y, want_i, want_g, *w)
        xs.copy_(v)
        for graph, y, z in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, y, z in graphs:
            assert torch.equal(y, want_y) and torch.equal(z, want_z)


def test_an_expired_wait_is_reported_and_the_next_call_is_whole(gk):
    from gaudi_kernels_b200 import _lib
    args = _problem(9, 3, 4, 640, 528)
    with pytest.raises(_lib.Bfp8Error, match="bounded wait"):
        _run(gk, args, wait_limit_cycles=1)
    _check(_run(gk, args), args, False)


@pytest.mark.parametrize("t", [2, 40])
@pytest.mark.parametrize("ctas", [1, 7, 100])
def test_the_layer_on_some_of_the_sms(gk, t, ctas):
    x, _, _, *w = [a.to(DEV) for a in _problem(t, 3, 24, 272, 144)]
    _, r, _ = _route_problem(1, 24, 272, seed=t)
    ids, weights = gk.route_topk(x, r.to(DEV), 3)
    want = gk.moe_block_fp8(x, ids, weights, *w, max_ctas=ctas)
    out, i2, w2 = gk.moe_layer_block_fp8(x, r.to(DEV), 3, *w, max_ctas=ctas)
    assert torch.equal(i2, ids) and torch.equal(w2, weights) and torch.equal(out, want)


def test_an_expired_wait_of_the_layer_is_reported_and_the_next_call_is_whole(gk):
    from gaudi_kernels_b200 import _lib
    x, _, _, *w = [a.to(DEV) for a in _problem(9, 3, 4, 640, 528)]
    _, r, _ = _route_problem(1, 4, 640)
    want = gk.moe_layer_block_fp8(x, r.to(DEV), 3, *w)
    with pytest.raises(_lib.Bfp8Error, match="bounded wait"):
        gk.moe_layer_block_fp8(x, r.to(DEV), 3, *w, wait_limit_cycles=1)
    assert all(torch.equal(a, b) for a, b in zip(gk.moe_layer_block_fp8(x, r.to(DEV), 3, *w), want))


def test_experts_after_the_quantizer_and_the_gemm_of_one_stream(gk):
    # a decode step: a block-FP8 projection, the routed layer on its result, another projection - against the same calls
    # with a wait between them
    x, ids, weights, *w = [a.to(DEV) for a in _problem(8, 2, 4, 256, 128)]
    gen = torch.Generator().manual_seed(3)
    pc, ps = fp8_codec_ref.quantize_block128(torch.randn((256, 256), generator=gen).numpy() * 0.05)
    pc, ps = torch.from_numpy(pc).to(DEV), torch.from_numpy(ps).to(DEV)

    def step(wait):
        y = x
        for _ in range(3):
            a, s = gk.quantize_act_1x128(y)
            y = gk.gemm_block_fp8(a, s, pc, ps, check=False)
            if wait:
                torch.cuda.synchronize()
            y = gk.moe_block_fp8(y, ids, weights, *w, check=False)
            if wait:
                torch.cuda.synchronize()
        return y

    want = step(True)
    for _ in range(5):
        assert torch.equal(step(False), want)


# ---- router ---------------------------------------------------------------------------------------------------------

ROUTES = [
    # t, e, h, k
    (1, 1, 8, 1), (1, 64, 2048, 8), (3, 33, 72, 5), (4, 8, 77, 8), (5, 60, 400, 4), (9, 256, 1024, 8), (130, 512, 160, 32),
    (17, 31, 4096, 6),
]


def _route_problem(t, e, h, seed=0):
    gen = torch.Generator().manual_seed(t + 7 * e + 13 * h + seed)
    x = torch.randn((t, h), generator=gen).to(torch.bfloat16)
    r = (torch.randn((e, h), generator=gen) / h ** 0.5).to(torch.bfloat16)
    return x, r, torch.randn(e, generator=gen) * 0.1


def _check_route(got, want, gap, scale):
    ids, weights = got
    assert gap > 1e-7, "the test's own inputs leave the order open"
    assert torch.equal(ids.cpu(), want[0])
    # scores are fp32 roundings of sums held to 1e-8; |score| <= 8 here, so an exponent is off by at most 2^-21 + 2^-23
    # and expf, the sum of up to 512 terms in 32 lanes and the divisions add some 2^-24 each: 2^-18 in all
    assert torch.allclose(weights.double().cpu(), want[1], rtol=2.0 ** -18, atol=scale * 1e-30)


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,h,k", ROUTES)
def test_route_matches_the_definition(gk, t, e, h, k, scoring, renorm):
    x, r, bias = _route_problem(t, e, h)
    bias = bias if scoring == "sigmoid" and e % 2 == 0 else None
    ids, w, gap = moe_ref.route(x, r, k, scoring, renorm, bias, 2.5)
    got = gk.route_topk(x.to(DEV), r.to(DEV), k, scoring=scoring, renormalize=renorm,
                        bias=None if bias is None else bias.to(DEV), scale=2.5)
    _check_route(got, (ids, w), gap, 2.5)


@pytest.mark.parametrize("t,e,h", [(40, 250, 264), (40, 250, 77), (70, 500, 96), (6, 7, 2056), (200, 24, 40), (3, 511, 4104), (2, 1, 300)])
def test_route_for_every_way_to_cut_the_work(gk, t, e, h):
    x, r, bias = _route_problem(t, e, h)
    k = min(e, 9)
    want = moe_ref.route(x, r, k, "sigmoid", True, bias, 2.5)
    _check_route(gk.route_topk(x.to(DEV), r.to(DEV), k, scoring="sigmoid", bias=bias.to(DEV), scale=2.5), want[:2], want[2], 2.5)


@pytest.mark.parametrize("t", [1, 4, 5, 40, 300])
def test_router_sums_are_exact_where_large_terms_cancel(gk, t):
    # two columns of every token a thousand times the others, with products that cancel: what is left is the sum of the small
    # terms, which fp32 sums lose to 2^-24 of the large ones
    gen = torch.Generator().manual_seed(t)
    e, h, k = 200, 2048, 8
    x = torch.randn((t, h), generator=gen).to(torch.bfloat16)
    r = (torch.randn((e, h), generator=gen) / h ** 0.5).to(torch.bfloat16)
    x[:, 7] *= 1000
    x[:, 1500] = -x[:, 7]
    r[:, 1500] = r[:, 7]
    l64 = x.double() @ r.double().t()
    order = torch.sort(l64.float(), dim=1, descending=True, stable=True).indices[:, :k]
    want = torch.sigmoid(l64.gather(1, order))
    assert (l64.gather(1, order) > 0).all()
    ids, w = gk.route_topk(x.to(DEV), r.to(DEV), k, scoring="sigmoid", renormalize=False)
    # l and its sigmoid are rounded to fp32, half a step each: 2^-24 relative, the first times l (1 - sigmoid(l)) <= 0.28;
    # sums of 2048 fp64 terms are off by 2048 2^-53 of their magnitudes' sum, about 200 here, which is far below
    assert torch.equal(ids.cpu().long(), order)
    assert ((w.double().cpu() - want).abs() <= 1.29 * 2.0 ** -24 * want).all()
    # and no token's choice depends on how many others there are
    for n in (1, 2, 5, 17):
        part = gk.route_topk(x[:n].to(DEV), r.to(DEV), k, scoring="sigmoid", renormalize=False)
        assert torch.equal(part[0], ids[:n]) and torch.equal(part[1], w[:n])


def test_route_ties_go_to_the_lower_index(gk):
    x, r, _ = _route_problem(6, 40, 256)
    r[11], r[30], r[5] = r[2], r[2], r[39]
    r[20] = 0.0
    r[21] = -r[20]
    ids, w, _ = moe_ref.route(x, r, 32, "softmax")
    got = gk.route_topk(x.to(DEV), r.to(DEV), 32)
    assert torch.equal(got[0].cpu(), ids)


def test_route_masks_and_nonfinite_scores(gk):
    x, r, bias = _route_problem(5, 12, 128)
    bias[[0, 3, 4, 7]] = float("-inf")                  # masked experts
    bias[9] = torch.finfo(torch.float32).min
    ids, w, _ = moe_ref.route(x, r, 7, "sigmoid", True, bias)
    got = gk.route_topk(x.to(DEV), r.to(DEV), 7, scoring="sigmoid", bias=bias.to(DEV))
    assert torch.equal(got[0].cpu(), ids) and torch.allclose(got[1].double().cpu(), w, rtol=2.0 ** -18)
    bias[:] = float("-inf")                             # nothing is left: the lowest indexes, in order
    got = gk.route_topk(x.to(DEV), r.to(DEV), 7, scoring="sigmoid", bias=bias.to(DEV))
    assert got[0].cpu().tolist() == [list(range(7))] * 5
    r[2, 5] = float("nan")                              # one expert's scores are NaN: it ranks last, the weights follow
    got = gk.route_topk(x.to(DEV), r.to(DEV), 12)
    assert (got[0][:, 11] == 2).all() and (got[0][:, :11] != 2).all()
    got = gk.route_topk(x.to(DEV), r.to(DEV), 11)
    assert torch.isfinite(got[1]).all()


def test_route_reads_strided_rows(gk):
    x, r, _ = _route_problem(5, 24, 128)
    want = gk.route_topk(x.to(DEV), r.to(DEV), 4)
    wx, wr = torch.zeros((5, 140), dtype=torch.bfloat16, device=DEV), torch.zeros((24, 131), dtype=torch.bfloat16, device=DEV)
    wx[:, 3:131], wr[:, 1:129] = x.to(DEV), r.to(DEV)
    got = gk.route_topk(wx[:, 3:131], wr[:, 1:129], 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("t", [1, 5, 20, 128])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_layer_is_route_then_experts(gk, t, scoring):
    x, _, _, *w = [a.to(DEV) for a in _problem(t, 3, 40, 272, 144)]
    _, r, bias = _route_problem(1, 40, 272, seed=t)
    r, bias = r.to(DEV), bias.to(DEV) if scoring == "sigmoid" else None
    for half in (False, True):
        ids, weights = gk.route_topk(x, r, 3, scoring=scoring, bias=bias, scale=1.5)
        want = gk.moe_block_fp8(x, ids, weights, *w, native_half=half)
        out, i2, w2 = gk.moe_layer_block_fp8(x, r, 3, *w, scoring=scoring, bias=bias, scale=1.5, native_half=half)
        assert torch.equal(i2, ids) and torch.equal(w2, weights) and torch.equal(out, want)
