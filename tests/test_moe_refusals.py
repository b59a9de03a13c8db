"""What the routed experts and the router refuse, checked without a GPU: the C entry points' argument checks, and the
Python ones' on fake tensors with a stand-in library that records the calls."""

import pytest
import torch

from gaudi_kernels_b200 import _lib
from test_call_routes import lib  # noqa: F401  (the recording library and its fake tensors)

A = 4096                                                   # an aligned address that is never read


@pytest.fixture(scope="module")
def so():
    from gaudi_kernels_b200 import build
    build.build()
    return _lib.load()


def _experts(so, **over):
    a = dict(x=A, ldx=256, ids=A, weights=A, w13=A, s13=A, w2=A, s2=A, out=A, ldo=256, t=4, k=2, e=8, h=256, i=128, half=0,
             ws=A, bytes=1 << 40, status=A)
    a.update(over)
    return so.bfp8_moe_block128(a["x"], a["ldx"], a["ids"], a["weights"], a["w13"], a["s13"], a["w2"], a["s2"], a["out"],
                                a["ldo"], a["t"], a["k"], a["e"], a["h"], a["i"], a["half"], a["ws"], a["bytes"], a["status"],
                                None, 0, 0)


@pytest.mark.parametrize("over,code", [
    ({"x": None}, -1), ({"ids": None}, -1), ({"weights": None}, -1), ({"w13": None}, -1), ({"s2": None}, -1), ({"out": None}, -1),
    ({"ws": None}, -1), ({"status": None}, -1),
    ({"w13": A + 8}, -2), ({"w2": A + 4}, -2), ({"out": A + 4}, -2), ({"ldo": 258}, -2), ({"ws": A + 128}, -2), ({"x": A + 1}, -2),
    ({"t": 0}, -3), ({"k": 0}, -3), ({"e": 0}, -3), ({"h": 0}, -3), ({"i": -16}, -3), ({"ldx": 128}, -3), ({"ldo": 128}, -3),
    ({"t": 129}, -6), ({"k": 33}, -6), ({"t": 128, "k": 17}, -6), ({"e": 513}, -6), ({"h": 248}, -6), ({"i": 120}, -6),
    ({"bytes": 1000}, -4),
])
def test_experts_argument_checks(so, over, code):
    assert _experts(so, **over) == code


def _route(so, **over):
    a = dict(x=A, ldx=64, r=A, ldr=64, bias=None, t=4, h=64, e=8, k=2, scoring=0, ids=A, weights=A, ws=A, bytes=4 * 8 * 4)
    a.update(over)
    return so.bfp8_moe_route(a["x"], a["ldx"], a["r"], a["ldr"], a["bias"], a["t"], a["h"], a["e"], a["k"], a["scoring"], 1, 1.0,
                             a["ids"], a["weights"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("over,code", [
    ({"x": None}, -1), ({"r": None}, -1), ({"ids": None}, -1), ({"weights": None}, -1), ({"ws": None}, -1),
    ({"t": 0}, -3), ({"k": 9}, -3), ({"k": 0}, -3), ({"ldx": 63}, -3), ({"ldr": 32}, -3), ({"scoring": 2}, -3),
    ({"bias": A}, -6), ({"e": 513, "bytes": 1 << 30}, -6), ({"e": 64, "k": 33, "bytes": 1 << 30}, -6),
    ({"x": A + 1}, -2), ({"ids": A + 2}, -2), ({"bytes": 100}, -4),
])
def test_route_argument_checks(so, over, code):
    assert _route(so, **over) == code


def test_workspace_sizes(so):
    assert so.bfp8_moe_route_workspace_bytes(3, 8) == 96
    need = so.bfp8_moe_block128_workspace_bytes(4, 2, 8, 256, 128)
    assert need > 0 and _experts(so, bytes=need - 1) == -4
    assert so.bfp8_moe_block128_workspace_bytes(129, 2, 8, 256, 128) == 0
    assert so.bfp8_moe_block128_workspace_bytes(0, 2, 8, 256, 128) == 0


def _operands(t=4, k=2, e=8, h=256, i=144):
    d = "cuda:0"
    return dict(x=torch.empty((t, h), dtype=torch.bfloat16, device=d), ids=torch.empty((t, k), dtype=torch.int32, device=d),
                weights=torch.empty((t, k), device=d), w_gate_up=torch.empty((e, 2, i, h), dtype=torch.uint8, device=d),
                s_gate_up=torch.empty((e, 2, (i + 127) // 128, (h + 127) // 128), device=d),
                w_down=torch.empty((e, h, i), dtype=torch.uint8, device=d),
                s_down=torch.empty((e, (h + 127) // 128, (i + 127) // 128), device=d))


BAD = [
    ("x", lambda t: t.float()), ("x", lambda t: t[0]), ("x", lambda t: t.t()), ("x", lambda t: t.cpu()),
    ("ids", lambda t: t.long()), ("ids", lambda t: t[:3]), ("ids", lambda t: t[:, :0]), ("ids", lambda t: t.t().contiguous().t()),
    ("weights", lambda t: t.double()), ("weights", lambda t: t[:, :1]), ("weights", lambda t: t.cpu()),
    ("w_gate_up", lambda t: t.float()), ("w_gate_up", lambda t: t[:, :1]), ("w_gate_up", lambda t: t.transpose(2, 3)),
    ("w_gate_up", lambda t: t.flatten(1, 2)), ("w_down", lambda t: t[:, :128]), ("w_down", lambda t: t.cpu()),
    ("s_gate_up", lambda t: t[:, :, :1]), ("s_gate_up", lambda t: t.to(torch.bfloat16)), ("s_down", lambda t: t.transpose(1, 2)),
]


@pytest.mark.parametrize("name,change", BAD)
def test_experts_refuse(lib, name, change):                # noqa: F811
    import gaudi_kernels_b200 as gk
    ops = _operands()
    ops[name] = change(ops[name])
    with pytest.raises(ValueError):
        gk.moe_block_fp8(**ops, check=False)
    assert not lib.calls


@pytest.mark.parametrize("sizes", [{"t": 129}, {"t": 128, "k": 17}, {"t": 2, "k": 33}, {"e": 513, "h": 16, "i": 16}, {"h": 248}, {"i": 136}])
def test_experts_refuse_sizes(lib, sizes):                 # noqa: F811
    import gaudi_kernels_b200 as gk
    with pytest.raises(ValueError):
        gk.moe_block_fp8(**_operands(**sizes), check=False)
    assert not lib.calls


def test_outputs_that_do_not_fit(lib):                     # noqa: F811
    import gaudi_kernels_b200 as gk
    ops = _operands()
    for out in (torch.empty((4, 256), device="cuda:0"), torch.empty((4, 255), dtype=torch.bfloat16, device="cuda:0"),
                torch.empty((256, 4), dtype=torch.bfloat16, device="cuda:0").t(),
                torch.empty((4, 258), dtype=torch.bfloat16, device="cuda:0")[:, :256],
                torch.empty((1, 256), dtype=torch.bfloat16, device="cuda:0").expand(4, 256)):
        with pytest.raises(ValueError):
            gk.moe_block_fp8(**ops, out=out, check=False)
    assert not lib.calls


@pytest.mark.parametrize("over", [
    {"top_k": 0}, {"top_k": 9}, {"scoring": "tanh"}, {"bias": "softmax"}, {"bias": "short"}, {"bias": "half"}, {"router": "float"},
    {"router": "narrow"}, {"router": "cpu"}, {"router": "experts"},
])
def test_routers_refuse(lib, over):                        # noqa: F811
    import gaudi_kernels_b200 as gk
    ops = _operands()
    d = "cuda:0"
    router = {"float": torch.empty((8, 256), device=d), "narrow": torch.empty((8, 240), dtype=torch.bfloat16, device=d),
              "cpu": torch.empty((8, 256), dtype=torch.bfloat16), "experts": torch.empty((513, 256), dtype=torch.bfloat16, device=d)
              }.get(over.get("router"), torch.empty((8, 256), dtype=torch.bfloat16, device=d))
    bias = {"softmax": torch.empty(8, device=d), "short": torch.empty(7, device=d),
            "half": torch.empty(8, dtype=torch.bfloat16, device=d)}.get(over.get("bias"))
    scoring = over.get("scoring", "sigmoid" if over.get("bias") in ("short", "half") else "softmax")
    kw = dict(scoring=scoring, bias=bias)
    w = [ops[n] for n in ("w_gate_up", "s_gate_up", "w_down", "s_down")]
    with pytest.raises(ValueError):
        gk.route_topk(ops["x"], router, over.get("top_k", 2), **kw)
    with pytest.raises(ValueError):
        gk.moe_layer_block_fp8(ops["x"], router, over.get("top_k", 2), *w, check=False, **kw)
    assert not lib.calls


def test_strides_and_arguments_of_the_calls(lib):          # noqa: F811
    import gaudi_kernels_b200 as gk
    ops = _operands(t=1)
    ops["x"] = torch.empty((1, 999), dtype=torch.bfloat16, device="cuda:0")[:, 5:261]
    gk.moe_block_fp8(**ops, native_half=True, check=False, max_ctas=3)
    args = lib.named("bfp8_moe_block128")[0]
    assert args[1] == 256 and args[9] == 256               # one row: the stride is free, the width is given
    assert args[10:16] == (1, 2, 8, 256, 144, 1) and args[20] == 3


def test_the_layer_takes_the_experts_controls(lib):        # noqa: F811
    import gaudi_kernels_b200 as gk
    ops = _operands()
    router = torch.empty((8, 256), dtype=torch.bfloat16, device="cuda:0")
    w = [ops[n] for n in ("w_gate_up", "s_gate_up", "w_down", "s_down")]
    gk.moe_layer_block_fp8(ops["x"], router, 2, *w, check=False, max_ctas=100, wait_limit_cycles=7)
    gk.moe_layer_block_fp8(ops["x"], router, 2, *w, check=False)
    assert [a[-2:] for a in lib.named("bfp8_moe_layer_block128_ex")] == [(100, 7), (0, 0)]


def test_misaligned_choices(so):
    assert _experts(so, ids=A + 2) == -2 and _experts(so, weights=A + 1) == -2
