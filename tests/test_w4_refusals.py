"""What the 4-bit products and their quantizer refuse, checked without a GPU: the C entry points' argument checks, and the
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


@pytest.mark.parametrize("over,code", [
    ({"x": None}, -1), ({"codes": None}, -1), ({"scales": None}, -1), ({"out": None}, -1), ({"status": None}, -1),
    ({"m": 0}, -3), ({"n": 0}, -3), ({"k": 0}, -3), ({"ldx": 56}, -3), ({"ldo": 15}, -3), ({"dtype": 2}, -3), ({"m": (1 << 20) + 1}, -3),
    ({"group": 16}, -6), ({"group": 96}, -6), ({"k": 48}, -6), ({"k": 16}, -6),
    ({"x": A + 8}, -2), ({"codes": A + 4}, -2), ({"ldx": 68}, -2), ({"scales": A + 1}, -2), ({"out": A + 1}, -2),
    ({"out": A + 2, "f32": 1}, -2), ({"bias": A + 2}, -2), ({"status": A + 1}, -2),
])
def test_product_argument_checks(so, over, code):
    a = dict(x=A, ldx=64, dtype=0, codes=A, scales=A, zeros=None, group=64, bias=None, out=A, f32=0, ldo=16, m=2, n=16, k=64, status=A)
    a.update(over)
    assert so.bfp8_gemm_group_w4(a["x"], a["ldx"], a["dtype"], a["codes"], a["scales"], a["zeros"], a["group"], a["bias"], a["out"],
                                 a["f32"], a["ldo"], a["m"], a["n"], a["k"], a["status"], None, 0) == code


@pytest.mark.parametrize("over,code", [
    ({"w": None}, -1), ({"codes": None}, -1), ({"scales": None}, -1), ({"n": 0}, -3), ({"ldw": 32}, -3), ({"dtype": 3}, -3),
    ({"group": 256}, -6), ({"k": 40}, -6), ({"w": A + 2}, -2), ({"scales": A + 1}, -2),
])
def test_quantizer_argument_checks(so, over, code):
    a = dict(w=A, n=4, k=64, ldw=64, group=32, codes=A, scales=A, zeros=A, dtype=0)
    a.update(over)
    assert so.bfp8_quant_group_w4_f32(a["w"], a["n"], a["k"], a["ldw"], a["group"], a["codes"], a["scales"], a["zeros"],
                                      a["dtype"], None) == code


def _operands(m=3, n=40, k=128, group=64, dtype=torch.bfloat16):
    d = "cuda:0"
    return dict(x=torch.empty((m, k), dtype=dtype, device=d), codes=torch.empty((n, k // 2), dtype=torch.uint8, device=d),
                scales=torch.empty((n, k // group), dtype=dtype, device=d),
                zeros=torch.empty((n, k // group), dtype=torch.uint8, device=d), group=group,
                bias=torch.empty(n, device=d))


BAD = [
    ("x", lambda t: t.float()), ("x", lambda t: t[0]), ("x", lambda t: t.cpu()), ("x", lambda t: t[:, :96]),
    ("x", lambda t: t.to(torch.float16)), ("x", lambda t: torch.empty((128, 3), dtype=t.dtype, device=t.device).t()),
    ("codes", lambda t: t.to(torch.int8)), ("codes", lambda t: t[:, :32]), ("codes", lambda t: t[:0]), ("codes", lambda t: t.cpu()),
    ("codes", lambda t: t[::2]),
    ("scales", lambda t: t.float()), ("scales", lambda t: t[:, :1]), ("scales", lambda t: t[:39]), ("scales", lambda t: t.cpu()),
    ("zeros", lambda t: t.float()), ("zeros", lambda t: t[:, :1]), ("zeros", lambda t: t.cpu()),
    ("bias", lambda t: t.double()), ("bias", lambda t: t[:39]), ("bias", lambda t: t.cpu()),
    ("group", lambda g: 16), ("group", lambda g: 32),
]


@pytest.mark.parametrize("name,change", BAD)
def test_products_refuse(lib, name, change):               # noqa: F811
    import gaudi_kernels_b200 as gk
    ops = _operands()
    ops[name] = change(ops[name])
    with pytest.raises(ValueError):
        gk.gemm_group_w4(**ops)
    assert not lib.calls


def test_outputs_and_sizes_that_do_not_fit(lib):           # noqa: F811
    import gaudi_kernels_b200 as gk
    ops, d = _operands(), "cuda:0"
    with pytest.raises(ValueError):
        gk.gemm_group_w4(**ops, out_dtype=torch.float16)
    for out in (torch.empty((3, 39), dtype=torch.bfloat16, device=d), torch.empty((3, 40), dtype=torch.float16, device=d),
                torch.empty((40, 3), dtype=torch.bfloat16, device=d).t(), torch.empty((3, 40), dtype=torch.bfloat16),
                torch.empty((1, 40), dtype=torch.bfloat16, device=d).expand(3, 40)):
        with pytest.raises(ValueError):
            gk.gemm_group_w4(**ops, out=out)
    for k in (16, 48):
        x = torch.empty((2, k), dtype=torch.bfloat16, device=d)
        with pytest.raises(ValueError):
            gk.gemm_group_w4(x, torch.empty((4, k // 2), dtype=torch.uint8, device=d), torch.empty((4, 1), dtype=torch.bfloat16, device=d), group=64)
    assert not lib.calls


def test_quantizer_refuses(lib):                           # noqa: F811
    import gaudi_kernels_b200 as gk
    w = torch.empty((4, 64), device="cuda:0")
    for bad in (w.to(torch.bfloat16), w[0], w[:0], w.t(), w[:, :48]):
        with pytest.raises(ValueError):
            gk.quantize_group_w4(bad, 32)
    with pytest.raises(ValueError):
        gk.quantize_group_w4(w, 48)
    with pytest.raises(ValueError):
        gk.quantize_group_w4(w, 32, scale_dtype=torch.float32)
    assert not lib.calls


def test_rows_and_strides_of_the_call(lib):                # noqa: F811
    import gaudi_kernels_b200 as gk
    ops = _operands()
    ops["x"] = torch.empty((3, 136), dtype=torch.bfloat16, device="cuda:0")[:, :128]
    out = torch.empty((3, 50), dtype=torch.float32, device="cuda:0")[:, :40]
    gk.gemm_group_w4(**ops, out=out)
    args = lib.named("bfp8_gemm_group_w4")[0]
    assert args[1] == 136 and args[2] == 0 and args[6] == 64 and args[9] == 1 and args[10] == 50 and args[11:14] == (3, 40, 128)


def test_what_shares_memory():
    from gaudi_kernels_b200.w4 import _share_memory
    base = torch.empty((6, 64), dtype=torch.bfloat16)

    def really(a, b):
        def taken(t):
            first = t.data_ptr()
            return {first + 2 * (r * t.stride(0) + c) for r in range(t.shape[0]) for c in range(t.shape[1])}
        return bool(taken(a) & taken(b))

    views = [base[:3, :32], base[3:, :32], base[:3, 32:], base[1:4, 8:40], base[1:4, 40:64], base[:1, :32], base[2:3, 16:48],
             base.view(12, 32)[:3], base.view(12, 32)[5:8, :16], base[:3, 31:63], base[:3]]
    for a in views:
        for b in views:
            if a.shape[0] == b.shape[0]:
                assert _share_memory(a, b) or not really(a, b)
                if a.stride(0) == b.stride(0) and a.shape[0] > 1:          # rows of one pitch: exactly
                    span = lambda t: (t.data_ptr(), t.data_ptr() + 2 * ((t.shape[0] - 1) * t.stride(0) + t.shape[1]))    # noqa: E731
                    apart = span(a)[1] <= span(b)[0] or span(b)[1] <= span(a)[0]
                    columns = {(c + a.data_ptr() // 2) % a.stride(0) for c in range(a.shape[1])} & {
                        (c + b.data_ptr() // 2) % b.stride(0) for c in range(b.shape[1])}
                    assert _share_memory(a, b) == (bool(columns) and not apart)
    assert not _share_memory(torch.empty((3, 8)), torch.empty((3, 8)))


def test_fresh_codes_reach_the_call(lib, so):              # noqa: F811
    import gaudi_kernels_b200 as gk
    ops = _operands(dtype=torch.float16)
    gk.gemm_group_w4(**ops)
    gk.gemm_group_w4(**ops, fresh_codes=True)
    assert [a[2] for a in lib.named("bfp8_gemm_group_w4")] == [1, 1 | 0x100]
    args = [A, 64, 0x100, A, A, None, 64, None, A, 0, 16, 2, 16, 64, A + 1, None, 0]
    assert so.bfp8_gemm_group_w4(*args) == -2              # the type under the flag is accepted: only the status word is misaligned
    args[2] = 0x102
    assert so.bfp8_gemm_group_w4(*args) == -3


@pytest.mark.parametrize("m", [65535 * 16 + 1, 1 << 20])
def test_more_rows_than_the_grid_holds(so, m):
    assert so.bfp8_gemm_group_w4(A, 64, 0, A, A, None, 64, None, A, 0, 16, m, 16, 64, A, None, 0) == -3
