"""Routed experts of a decode step: the router's choice and a whole block-FP8 mixture-of-experts layer for a few tokens.

The experts' weights are E4M3 codes with a scale per 128 x 128 block, the format of gemm_block_fp8; activations and the
intermediate h are quantized to E4M3 in groups of 128 columns as quantize_act_1x128 does.  A layer is two kernels whatever
the routing is: the router's products with the activation quantizer, and the experts (libbfp8.so, csrc/moe.cu).  The
reference has no mixture-of-experts kernels.
"""

import functools

import torch

from . import _lib
from .block_fp8_gemm import _WAIT_TIMEOUT_MSG
from .fp8_codec import BLOCK, _device_guard, _empty, _read_status, _status_buffer, _status_sink, _stream_ptr

MAX_TOKENS, MAX_TOP_K, MAX_SLOTS, MAX_EXPERTS, MAX_WIDTH = 128, 32, 2048, 512, 1 << 16
_SCORING = {"softmax": 0, "sigmoid": 1}
_E4M3 = (torch.float8_e4m3fn, torch.uint8)
_BF16, _F32, _I32, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8


@functools.lru_cache(maxsize=None)
def _workspace_bytes(t, k, experts, h, inter):
    """A pure function of the sizes; the C call takes longer than looking it up."""
    return _lib.load().bfp8_moe_block128_workspace_bytes(t, k, experts, h, inter)


# A decode step's calls are bound by the host where the batch is small, so the checks below touch each property once and
# build their messages only when they fail.

def _check_rows(x):
    if (not isinstance(x, torch.Tensor) or x.dtype != _BF16 or x.ndim != 2 or not x.is_cuda or x.shape[1] < 1
            or (x.stride(1) != 1 and x.shape[1] > 1)):
        raise ValueError("x must be a bf16 [T, H] CUDA tensor with unit column stride")


def _check_router(dev, h, router_weight, top_k, scoring, bias):
    """Checked arguments of a router: the number of experts."""
    if (not isinstance(router_weight, torch.Tensor) or router_weight.dtype != _BF16 or router_weight.ndim != 2
            or router_weight.device != dev):
        raise ValueError("router_weight must be bf16 [E, H] on x's device")
    experts, width = router_weight.shape
    if width != h or experts < 1 or (router_weight.stride(1) != 1 and h > 1):
        raise ValueError("router_weight must be [E, H] with x's H and unit column stride")
    if scoring not in _SCORING:
        raise ValueError("scoring must be 'softmax' or 'sigmoid'")
    if not 1 <= top_k <= min(experts, MAX_TOP_K) or experts > MAX_EXPERTS:
        raise ValueError("1 <= top_k <= min(E, %d) and E <= %d required" % (MAX_TOP_K, MAX_EXPERTS))
    if bias is not None:
        if scoring != "sigmoid":
            raise ValueError("a bias on the choice goes with sigmoid scoring")
        if bias.dtype != _F32 or bias.shape != (experts,) or not bias.is_contiguous() or bias.device != dev:
            raise ValueError("bias must be contiguous FP32 [E] on x's device")
    return experts


def _row_stride(t, rows, width):
    return t.stride(0) if rows > 1 else width


def _rows_apart(t, rows, width):
    """t itself, or a copy where its rows overlap (a broadcast one): the kernels take any pitch from the width on."""
    return t.contiguous() if rows > 1 and t.stride(0) < width else t


def route_topk(x, router_weight, top_k, *, scoring="softmax", renormalize=True, bias=None, scale=1.0):
    """(ids int32 [T, top_k], weights fp32 [T, top_k]): the experts of every token, in descending order of their score.

    l = fp32(x . router_weight^T), the sum formed in fp64.  scoring "softmax": the largest l,
    weights softmax(l) at them, over the chosen ones alone with `renormalize`.  "sigmoid": the largest
    fp32(sigmoid(l) + bias), weights sigmoid(l) at them, divided by their sum with `renormalize`.  Weights are multiplied by
    `scale`.  Ties go to the lower index; a NaN ranks last.  x bf16 [T, H], router_weight bf16 [E, H], E <= 512, any T.
    """
    _check_rows(x)
    t, h = x.shape
    dev = x.device
    experts = _check_router(dev, h, router_weight, top_k, scoring, bias)
    lib = _lib.load()
    with _device_guard(dev):
        x, router_weight = _rows_apart(x, t, h), _rows_apart(router_weight, experts, h)
        ids = _empty(t, top_k, _I32, dev)
        weights = _empty(t, top_k, _F32, dev)
        if t == 0:
            return ids, weights
        scores = _empty(t, experts, _F32, dev)
        rc = lib.bfp8_moe_route(x.data_ptr(), _row_stride(x, t, h), router_weight.data_ptr(),
                                _row_stride(router_weight, experts, h), None if bias is None else bias.data_ptr(), t, h, experts,
                                top_k, _SCORING[scoring], 1 if renormalize else 0, scale, ids.data_ptr(), weights.data_ptr(),
                                scores.data_ptr(), t * experts * 4, _stream_ptr(dev))
        if rc:
            _lib.check(rc, "bfp8_moe_route")
    return ids, weights


def _check_experts(dev, t, h, top_k, w_gate_up, s_gate_up, w_down, s_down, out):
    """Checked arguments of the experts: (E, I)."""
    if (not isinstance(w_gate_up, torch.Tensor) or w_gate_up.dtype not in _E4M3 or w_gate_up.ndim != 4
            or not w_gate_up.is_contiguous() or w_gate_up.device != dev):
        raise ValueError("w_gate_up must be a contiguous 4-D E4M3 tensor on x's device")
    if (not isinstance(w_down, torch.Tensor) or w_down.dtype not in _E4M3 or not w_down.is_contiguous()
            or w_down.device != dev):
        raise ValueError("w_down must be a contiguous 3-D E4M3 tensor on x's device")
    experts, two, inter, width = w_gate_up.shape
    if two != 2 or width != h or w_down.shape != (experts, h, inter) or experts < 1 or inter < 1:
        raise ValueError("w_gate_up [E, 2, I, H] and w_down [E, H, I] must agree with x [T, H]")
    gh, gi = (h + BLOCK - 1) // BLOCK, (inter + BLOCK - 1) // BLOCK
    if (not isinstance(s_gate_up, torch.Tensor) or s_gate_up.dtype != _F32 or s_gate_up.shape != (experts, 2, gi, gh)
            or not s_gate_up.is_contiguous() or s_gate_up.device != dev):
        raise ValueError("s_gate_up must be contiguous FP32 %s on x's device" % ((experts, 2, gi, gh),))
    if (not isinstance(s_down, torch.Tensor) or s_down.dtype != _F32 or s_down.shape != (experts, gh, gi)
            or not s_down.is_contiguous() or s_down.device != dev):
        raise ValueError("s_down must be contiguous FP32 %s on x's device" % ((experts, gh, gi),))
    if h % 16 or inter % 16 or h > MAX_WIDTH or inter > MAX_WIDTH:
        raise ValueError("H and I must be multiples of 16 and at most %d" % MAX_WIDTH)
    if t > MAX_TOKENS or top_k > MAX_TOP_K or t * top_k > MAX_SLOTS or experts > MAX_EXPERTS:
        raise ValueError("at most %d tokens, %d choices per token, %d in all and %d experts"
                         % (MAX_TOKENS, MAX_TOP_K, MAX_SLOTS, MAX_EXPERTS))
    if out is not None and (out.dtype != _BF16 or out.shape != (t, h) or out.stride(1) != 1 or out.device != dev
                            or (t > 1 and (out.stride(0) < h or out.stride(0) % 4)) or out.data_ptr() % 8):
        raise ValueError("out must be bf16 [T, H] on x's device, rows of unit stride starting on 8-byte boundaries")
    return experts, inter


def _raise_for(status):
    status = _read_status(status)[1]
    if status & _lib.STATUS_WAIT_TIMEOUT:
        raise _lib.Bfp8Error(_WAIT_TIMEOUT_MSG)
    if status & _lib.STATUS_BAD_INDEX:
        raise ValueError("an expert index is beyond the last expert")


def moe_block_fp8(x, ids, weights, w_gate_up, s_gate_up, w_down, s_down, *, native_half=False, out=None, check=True,
                  status=None, max_ctas=0, wait_limit_cycles=0):
    """bf16 [T, H]: out[t] = sum_j weights[t, j] * expert ids[t, j] of x[t], expert e of v = down(silu(gate(v)) * up(v)).

    x          bf16 [T, H], T <= 128, rows of unit stride;  ids int32 [T, k];  weights fp32 [T, k]
    w_gate_up  E4M3 [E, 2, I, H] (gate, then up), s_gate_up fp32 [E, 2, ceil(I/128), ceil(H/128)]
    w_down     E4M3 [E, H, I],                    s_down    fp32 [E, ceil(H/128), ceil(I/128)]
    H and I are multiples of 16.  x, and silu(gate) * up in fp32, are quantized as quantize_act_1x128(native_half) does.
    A negative id adds nothing (an expert that another GPU holds); one beyond the last expert adds nothing either and,
    with `check`, raises ValueError.  An expert may occur several times in a token.  check, status, max_ctas and
    wait_limit_cycles as in gemm_block_fp8.  Calls need no workspace of the caller's and may overlap; out may be x.
    """
    _check_rows(x)
    t, h = x.shape
    dev = x.device
    if (not isinstance(ids, torch.Tensor) or ids.dtype != _I32 or ids.ndim != 2 or not ids.is_contiguous()
            or ids.device != dev):
        raise ValueError("ids must be contiguous INT32 [T, k] on x's device")
    rows, k = ids.shape
    if rows != t or k < 1:
        raise ValueError("ids must be [T, k] with x's T and at least one choice")
    if (not isinstance(weights, torch.Tensor) or weights.dtype != _F32 or weights.shape != (t, k)
            or not weights.is_contiguous() or weights.device != dev):
        raise ValueError("weights must be contiguous FP32 [T, k] on x's device")
    experts, inter = _check_experts(dev, t, h, k, w_gate_up, s_gate_up, w_down, s_down, out)
    lib = _lib.load()
    with _device_guard(dev):
        x = _rows_apart(x, t, h)
        if out is None:
            out = _empty(t, h, _BF16, dev)
        if t == 0:
            return out
        nbytes = _workspace_bytes(t, k, experts, h, inter)
        ws = torch.empty_strided((nbytes,), (1,), dtype=_U8, device=dev)
        st = status if status is not None else _status_buffer(dev) if check else _status_sink(dev)
        rc = lib.bfp8_moe_block128(x.data_ptr(), _row_stride(x, t, h), ids.data_ptr(), weights.data_ptr(), w_gate_up.data_ptr(),
                                   s_gate_up.data_ptr(), w_down.data_ptr(), s_down.data_ptr(), out.data_ptr(),
                                   _row_stride(out, t, h), t, k, experts, h, inter, 1 if native_half else 0, ws.data_ptr(), nbytes,
                                   st.data_ptr() + 8, _stream_ptr(dev), max_ctas, wait_limit_cycles)
        if rc:
            _lib.check(rc, "bfp8_moe_block128")
        if check:
            _raise_for(st)
    return out


def moe_layer_block_fp8(x, router_weight, top_k, w_gate_up, s_gate_up, w_down, s_down, *, scoring="softmax", renormalize=True,
                        bias=None, scale=1.0, native_half=False, out=None, check=True, status=None, max_ctas=0,
                        wait_limit_cycles=0):
    """(out bf16 [T, H], ids, weights): route_topk and moe_block_fp8 on its choice as two kernels, the same bits.

    Arguments as theirs; max_ctas and wait_limit_cycles are the experts' kernel's.
    """
    _check_rows(x)
    t, h = x.shape
    dev = x.device
    experts = _check_router(dev, h, router_weight, top_k, scoring, bias)
    held, inter = _check_experts(dev, t, h, top_k, w_gate_up, s_gate_up, w_down, s_down, out)
    if held != experts:
        raise ValueError("router_weight [E, H] and w_gate_up [E, 2, I, H] must share E")
    lib = _lib.load()
    with _device_guard(dev):
        x, router_weight = _rows_apart(x, t, h), _rows_apart(router_weight, experts, h)
        if out is None:
            out = _empty(t, h, _BF16, dev)
        ids = _empty(t, top_k, _I32, dev)
        weights = _empty(t, top_k, _F32, dev)
        if t == 0:
            return out, ids, weights
        nbytes = _workspace_bytes(t, top_k, experts, h, inter)
        ws = torch.empty_strided((nbytes,), (1,), dtype=_U8, device=dev)
        st = status if status is not None else _status_buffer(dev) if check else _status_sink(dev)
        rc = lib.bfp8_moe_layer_block128_ex(x.data_ptr(), _row_stride(x, t, h), router_weight.data_ptr(),
                                            _row_stride(router_weight, experts, h), None if bias is None else bias.data_ptr(),
                                            _SCORING[scoring], 1 if renormalize else 0, scale, ids.data_ptr(), weights.data_ptr(),
                                            w_gate_up.data_ptr(), s_gate_up.data_ptr(), w_down.data_ptr(), s_down.data_ptr(),
                                            out.data_ptr(), _row_stride(out, t, h), t, top_k, experts, h, inter,
                                            1 if native_half else 0, ws.data_ptr(), nbytes, st.data_ptr() + 8, _stream_ptr(dev),
                                            max_ctas, wait_limit_cycles)
        if rc:
            _lib.check(rc, "bfp8_moe_layer_block128")
        if check:
            _raise_for(st)
    return out, ids, weights
