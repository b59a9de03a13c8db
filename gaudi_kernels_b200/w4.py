"""4-bit weights with a scale (and a zero point) per group of k, for products of a few activation rows.

W[n, k] = (q[n, k] - z[n, k // group]) * s[n, k // group], q packed two to a byte (even k in the low four bits).  The weight is
read as it is stored: no repacked copy.  Kernels: libbfp8.so, csrc/w4.cu.  The reference has no 4-bit weights.
"""

import torch

from . import _lib
from .block_fp8_gemm import _WAIT_TIMEOUT_MSG
from .fp8_codec import _device_for, _device_guard, _empty, _read_status, _status_buffer, _status_sink, _stream_ptr

GROUPS = (32, 64, 128)
_DTYPE = {torch.bfloat16: 0, torch.float16: 1}


def quantize_group_w4(w, group=128, zeros=True, scale_dtype=torch.bfloat16):
    """fp32 [N, K] -> (codes uint8 [N, K / 2], scales [N, ceil(K / group)], zeros uint8 of that shape or None).

    With zeros: s = round((max(w, 0) - min(w, 0)) / 15), z = clamp(rne(-min / s), 0, 15); without: s = round(max|w| / 7) and
    z = 8 everywhere.  q = clamp(rne(w / s) + z, 0, 15).  Scales are rounded to scale_dtype (bfloat16 or float16) before they
    are used.  K is a multiple of 32.  A group of zeros gets s = 1, one with a NaN s = NaN, one with an infinity (or a range
    beyond fp32, or a scale beyond scale_dtype) s = inf: such a group does not read back as finite numbers.
    """
    if not isinstance(w, torch.Tensor) or w.dtype != torch.float32 or w.ndim != 2 or not w.numel() or w.stride(1) != 1:
        raise ValueError("expected a nonempty FP32 [N, K] tensor with unit stride along the last dimension")
    if group not in GROUPS or w.shape[1] % 32:
        raise ValueError("group must be 32, 64 or 128 and K a multiple of 32")
    if scale_dtype not in _DTYPE:
        raise ValueError("scale_dtype must be bfloat16 or float16")
    lib = _lib.load()
    dev = _device_for(w)
    on_host = w.device.type == "cpu"
    with _device_guard(dev):
        wd = w.to(dev, non_blocking=True) if on_host else w
        n, k = wd.shape
        g = (k + group - 1) // group
        codes, scales = _empty(n, k // 2, torch.uint8, dev), _empty(n, g, scale_dtype, dev)
        z = _empty(n, g, torch.uint8, dev) if zeros else None
        rc = lib.bfp8_quant_group_w4_f32(wd.data_ptr(), n, k, wd.stride(0) if n > 1 else k, group, codes.data_ptr(),
                                         scales.data_ptr(), None if z is None else z.data_ptr(), _DTYPE[scale_dtype],
                                         _stream_ptr(dev))
        _lib.check(rc, "bfp8_quant_group_w4_f32")
    if on_host:
        codes, scales, z = codes.cpu(), scales.cpu(), None if z is None else z.cpu()
    return codes, scales, z


def _share_memory(x, out):
    """Whether matrices with unit column stride may have bytes in common (rows of one pitch are compared by their columns)."""
    a, b = x.data_ptr(), out.data_ptr()
    wide_a, wide_b = x.shape[1] * x.element_size(), out.shape[1] * out.element_size()
    pitch_a, pitch_b = x.stride(0) * x.element_size(), out.stride(0) * out.element_size()
    rows = x.shape[0]
    if not a or not b or a + (rows - 1) * pitch_a + wide_a <= b or b + (rows - 1) * pitch_b + wide_b <= a:
        return False                                       # apart, or without memory
    off = (b - a) % pitch_a if rows > 1 and pitch_a == pitch_b else 0
    return off < wide_a or off + wide_b > pitch_a


def gemm_group_w4(x, codes, scales, zeros=None, *, group, bias=None, out=None, out_dtype=None, check=False, status=None,
                  wait_limit_cycles=0, fresh_codes=False):
    """[M, N] = x . W^T (+ bias), W[n, k] = (q[n, k] - z[n, k // group]) * scales[n, k // group].

    x      bf16 or fp16 [M, K], K a multiple of 32; M <= 1048560, made for few rows (the weight is read once per 16 or 32;
           from about 32 rows on gemm_block_fp8 is faster)
    codes  uint8 [N, K / 2], q of even k in the low four bits;  scales of x's type [N, ceil(K / group)]
    zeros  uint8 of scales' shape, 0 .. 15, or None: 8;  bias fp32 [N] or None;  group 32, 64 or 128
    out    of x's type, or float32 with out_dtype=torch.float32; where it overlaps x, x is copied first
    check  read the status word after the launch (one synchronisation) and raise if a bounded wait expired; status as in
           gemm_block_fp8.  The bounded waits are for the kernel's own copies, which begin when the previous kernel has
           ended; CTAs of a cluster also wait for one another, each to its end.  So calls are unchecked by default.
    fresh_codes  the codes were written by a kernel enqueued just before this call (quantize_group_w4, a copy) and are not taken
           to be at rest where set_weights_at_rest is on
    """
    kind = _DTYPE.get(x.dtype) if isinstance(x, torch.Tensor) else None
    if kind is None or x.ndim != 2 or not x.is_cuda or (x.stride(1) != 1 and x.shape[1] > 1):
        raise ValueError("x must be a bf16 or fp16 [M, K] CUDA tensor with unit column stride")
    m, k = x.shape
    dev = x.device
    if group not in GROUPS or k < 32 or k % 32:
        raise ValueError("group must be 32, 64 or 128 and K a multiple of 32")
    if (not isinstance(codes, torch.Tensor) or codes.dtype != torch.uint8 or codes.ndim != 2 or not codes.is_contiguous()
            or codes.device != dev):
        raise ValueError("codes must be contiguous uint8 [N, K / 2] on x's device")
    n, packed = codes.shape
    if packed * 2 != k or n < 1:
        raise ValueError("codes must be [N, K / 2] with x's K")
    shape = (n, (k + group - 1) // group)
    if (not isinstance(scales, torch.Tensor) or scales.dtype != x.dtype or scales.shape != shape
            or not scales.is_contiguous() or scales.device != dev):
        raise ValueError("scales must be contiguous [N, ceil(K / group)] of x's type on x's device")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != shape or not zeros.is_contiguous()
                              or zeros.device != dev):
        raise ValueError("zeros must be contiguous uint8 of the scales' shape on x's device")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous()
                             or bias.device != dev):
        raise ValueError("bias must be contiguous FP32 [N] on x's device")
    if out_dtype is None:
        out_dtype = x.dtype if out is None else out.dtype
    if out_dtype != x.dtype and out_dtype != torch.float32:
        raise ValueError("out_dtype must be x's type or float32")
    if out is not None and (out.dtype != out_dtype or out.shape != (m, n) or (n > 1 and out.stride(1) != 1)
                            or (m > 1 and out.stride(0) < n) or out.device != dev):
        raise ValueError("out must be [M, N] of out_dtype on x's device with unit column stride and rows apart")
    lib = _lib.load()
    with _device_guard(dev):
        given = out is not None
        if not given:
            out = _empty(m, n, out_dtype, dev)
        if m == 0:
            return out
        if x.data_ptr() % 16 or (m > 1 and (x.stride(0) % 8 or x.stride(0) < k)) or (given and _share_memory(x, out)):
            # TMA reads rows from 16-byte boundaries, each its own, and reads on while outputs are stored
            x = x.contiguous() if not x.is_contiguous() else x.clone()
        st = status if status is not None else _status_buffer(dev) if check else _status_sink(dev)
        rc = lib.bfp8_gemm_group_w4(x.data_ptr(), x.stride(0) if m > 1 else k,
                                    kind | (_lib.W4_FRESH_CODES if fresh_codes else 0), codes.data_ptr(),
                                    scales.data_ptr(), None if zeros is None else zeros.data_ptr(), group,
                                    None if bias is None else bias.data_ptr(), out.data_ptr(),
                                    1 if out_dtype == torch.float32 else 0, out.stride(0) if m > 1 else n, m, n, k,
                                    st.data_ptr() + 8, _stream_ptr(dev), wait_limit_cycles)
        if rc:
            _lib.check(rc, "bfp8_gemm_group_w4")
        if check and _read_status(st)[1] & _lib.STATUS_WAIT_TIMEOUT:
            raise _lib.Bfp8Error(_WAIT_TIMEOUT_MSG)
    return out
