"""Quantised linear layers and the norm that feeds them, on torch tensors.

    wq, ws = quantize_q8(w)                                 # once, when the weights are loaded
    q, s, h = rms_norm_q8(x, norm_w, residual=h)            # h = x + h;  8-bit rows of the norm of h
    y = linear_q8(q, s, wq, ws, bias=b, dtype=x.dtype)

    w4, sc, z = quantize_q4(w, group=128, zeros=True)       # once
    y, h = rms_norm(x, norm_w, residual=h)
    y = linear_q4(y, w4, sc, 128, zeros=z, bias=b)          # for few rows

Tensors are 2-D CUDA tensors [rows, columns] whose columns are adjacent (any
row stride), in float32, float16 or bfloat16; what a call reads and writes
stands at the entry points of include/rk_b200.h.  Results are new tensors on
the current stream of the inputs' device.  Arguments that do not fit raise
ValueError before anything is enqueued.  The operators are for serving and have
no gradients: an input that requires one is refused while gradients are
recorded.  There is no other path than librokoko_b200.so.
"""
from __future__ import annotations

import torch

from . import lib

DTYPES = {torch.float32: lib.RK_DTYPE_F32, torch.float16: lib.RK_DTYPE_F16, torch.bfloat16: lib.RK_DTYPE_BF16}
Q8 = torch.float8_e4m3fn


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _rows(t, name: str, dtype, device, shape=None) -> int:
    """Checks a 2-D tensor and returns its row stride in elements."""
    _need(t.dim() == 2, f"{name}: 2-D tensor expected, got {t.dim()}-D")
    _need(t.is_cuda and t.device == device, f"{name}: expected a tensor on {device}, got {t.device}")
    _need(t.dtype == dtype, f"{name}: expected {dtype}, got {t.dtype}")
    _need(shape is None or t.shape == shape, f"{name}: expected shape {shape}, got {tuple(t.shape)}")
    rows, cols = t.shape
    ld, step = t.stride()
    _need(cols <= 1 or step == 1, f"{name}: columns must be adjacent (stride {step})")
    _need(rows <= 1 or ld >= cols, f"{name}: rows overlap (stride {ld}, {cols} columns)")
    _need(not (t.requires_grad and torch.is_grad_enabled()), f"{name} requires a gradient; this operator has none")
    return ld if rows > 1 else max(ld, cols)


def _vector(t, name: str, dtype, device, n: int) -> int:
    _need(t.dim() == 1 and t.shape[0] == n, f"{name}: expected shape ({n},), got {tuple(t.shape)}")
    _need(t.is_cuda and t.device == device, f"{name}: expected a tensor on {device}, got {t.device}")
    _need(t.dtype == dtype, f"{name}: expected {dtype}, got {t.dtype}")
    _need(n <= 1 or t.stride(0) == 1, f"{name}: elements must be adjacent")
    _need(not (t.requires_grad and torch.is_grad_enabled()), f"{name} requires a gradient; this operator has none")
    return t.data_ptr()


def _activation(x, name: str = "x") -> int:
    _need(isinstance(x, torch.Tensor), f"{name}: a tensor is expected")
    _need(x.dtype in DTYPES, f"{name}: float32, float16 or bfloat16 expected, got {x.dtype}")
    _need(x.is_cuda, f"{name}: a CUDA tensor is expected")
    return DTYPES[x.dtype]


def _call(name: str, device, *args) -> None:
    """The entry point with the current stream of `device`, on that device."""
    fn = getattr(lib.load(), name)
    if torch.cuda.current_device() == device.index:
        st = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            st = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if st != lib.RK_OK:
        lib.check(st, name)


def _q8_rows(rows: int, cols: int, device):
    """8-bit rows of a multiple of 16 bytes."""
    return torch.empty(rows, (cols + 15) // 16 * 16, dtype=Q8, device=device)[:, :cols]


def _norm_args(x, weight, residual, out, sum_out):
    dt = _activation(x)
    ldx = _rows(x, "x", x.dtype, x.device)
    rows, cols = x.shape
    _need(cols >= 1, "x: at least one column")
    wp = _vector(weight, "weight", x.dtype, x.device, cols)
    rp, ldr = None, 0
    if residual is not None:
        ldr = _rows(residual, "residual", x.dtype, x.device, x.shape)
        rp = residual.data_ptr()
    if sum_out is None and residual is not None:
        sum_out = torch.empty(rows, cols, dtype=x.dtype, device=x.device)
    sp, lds = None, 0
    if sum_out is not None:
        lds = _rows(sum_out, "sum_out", x.dtype, x.device, x.shape)
        sp = sum_out.data_ptr()
    return dt, rows, cols, sum_out, (x.data_ptr(), ldx, rp, ldr, wp, sp, lds)


def rms_norm(x, weight, residual=None, eps: float = 1e-6, out=None, sum_out=None):
    """y = h / sqrt(mean(h^2) + eps) * weight over the rows of h = x + residual.

    Returns y, or (y, h) when there is a residual (h in x's type; y comes from the unrounded sum).  `out` and `sum_out`
    may name tensors to write y and h to, x and residual themselves among them."""
    dt, rows, cols, h, args = _norm_args(x, weight, residual, out, sum_out)
    if out is None:
        out = torch.empty(rows, cols, dtype=x.dtype, device=x.device)
    ldy = _rows(out, "out", x.dtype, x.device, x.shape)
    _need(h is None or h.data_ptr() != out.data_ptr() or rows == 0, "out and sum_out are the same memory")
    _call("rk_rms_norm", x.device, *args, out.data_ptr(), ldy, rows, cols, eps, dt)
    return out if h is None else (out, h)


def rms_norm_q8(x, weight, residual=None, eps: float = 1e-6, sum_out=None):
    """rms_norm with 8-bit rows: returns (q, scale), or (q, scale, h) when there is a residual; y is about
    q.float() * scale[:, None]."""
    dt, rows, cols, h, args = _norm_args(x, weight, residual, None, sum_out)
    q = _q8_rows(rows, cols, x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    _call("rk_rms_norm_q8", x.device, *args, q.data_ptr(), q.stride(0), scale.data_ptr(), rows, cols, eps, dt)
    return (q, scale) if h is None else (q, scale, h)


def quantize_q8(x):
    """8-bit rows of x: (q [rows, columns], scale [rows])."""
    dt = _activation(x)
    ldx = _rows(x, "x", x.dtype, x.device)
    rows, cols = x.shape
    _need(cols >= 1, "x: at least one column")
    q = _q8_rows(rows, cols, x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    _call("rk_quantize_q8", x.device, x.data_ptr(), ldx, q.data_ptr(), q.stride(0), scale.data_ptr(), rows, cols, dt)
    return q, scale


def _finish_args(rows: int, n: int, dtype, device, bias, residual, out):
    bp = _vector(bias, "bias", torch.float32, device, n) if bias is not None else None
    rp, ldr = None, 0
    if residual is not None:
        ldr = _rows(residual, "residual", dtype, device, (rows, n))
        rp = residual.data_ptr()
    if out is None:
        out = torch.empty(rows, n, dtype=dtype, device=device)
    ldy = _rows(out, "out", dtype, device, (rows, n))
    return out, (bp, rp, ldr, out.data_ptr(), ldy)


def _q8_operand(t, name: str, device) -> int:
    ld = _rows(t, name, Q8, device)
    _need(t.shape[1] >= 1, f"{name}: at least one column")
    _need(t.shape[0] == 0 or (t.data_ptr() % 16 == 0 and (t.shape[0] == 1 or ld % 16 == 0)),
          f"{name}: 8-bit rows start on 16-byte boundaries (quantize_q8 and rms_norm_q8 lay them out so)")
    return ld


def linear_q8(x, x_scale, w, w_scale, bias=None, residual=None, dtype=torch.float32, out=None):
    """x w^T + bias + residual for 8-bit rows x [rows, k] and w [n, k] with their scales; the result in `dtype`.

    bias is float32 [n], residual [rows, n] in `dtype`; `out` may name the tensor to write, residual itself among them."""
    _need(isinstance(x, torch.Tensor) and x.is_cuda, "x: a CUDA tensor is expected")
    _need(dtype in DTYPES, f"dtype: float32, float16 or bfloat16 expected, got {dtype}")
    device = x.device
    ldx = _q8_operand(x, "x", device)
    ldw = _q8_operand(w, "w", device)
    rows, k = x.shape
    n = w.shape[0]
    _need(n >= 1 and w.shape[1] == k, f"w: expected {k} columns and at least one row, got {tuple(w.shape)}")
    sx = _vector(x_scale, "x_scale", torch.float32, device, rows)
    sw = _vector(w_scale, "w_scale", torch.float32, device, n)
    out, tail = _finish_args(rows, n, dtype, device, bias, residual, out)
    _call("rk_linear_q8", device, x.data_ptr(), ldx, sx, w.data_ptr(), ldw, sw, *tail, rows, n, k, DTYPES[dtype])
    return out


def quantize_q4(w, group: int = 128, zeros: bool = False, scale_dtype=torch.float32):
    """4-bit weights of w [n, k]: (codes uint8 [n, ceil(k / 32) * 16], scales [n, groups], zero points uint8 [n, groups] or
    None).  `group` is 32, 64 or a multiple of 128."""
    dt = _activation(w, "w")
    _need(scale_dtype in DTYPES, f"scale_dtype: float32, float16 or bfloat16 expected, got {scale_dtype}")
    _need(group in (32, 64) or (group >= 128 and group % 128 == 0),
          f"group: 32, 64 or a multiple of 128 expected, got {group}")
    ldw = _rows(w, "w", w.dtype, w.device)
    n, k = w.shape
    _need(k >= 1, "w: at least one column")
    groups = -(-k // group)
    q = torch.empty(n, (k + 31) // 32 * 16, dtype=torch.uint8, device=w.device)
    s = torch.empty(n, groups, dtype=scale_dtype, device=w.device)
    z = torch.empty(n, groups, dtype=torch.uint8, device=w.device) if zeros else None
    _call("rk_quantize_q4", w.device, w.data_ptr(), ldw, q.data_ptr(), q.stride(0), s.data_ptr(),
          z.data_ptr() if zeros else None, n, k, group, dt, DTYPES[scale_dtype])
    return q, s, z


def linear_q4(x, w, scales, group: int, zeros=None, bias=None, residual=None, out=None):
    """x w^T + bias + residual for x [rows, k] and 4-bit weights (codes [n, ceil(k / 32) * 16], scales [n, ceil(k /
    group)], zeros of the same shape or None); the result in x's type.

    bias is float32 [n], residual [rows, n] in x's type; `out` may name the tensor to write, residual itself among
    them.  For few rows: the cost is the weights' bytes."""
    dt = _activation(x)
    device = x.device
    ldx = _rows(x, "x", x.dtype, device)
    rows, k = x.shape
    _need(k >= 1, "x: at least one column")
    _need(group in (32, 64) or (group >= 128 and group % 128 == 0),
          f"group: 32, 64 or a multiple of 128 expected, got {group}")
    ldw = _rows(w, "w", torch.uint8, device)
    n, groups = w.shape[0], -(-k // group)
    _need(n >= 1 and w.shape[1] == (k + 31) // 32 * 16,
          f"w: expected {(k + 31) // 32 * 16} bytes a row and at least one row, got {tuple(w.shape)}")
    _need(w.data_ptr() % 16 == 0 and (n == 1 or ldw % 16 == 0), "w: rows start on 16-byte boundaries")
    _need(scales.dtype in DTYPES, f"scales: float32, float16 or bfloat16 expected, got {scales.dtype}")
    _rows(scales, "scales", scales.dtype, device, (n, groups))
    _need(scales.is_contiguous(), "scales: a contiguous tensor is expected")
    zp = None
    if zeros is not None:
        _rows(zeros, "zeros", torch.uint8, device, (n, groups))
        _need(zeros.is_contiguous(), "zeros: a contiguous tensor is expected")
        zp = zeros.data_ptr()
    out, tail = _finish_args(rows, n, x.dtype, device, bias, residual, out)
    _call("rk_linear_q4", device, x.data_ptr(), ldx, w.data_ptr(), ldw, scales.data_ptr(), zp, *tail, rows, n, k,
          group, dt, DTYPES[scales.dtype])
    return out
