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
the current stream of the inputs' device, or the ones that `out` and `sum_out`
name; these may be an input itself where a function says so and otherwise share
no memory with an input or each other.  Arguments that do not fit raise
ValueError before anything is enqueued.  The operators are for serving and have
no gradients: an input that requires one while gradients are recorded, or carries
a forward-mode tangent, is refused.  There is no other path than librokoko_b200.so.
"""
from __future__ import annotations

import functools

import torch
import torch.autograd.forward_ad as forward_ad

from . import lib

DTYPES = {torch.float32: lib.RK_DTYPE_F32, torch.float16: lib.RK_DTYPE_F16, torch.bfloat16: lib.RK_DTYPE_BF16}
Q8 = torch.float8_e4m3fn
MOST = 1 << 30  # rows, columns and groups: the entry points take 32-bit sizes, and ctypes would cut larger ones short


# The current stream of a device as a plain number: the same as torch.cuda.current_stream(i).cuda_stream, without the
# Stream object (a microsecond a call, which a token's layer pays seven times).
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _place(t, name: str, dtype, dev: int) -> None:
    """Raises for what _odd found, where it is not a tensor of this type on this device or not to be read as it lies."""
    _need(isinstance(t, torch.Tensor), f"{name}: a tensor is expected")
    _need(t.get_device() == dev, f"{name}: expected a tensor on cuda:{dev}, got {t.device}")
    _need(t.dtype is dtype, f"{name}: expected {dtype}, got {t.dtype}")
    _need(not (t.requires_grad and torch.is_grad_enabled()), f"{name} requires a gradient; this operator has none")
    _need(forward_ad.unpack_dual(t).tangent is None, f"{name} carries a tangent; this operator has no derivatives")
    _need(not t.is_neg(), f"{name}: a view of negated values; resolve_neg() makes a tensor of them")


def _odd(t, dtype, dev: int) -> bool:
    """Whether _place has to look at it: anything but plain values in the memory of this device."""
    return (t.__class__ is not torch.Tensor or t.dtype is not dtype or t.get_device() != dev or t.requires_grad or
            forward_ad._current_level >= 0 or t.is_neg())


def _rows(t, name: str, dtype, dev: int, rows: int, cols: int) -> int:
    """Checks a [rows, cols] tensor of this type on this device and returns its row stride in elements."""
    if _odd(t, dtype, dev):
        _place(t, name, dtype, dev)
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{name}: 2-D tensor expected, got {len(shape)}-D")
    if shape[0] != rows or shape[1] != cols:
        raise ValueError(f"{name}: expected shape {(rows, cols)}, got {tuple(shape)}")
    ld, step = t.stride()
    if (step != 1 and cols > 1) or (ld < cols and rows > 1):
        if not (cols <= 1 or step == 1):
            raise ValueError(f"{name}: columns must be adjacent (stride {step})")
        raise ValueError(f"{name}: rows overlap (stride {ld}, {cols} columns)")
    return ld if rows > 1 else max(ld, cols)


def _vector(t, name: str, dtype, dev: int, n: int) -> int:
    if _odd(t, dtype, dev):
        _place(t, name, dtype, dev)
    if t.shape != (n,):
        raise ValueError(f"{name}: expected shape ({n},), got {tuple(t.shape)}")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{name}: elements must be adjacent")
    return t.data_ptr()


def _apart(out, other, what: str, itself: bool = False) -> None:
    """Refuses an output that shares memory with `other`, a vector or a tensor of rows; `itself`: the very same rows may.
    Columns of one buffer beside each other are apart."""
    if out is None or other is None or not (out.numel() and other.numel()):
        return
    a, b = out.data_ptr(), other.data_ptr()
    na, nb = out.shape[0], other.shape[0] if other.dim() > 1 else 1
    lda, ldb = out.stride(0) * out.element_size(), other.stride(0) * other.element_size()
    wa, wb = out.shape[1] * out.element_size(), other.shape[-1] * other.element_size()
    if itself and a == b and (na == 1 or lda == ldb):
        return
    if a + (na - 1) * lda + wa <= b or b + (nb - 1) * ldb + wb <= a:
        return
    pitch = 0 if na == 1 == nb else lda if nb == 1 or na > 1 and lda == ldb else ldb if na == 1 else 0
    if pitch:
        at = (b - a) % pitch
        if at >= wa and at + wb <= pitch:
            return
    raise ValueError(f"{what} overlap")


def _activation(x, name: str = "x"):
    """(dtype code, device, rows, columns) of the tensor that sets them for a call."""
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{name}: a tensor is expected")
    dt = DTYPES.get(x.dtype)
    if dt is None:
        raise ValueError(f"{name}: float32, float16 or bfloat16 expected, got {x.dtype}")
    dev = x.get_device()
    if dev < 0:
        raise ValueError(f"{name}: a CUDA tensor is expected")
    shape = x.shape
    if len(shape) != 2:
        raise ValueError(f"{name}: 2-D tensor expected, got {len(shape)}-D")
    if shape[1] < 1:
        raise ValueError(f"{name}: at least one column")
    if shape[0] > MOST or shape[1] > MOST:
        raise ValueError(f"{name}: at most 2^30 rows and columns, got {tuple(shape)}")
    return dt, dev, shape[0], shape[1]


def _call(name: str, dev: int, *args, wrote=()) -> None:
    """The entry point with the current stream of device `dev`, on that device.  `wrote`: the caller's tensors (or None)
    that it writes, which autograd is told of."""
    fn = getattr(lib.load(), name)
    if torch.cuda.current_device() == dev:
        st = fn(*args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, _stream(dev))
    if st != lib.RK_OK:
        lib.check(st, name)
    for t in wrote:
        if t is not None:
            torch.autograd.graph.increment_version(t)


def _q8_rows(like, rows: int, cols: int):
    """8-bit rows of a multiple of 16 bytes, and their pitch."""
    if cols % 16 == 0:
        return like.new_empty((rows, cols), dtype=Q8), cols
    ld = (cols + 15) // 16 * 16
    return like.new_empty((rows, ld), dtype=Q8)[:, :cols], ld


def _norm_args(x, weight, residual, sum_out):
    dt, dev, rows, cols = _activation(x)
    ldx = _rows(x, "x", x.dtype, dev, rows, cols)
    wp = _vector(weight, "weight", x.dtype, dev, cols)
    rp, ldr, sp, lds = None, 0, None, 0
    if residual is not None:
        ldr = _rows(residual, "residual", x.dtype, dev, rows, cols)
        rp = residual.data_ptr()
    if sum_out is not None:
        lds = _rows(sum_out, "sum_out", x.dtype, dev, rows, cols)
        sp = sum_out.data_ptr()
        _apart(sum_out, x, "sum_out and x", itself=True)
        _apart(sum_out, residual, "sum_out and residual", itself=True)
        _apart(sum_out, weight, "sum_out and weight")
    elif residual is not None:
        sum_out, lds = x.new_empty((rows, cols)), cols
        sp = sum_out.data_ptr()
    return dt, dev, rows, cols, sum_out, (x.data_ptr(), ldx, rp, ldr, wp, sp, lds)


def rms_norm(x, weight, residual=None, eps: float = 1e-6, out=None, sum_out=None):
    """y = h / sqrt(mean(h^2) + eps) * weight over the rows of h = x + residual.

    Returns y, or (y, h) when there is a residual or a `sum_out` (h in x's type; y comes from the unrounded sum).  `out`
    and `sum_out` may name tensors to write y and h to, x and residual themselves among them."""
    dt, dev, rows, cols, h, args = _norm_args(x, weight, residual, sum_out)
    wrote = (out, sum_out)
    if out is None:
        out, ldy = x.new_empty((rows, cols)), cols
    else:
        ldy = _rows(out, "out", x.dtype, dev, rows, cols)
        if not (h is None or h.data_ptr() != out.data_ptr() or rows == 0):
            raise ValueError("out and sum_out are the same memory")
        _apart(out, sum_out, "out and sum_out")
        _apart(out, x, "out and x", itself=True)
        _apart(out, residual, "out and residual", itself=True)
        _apart(out, weight, "out and weight")
    _call("rk_rms_norm", dev, *args, out.data_ptr(), ldy, rows, cols, eps, dt, wrote=wrote)
    return out if h is None else (out, h)


def rms_norm_q8(x, weight, residual=None, eps: float = 1e-6, sum_out=None):
    """rms_norm with 8-bit rows: returns (q, scale), or (q, scale, h) when there is a residual or a `sum_out`; y is about
    q.float() * scale[:, None]."""
    dt, dev, rows, cols, h, args = _norm_args(x, weight, residual, sum_out)
    q, ldq = _q8_rows(x, rows, cols)
    scale = x.new_empty((rows,), dtype=torch.float32)
    _call("rk_rms_norm_q8", dev, *args, q.data_ptr(), ldq, scale.data_ptr(), rows, cols, eps, dt,
          wrote=(sum_out,))
    return (q, scale) if h is None else (q, scale, h)


def quantize_q8(x):
    """8-bit rows of x: (q [rows, columns], scale [rows])."""
    dt, dev, rows, cols = _activation(x)
    ldx = _rows(x, "x", x.dtype, dev, rows, cols)
    q, ldq = _q8_rows(x, rows, cols)
    scale = x.new_empty((rows,), dtype=torch.float32)
    _call("rk_quantize_q8", dev, x.data_ptr(), ldx, q.data_ptr(), ldq, scale.data_ptr(), rows, cols, dt)
    return q, scale


def _finish_args(rows: int, n: int, dtype, dev: int, bias, residual, out, **inputs):
    """bias, residual and the output of a linear layer; `inputs`: by name, what else the output has to be apart from."""
    bp = _vector(bias, "bias", torch.float32, dev, n) if bias is not None else None
    rp, ldr = None, 0
    if residual is not None:
        ldr = _rows(residual, "residual", dtype, dev, rows, n)
        rp = residual.data_ptr()
    if out is None:
        out, ldy = inputs["x"].new_empty((rows, n), dtype=dtype), n
    else:
        ldy = _rows(out, "out", dtype, dev, rows, n)
        _apart(out, residual, "out and residual", itself=True)
        _apart(out, bias, "out and bias")
        for name, t in inputs.items():
            _apart(out, t, f"out and {name}")
    return out, (bp, rp, ldr, out.data_ptr(), ldy)


def _q8_operand(t, name: str, dev: int, rows: int, cols: int):
    ld, p = _rows(t, name, Q8, dev, rows, cols), t.data_ptr()
    if p % 16 or (rows > 1 and ld % 16):
        raise ValueError(f"{name}: 8-bit rows start on 16-byte boundaries (quantize_q8 and rms_norm_q8 lay them out so)")
    return p, ld


def linear_q8(x, x_scale, w, w_scale, bias=None, residual=None, dtype=torch.float32, out=None):
    """x w^T + bias + residual for 8-bit rows x [rows, k] and w [n, k] with their scales; the result in `dtype`.

    bias is float32 [n], residual [rows, n] in `dtype`; `out` may name the tensor to write, residual itself among them."""
    for t, name in ((x, "x"), (w, "w")):
        if not (isinstance(t, torch.Tensor) and t.dim() == 2):
            raise ValueError(f"{name}: a 2-D tensor is expected")
    dev = x.get_device()
    if dev < 0:
        raise ValueError("x: a CUDA tensor is expected")
    dt = DTYPES.get(dtype)
    if dt is None:
        raise ValueError(f"dtype: float32, float16 or bfloat16 expected, got {dtype}")
    rows, k = x.shape
    n = w.shape[0]
    if k < 1:
        raise ValueError("x: at least one column")
    if not (n >= 1 and w.shape[1] == k):
        raise ValueError(f"w: expected {k} columns and at least one row, got {tuple(w.shape)}")
    if rows > MOST or n > MOST or k > MOST:
        raise ValueError(f"x and w: at most 2^30 rows and columns, got {tuple(x.shape)} and {tuple(w.shape)}")
    px, ldx = _q8_operand(x, "x", dev, rows, k)
    pw, ldw = _q8_operand(w, "w", dev, n, k)
    sx = _vector(x_scale, "x_scale", torch.float32, dev, rows)
    sw = _vector(w_scale, "w_scale", torch.float32, dev, n)
    y, tail = _finish_args(rows, n, dtype, dev, bias, residual, out, x=x, w=w, x_scale=x_scale, w_scale=w_scale)
    _call("rk_linear_q8", dev, px, ldx, sx, pw, ldw, sw, *tail, rows, n, k, dt, wrote=(out,))
    return y


@functools.lru_cache(maxsize=4096)
def _q4_workspace(rows: int, n: int, k: int, group: int, dt: int) -> int:
    return lib.load().rk_linear_q4_workspace_size(rows, n, k, group, dt)


def _check_group(group) -> None:
    if not (group in (32, 64) or (128 <= group <= MOST and group % 128 == 0)):
        raise ValueError(f"group: 32, 64 or a multiple of 128 up to 2^30 expected, got {group}")


def quantize_q4(w, group: int = 128, zeros: bool = False, scale_dtype=torch.float32):
    """4-bit weights of w [n, k]: (codes uint8 [n, ceil(k / 32) * 16], scales [n, groups], zero points uint8 [n, groups] or
    None).  `group` is 32, 64 or a multiple of 128 up to 2^30."""
    dt, dev, n, k = _activation(w, "w")
    if not (scale_dtype in DTYPES):
        raise ValueError(f"scale_dtype: float32, float16 or bfloat16 expected, got {scale_dtype}")
    _check_group(group)
    ldw = _rows(w, "w", w.dtype, dev, n, k)
    groups = -(-k // group)
    ldq = (k + 31) // 32 * 16
    q = w.new_empty((n, ldq), dtype=torch.uint8)
    s = w.new_empty((n, groups), dtype=scale_dtype)
    z = w.new_empty((n, groups), dtype=torch.uint8) if zeros else None
    _call("rk_quantize_q4", dev, w.data_ptr(), ldw, q.data_ptr(), ldq, s.data_ptr(), z.data_ptr() if zeros else None,
          n, k, group, dt, DTYPES[scale_dtype])
    return q, s, z


def linear_q4(x, w, scales, group: int, zeros=None, bias=None, residual=None, out=None):
    """x w^T + bias + residual for x [rows, k] and 4-bit weights (codes [n, ceil(k / 32) * 16], scales [n, ceil(k /
    group)], zeros of the same shape or None); the result in x's type.

    bias is float32 [n], residual [rows, n] in x's type; `out` may name the tensor to write, residual itself among
    them.  For few rows: the cost is the weights' bytes.  A row of x whose magnitudes lie too far apart (2^30, half 2^27),
    with an infinity or a NaN takes far longer (include/rk_b200.h)."""
    dt, dev, rows, k = _activation(x)
    dtype = x.dtype
    ldx = _rows(x, "x", dtype, dev, rows, k)
    _check_group(group)
    if not (isinstance(w, torch.Tensor) and w.dim() == 2):
        raise ValueError("w: a 2-D tensor is expected")
    n, groups, row_bytes = w.shape[0], -(-k // group), (k + 31) // 32 * 16
    if not (n >= 1 and w.shape[1] == row_bytes):
        raise ValueError(f"w: expected {row_bytes} bytes a row and at least one row, got {tuple(w.shape)}")
    if n > MOST:
        raise ValueError(f"w: at most 2^30 rows, got {n}")
    ldw, pw = _rows(w, "w", torch.uint8, dev, n, row_bytes), w.data_ptr()
    if not (pw % 16 == 0 and (n == 1 or ldw % 16 == 0)):
        raise ValueError("w: rows start on 16-byte boundaries")
    if not (isinstance(scales, torch.Tensor)):
        raise ValueError("scales: a tensor is expected")
    st = DTYPES.get(scales.dtype)
    if st is None:
        raise ValueError(f"scales: float32, float16 or bfloat16 expected, got {scales.dtype}")
    lds = _rows(scales, "scales", scales.dtype, dev, n, groups)
    if not (lds == groups or n == 1):
        raise ValueError("scales: a contiguous tensor is expected")
    zp = None
    if zeros is not None:
        ldz = _rows(zeros, "zeros", torch.uint8, dev, n, groups)
        if not (ldz == groups or n == 1):
            raise ValueError("zeros: a contiguous tensor is expected")
        zp = zeros.data_ptr()
    y, tail = _finish_args(rows, n, dtype, dev, bias, residual, out, x=x, w=w, scales=scales, zeros=zeros)
    size = _q4_workspace(rows, n, k, group, dt)
    ws = x.new_empty((size,), dtype=torch.uint8)  # torch's blocks start on 512-byte boundaries
    _call("rk_linear_q4", dev, x.data_ptr(), ldx, pw, ldw, scales.data_ptr(), zp, *tail, ws.data_ptr(), size, rows, n, k,
          group, dt, st, wrote=(out,))
    return y


def check(device: int | None = None) -> None:
    """Waits for the current stream of a device and raises RkError if a bounded device-side wait of a call above gave up
    since the last check (its result is then incomplete)."""
    dev = torch.cuda.current_device() if device is None else torch.device("cuda", device).index
    _call("rk_linear_check", dev)
