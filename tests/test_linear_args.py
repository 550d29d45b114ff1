"""Argument checks of the quantised linear layers and norms at the C ABI (no
GPU): every unsupported argument is refused with a status and a reason before
any CUDA call, and zero rows are no work.  The pointers are never read."""
import ctypes

import pytest

P = 1 << 20  # a 16-byte aligned address that nothing dereferences
F32, F16, BF16 = 0, 1, 2
REFUSED = -1


def _norm(L, name="rk_rms_norm", x=P, ldx=64, res=None, ldr=0, w=P, h=None, ldh=0, y=P, ldy=64, rows=4, cols=64,
          dtype=F32, scale=P):
    if name == "rk_rms_norm":
        return L.rk_rms_norm(x, ldx, res, ldr, w, h, ldh, y, ldy, rows, cols, 1e-6, dtype, None)
    if name == "rk_rms_norm_q8":
        return L.rk_rms_norm_q8(x, ldx, res, ldr, w, h, ldh, y, ldy, scale, rows, cols, 1e-6, dtype, None)
    return L.rk_quantize_q8(x, ldx, y, ldy, scale, rows, cols, dtype, None)


NORM_BAD = [dict(x=None), dict(y=None), dict(cols=0), dict(rows=-1), dict(dtype=3), dict(dtype=-1), dict(ldx=63),
            dict(ldy=63), dict(x=P + 2), dict(x=P + 1, dtype=BF16)]


@pytest.mark.parametrize("name", ["rk_rms_norm", "rk_rms_norm_q8", "rk_quantize_q8"])
@pytest.mark.parametrize("bad", NORM_BAD, ids=str)
def test_norm_refuses(rk_lib, name, bad):
    assert _norm(rk_lib, name, **bad) == REFUSED
    assert name.encode() in rk_lib.rk_last_error()


@pytest.mark.parametrize("bad", [dict(w=None), dict(res=P, ldr=10), dict(h=P, ldh=10), dict(w=P + 2), dict(h=P + 3, ldh=64)],
                         ids=str)
def test_norm_refuses_residual_and_weight(rk_lib, bad):
    assert _norm(rk_lib, "rk_rms_norm", **bad) == REFUSED
    assert _norm(rk_lib, "rk_rms_norm_q8", **bad) == REFUSED


def test_q8_rows_need_a_scale(rk_lib):
    assert _norm(rk_lib, "rk_rms_norm_q8", scale=None) == REFUSED
    assert _norm(rk_lib, "rk_quantize_q8", scale=None) == REFUSED
    assert _norm(rk_lib, "rk_quantize_q8", scale=P + 1) == REFUSED


def _q8(L, x=P, ldx=64, sx=P, w=P, ldw=64, sw=P, b=None, r=None, ldr=0, y=P, ldy=32, rows=4, n=32, k=64, dtype=F32):
    return L.rk_linear_q8(x, ldx, sx, w, ldw, sw, b, r, ldr, y, ldy, rows, n, k, dtype, None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(sx=None), dict(w=None), dict(sw=None), dict(y=None), dict(ldx=48),
                                 dict(ldw=48), dict(ldy=31), dict(r=P, ldr=31), dict(rows=-1), dict(n=0), dict(k=0),
                                 dict(dtype=3), dict(x=P + 8), dict(w=P + 8), dict(ldx=72), dict(ldw=72), dict(y=P + 2),
                                 dict(b=P + 2), dict(r=P + 2, ldr=32)], ids=str)
def test_linear_q8_refuses(rk_lib, bad):
    assert _q8(rk_lib, **bad) == REFUSED
    assert b"rk_linear_q8" in rk_lib.rk_last_error()


def _q4(L, x=P, ldx=96, w=P, ldw=48, s=P, z=None, b=None, r=None, ldr=0, y=P, ldy=32, rows=4, n=32, k=96, group=32,
        dtype=F32, sdtype=F32, ws=P, size=1 << 40):
    return L.rk_linear_q4(x, ldx, w, ldw, s, z, b, r, ldr, y, ldy, ws, size, rows, n, k, group, dtype, sdtype, None)


Q4_BAD = [dict(x=None), dict(w=None), dict(s=None), dict(y=None), dict(ldx=95), dict(ldw=32), dict(ldw=56), dict(ldy=31),
          dict(rows=-1), dict(n=0), dict(k=0), dict(dtype=3), dict(sdtype=3), dict(group=0), dict(group=16),
          dict(group=96), dict(group=192), dict(group=-128), dict(w=P + 8), dict(x=P + 2), dict(s=P + 2),
          dict(r=P, ldr=31), dict(b=P + 1)]


@pytest.mark.parametrize("bad", Q4_BAD, ids=str)
def test_linear_q4_refuses(rk_lib, bad):
    assert _q4(rk_lib, **bad) == REFUSED
    assert b"rk_linear_q4" in rk_lib.rk_last_error()


def test_linear_q4_workspace(rk_lib):
    """The size is pure arithmetic: it grows with rows and k, and a smaller, missing or misaligned one is refused."""
    size = rk_lib.rk_linear_q4_workspace_size
    assert size(0, 32, 96, 32, F32) == 0
    for bad in [(-1, 32, 96, 32, F32), (1, 0, 96, 32, F32), (1, 32, 0, 32, F32), (1, 32, 96, 48, F32), (1, 32, 96, 32, 5)]:
        assert size(*bad) == 0
    assert 0 < size(1, 32, 96, 32, F16) < size(1, 32, 96, 32, F32) < size(1, 32, 4096, 32, F32) < size(33, 32, 4096, 32, F32)
    need = size(4, 32, 96, 32, F32)
    assert need % 256 == 0
    for bad in (dict(ws=None), dict(ws=P + 128), dict(size=need - 1)):
        assert _q4(rk_lib, **bad) == -2


@pytest.mark.parametrize("bad", [dict(w=None), dict(q=None), dict(s=None), dict(ldw=95), dict(ldq=32), dict(ldq=56),
                                 dict(n=-1), dict(k=0), dict(group=48), dict(dtype=4), dict(sdtype=4), dict(q=P + 4),
                                 dict(n=1 << 30, k=1 << 20, ldw=1 << 20, ldq=1 << 19)], ids=str)
def test_quantize_q4_refuses(rk_lib, bad):
    a = dict(w=P, ldw=96, q=P, ldq=48, s=P, z=None, n=32, k=96, group=32, dtype=F32, sdtype=F32) | bad
    assert rk_lib.rk_quantize_q4(a["w"], a["ldw"], a["q"], a["ldq"], a["s"], a["z"], a["n"], a["k"], a["group"],
                                 a["dtype"], a["sdtype"], None) == REFUSED
    assert b"rk_quantize_q4" in rk_lib.rk_last_error()


BIG = (1 << 30) + 1


def test_more_than_2_30_rows_or_columns_are_refused(rk_lib):
    """32-bit indices would step past the end by a block's width."""
    for name in ("rk_rms_norm", "rk_rms_norm_q8", "rk_quantize_q8"):
        assert _norm(rk_lib, name, cols=BIG, ldx=2 * BIG, ldy=2 * BIG) == REFUSED
        assert _norm(rk_lib, name, rows=BIG) == REFUSED
    for bad in (dict(rows=BIG), dict(n=BIG, ldy=2 * BIG), dict(k=BIG, ldx=1 << 32, ldw=1 << 32)):
        assert _q8(rk_lib, **bad) == REFUSED
        assert _q4(rk_lib, **bad) == REFUSED
        a = dict(rows=1, n=32, k=96) | {k: v for k, v in bad.items() if k in ("rows", "n", "k")}
        assert rk_lib.rk_linear_q4_workspace_size(a["rows"], a["n"], a["k"], 32, F32) == 0
    assert rk_lib.rk_quantize_q4(P, 1 << 32, P, 1 << 32, P, None, 1, BIG, 1 << 30, F32, F32, None) == REFUSED
    assert rk_lib.rk_quantize_q4(P, 96, P, 48, P, None, BIG, 96, 128, F32, F32, None) == REFUSED


def test_zero_rows_are_no_work(rk_lib):
    for name in ("rk_rms_norm", "rk_rms_norm_q8", "rk_quantize_q8"):
        assert _norm(rk_lib, name, rows=0, x=None, y=None) == 0
    assert _q8(rk_lib, rows=0, x=None, y=None) == 0
    assert _q4(rk_lib, rows=0, x=None, y=None) == 0
    assert rk_lib.rk_quantize_q4(None, 0, None, 0, None, None, 0, 96, 32, F32, F32, None) == 0


def test_python_front_end_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    from rokoko_b200 import linear
    x, w = torch.zeros(4, 64), torch.ones(64)
    with pytest.raises(ValueError, match="x: a CUDA tensor"):
        linear.rms_norm(x, w)
    with pytest.raises(ValueError, match="x: a CUDA tensor"):
        linear.rms_norm_q8(x, w)
    with pytest.raises(ValueError, match="x: a CUDA tensor"):
        linear.quantize_q8(x)
    with pytest.raises(ValueError, match="x: a CUDA tensor"):
        linear.linear_q8(x, w, x, w)
    with pytest.raises(ValueError, match="w: a CUDA tensor"):
        linear.quantize_q4(x)
    with pytest.raises(ValueError, match="x: a CUDA tensor"):
        linear.linear_q4(x, x, x, 32)
    with pytest.raises(ValueError, match="x: float32, float16 or bfloat16"):
        linear.rms_norm(x.double(), w)


def test_sizes_past_32_bits_are_refused_and_not_cut_short():
    """2^32 + 128 reaches a 32-bit argument as 128: a group that the scales were not made for."""
    pytest.importorskip("torch")
    from rokoko_b200 import linear
    for group in (32, 64, 128, 384, 1 << 30):
        linear._check_group(group)
    for group in ((1 << 32) + 32, (1 << 32) + 64, (1 << 32) + 128, (1 << 30) + 128, 1 << 31):
        with pytest.raises(ValueError, match="group"):
            linear._check_group(group)


def test_tensors_that_are_more_than_their_memory_are_refused():
    """A forward-mode tangent would be dropped, a negated view be read without its sign.  (On host tensors: device -1.)"""
    torch = pytest.importorskip("torch")
    import torch.autograd.forward_ad as fwd
    from rokoko_b200 import linear
    x, v = torch.randn(3, 4), torch.randn(4)

    def both(x, v):
        linear._rows(x, "x", torch.float32, -1, 3, 4)
        linear._vector(v, "v", torch.float32, -1, 4)
    both(x, v)
    with fwd.dual_level():
        both(x, v)
        with pytest.raises(ValueError, match="x carries a tangent"):
            both(fwd.make_dual(x, x), v)
        with pytest.raises(ValueError, match="v carries a tangent"):
            both(x, fwd.make_dual(v, v))
        with torch.no_grad(), pytest.raises(ValueError, match="x carries a tangent"):
            both(fwd.make_dual(x, x), v)

    def f(x, v):
        with pytest.raises(ValueError, match="carries a tangent"):
            both(x, v)
        return x.sum()
    torch.func.jvp(f, (x, v), (x, v))
    with pytest.raises(ValueError, match="x requires a gradient"):
        torch.func.grad(lambda x: both(x, v))(x)
    z = torch.randn(3, 1, dtype=torch.complex64).conj().imag
    with pytest.raises(ValueError, match="x: a view of negated values"):
        linear._rows(z, "x", torch.float32, -1, 3, 1)
    linear._rows(z.resolve_neg(), "x", torch.float32, -1, 3, 1)


def test_overlapping_rows():
    """Which rows the front end takes to share memory, against the sets of their elements."""
    torch = pytest.importorskip("torch")
    from rokoko_b200.linear import _apart
    buf = torch.zeros(400)
    seen = set()
    for rows, cols, la, lb, at in [(r, c, a, b, o) for r in (1, 3) for c in (4, 7) for a in (16, 20) for b in (16, 20)
                                   for o in (0, 1, 4, 7, 9, 12, 13, 16, 33, 60, 80)]:
        a, b = buf.as_strided((rows, cols), (la, 1), 100), buf.as_strided((rows, cols), (lb, 1), 100 + at)
        for x, y in ((a, b), (b, a)):
            where = [{(t.data_ptr() // 4 + i * t.stride(0) + j) for i in range(rows) for j in range(cols)} for t in (x, y)]
            try:
                _apart(x, y, "x and y")
                free = True
            except ValueError:
                free = False
            assert not (free and where[0] & where[1])                       # never let through
            assert free or where[0] & where[1] or (rows > 1 and la != lb)   # refused in vain for unlike pitches alone
            seen.add(free)
    assert seen == {True, False}
    _apart(buf.view(20, 20)[:, :4], buf.view(20, 20)[:, :4], "x and y", itself=True)


def test_rows_and_vectors_that_overlap():
    """The same for an output and a vector, of another element size too, or rows in another number."""
    torch = pytest.importorskip("torch")
    from rokoko_b200.linear import _apart
    buf = torch.zeros(400)
    seen = set()

    def where(t):
        step = t.element_size()
        rows, pitch = (t.shape[0], t.stride(0) * step) if t.dim() > 1 else (1, 0)
        return {t.data_ptr() + i * pitch + j for i in range(rows) for j in range(t.shape[-1] * step)}
    for rows, cols, ld in ((1, 7, 7), (1, 4, 30), (3, 7, 16), (3, 7, 7), (3, 4, 20)):
        out = buf.as_strided((rows, cols), (ld, 1), 100)
        others = [buf[at:at + n] for at in range(80, 165) for n in (1, 5, 9)]
        others += [t.view(torch.uint8) for t in others]
        others += [buf.as_strided((r, c), (p, 1), at) for at in range(60, 165, 3) for r in (1, 2, 5) for c in (1, 9)
                   for p in (ld, 11) if p >= c]
        for t in others:
            try:
                _apart(out, t, "out and other")
                free = True
            except ValueError:
                free = False
            meet = bool(where(out) & where(t))
            assert not (free and meet)
            many = t.dim() > 1 and t.shape[0] > 1
            assert free or meet or (many and rows > 1 and t.stride(0) != ld)  # in vain for unlike pitches alone
            seen.add((free, t.dim()))
    assert len(seen) == 4


def test_header_constants_match():
    from rokoko_b200 import lib
    assert (lib.RK_DTYPE_F32, lib.RK_DTYPE_F16, lib.RK_DTYPE_BF16) == (F32, F16, BF16)
    assert ctypes.sizeof(ctypes.c_longlong) == 8
