"""The quantised linear layers and norms (rokoko_b200.linear) against their
definitions in 64 bits.

Tolerances, per value.  u = 2^-24 is half a step of float32 relative to the
value; storing in type t adds eps(t) / 2 of it (plus half the smallest step).

norm     the sum of squares of a row is a tree of at most 32 + 15 additions (one more u per
         thousand columns past 32768 columns), half of its error reaches the root; the root's function is good to
         4u, and the sum h, the mean, the two products and the scale round once each: (24 + 4 + 6) u < 64 u.
q8       a code is off by half a step, 2^-4 of the value or 2^-10 of the scale, from a value good to 64 u.
linear   every partial sum lies below S = sum |x w| (scales taken in); a 16-bit or 8-bit matrix instruction
         adds 16 or 32 products and the carried sum with an error of at most 4u S however it aligns them, so
         K / 16 of them make K / 4 u S; the last scaling, bias and residual round once each.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
U = 2.0 ** -24
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}
EPS = 1e-6


def ids(v):
    return str(v).replace("torch.", "")


@pytest.fixture(scope="module")
def lin():
    from rokoko_b200 import linear
    return linear


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def close(got, ref, err, dtype):
    """|got - ref| within err plus the rounding to dtype, NaN and infinities in the same places."""
    got = got.double()
    assert got.shape == ref.shape
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    fin = torch.isfinite(ref)
    assert torch.equal(got[~fin & ~torch.isnan(ref)], ref[~fin & ~torch.isnan(ref)])
    tol = err + (ref.abs() + err) * (torch.finfo(dtype).eps / 2) + TINY[dtype]
    bad = (got - ref).abs() > tol
    bad &= fin
    assert not bad.any(), (int(bad.sum()), float(((got - ref).abs() / tol)[fin].max()))


# ------------------------------------------------------------------ norm

def norm_ref(x, w, r=None, norm=True):
    h = x.double() + (r.double() if r is not None else 0)
    if not norm:
        return h, h
    return h, h / (h.square().mean(1, keepdim=True) + EPS).sqrt() * w.double()


def check_q8(q, scale, y, rel=64 * U):
    top = y.abs().amax(1).clamp_min(1e-30)
    assert torch.allclose(scale.double(), top / 448, rtol=2 * rel, atol=0)
    s = scale.double()[:, None]
    back = q.double() * s
    tol = y.abs() * (2.0 ** -4 + 4 * rel) + s * 2.0 ** -10
    assert ((back - y).abs() <= tol).all()
    # the codes are the nearest ones: away from the middle between two, they are the code of the definition's own value
    v = y / s
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(-6) - 3)
    near = ((v / step).round() * step).clamp(-448, 448)
    off_middle = ((v / step - (v / step).floor()) - 0.5).abs() > 1e-3
    assert torch.equal(q.double()[off_middle], near[off_middle])


NORM_SIZES = [(1, 1), (1, 256), (11, 256), (3, 7), (5, 64), (2, 1000), (33, 1024), (4, 1025), (7, 2037), (1, 8192),
              (3, 8191), (2, 16384), (2, 20001), (2, 32768), (2, 40000), (2, 40003), (1000, 96), (4099, 100)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
def test_rms_norm(lin, rows, cols, dtype, residual):
    g = gen(rows * 7 + cols)
    x, w = randn(g, rows, cols, dtype=dtype) * 3, randn(g, cols, dtype=dtype)
    r = randn(g, rows, cols, dtype=dtype) if residual else None
    h_ref, y_ref = norm_ref(x, w, r)
    out = lin.rms_norm(x, w, residual=r, eps=EPS)
    y = out[0] if residual else out
    close(y, y_ref, y_ref.abs() * 64 * U, dtype)
    if residual:
        close(out[1], h_ref, h_ref.abs() * U, dtype)
    out = lin.rms_norm_q8(x, w, residual=r, eps=EPS)
    check_q8(out[0], out[1], y_ref)
    if residual:
        close(out[2], h_ref, h_ref.abs() * U, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,cols", [(1, 1), (300, 256), (5, 1001), (2, 40001)])
def test_quantize_q8(lin, rows, cols, dtype):
    x = randn(gen(5), rows, cols, dtype=dtype)
    q, s = lin.quantize_q8(x)
    assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and q.stride(0) % 16 == 0
    check_q8(q, s, x.double(), rel=2 * U)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("cols", [256, 1000, 1003, 8192])
def test_norm_strides_and_in_place(lin, dtype, cols):
    """Rows of wider buffers; y and h written over x and the residual; what lies between the rows stays."""
    g = gen(2)
    wide_x, wide_r = randn(g, 6, cols + 24, dtype=dtype), randn(g, 6, cols + 40, dtype=dtype)
    w = randn(g, cols + 3, dtype=dtype)[3:]
    for off in (0, 8, 3):
        bx, br = wide_x.clone(), wide_r.clone()
        x, r = bx[:, off:off + cols], br[:, off + 8:off + 8 + cols]
        y0, h0 = lin.rms_norm(x, w, residual=r, eps=EPS)
        q0, s0, _ = lin.rms_norm_q8(x, w, residual=r, eps=EPS)
        close(y0, norm_ref(x, w, r)[1], norm_ref(x, w, r)[1].abs() * 64 * U, dtype)
        y1, h1 = lin.rms_norm(x, w, residual=r, eps=EPS, out=x, sum_out=r)
        assert y1 is x and h1 is r and torch.equal(x, y0) and torch.equal(r, h0)
        bx2, br2 = wide_x.clone(), wide_r.clone()
        q1, s1, _ = lin.rms_norm_q8(bx2[:, off:off + cols], w, residual=br2[:, off + 8:off + 8 + cols], eps=EPS,
                                    sum_out=br2[:, off + 8:off + 8 + cols])
        assert torch.equal(q0.float(), q1.float()) and torch.equal(s0, s1) and torch.equal(br2, br)
        keep = torch.ones(cols + 24, dtype=torch.bool, device="cuda")
        keep[off:off + cols] = False
        assert torch.equal(bx[:, keep], wide_x[:, keep])
        keep = torch.ones(cols + 40, dtype=torch.bool, device="cuda")
        keep[off + 8:off + 8 + cols] = False
        assert torch.equal(br[:, keep], wide_r[:, keep])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("cols", [1025, 1536, 2037, 4099, 8185, 8191, 8192, 12001])
@pytest.mark.parametrize("off,gap,apart", [(0, 8, 0), (0, 0, 0), (1, 13, 0), (3, 16, 0), (4, 9, 0), (7, 7, 0), (2, 11, 8),
                                           (5, 11, 1)])
def test_norm_many_rows(lin, dtype, cols, off, gap, apart):
    """Rows enough for every block to work on several, from any place within 16 bytes, the residual's rows `apart`
    elements from there; NaN before and behind every row must not get in."""
    rows, ld = 1601, cols + gap
    g = gen(off * 11 + cols)
    flat = randn(g, 2, rows * ld + 32, dtype=dtype)
    x = flat[0].as_strided((rows, cols), (ld, 1), off)
    r = flat[1].as_strided((rows, cols), (ld, 1), flat.stride(0) + off + apart)
    xs, rs = x.clone(), r.clone()
    flat.fill_(float("nan"))
    x.copy_(xs)
    r.copy_(rs)
    w = randn(g, cols, dtype=dtype)
    h_ref, y_ref = norm_ref(xs, w, rs)
    q, s, h = lin.rms_norm_q8(x, w, residual=r, eps=EPS)
    check_q8(q, s, y_ref)
    close(h, h_ref, h_ref.abs() * U, dtype)
    q1, s1 = lin.rms_norm_q8(x, w, eps=EPS)
    check_q8(q1, s1, norm_ref(xs, w)[1])
    q2, s2 = lin.quantize_q8(x)
    check_q8(q2, s2, xs.double(), rel=2 * U)
    y, h = lin.rms_norm(x, w, residual=r, eps=EPS)
    close(y, y_ref, y_ref.abs() * 64 * U, dtype)
    close(h, h_ref, h_ref.abs() * U, dtype)
    y1, h1 = lin.rms_norm(x, w, residual=r, eps=EPS, out=x, sum_out=r)
    close(y1, y_ref, y_ref.abs() * 64 * U, dtype)
    assert torch.equal(h1, h)
    left = torch.ones(flat.shape, dtype=torch.bool, device="cuda")
    left[0].as_strided((rows, cols), (ld, 1), off).fill_(False)
    left[1].as_strided((rows, cols), (ld, 1), left.stride(0) + off + apart).fill_(False)
    assert torch.isnan(flat[left]).all() and not torch.isnan(flat[~left]).any()


@pytest.mark.parametrize("cols", [64, 513, 4096, 40000])
def test_norm_rows_of_zeros_nan_and_infinity(lin, cols):
    """A row's zeros, NaN or infinity stay in that row."""
    g = gen(3)
    x, w = randn(g, 7, cols), randn(g, cols).abs() + 0.1
    x[1] = 0
    x[2, cols // 2] = float("nan")
    x[3, cols - 1] = float("inf")
    x[4] = x[4] * 1e-25  # below eps: y = h / sqrt(eps) w
    y = lin.rms_norm(x, w, eps=EPS)
    q, s = lin.rms_norm_q8(x, w, eps=EPS)
    ref = norm_ref(x, w)[1]
    fine = [0, 1, 4, 5, 6]
    close(y[fine], ref[fine], ref[fine].abs() * 64 * U, F32)
    check_q8(q[[0, 5, 6]], s[[0, 5, 6]], ref[[0, 5, 6]])
    assert (q[1].float() == 0).all() and torch.isfinite(s[1])
    assert torch.isnan(y[2]).all() and torch.isnan(s[2])
    assert torch.isnan(y[3, cols - 1]) and torch.isnan(s[3])
    qz, sz = lin.quantize_q8(x)
    assert torch.isnan(sz[2]) and (qz[1].float() == 0).all() and sz[3] == float("inf")


def test_norm_far_offsets(lin):
    """Row offsets past 2^31 elements."""
    big = torch.empty((1 << 31) + (1 << 22), dtype=BF16, device="cuda")
    x = big.as_strided((3, 1024), ((1 << 30) + 8192, 1))
    g = gen(4)
    x.copy_(randn(g, 3, 1024))
    w = randn(g, 1024, dtype=BF16)
    ref = norm_ref(x, w)[1]
    close(lin.rms_norm(x, w, eps=EPS), ref, ref.abs() * 64 * U, BF16)
    out = lin.rms_norm(x.contiguous(), w, eps=EPS, out=x)
    close(out, ref, ref.abs() * 64 * U, BF16)


# ------------------------------------------------------------------ 8-bit linear

def q8_ref(x, sx, w, sw, bias, res):
    xd, wd = x.double() * sx.double()[:, None], w.double() * sw.double()[:, None]
    y, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    last = y.abs()
    if bias is not None:
        y, last = y + bias.double(), last + bias.double().abs()
    if res is not None:
        y, last = y + res.double(), last + res.double().abs()
    return y, size * ((x.shape[1] / 4 + 32) * U) + last * 4 * U


Q8_SIZES = [(1, 1, 1), (1, 64, 64), (1, 256, 1024), (2, 129, 127), (3, 1000, 2048), (11, 768, 256), (16, 257, 33),
            (17, 128, 128), (33, 515, 300), (64, 2048, 256), (65, 96, 4100), (127, 384, 640), (128, 128, 4096),
            (129, 130, 131), (200, 2304, 768), (256, 256, 256), (257, 1025, 515), (700, 768, 2048), (1031, 514, 1090),
            (4100, 256, 1024), (20000, 96, 64)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,n,k", Q8_SIZES)
@pytest.mark.parametrize("extra", ["none", "bias", "both"])
def test_linear_q8(lin, rows, n, k, dtype, extra):
    g = gen(rows + 3 * n + 5 * k)
    x, sx = lin.quantize_q8(randn(g, rows, k))
    w, sw = lin.quantize_q8(randn(g, n, k) * k ** -0.5)
    bias = randn(g, n) if extra != "none" else None
    res = randn(g, rows, n, dtype=dtype) if extra == "both" else None
    y = lin.linear_q8(x, sx, w, sw, bias=bias, residual=res, dtype=dtype)
    ref, err = q8_ref(x, sx, w, sw, bias, res)
    close(y, ref, err, dtype)
    assert torch.equal(y, lin.linear_q8(x, sx, w, sw, bias=bias, residual=res, dtype=dtype))


@pytest.mark.parametrize("rows", [1, 5, 300])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_linear_q8_strides_pads_and_in_place(lin, rows, dtype):
    """Rows of wider buffers on both sides; the bytes past a row's end count for nothing; y over the residual."""
    g, k, n = gen(9), 200, 333
    x, sx = lin.quantize_q8(randn(g, rows, k))
    w, sw = lin.quantize_q8(randn(g, n, k))
    bx = torch.full((rows, 512), 448.0, device="cuda").to(torch.float8_e4m3fn)
    bw = torch.full((n, 304), float("nan"), device="cuda").to(torch.float8_e4m3fn)
    bx[:, 256:256 + k] = x
    bw[:, 16:16 + k] = w
    by = torch.full((rows, n + 30), 7.0, dtype=dtype, device="cuda")
    res = by[:, 13:13 + n]
    res.copy_(randn(g, rows, n))
    ref, err = q8_ref(x, sx, w, sw, None, res)
    y0 = lin.linear_q8(x, sx, w, sw, residual=res.clone(), dtype=dtype)
    y1 = lin.linear_q8(bx[:, 256:256 + k], sx, bw[:, 16:16 + k], sw, residual=res, dtype=dtype, out=res)
    assert torch.equal(y0, y1)
    close(y0, ref, err, dtype)
    assert (by[:, :13] == 7).all() and (by[:, 13 + n:] == 7).all()


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_q8_scales_whose_product_is_out_of_range(lin, rows, bias):
    """Scales whose product is smaller than float's normal numbers or passes its largest, and results that do neither."""
    g, n, k = gen(22), 70, 2048
    bias = randn(g, n) * 1e-36 if bias else None
    x, sx = lin.quantize_q8(randn(g, rows, k) * 1e-22)
    w, sw = lin.quantize_q8(randn(g, n, k) * 1e-16)
    assert float(sx.max() * sw.max()) < 2.0 ** -126
    ref, err = q8_ref(x, sx, w, sw, bias, None)
    close(lin.linear_q8(x, sx, w, sw, bias=bias), ref, err, F32)
    big, small = torch.zeros(rows, k, device="cuda"), torch.zeros(n, k, device="cuda")
    big[:, ::2], small[:, 1::2] = 1e30, 1e20  # what one has is zero in the other
    x, sx = lin.quantize_q8(big)
    w, sw = lin.quantize_q8(small)
    sw = sw * 1e5
    assert torch.isinf(sx[0] * sw[0])
    assert (lin.linear_q8(x, sx, w, sw) == 0).all()


def test_linear_q8_nan_and_infinity_stay_in_their_row(lin):
    g = gen(10)
    for rows in (6, 200):
        xf = randn(g, rows, 160)
        w, sw = lin.quantize_q8(randn(g, 70, 160))
        xf[2, 5] = float("nan")
        x, sx = lin.quantize_q8(xf)
        y = lin.linear_q8(x, sx, w, sw)
        fine = [i for i in range(rows) if i != 2]
        ref, err = q8_ref(x[fine], sx[fine], w, sw, None, None)
        close(y[fine], ref, err, F32)
        assert torch.isnan(y[2]).all()


def test_linear_q8_far_offsets(lin):
    """Outputs and rows past 2^31 elements."""
    g = gen(11)
    x, sx = lin.quantize_q8(randn(g, 70000, 64))
    w, sw = lin.quantize_q8(randn(g, 32000, 64))
    y = lin.linear_q8(x, sx, w, sw, dtype=BF16)
    pick = torch.tensor([0, 1, 35000, 67108, 67109, 69998, 69999], device="cuda")
    ref, err = q8_ref(x[pick], sx[pick], w, sw, None, None)
    close(y[pick], ref, err, BF16)
    del y
    for rows in (2, 150):  # both operands in rows that lie far apart
        step = ((1 << 32) // (rows - 1) + 4096) // 16 * 16
        far = torch.empty(step * (rows - 1) + 64, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        xf = far.as_strided((rows, 64), (step, 1))
        xf.copy_(x[:rows])
        assert torch.equal(lin.linear_q8(xf, sx[:rows].contiguous(), w[:100], sw[:100].contiguous()),
                           lin.linear_q8(x[:rows], sx[:rows].contiguous(), w[:100], sw[:100].contiguous()))


# ------------------------------------------------------------------ 4-bit linear

def q4_values(w, s, z, k, group):
    q = torch.stack((w & 15, w >> 4), 2).flatten(1)[:, :k].double()
    at = torch.arange(k, device="cuda") // group
    return (q - (z.double()[:, at] if z is not None else 8)) * s.double()[:, at]


def q4_ref(x, w, s, z, group, bias, res):
    xd, wd = x.double(), q4_values(w, s, z, x.shape[1], group)
    y, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    last = y.abs()
    if bias is not None:
        y, last = y + bias.double(), last + bias.double().abs()
    if res is not None:
        y, last = y + res.double(), last + res.double().abs()
    return y, size * ((x.shape[1] / 4 + 32) * U) + last * 4 * U


def q4_case(g, n, k, group, sdtype, zeros):
    groups = -(-k // group)
    w = torch.randint(0, 256, (n, (k + 31) // 32 * 16), generator=g, device="cuda", dtype=torch.uint8)
    s = ((torch.rand(n, groups, generator=g, device="cuda") + 0.1) * k ** -0.5).to(sdtype)
    z = torch.randint(0, 16, (n, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return w, s, z


Q4_SIZES = [(1, 1, 1), (1, 16, 32), (1, 100, 31), (1, 1000, 4096), (1, 33, 16384), (2, 17, 129), (3, 768, 256),
            (5, 515, 1000), (8, 64, 2049), (9, 130, 515), (11, 2048, 256), (16, 257, 640), (24, 300, 1111),
            (31, 40, 4000), (33, 96, 300), (70, 50, 200), (300, 70, 260)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,n,k", Q4_SIZES)
@pytest.mark.parametrize("group", [32, 64, 128, 384])
@pytest.mark.parametrize("zeros", [False, True], ids=["sym", "zeros"])
def test_linear_q4(lin, rows, n, k, dtype, group, zeros):
    g = gen(rows + 3 * n + 5 * k + group)
    sdtype = TYPES[(rows + n + k) % 3]
    x = randn(g, rows, k, dtype=dtype)
    w, s, z = q4_case(g, n, k, group, sdtype, zeros)
    bias = randn(g, n) if zeros else None
    res = randn(g, rows, n, dtype=dtype) if group in (32, 128) else None
    y = lin.linear_q4(x, w, s, group, zeros=z, bias=bias, residual=res)
    ref, err = q4_ref(x, w, s, z, group, bias, res)
    close(y, ref, err, dtype)
    assert torch.equal(y, lin.linear_q4(x, w, s, group, zeros=z, bias=bias, residual=res))


def test_linear_q4_keeps_32_bit_inputs(lin):
    """x of values whose 16-bit parts do not hold them, in magnitudes from 1e-30 to 1e30."""
    g = gen(12)
    x = randn(g, 4, 512) * torch.tensor([1e-30, 1.0, 1e30, 3e4], device="cuda")[:, None]
    w, s, _ = q4_case(g, 40, 512, 64, F32, False)
    ref, err = q4_ref(x, w, s, None, 64, None, None)
    close(lin.linear_q4(x, w, s, 64), ref, err, F32)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows", [3, 40])
def test_linear_q4_uneven_magnitudes(lin, dtype, rows):
    """Rows of zeros, of the type's smallest numbers, of magnitudes around and beyond 2^30 apart, each beside ordinary
    rows: the ones that the 8-bit parts hold and the ones that they do not."""
    g = gen(17)
    k = 700
    x = randn(g, rows, k, dtype=dtype)
    x[0] = 0
    x[1, ::3] *= 2.0 ** -14
    x[2, 5] = 2.0 ** 15 if dtype == F16 else 2.0 ** 60
    x[2, 6:] *= 2.0 ** -10
    x[rows - 1] = (x[rows - 1] * TINY[dtype] * 8).to(dtype)
    w, s, z = q4_case(g, 60, k, 64, F32, True)
    ref, err = q4_ref(x, w, s, z, 64, None, None)
    close(lin.linear_q4(x, w, s, 64, zeros=z), ref, err + TINY[F32] * k, dtype)
    lin.check()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True], ids=["sym", "zeros"])
def test_linear_q4_large_values_at_the_zero_point(lin, dtype, group, zeros):
    """One value of a row up to 2^29 times the others, where every weight is zero (its code is the zero point): it has
    no part in sum |x w|, so nothing of it may show."""
    g, rows, n, k = gen(18), 40, 150, 512
    spread = torch.tensor([0, 10, 13, 15] if dtype == F16 else [0, 10, 13, 17, 21, 25, 29], device="cuda").double()
    x = (torch.rand(rows, k, generator=g, device="cuda") * 1.5 + 0.5) * randn(g, rows, k).sign()
    w, s, z = q4_case(g, n, k, group, F32, zeros)
    for at in (5, k - 2):  # one in a high half of a byte, one in a low half
        x[:, at] = torch.exp2(spread[torch.arange(rows, device="cuda") % len(spread)]).float()
        code = z[:, at // group] if zeros else torch.full((n,), 8, dtype=torch.uint8, device="cuda")
        low, high = w[:, at // 2] & 15, w[:, at // 2] >> 4
        w[:, at // 2] = code | high << 4 if at % 2 == 0 else low | code << 4
    x = x.to(dtype)
    for r in (3, rows):
        ref, err = q4_ref(x[:r], w, s, z, group, None, None)
        close(lin.linear_q4(x[:r], w, s, group, zeros=z), ref, err, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("binades", [26, 27, 28, 29, 30, 31])
def test_linear_q4_small_values_keep_their_bits(lin, dtype, binades):
    """Values that far below their row's largest, which meets a weight of zero: the small ones alone are the result.
    Parts of 32-bit x may lose 8 last places of a value, 16 u of it and so of sum |x w|; the bound of `linear` has 32 u
    beside its K / 4 u for the last roundings, of which there are fewer than 8."""
    g, rows, n, k = gen(19), 4, 80, 32
    if dtype == F16 and binades > 29:
        pytest.skip("half has no normal numbers so far apart")
    top = 2.0 ** (15 if dtype == F16 else 40)
    x = (torch.rand(rows, k, generator=g, device="cuda", dtype=torch.float64) * 0.99 + 1) * top * 2.0 ** -binades
    x = x.to(dtype) * randn(g, rows, k).sign().to(dtype)
    x[:, 7] = top
    w, s, _ = q4_case(g, n, k, 32, F32, False)
    w[:, 3] = 8 << 4 | w[:, 3] & 15
    s *= 1024.0  # results beyond half's smallest numbers
    ref, err = q4_ref(x, w, s, None, 32, None, None)
    close(lin.linear_q4(x, w, s, 32), ref, err, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=ids)
@pytest.mark.parametrize("small", [1.0, 2.0 ** -20], ids=["even", "uneven"])
def test_linear_q4_values_near_the_largest_float(lin, dtype, small):
    """A value that passes the largest float when it is multiplied by its code, and not when by its weight."""
    g = gen(21)
    x = randn(g, 3, 96, dtype=dtype) * small
    x[1] = 2.0 ** 100
    x[1, 3] = 2.0 ** 126
    if small != 1:
        x[1, 50] = small
    w, s, z = q4_case(g, 70, 96, 32, F32, True)
    w[:, 1] = 0xf0 | w[:, 1] & 15
    z[:, 0] = 0
    ref, err = q4_ref(x, w, s, z, 32, None, None)
    assert torch.isfinite(ref.float()).all()
    close(lin.linear_q4(x, w, s, 32, zeros=z), ref, err, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_linear_q4_strides_pads_and_in_place(lin, dtype):
    g, rows, n, k = gen(13), 5, 45, 250
    x = randn(g, rows, k, dtype=dtype)
    w, s, z = q4_case(g, n, k, 64, F16, True)
    bx = torch.full((rows, 300), float("nan"), dtype=dtype, device="cuda")
    bx[:, 3:3 + k] = x
    bw = torch.full((n, 256), 255, dtype=torch.uint8, device="cuda")
    bw[:, 16:16 + 128] = w
    by = torch.full((rows, n + 9), 7.0, dtype=dtype, device="cuda")
    res = by[:, 4:4 + n]
    res.copy_(randn(g, rows, n))
    ref, err = q4_ref(x, w, s, z, 64, None, res)
    y0 = lin.linear_q4(x, w, s, 64, zeros=z, residual=res.clone())
    w2 = w.clone()
    w2[:, 125:] = 0  # past column 250
    assert torch.equal(y0, lin.linear_q4(x, w2, s, 64, zeros=z, residual=res.clone()))
    y1 = lin.linear_q4(bx[:, 3:3 + k], bw[:, 16:16 + 128], s, 64, zeros=z, residual=res, out=res)
    assert torch.equal(y0, y1)
    close(y0, ref, err, dtype)
    assert (by[:, :4] == 7).all() and (by[:, 4 + n:] == 7).all()


def test_linear_q4_nan_and_infinity_stay_in_their_row(lin):
    g = gen(14)
    for dtype in TYPES:
        x = randn(g, 6, 300, dtype=dtype)
        w, s, _ = q4_case(g, 50, 300, 128, F32, False)
        w[:] = torch.where((w & 15) == 8, w + 1, w)  # no weight is zero in the low halves: inf gives inf
        x[2, 4] = float("inf")
        x[4, 5] = float("nan")
        y = lin.linear_q4(x, w, s, 128)
        fine = [0, 1, 3, 5]
        ref, err = q4_ref(x[fine], w, s, None, 128, None, None)
        close(y[fine], ref, err, dtype)
        assert torch.isnan(y[4]).all()
        q = ((w[:, 2] & 15).double() - 8)
        assert torch.equal(y[2].double(), q.sign() * float("inf"))


def test_linear_q4_far_offsets(lin):
    """Weight rows past 2^32 bytes."""
    g = gen(15)
    n, k = 37, 256
    w, s, _ = q4_case(g, n, k, 128, F32, False)
    step = (1 << 32) // 36 // 16 * 16 + 4096
    far = torch.empty(step * (n - 1) + 128, dtype=torch.uint8, device="cuda").as_strided((n, 128), (step, 1))
    far.copy_(w)
    x = randn(g, 3, k)
    assert torch.equal(lin.linear_q4(x, far, s, 128), lin.linear_q4(x, w, s, 128))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("sdtype", TYPES, ids=ids)
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (40, 256, 32), (33, 300, 64), (17, 1000, 128), (5, 777, 256)])
@pytest.mark.parametrize("zeros", [False, True], ids=["sym", "zeros"])
def test_quantize_q4(lin, n, k, group, dtype, sdtype, zeros):
    """Every weight is within half a scale (and the scale's own rounding) of the value its code stands for."""
    g = gen(16)
    w = randn(g, n, k, dtype=dtype) + (0.5 if zeros else 0)
    w[0] = 0
    q, s, z = lin.quantize_q4(w, group, zeros=zeros, scale_dtype=sdtype)
    assert q.shape == (n, (k + 31) // 32 * 16) and s.shape == (n, -(-k // group)) and (z is None) == (not zeros)
    back = q4_values(q, s, z, k, group)
    at = torch.arange(k, device="cuda") // group
    sd = s.double()[:, at]
    # half a step, a rounded zero point (zeros: half a step more at the ends, 15 steps of the scale's rounding)
    tol = sd * (0.5 + (0.5 if zeros else 0) + 15 * torch.finfo(sdtype).eps / 2 + 64 * U)
    assert ((back - w.double()).abs() <= tol).all()
    assert (back[0] == 0).all()
    if k % 32:
        pad = torch.stack((q & 15, q >> 4), 2).flatten(1)[:, k:]
        assert (pad == 0).all()


# ------------------------------------------------------------------ together

def test_norm_then_linears(lin):
    """A layer's steps as they are used: norm with the residual, 8-bit projection, norm, 4-bit projection onto the
    residual, against the same in 64 bits from the codes that were made."""
    g, rows, d, ff = gen(20), 37, 256, 640
    x, h = randn(g, rows, d), randn(g, rows, d)
    nw = randn(g, d) * 0.1 + 1
    w1, w2 = randn(g, ff, d) * d ** -0.5, randn(g, d, ff) * ff ** -0.5
    b1, n2 = randn(g, ff), randn(g, ff) * 0.1 + 1
    w1q, s1 = lin.quantize_q8(w1)
    w2q, s2, z2 = lin.quantize_q4(w2, 64, zeros=True)
    q, s, h1 = lin.rms_norm_q8(x, nw, residual=h)
    y = lin.linear_q8(q, s, w1q, s1, bias=b1)
    m = lin.rms_norm(y, n2)
    out = lin.linear_q4(m, w2q, s2, 64, zeros=z2, residual=h1)
    h_ref, y_ref = norm_ref(x, nw, h)
    check_q8(q, s, y_ref)
    ref, err = q8_ref(q, s, w1q, s1, b1, None)
    close(y, ref, err, F32)
    m_ref = norm_ref(y, n2)[1]
    close(m, m_ref, m_ref.abs() * 64 * U, F32)
    ref, err = q4_ref(m, w2q, s2, z2, 64, None, h1)
    close(out, ref, err, F32)
    # and near the unquantised layer: 8-bit operands are off by 2^-4 / sqrt(3) a value at most, 4-bit ones by less
    lin.check()
    full = norm_ref(y_ref @ w1.double().t() + b1.double(), n2)[1] @ w2.double().t() + h_ref
    assert float((out.double() - full).norm() / full.norm()) < 0.1


def _layer(lin, s):
    q, sc, h = lin.rms_norm_q8(s["x"], s["nw"], residual=s["h"])
    y = lin.linear_q8(q, sc, *s["w1"], bias=s["b"])
    return lin.linear_q4(lin.rms_norm(y, s["n2"]), *s["w2"][:2], 64, zeros=s["w2"][2], residual=h), q


def _layer_state(lin, seed, rows, d=256, ff=640):
    g = gen(seed)
    return {"x": randn(g, rows, d), "h": randn(g, rows, d), "nw": randn(g, d), "n2": randn(g, ff), "b": randn(g, ff),
            "w1": lin.quantize_q8(randn(g, ff, d)), "w2": lin.quantize_q4(randn(g, d, ff), 64, zeros=True)}


@pytest.mark.parametrize("rows", [1, 9, 300])
def test_streams_and_graphs(lin, rows):
    """The same bits eagerly, on two streams at once, and from two captured graphs replayed with new inputs."""
    states = [_layer_state(lin, 30 + i, rows) for i in range(2)]
    want = [_layer(lin, s)[0].clone() for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = []
    for st, s in zip(streams, states):
        with torch.cuda.stream(st):
            for _ in range(20):
                r = _layer(lin, s)[0]
            got.append(r)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for st, s in zip(streams, states):
        with torch.cuda.stream(st):
            _layer(lin, s)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            outs.append(_layer(lin, s))
        graphs.append(gr)
    for i in range(2):  # swap the inputs: the graphs read what lies in their tensors at replay
        a, b = states[0]["x"].clone(), states[1]["x"].clone()
        states[0]["x"].copy_(b)
        states[1]["x"].copy_(a)
        want = [_layer(lin, s)[0].clone() for s in states]
        torch.cuda.synchronize()
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o[0], w) for o, w in zip(outs, want))


# ------------------------------------------------------------------ refusals of the Python front end

def test_refusals(lin):
    d = torch.device("cuda:0")
    x, w = torch.zeros(4, 64, device=d), torch.ones(64, device=d)
    for bad, match in [(dict(x=x.t()), "columns must be adjacent"), (dict(x=x[0]), "2-D"),
                       (dict(weight=w[:10]), "weight: expected shape"), (dict(weight=w.half()), "weight: expected torch.float32"),
                       (dict(residual=x[:2]), "residual: expected shape"), (dict(residual=x.half()), "residual: expected"),
                       (dict(x=x[:1].expand(4, 64)), "rows overlap"), (dict(x=x[:, :0]), "at least one column"),
                       (dict(weight=w.cpu()), "weight: expected a tensor on"),
                       (dict(x=x.clone().requires_grad_()), "requires a gradient"),
                       (dict(weight=w.clone().requires_grad_()), "requires a gradient")]:
        a = dict(x=x, weight=w) | bad
        for f in (lin.rms_norm, lin.rms_norm_q8):
            with pytest.raises(ValueError, match=match):
                f(**a)
    with pytest.raises(ValueError, match="same memory"):
        lin.rms_norm(x, w, residual=x, out=x, sum_out=x)
    with torch.no_grad():
        lin.rms_norm(x.clone().requires_grad_(), w)
    q, s = lin.quantize_q8(x)
    wq, ws = lin.quantize_q8(torch.zeros(8, 64, device=d))
    ok = dict(x=q, x_scale=s, w=wq, w_scale=ws)
    for bad, match in [(dict(x=x), "x: expected torch.float8"), (dict(w=wq[:, :32]), "w: expected 64 columns"),
                       (dict(x_scale=ws), "x_scale: expected shape"), (dict(w_scale=s), "w_scale: expected shape"),
                       (dict(bias=w), "bias: expected shape"), (dict(bias=ws.half()), "bias: expected torch.float32"),
                       (dict(residual=x), "residual: expected shape"), (dict(dtype=torch.float64), "dtype: "),
                       (dict(w=wq[:0]), "at least one row"), (dict(x=q[:, 1:33], w=wq[:, :32]), "16-byte boundaries"),
                       (dict(out=torch.zeros(4, 8, device=d, dtype=F16)), "out: expected torch.float32"),
                       (dict(w=torch.zeros(8, 72, device=d).to(lin.Q8)[:, :64]), "16-byte boundaries")]:
        with pytest.raises(ValueError, match=match):
            lin.linear_q8(**(ok | bad))
    p4, s4, z4 = lin.quantize_q4(torch.zeros(8, 64, device=d), 32, zeros=True)
    ok = dict(x=x, w=p4, scales=s4, group=32, zeros=z4)
    for bad, match in [(dict(group=48), "group"), (dict(group=64), "scales: expected shape"), (dict(w=p4[:, :16]), "w: expected 32 bytes"),
                       (dict(scales=s4.double()), "scales: float32"), (dict(zeros=z4.int()), "zeros: expected torch.uint8"),
                       (dict(zeros=z4[:, :1]), "zeros: expected shape"), (dict(x=x.double()), "x: float32"),
                       (dict(scales=s4.t().contiguous().t()), "columns must be adjacent"),
                       (dict(residual=x), "residual: expected shape"), (dict(bias=w), "bias: expected shape")]:
        with pytest.raises(ValueError, match=match):
            lin.linear_q4(**(ok | bad))
    with pytest.raises(ValueError, match="group"):
        lin.quantize_q4(x, 100)


def test_sizes_past_32_bits_are_refused(lin):
    """2^32 rows reach a 32-bit argument as none: the call would return whatever its output's memory held."""
    d = torch.device("cuda:0")
    x = torch.empty((1 << 32, 1), dtype=F16, device=d)
    w = torch.ones(1, dtype=F16, device=d)
    for f in (lambda: lin.rms_norm(x, w), lambda: lin.rms_norm_q8(x, w), lambda: lin.quantize_q8(x),
              lambda: lin.quantize_q4(x)):
        with pytest.raises(ValueError, match="2\\^30"):
            f()
    del x
    wide = torch.empty((1, (1 << 32) + 64), dtype=torch.uint8, device=d)
    small = torch.zeros((1, 64), device=d)
    q, s = wide.view(lin.Q8), torch.ones(1, device=d)
    with pytest.raises(ValueError, match="2\\^30"):
        lin.linear_q8(q, s, q, s)
    with pytest.raises(ValueError, match="group"):
        lin.linear_q4(small, wide[:, :32], s[:, None], (1 << 32) + 128)
    with pytest.raises(ValueError, match="group"):
        lin.quantize_q4(small, (1 << 32) + 128)


def test_outputs_that_overlap_inputs_are_refused(lin):
    """Rows are worked on side by side, so an output may share memory with an input only row on row."""
    g = gen(9)
    buf = randn(g, 9, 200)
    w, x, side = randn(g, 64), buf[:8, :64], buf[:8, 64:128]
    with pytest.raises(ValueError, match="out and x overlap"):
        lin.rms_norm(x, w, out=buf[1:, :64])
    with pytest.raises(ValueError, match="out and x overlap"):
        lin.rms_norm(x, w, out=buf[:8, 32:96])
    with pytest.raises(ValueError, match="out and residual overlap"):
        lin.rms_norm(x.clone(), w, residual=x, out=buf[:8, 1:65])
    with pytest.raises(ValueError, match="sum_out and x overlap"):
        lin.rms_norm_q8(x, w, sum_out=buf[1:, :64])
    with pytest.raises(ValueError, match="sum_out and residual overlap"):
        lin.rms_norm_q8(x.clone(), w, residual=x, sum_out=buf[:8, 1:65])
    with pytest.raises(ValueError, match="out and sum_out overlap"):
        lin.rms_norm(x.clone(), w, out=x, sum_out=buf[:8, 32:96])
    p4, s4, _ = lin.quantize_q4(randn(g, 64, 64), 32)
    with pytest.raises(ValueError, match="out and x overlap"):
        lin.linear_q4(x, p4, s4, 32, out=x)
    with pytest.raises(ValueError, match="out and residual overlap"):
        lin.linear_q4(x.clone(), p4, s4, 32, residual=x, out=buf[1:, :64])
    # beside each other, the columns between them of others, they are apart
    ref = lin.rms_norm(x.clone(), w)
    assert torch.equal(lin.rms_norm(x, w, out=side), ref)
    ref = lin.linear_q4(x.clone(), p4, s4, 32)
    assert torch.equal(lin.linear_q4(x, p4, s4, 32, out=side), ref)
    assert torch.equal(lin.linear_q4(x, p4, s4, 32, out=buf[:8, 136:]), ref)
    one = buf[8:]
    assert torch.equal(lin.linear_q4(one[:, :64], p4, s4, 32, out=one[:, 64:128]), lin.linear_q4(one[:, :64], p4, s4, 32))
    with pytest.raises(ValueError, match="out and x overlap"):
        lin.linear_q4(one[:, :64], p4, s4, 32, out=one[:, 63:127])


def test_outputs_that_overlap_weights_are_refused(lin):
    """Every row reads them, so no output may share their memory, not even row on row."""
    g = gen(23)
    x = randn(g, 64, 64)
    w = randn(g, 64)
    with pytest.raises(ValueError, match="out and weight overlap"):
        lin.rms_norm(x, x[0], out=x)
    for f in (lin.rms_norm, lin.rms_norm_q8):
        with pytest.raises(ValueError, match="sum_out and weight overlap"):
            f(x, x[3], sum_out=x)
    before = x.clone()
    q, s = lin.quantize_q8(x)
    bytes_ = torch.empty((64, 64 * 4), dtype=torch.uint8, device="cuda")
    wq = bytes_[:, :64].view(lin.Q8)
    wq.copy_(q)
    over = bytes_.view(F32)
    for a in (dict(w=wq, out=over), dict(w_scale=x[0], out=x), dict(x_scale=x[5], out=x), dict(bias=x[63], out=x)):
        name = [k for k in a if k != "out"][0]
        with pytest.raises(ValueError, match=f"out and {name} overlap"):
            lin.linear_q8(**(dict(x=q, x_scale=s, w=q, w_scale=s) | a))
    p4, s4, z4 = lin.quantize_q4(x, 32, zeros=True)
    held = torch.empty((64, 64 * 4), dtype=torch.uint8, device="cuda")
    p5, z5, s5 = held[:, 16:48], held.view(-1)[128:256].view(64, 2), held.view(F32).view(-1)[64:192].view(64, 2)
    for a in (dict(w=p5), dict(zeros=z5), dict(scales=s5), dict(bias=held.view(F32)[2])):
        with pytest.raises(ValueError, match=f"out and {list(a)[0]} overlap"):
            lin.linear_q4(**(dict(x=x, w=p4, scales=s4, group=32, zeros=z4, out=held.view(F32)) | a))
    assert torch.equal(x, before)


def test_autograd_is_told_of_tensors_written_in_place(lin):
    """A tensor that autograd saved and a call then wrote to fails in the backward pass, as with torch's own functions."""
    g = gen(24)
    x, w = randn(g, 64, 64), randn(g, 64)
    q, s = lin.quantize_q8(x)
    p4, s4, _ = lin.quantize_q4(x, 32)
    calls = [lambda t: lin.rms_norm(x, w, out=t), lambda t: lin.rms_norm(x, w, sum_out=t),
             lambda t: lin.rms_norm(t, w, residual=x, sum_out=t), lambda t: lin.rms_norm_q8(x, w, sum_out=t),
             lambda t: lin.linear_q8(q, s, q, s, out=t), lambda t: lin.linear_q4(x, p4, s4, 32, out=t),
             lambda t: lin.linear_q4(x, p4, s4, 32, residual=t, out=t)]
    for call in calls:
        leaf = randn(g, 64, 64).requires_grad_()
        saved = leaf.exp()  # its backward needs the result
        with torch.no_grad():
            call(saved)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.sum().backward()
    before = x._version
    lin.rms_norm(x, w, residual=x)
    assert x._version == before
    with torch.inference_mode():
        lin.rms_norm(x.clone(), w, out=torch.empty_like(x))


def test_zero_rows(lin):
    x, w = torch.zeros(0, 64, device="cuda"), torch.ones(64, device="cuda")
    assert lin.rms_norm(x, w).shape == (0, 64)
    q, s, h = lin.rms_norm_q8(x, w, residual=x)
    assert q.shape == (0, 64) and s.shape == (0,) and h.shape == (0, 64)
    wq, ws = lin.quantize_q8(torch.zeros(8, 64, device="cuda"))
    assert lin.linear_q8(q, s, wq, ws).shape == (0, 8)
    p, s4, _ = lin.quantize_q4(torch.zeros(8, 64, device="cuda"))
    assert lin.linear_q4(x, p, s4, 128).shape == (0, 8)
