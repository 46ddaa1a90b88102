"""The 8-bit linear path on the GPU against plain 64-bit forms of the same operators.

Tolerances count roundings. u = 2^-24 is half a step of fp32 relative to the value, h half a
step of the 16-bit type (fp16 2^-11, bf16 2^-8), 2^-25 half fp16's smallest subnormal:
  * quantize_i8: 127 / top is off by up to 5 * 2^-23 = 10 u, so q is the integer nearest to
    x * 127 / top up to 127 * 10 u beyond the half step; the scale is one division (u).
  * rmsnorm_i8: x + residual and * weight (the element and the row's maximum), and 10 u: 14 u.
  * rstd: a sum of D non-negative terms as chains of at most 64 fmas and 10 additions (74 u,
    halved by the root), a division, an addition, rsqrt (2 steps = 4 u): under 45 u; y adds two
    products, the 8-bit scale one product and one division: 50 u.
  * linear_i8: the sum is exact; int -> fp32, * a_scale, * w_scale + bias: 3 u of the product.
"""
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
DTYPES = [torch.float16, torch.bfloat16]
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    import bbh

    assert bbh.linear_i8_device_error() == 0


def gen(*key):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(key).encode()))


def rows16(M, D, dtype, g, ld=None, offset=0):
    """[M, D] with row stride ld, starting `offset` elements into its buffer."""
    ld = D if ld is None else ld
    buf = torch.empty(offset + M * ld, dtype=dtype, device=DEV)
    x = buf[offset:].as_strided((M, D), (ld, 1))
    x.copy_(torch.randn(M, D, generator=g, device=DEV) * torch.exp(torch.randn(M, 1, generator=g, device=DEV)))
    return x


def assert_close16(got, want, rel32, dtype):
    """got (16 bit) against want (float64): one 16-bit rounding on top of rel32 * u."""
    tol = want.abs() * (HALF[dtype] * (1 + 1e-6) + rel32 * U) + TINY[dtype]
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{(err / tol).max().item():.3f} of the tolerance"


def check_quantized(q, scale, y, ulps_q, ulps_s):
    """q, scale against the real values y (float64, before quantisation)."""
    top = y.abs().amax(1)
    want_s = top / 127
    assert bool(((scale.double() - want_s).abs() <= want_s * ulps_s * U).all())
    t = torch.where(top[:, None] > 0, y * 127 / top[:, None], 0.0)
    off = (q.double() - t).abs()
    assert off.max().item() <= 0.5 + 127 * ulps_q * U, off.max().item()
    assert int(q.to(torch.int32).abs().max()) <= 127
    assert bool((q.abs().amax(1)[top > 0] == 127).all())


SHAPES = [(1, 1), (1, 7), (2, 8), (3, 16), (5, 127), (9, 128), (1, 384), (1000, 384), (77, 1000), (33, 1023),
          (4, 1024), (300, 4096), (700, 1025), (3, 16384), (301, 16400), (2, 32768), (1, 32767), (310, 32760)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D", SHAPES)
def test_quantize_i8(M, D, dtype):
    import bbh

    x = rows16(M, D, dtype, gen("quant", M, D))
    q, scale = bbh.quantize_i8(x)
    assert q.shape == (M, D) and q.dtype == torch.int8 and q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0
    check_quantized(q, scale, x.double(), 10, 1)
    y = bbh.dequantize_i8(q, scale, dtype)
    assert_close16(y, q.double() * scale.double()[:, None], 1, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_i8_rounds_half_to_even(dtype):
    """x * 127 / top of 16-bit values is exactly a half for x = top / 2 (63.5) and others: with 11
    bits a value that is not a half is 2^-20 of itself away from one, so the integers are those of the
    64-bit quotient, all of them."""
    import bbh

    g = gen("ties")
    x = rows16(4000, 256, dtype, g)
    x[:, 1] = x.abs().amax(1) / 2
    x[:, 2] = -x[:, 1]
    x[:2000, 3:] = (torch.randint(-127, 128, (2000, 253), generator=g, device=DEV) * 0.5).to(dtype)
    x[:2000, 0] = 127.0
    q, _ = bbh.quantize_i8(x)
    top = x.double().abs().amax(1, keepdim=True)
    want = torch.round(x.double() * 127 / top)
    assert torch.equal(q.double(), want)
    assert bool((x[:2000, 3:].double() * 2 % 2 == 1).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D,ld,offset", [(5, 64, 72, 0), (5, 64, 64, 1), (7, 100, 101, 3), (40, 384, 1152, 384),
                                           (40, 384, 1152, 8), (6, 9, 4096, 5), (3, 1000, 1001, 0)])
def test_row_strides_and_alignments(M, D, ld, offset, dtype):
    """Slices of wider buffers (a head's part of a QKV row, a row that starts anywhere)."""
    import bbh

    g = gen("stride", M, D, ld)
    x, r = rows16(M, D, dtype, g, ld, offset), rows16(M, D, dtype, g, ld + 3, offset + 1)
    w = torch.randn(D, generator=g, device=DEV).to(dtype)
    q, scale = bbh.quantize_i8(x)
    q0, scale0 = bbh.quantize_i8(x.contiguous())
    assert torch.equal(q, q0) and torch.equal(scale, scale0)
    y, v = bbh.rmsnorm(x, w, residual=r)
    want = x.double() + r.double()
    rms = (want.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    assert_close16(y, want * rms * w.double(), 50, dtype)
    assert_close16(v, want, 1, dtype)
    # outputs with strides and offsets of their own, and what lies between the rows left alone
    for view_ld, view_off in ((ld + 5, 3), (ld + 8 - ld % 8, 8)):
        buf = torch.full((view_off + M * view_ld,), 7.0, dtype=dtype, device=DEV)
        out = buf[view_off:].as_strided((M, D), (view_ld, 1))
        bbh.rmsnorm(x, w, residual=r, out=out)
        assert_close16(out, want * rms * w.double(), 50, dtype)
        out.fill_(7.0)
        assert bool((buf == 7.0).all())
        bbh.dequantize_i8(q, scale, out=out)
        assert torch.equal(out, bbh.dequantize_i8(q, scale, dtype))
        out.fill_(7.0)
        assert bool((buf == 7.0).all())


@pytest.mark.parametrize("D", [5, 8, 63, 384, 1023, 4095, 16381, 32761])
def test_every_alignment_of_a_row(D):
    """Rows that start 0 to 7 elements behind a 16-byte boundary, alone and as the rows of one call of odd
    width, and a weight at an odd address. Sums (not the order of the mean's terms), integers and what is
    read back are the bits of the same rows elsewhere."""
    import bbh

    f16 = torch.float16
    g = gen("align", D)
    x, r = rows16(16, D, f16, g), rows16(16, D, f16, g)
    w = torch.randn(D, generator=g, device=DEV).half()
    t = x.double() + r.double()
    want = t / (t.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    want_s = want.abs().amax(1) / 127
    y, v = bbh.rmsnorm(x, w, residual=r)
    assert_close16(y, want, 50, f16)
    q, s, _ = bbh.rmsnorm_i8(x, w, residual=r)
    check_quantized(q, s, want, 14, 55)
    q2, s2 = bbh.quantize_i8(x)
    z = bbh.dequantize_i8(q2, s2)
    for off in range(8):
        one = lambda t, i: torch.cat([t.new_empty(off), t[i]])[off:].view(1, D)
        i = (3 * off + 1) % 16
        xo, ro = one(x, i), one(r, i)
        assert (xo.data_ptr() // 2) % 8 == off
        out, so = one(y, 0), one(y, 0)
        bbh.rmsnorm(xo, w, residual=ro, out=out, sum_out=so)
        assert_close16(out[0], want[i], 50, f16)
        assert torch.equal(so[0], v[i])
        a, b, c = bbh.rmsnorm_i8(xo, w, residual=ro, sum_out=so)
        assert torch.equal(a[0], q[i]) and torch.equal(c[0], v[i])
        assert abs(b[0].double() - want_s[i]) <= 55 * U * want_s[i]
        a, b = bbh.quantize_i8(xo)
        assert torch.equal(a[0], q2[i]) and b[0] == s2[i]
        bbh.dequantize_i8(a, b, out=out)
        assert torch.equal(out[0], z[i])
    w1 = torch.cat([w[:1], w])[1:]
    assert_close16(bbh.rmsnorm(x, w1, residual=r)[0], want, 50, f16)
    a, b, _ = bbh.rmsnorm_i8(x, w1, residual=r)
    assert torch.equal(a, q) and bool(((b.double() - want_s).abs() <= 55 * U * want_s).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,D", SHAPES)
def test_rmsnorm(M, D, residual, dtype):
    import bbh

    g = gen("norm", M, D)
    x = rows16(M, D, dtype, g)
    r = rows16(M, D, dtype, g) if residual else None
    w = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dtype)
    v = x.double() + (r.double() if residual else 0)
    for weight in (w, None):
        y = v / (v.square().mean(1, keepdim=True) + 1e-5).sqrt() * (1.0 if weight is None else weight.double())
        got = bbh.rmsnorm(x, weight, 1e-5, residual=r)
        if residual:
            got, s = got
            assert_close16(s, v, 1, dtype)
        assert_close16(got, y, 50, dtype)
        q, scale, *s = bbh.rmsnorm_i8(x, weight, 1e-5, residual=r)
        if residual:
            assert_close16(s[0], v, 1, dtype)
        check_quantized(q, scale, y, 14, 55)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D", [(3, 384), (500, 1024), (11, 77)])
def test_rmsnorm_in_place(M, D, dtype):
    """The residual stream updated in place, and y over x: the same bits as fresh outputs."""
    import bbh

    g = gen("inplace", M, D)
    x, r = rows16(M, D, dtype, g), rows16(M, D, dtype, g)
    y, v = bbh.rmsnorm(x, residual=r)
    x1, r1 = x.clone(), r.clone()
    y1, v1 = bbh.rmsnorm(x1, residual=r1, out=x1, sum_out=r1)
    assert y1 is x1 and v1 is r1 and torch.equal(y, x1) and torch.equal(v, r1)
    x2, r2 = x.clone(), r.clone()
    bbh.rmsnorm(x2, residual=r2, out=r2, sum_out=x2)
    assert torch.equal(y, r2) and torch.equal(v, x2)
    q, s, v3 = bbh.rmsnorm_i8(x, residual=r)
    r4 = r.clone()
    q4, s4, v4 = bbh.rmsnorm_i8(x, residual=r4, sum_out=r4)
    assert torch.equal(q, q4) and torch.equal(s, s4) and torch.equal(v3, r4) and v4 is r4


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [8, 384, 1023, 20000])
def test_special_rows(D, dtype):
    """Zero rows, the type's lowest and smallest values, NaN and infinities: each row by itself."""
    import bbh

    x = rows16(8, D, dtype, gen("special", D))
    x[1] = 0
    x[2] = torch.finfo(dtype).min
    x[3, D // 2] = float("nan")
    x[4, D - 1] = float("inf")
    x[5, 0] = float("-inf")
    x[6] = torch.finfo(dtype).smallest_normal
    ref, ref_s = bbh.quantize_i8(x[[0, 7]].contiguous())
    q, s = bbh.quantize_i8(x)
    assert torch.equal(q[[0, 7]], ref) and torch.equal(s[[0, 7]], ref_s)
    assert bool((q[1] == 0).all()) and s[1].item() == 0
    assert bool((q[2] == -127).all())
    assert bool(torch.isnan(s[3:6]).all()) and bool((q[3:6] == 0).all())
    y = bbh.dequantize_i8(q, s, dtype)
    assert bool(torch.isnan(y[3:6]).all()) and bool(torch.isfinite(y[[0, 1, 7]]).all())
    if dtype is torch.float16:
        assert bool((q[6] == 127).all())
    else:  # 2^-126: under 2^-120, stored as zeros
        assert bool((q[6] == 0).all()) and s[6].item() == 0
    x[2] = 100  # (the square of bf16's lowest value is not an fp32 number)
    y = bbh.rmsnorm(x)
    assert bool(torch.isnan(y[3:6]).any(1).all()) and bool(torch.isfinite(y[[0, 1, 2, 6, 7]]).all())
    assert bool((y[1] == 0).all())
    q, s = bbh.rmsnorm_i8(x)
    assert bool(torch.isnan(s[3:6]).all()) and bool((q[3:6] == 0).all())
    assert s[1].item() == 0 and bool((q[1] == 0).all())
    assert bool((q[2] == 127).all()) and abs(s[2].item() * 127 - 1) < 1e-5
    # a NaN scale reaches every output of the row and no other
    w, ws = bbh.quantize_i8(rows16(24, D, dtype, gen("w", D)))
    c = bbh.linear_i8(q, s, w, ws, dtype=dtype)
    assert bool(torch.isnan(c[3:6]).all()) and bool(torch.isfinite(c[[0, 1, 2, 6, 7]]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 77, 4096])
def test_zero_rows_with_eps_zero(D, dtype):
    """1 / sqrt(0) is infinite; a zero row still gets scale 0 and zeros."""
    import bbh

    x = rows16(5, D, dtype, gen("zeros", D))
    x[[1, 4]] = 0
    q, s, v = bbh.rmsnorm_i8(x, eps=0.0, residual=torch.zeros_like(x))
    assert s[[1, 4]].tolist() == [0, 0] and bool((q[[1, 4]] == 0).all()) and torch.equal(v, x)
    assert bool((s[[0, 2, 3]] > 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D", [(1, 64), (7, 384), (300, 1000)])
def test_columns_of_one_matrix(M, D, dtype):
    """Operands that are columns of the same matrix: the same bits as separate ones, nothing else written."""
    import bbh

    g = gen("columns", M, D)
    x, r = rows16(M, D, dtype, g), rows16(M, D, dtype, g)
    y, v = bbh.rmsnorm(x, residual=r)
    wide = torch.full((M, 4 * D + 8), 7, dtype=dtype, device=DEV)
    part = [wide[:, i * D:(i + 1) * D] for i in range(4)]
    part[0].copy_(x)
    part[2].copy_(r)
    bbh.rmsnorm(part[0], residual=part[2], out=part[1], sum_out=part[3])
    assert all(torch.equal(a, b) for a, b in zip(part, (x, y, r, v))) and bool((wide[:, 4 * D:] == 7).all())


def test_rows_past_32_bit_offsets():
    """2.25 G elements: the last rows are those of a small call."""
    import bbh

    M, D = 2_200_000, 1024
    x = torch.zeros(M, D, dtype=torch.float16, device=DEV)
    tail = rows16(5, D, torch.float16, gen("tail"))
    x[-5:] = tail
    q, s = bbh.quantize_i8(x)
    q0, s0 = bbh.quantize_i8(tail)
    assert torch.equal(q[-5:], q0) and torch.equal(s[-5:], s0) and int(q[:1000].abs().max()) == 0
    y = bbh.dequantize_i8(q, s)
    assert torch.equal(y[-5:], bbh.dequantize_i8(q0, s0))
    del q, y
    y, v = bbh.rmsnorm(x, residual=x)
    y0, v0 = bbh.rmsnorm(tail, residual=tail)
    assert torch.equal(y[-5:], y0) and torch.equal(v[-5:], v0)


# ------------------------------------------------------------------------------ linear
def int8_rows(R, K, g, ld=None, low=-127):
    ld = (K + 15) // 16 * 16 if ld is None else ld
    q = torch.randint(-99, 99, (R, ld), generator=g, device=DEV, dtype=torch.int8)  # the padding too
    q[:, :K] = torch.randint(low, 128, (R, K), generator=g, device=DEV, dtype=torch.int8)
    return q[:, :K]


def linear64(a, sa, w, sw, bias):
    p = (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()
    return p, p + (0 if bias is None else bias.double())


def make_linear(M, N, K, dtype, bias, seed=0):
    g = gen("linear", M, N, K, seed)
    a, w = int8_rows(M, K, g), int8_rows(N, K, g)
    sa = torch.rand(M, generator=g, device=DEV) * 0.02 + 1e-4
    sw = (torch.rand(N, generator=g, device=DEV) + 0.1) / K**0.5
    b = torch.randn(N, generator=g, device=DEV).to(dtype) if bias else None
    return a, sa, w, sw, b


def assert_linear(c, a, sa, w, sw, b, dtype):
    p, want = linear64(a, sa, w, sw, b)
    tol = (p.abs() * 2 + want.abs()) * U + want.abs() * HALF[dtype] * (1 + 1e-6) + TINY[dtype]
    err = (c.double() - want).abs()
    assert bool((err <= tol).all()), f"{(err / tol).max().item():.3f} of the tolerance"


def assert_linear_gelu(c, a, sa, w, sw, b, dtype):
    """x Phi(x) = max(x, 0) - |x| Phi(-|x|): Phi(-|x|) is within 5.8e-6 of itself by its fit and 2^-21 by
    ex2, in all 6.3e-6; the input's error (as without GELU) grows by the GELU's steepest slope, 1.13; two
    fp32 roundings follow, then the 16-bit one."""
    p, z = linear64(a, sa, w, sw, b)
    tail = 0.5 * torch.special.erfc(z.abs() / 2**0.5)
    want = z.clamp(min=0) - z.abs() * tail
    tol = 1.13 * U * (2 * p.abs() + z.abs()) + 6.3e-6 * z.abs() * tail + (2 * U + HALF[dtype]) * want.abs() + TINY[dtype]
    err = (c.double() - want).abs()
    assert bool((err <= tol * (1 + 1e-6)).all()), f"{(err / tol).max().item():.3f} of the tolerance"


LINEAR = [(1, 1, 1), (1, 16, 16), (1, 384, 384), (2, 130, 100), (5, 1000, 31), (16, 128, 128), (17, 127, 129),
          (32, 4096, 1024), (33, 256, 4096), (64, 1152, 384), (65, 1536, 384), (127, 999, 1537), (128, 384, 1536),
          (129, 8, 5000), (200, 257, 640), (1000, 1152, 384), (1024, 1024, 1024), (777, 1001, 333), (3000, 384, 1536),
          (2500, 1536, 384), (2049, 2047, 127), (4100, 1344, 200), (3001, 1152, 17), (70000, 24, 64), (24, 70000, 64),
          (9, 64, 131071), (1, 4096, 4096), (4, 5000, 2048), (8, 300, 8000), (8, 33, 65), (7, 15, 515), (9, 17, 1000),
          (16, 1024, 1040), (1, 70001, 48), (3, 2000, 4104)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", LINEAR)
def test_linear_i8(M, N, K, dtype):
    import bbh

    a, sa, w, sw, b = make_linear(M, N, K, dtype, (M + N) % 2 == 0)
    c = bbh.linear_i8(a, sa, w, sw, b, dtype=dtype)
    assert c.shape == (M, N) and c.dtype is dtype
    assert_linear(c, a, sa, w, sw, b, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(3, 200, 96), (64, 384, 384), (300, 513, 384), (3000, 1536, 384), (2500, 1341, 64),
                                   (2600, 1152, 384)])
def test_linear_i8_gelu(M, N, K, dtype):
    import bbh

    a, sa, w, sw, b = make_linear(M, N, K, dtype, True)
    assert_linear_gelu(bbh.linear_i8(a, sa, w, sw, b, gelu=True, dtype=dtype), a, sa, w, sw, b, dtype)


# one size for each tile and split (on a GPU of 148 SMs): SM pairs with 128, 192 and 256 columns, the last with
# each number of epilogue warps, stores by TMA or not, and several rounds of tiles; 16 to 128 tokens, K in 1 to 8 parts
EVERY_KERNEL = [(180, 8304, 65), (161, 8431, 130), (1285, 1680, 200), (556, 6853, 100), (338, 8928, 129), (292, 8235, 90),
                (2600, 7200, 300), (808, 7200, 1203), (779, 7115, 1233), (3837, 2081, 33), (5000, 4104, 1500),
                (263, 5104, 100), (2411, 131, 5293), (2598, 142, 5268), (39, 816, 100), (257, 144, 1430), (115, 168, 927),
                (18, 114, 941), (54, 6464, 100), (18, 4874, 2210), (17, 2256, 1851), (121, 139, 3908), (113, 152, 4890),
                (3685, 149, 33), (1591, 134, 2975), (1302, 141, 3582), (33, 3192, 3547), (596, 155, 5055)]


@pytest.mark.parametrize("M,N,K", EVERY_KERNEL)
def test_linear_i8_every_kernel(M, N, K):
    import bbh

    dtype = DTYPES[(M + K) % 2]
    a, sa, w, sw, b = make_linear(M, N, K, dtype, True)
    assert_linear(bbh.linear_i8(a, sa, w, sw, b, dtype=dtype), a, sa, w, sw, b, dtype)
    assert_linear_gelu(bbh.linear_i8(a, sa, w, sw, b, gelu=True, dtype=dtype), a, sa, w, sw, b, dtype)
    assert bbh.linear_i8_device_error() == 0


def test_linear_i8_gelu_over_the_range():
    """GELU of every 16-bit value from -20 to 20 (the weight is the identity, the scale the value) and
    of NaN."""
    import bbh

    x = torch.cat([torch.linspace(-20, 20, 40001, device=DEV), torch.tensor([6e4, -6e4, float("nan")], device=DEV)])
    a = torch.zeros(x.numel(), 16, dtype=torch.int8, device=DEV)
    a[:, 0] = 1
    w = torch.zeros(8, 16, dtype=torch.int8, device=DEV)
    w[:, 0] = 1
    for dtype in DTYPES:
        c = bbh.linear_i8(a, x, w, torch.ones(8, device=DEV), gelu=True, dtype=dtype)[:, 0]
        z = x.double()[:-1]
        tail = 0.5 * torch.special.erfc(z.abs() / 2**0.5)
        want = z.clamp(min=0) - z.abs() * tail
        # beyond the fit's 5.75 Phi is only known to be small: |x| Phi(-|x|) < 2e-8 there
        tol = 6.3e-6 * z.abs() * tail + (2 * U + HALF[dtype]) * want.abs() + TINY[torch.float16]
        assert bool(((c[:-1].double() - want).abs() <= tol).all())
        assert bool(torch.isnan(c[-1]))


@pytest.mark.parametrize("fill", [-128, 127])
def test_linear_i8_extreme_sums(fill):
    """The largest sums int32 has to hold: K = 131,071 products of -128 * -128 (2,147,467,264) or of
    -128 * 127."""
    import bbh

    K = 131071
    a = torch.full((3, 131072), -128, dtype=torch.int8, device=DEV)[:, :K]
    w = torch.full((5, 131072), fill, dtype=torch.int8, device=DEV)[:, :K]
    one, tiny = torch.ones(3, device=DEV), torch.full((5,), 2.0**-20, device=DEV)
    c = bbh.linear_i8(a, one, w, tiny, dtype=torch.float16)
    want = torch.full((3, 5), -128.0 * fill * K * 2.0**-20, dtype=torch.float64)
    assert torch.equal(c.double().cpu(), want.to(torch.float32).to(torch.float16).double())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,K", [(384, 1536), (1152, 384), (777, 100), (4096, 640)])
def test_linear_i8_bits_do_not_depend_on_the_batch(N, K, dtype):
    """Every kernel and split gives the same bits for the same row, with and without GELU."""
    import bbh

    a, sa, w, sw, b = make_linear(5000, N, K, dtype, True)
    for gelu in (False, True):
        full = bbh.linear_i8(a, sa, w, sw, b, gelu=gelu, dtype=dtype)
        for m in (1, 8, 11, 15, 32, 50, 128, 300, 1100):
            part = bbh.linear_i8(a[:m], sa[:m], w, sw, b, gelu=gelu, dtype=dtype)
            assert torch.equal(part, full[:m]), (m, gelu)


@pytest.mark.parametrize("M,N,ldc,offset", [(5, 100, 128, 0), (5, 100, 101, 1), (300, 384, 400, 8), (3000, 1536, 1544, 0),
                                            (3000, 1500, 1537, 3), (2900, 1152, 1156, 0), (3000, 1529, 1536, 0),
                                            (3786, 2095, 2096, 8), (2900, 1340, 1344, 0)])
def test_linear_i8_output_strides(M, N, ldc, offset):
    """C of any stride and alignment; what lies around it stays."""
    import bbh

    a, sa, w, sw, b = make_linear(M, N, 200, torch.float16, True)
    want = bbh.linear_i8(a, sa, w, sw, b)
    buf = torch.full((offset + (M + 300) * ldc,), 7.0, dtype=torch.float16, device=DEV)
    out = buf[offset:].as_strided((M, N), (ldc, 1))
    bbh.linear_i8(a, sa, w, sw, b, out=out)
    assert torch.equal(out, want)
    out.fill_(7.0)
    assert bool((buf == 7.0).all())


def test_linear_i8_past_32_bit_offsets():
    """An output of 2.3 G elements and an operand whose rows lie 2.2 GB apart."""
    import bbh

    M, N, K = 140_000, 16_400, 32
    a, sa, w, sw, _ = make_linear(M, N, K, torch.float16, False)
    c = bbh.linear_i8(a, sa, w, sw)
    assert_linear(c[-300:], a[-300:], sa[-300:], w, sw, None, torch.float16)
    del c
    far = torch.empty(2_200_000_000 // 16 * 16 + 64, dtype=torch.int8, device=DEV)
    two = far.as_strided((2, 48), (2_200_000_000 // 16 * 16, 1))
    two.copy_(a[:2, :1].expand(2, 48))
    w2 = int8_rows(70, 48, gen("far"))
    c = bbh.linear_i8(two, sa[:2], w2, sw[:70])
    assert_linear(c, two, sa[:2], w2, sw[:70], None, torch.float16)


def test_scales_of_zero_and_views_of_scales():
    """A zero scale leaves the bias; scale vectors may start at any element."""
    import bbh

    a, sa, w, sw, b = make_linear(200, 300, 64, torch.float16, True)
    sa[3] = 0
    sa_view = torch.cat([torch.zeros(1, device=DEV), sa])[1:]
    sw_view = torch.cat([torch.zeros(3, device=DEV), sw])[3:]
    b_view = torch.cat([torch.zeros(1, dtype=torch.float16, device=DEV), b])[1:]
    c = bbh.linear_i8(a, sa_view, w, sw_view, b_view)
    assert torch.equal(c[3], b)
    assert torch.equal(c, bbh.linear_i8(a, sa, w, sw, b))


def test_empty_calls():
    import bbh

    x = torch.empty(0, 384, dtype=torch.float16, device=DEV)
    assert bbh.rmsnorm(x).shape == (0, 384)
    q, s = bbh.quantize_i8(x)
    assert q.shape == (0, 384) and s.shape == (0,)
    assert bbh.dequantize_i8(q, s).shape == (0, 384)
    w, ws = bbh.quantize_i8(torch.ones(8, 384, dtype=torch.float16, device=DEV))
    assert bbh.linear_i8(q, s, w, ws).shape == (0, 8)
    assert bbh.linear_i8(w, ws, q, s).shape == (8, 0)


# ------------------------------------------------------------------------------ together
def ffn(bbh, x, r, norm_w, up, down):
    """Pre-norm feed-forward block in 8 bits: (output, residual stream)."""
    q, s, v = bbh.rmsnorm_i8(x, norm_w, residual=r)
    h = bbh.linear_i8(q, s, *up, gelu=True, dtype=x.dtype)
    q, s = bbh.quantize_i8(h)
    return bbh.linear_i8(q, s, *down, dtype=x.dtype), v


def make_ffn(bbh, M, D, F, dtype):
    g = gen("ffn", M, D, F)
    x, r = torch.randn(M, D, generator=g, device=DEV).to(dtype), torch.randn(M, D, generator=g, device=DEV).to(dtype)
    nw = (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(dtype)
    wu = (torch.randn(F, D, generator=g, device=DEV) / D**0.5).to(dtype)
    wd = (torch.randn(D, F, generator=g, device=DEV) / F**0.5).to(dtype)
    bu, bd = (0.1 * torch.randn(n, generator=g, device=DEV).to(dtype) for n in (F, D))
    return x, r, nw, (*bbh.quantize_i8(wu), bu), (*bbh.quantize_i8(wd), bd), wu, wd


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D,F", [(1, 384, 1536), (64, 384, 1536), (3000, 384, 1536), (333, 500, 1001)])
def test_ffn_block(M, D, F, dtype):
    """norm -> up + GELU -> quantise -> down against the unquantised block in 64 bits. Rounding
    normal values to 127 steps of their row's maximum (at most 6 sigma here) is off by a step /
    sqrt(12) = 6 / 127 / 3.5 = 1.4 % of their size, four operands in all: under 3 % together."""
    import bbh

    x, r, nw, up, down, wu, wd = make_ffn(bbh, M, D, F, dtype)
    y, v = ffn(bbh, x, r, nw, up, down)
    d = lambda t: t.double()
    s = d(x) + d(r)
    z = s / (s.square().mean(1, keepdim=True) + 1e-6).sqrt() * d(nw)
    h = z @ d(wu).T + d(up[2])
    want = (h * 0.5 * torch.special.erfc(-h / 2**0.5)) @ d(wd).T + d(down[2])
    assert_close16(v, s, 1, dtype)
    assert ((y.double() - want).norm() / want.norm()).item() < 0.03


def test_encoder_ffn_in_8_bits_next_to_fp16():
    """The encoder's own layer order: residual LayerNorm GEMM -> (quantise -> linear + GELU -> quantise ->
    linear) against bbh.linear on the same fp16 tensors (3 %, as above)."""
    import bbh

    g = gen("encoder")
    h = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g, device=DEV) * scale).half()
    ctx, res = h(700, 384), h(700, 384)
    wo, bo, gam, bet = h(384, 384, scale=0.05), h(384, scale=0.1), 1 + h(384, scale=0.1), h(384, scale=0.1)
    w1, b1, w2, b2 = h(1536, 384, scale=0.05), h(1536, scale=0.1), h(384, 1536, scale=0.03), h(384, scale=0.1)
    y = bbh.linear_residual_layernorm(ctx, wo, bo, res, gam, bet)
    want = bbh.linear(bbh.linear(y, w1, b1, gelu=True), w2, b2)
    q1, s1 = bbh.quantize_i8(w1)
    q2, s2 = bbh.quantize_i8(w2)
    t = bbh.linear_i8(*bbh.quantize_i8(y), q1, s1, b1, gelu=True)
    got = bbh.linear_i8(*bbh.quantize_i8(t), q2, s2, b2)
    assert ((got.double() - want.double()).norm() / want.double().norm()).item() < 0.03


@pytest.mark.parametrize("M", [1, 40, 2000])
def test_captured_and_replayed(M):
    """The block in a CUDA graph, replayed on new inputs, equals the eager calls; two graphs of
    different sizes replayed in turn do not disturb one another."""
    import bbh

    graphs = []
    for m in (M, M + 3):
        x, r, nw, up, down, *_ = make_ffn(bbh, m, 384, 1536, torch.float16)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ffn(bbh, x, r, nw, up, down)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, v = ffn(bbh, x, r, nw, up, down)
        graphs.append((graph, x, r, nw, up, down, y, v))
    for k in range(3):
        for graph, x, r, nw, up, down, y, v in graphs:
            x.copy_(torch.randn(x.shape, generator=gen(k), device=DEV))
            graph.replay()
        for graph, x, r, nw, up, down, y, v in graphs:
            y0, v0 = ffn(bbh, x, r, nw, up, down)
            assert torch.equal(y, y0) and torch.equal(v, v0)


@pytest.mark.parametrize("M", [1, 24, 200])
def test_weights_written_by_the_kernel_in_front(M):
    """Weights that the call before has just quantised, into the same memory every time: a launch that starts
    early must not see the old ones."""
    import bbh

    N, K, rounds = 1024, 2048, 40
    g = gen("rewritten", M)
    ws = rows16(rounds * N, K, torch.float16, g).view(rounds, N, K)
    a, sa = int8_rows(M, K, g), torch.rand(M, generator=g, device=DEV)
    outs = torch.empty(rounds, M, N, dtype=torch.float16, device=DEV)
    pointers = set()
    for i in range(rounds):
        wq, s = bbh.quantize_i8(ws[i])
        bbh.linear_i8(a, sa, wq, s, out=outs[i])
        pointers.add(wq.data_ptr())
        del wq, s
    assert len(pointers) <= 2
    for i in range(rounds):
        wq, s = bbh.quantize_i8(ws[i])
        torch.cuda.synchronize()
        assert torch.equal(bbh.linear_i8(a, sa, wq, s), outs[i])


_FIRST_CALLS = """
import sys
sys.path[:0] = [{here!r}]
import torch, bbh
g = torch.Generator().manual_seed(1)
x = torch.randn(40, 256, generator=g).half().cuda()
w = torch.randn(512, 256, generator=g).half().cuda()
many = x.repeat(60, 1)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    wq, ws = bbh.quantize_i8(w)
    outs = [bbh.linear_i8(*bbh.rmsnorm_i8(t), wq, ws, gelu=True) for t in (x[:1], x, many)]
    outs.append(bbh.dequantize_i8(wq, ws))
graph.replay()
wq, ws = bbh.quantize_i8(w)
eager = [bbh.linear_i8(*bbh.rmsnorm_i8(t), wq, ws, gelu=True) for t in (x[:1], x, many)]
eager.append(bbh.dequantize_i8(wq, ws))
assert all(torch.equal(a, b) for a, b in zip(outs, eager))
assert bbh.linear_i8_device_error() == 0
print("same")
"""


def test_first_calls_of_a_process_captured():
    """What a kernel's first launch sets up once may happen while a stream is captured."""
    import os
    import subprocess
    import sys

    import bbh

    code = _FIRST_CALLS.format(here=os.path.dirname(os.path.abspath(bbh.__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stdout + r.stderr


def test_two_streams_at_once():
    """Calls in flight on two streams, given as argument and as the current stream."""
    import bbh

    sets = [make_ffn(bbh, m, 384, 1536, torch.float16)[:5] for m in (37, 1500)]
    want = [ffn(bbh, *s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(20):
        for i, s in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i] = ffn(bbh, *s)
    torch.cuda.synchronize()
    for (y, v), (y0, v0) in zip(got, want):
        assert torch.equal(y, y0) and torch.equal(v, v0)
    x, r, nw, up, down = sets[1]
    q, s, v = bbh.rmsnorm_i8(x, nw, residual=r, stream=streams[0])
    h = bbh.linear_i8(q, s, *up, gelu=True, stream=streams[0])
    q, s = bbh.quantize_i8(h, stream=streams[0])
    y = bbh.linear_i8(q, s, *down, stream=streams[0])
    z = bbh.dequantize_i8(q, s, stream=streams[0])
    n, _ = bbh.rmsnorm(x, nw, residual=r, stream=streams[0])
    streams[0].synchronize()
    assert torch.equal(y, want[1][0]) and torch.equal(v, want[1][1])
    assert torch.equal(z, bbh.dequantize_i8(q, s)) and torch.equal(n, bbh.rmsnorm(x, nw, residual=r)[0])


def test_python_refusals():
    import bbh

    f = lambda *s: torch.zeros(*s, dtype=torch.float16, device=DEV)
    x, q = f(4, 64), torch.zeros(4, 64, dtype=torch.int8, device=DEV)
    s = torch.ones(4, device=DEV)
    cases = [
        (TypeError, lambda: bbh.rmsnorm(x.float())), (ValueError, lambda: bbh.rmsnorm(x[0])),
        (ValueError, lambda: bbh.rmsnorm(x.t())), (TypeError, lambda: bbh.rmsnorm(x, f(64).bfloat16())),
        (ValueError, lambda: bbh.rmsnorm(x, f(63))), (ValueError, lambda: bbh.rmsnorm(x, f(128)[::2])),
        (ValueError, lambda: bbh.rmsnorm(x, residual=f(4, 63))), (TypeError, lambda: bbh.rmsnorm(x, residual=x.bfloat16())),
        (ValueError, lambda: bbh.rmsnorm(x, sum_out=f(4, 64))), (ValueError, lambda: bbh.rmsnorm(x, out=f(5, 64))),
        (ValueError, lambda: bbh.rmsnorm(x, residual=x.cpu())), (bbh.BBHError, lambda: bbh.rmsnorm(x, eps=-1.0)),
        (bbh.BBHError, lambda: bbh.rmsnorm(f(1, 64).expand(4, 64))),
        (ValueError, lambda: bbh.rmsnorm_i8(x, sum_out=f(4, 64))), (TypeError, lambda: bbh.quantize_i8(q)),
        (bbh.BBHError, lambda: bbh.quantize_i8(f(2, 32769))), (TypeError, lambda: bbh.dequantize_i8(x, s)),
        (TypeError, lambda: bbh.dequantize_i8(q, s, torch.float32)), (ValueError, lambda: bbh.dequantize_i8(q, s[:3])),
        (TypeError, lambda: bbh.dequantize_i8(q, s.double())), (ValueError, lambda: bbh.linear_i8(q, s, q[:, :32], s)),
        (ValueError, lambda: bbh.linear_i8(q, s[:3], q, s)), (ValueError, lambda: bbh.linear_i8(q, s, q, s, f(5))),
        (TypeError, lambda: bbh.linear_i8(q, s, q, s, f(4).bfloat16())), (TypeError, lambda: bbh.linear_i8(x, s, q, s)),
        (bbh.BBHError, lambda: bbh.linear_i8(torch.zeros(4, 40, dtype=torch.int8, device=DEV), s, q[:, :40], s)),
        (bbh.BBHError, lambda: bbh.linear_i8(q[:, 8:40], s, q[:, :32], s)),
        (ValueError, lambda: bbh.linear_i8(q, s, q, s, out=f(4, 5))),
        (TypeError, lambda: bbh.linear_i8(q, s, q, s, dtype=torch.float32)),
        (ValueError, lambda: bbh.linear_i8(q, s, q.cpu(), s)),
    ]
    for i, (err, call) in enumerate(cases):
        with pytest.raises(err):
            call()
            pytest.fail(f"case {i} was accepted")


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one device")
def test_tensors_on_another_device():
    import bbh

    x = torch.randn(5, 384, device="cuda:1").half()
    q, s = bbh.quantize_i8(x)
    w, ws = bbh.quantize_i8(torch.randn(64, 384, device="cuda:1").half())
    c = bbh.linear_i8(q, s, w, ws)
    assert c.device == x.device and bool(torch.isfinite(c).all())
