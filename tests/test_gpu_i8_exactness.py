"""Exactness of the 8-bit linear path on the GPU, finer than one rounding of its 16-bit outputs shows: an output
is compared with the 64-bit value rounded once, wherever that value lies further from the border between two
16-bit neighbours than the kernel's 32-bit arithmetic may be off. u = 2^-24 is half a step of fp32."""
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
DTYPES = [torch.float16, torch.bfloat16]
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def gen(*key):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(key).encode()))


def gelu_error(z):
    """(64-bit GELU of z, how far the 32-bit one may be from it), |z| <= 5.75. Of Phi(-a): the fit (1.8e-7 of
    itself up to a = 4, 2e-6 above), ex2 (2^-22) and the polynomial's fmas in the exponent, each half a step of a
    partial sum: those partial sums together are under 1 + 3 a + 3 a^2. One rounding of the result follows."""
    a = z.abs()
    tail = 0.5 * torch.special.erfc(a / 2**0.5)
    want = z.clamp(min=0) - a * tail
    rel = torch.where(a <= 4, 1.8e-7, 2e-6) + 2.0**-22 + 0.6932 * U * (1 + 3 * a + 3 * a * a)
    return want, a * tail * rel + U * want.abs() * 1.001


def decided(want, off, dtype):
    """Where every value within `off` of `want` has one 16-bit rounding: that of both ends of the interval, since the
    conversion does not decrease."""
    lo, hi = (want - off).to(dtype), (want + off).to(dtype)
    return lo == hi


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [0.5, 1.0, 2.5])
@pytest.mark.parametrize("kernel", ["pair", "few rows", "one token"])
def test_gelu_to_32_bits(kernel, size, dtype):
    """A product of one term: the scale vectors give the GELU's argument to the bit (a_scale or w_scale the value,
    the others 1)."""
    import bbh

    count = {"pair": 400_000, "few rows": 60, "one token": 8}[kernel]
    columns = {"pair": 8, "few rows": 9000, "one token": 70_000}[kernel]
    g = gen("gelu", kernel, size)
    a = torch.zeros(count, 16, dtype=torch.int8, device=DEV)
    w = torch.zeros(columns, 16, dtype=torch.int8, device=DEV)
    a[:, 0] = 1
    w[:, 0] = 1
    wide = kernel != "pair"
    x = (size * torch.randn(columns if wide else count, generator=g, device=DEV)).clamp(-5.75, 5.75)
    one = torch.ones(count if wide else columns, device=DEV)
    c = bbh.linear_i8(a, one, w, x, gelu=True, dtype=dtype) if wide else bbh.linear_i8(a, x, w, one, gelu=True, dtype=dtype)
    c = c if wide else c.t()
    assert torch.equal(c, c[:1].expand_as(c))
    want, off = gelu_error(x.double())
    sure = decided(want, off, dtype)
    assert sure.double().mean().item() > 0.99
    assert torch.equal(c[0][sure], want.to(dtype)[sure])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D,F", [(1, 384, 1536), (50, 384, 1536), (1024, 1024, 4096), (1000, 333, 1001)])
def test_ffn_block_stage_by_stage(M, D, F, dtype):
    """norm -> up + GELU -> quantise -> down, each stage in 64 bits from what the stage in front returned: a 16-bit
    output is the 64-bit value's rounding wherever 32-bit arithmetic leaves no doubt, and the integers of the GELU's
    output are those of the 64-bit quotient, all of them."""
    import bbh

    g = gen("stages", M, D, F)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x, r = rand(M, D).to(dtype), rand(M, D).to(dtype)
    nw = (1 + 0.1 * rand(D)).to(dtype)
    up, up_s = bbh.quantize_i8((rand(F, D) / D**0.5).to(dtype))
    down, down_s = bbh.quantize_i8((rand(D, F) / F**0.5).to(dtype))
    bu, bd = (0.1 * rand(F)).to(dtype), (0.1 * rand(D)).to(dtype)
    q, s, v = bbh.rmsnorm_i8(x, nw, residual=r)
    h = bbh.linear_i8(q, s, up, up_s, bu, gelu=True, dtype=dtype)
    q2, s2 = bbh.quantize_i8(h)
    y = bbh.linear_i8(q2, s2, down, down_s, bd, dtype=dtype)
    product = lambda a, sa, w, sw: (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()
    p = product(q, s, up, up_s)
    z = p + bu.double()
    # int -> fp32, * a_scale, * w_scale + bias: three roundings, the first two of the product alone; GELU's slope is
    # under 1.13
    want, off = gelu_error(z)
    off = off + 1.13 * U * (2 * p.abs() + z.abs()) * 1.001
    sure = decided(want, off, dtype) & (z.abs() <= 5.75)
    assert sure.double().mean().item() > 0.99
    assert torch.equal(h[sure], want.to(dtype)[sure])
    t = h.double()
    assert torch.equal(q2.double(), torch.round(t * 127 / t.abs().amax(1, keepdim=True)))
    p = product(q2, s2, down, down_s)
    want = p + bd.double()
    sure = decided(want, U * (2 * p.abs() + want.abs()) * 1.001, dtype)
    assert sure.double().mean().item() > 0.99
    assert torch.equal(y[sure], want.to(dtype)[sure])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(1, 64), (3, 70_000), (40, 64), (300, 1000), (3000, 1001), (5000, 4096)])
def test_gelu_of_infinities(M, N, dtype):
    """x Phi(x) is +inf at +inf and 0 at -inf; NaN only of NaN. An infinite bias, an infinite scale, and finite values
    far out, each in columns of its own next to ordinary ones."""
    import bbh

    inf, nan = float("inf"), float("nan")
    g = gen("infinities", M, N)
    a = torch.randint(1, 100, (M, 16), generator=g, device=DEV, dtype=torch.int8)
    w = torch.randint(1, 100, (N, 16), generator=g, device=DEV, dtype=torch.int8)
    sa = torch.full((M,), 1e-3, device=DEV)
    sw = torch.full((N,), 1e-3, device=DEV)
    b = torch.zeros(N, dtype=dtype, device=DEV)
    plain = bbh.linear_i8(a, sa, w, sw, b, gelu=True, dtype=dtype)
    big = 6e4 if dtype is torch.float16 else 3e38
    b[1::9], b[3::9], b[5::9], b[7::9] = inf, -inf, nan, big
    sw[2::9], sw[6::9] = inf, -inf
    sw[8::9] = -3e38
    c = bbh.linear_i8(a, sa, w, sw, b, gelu=True, dtype=dtype)
    assert bool((c[:, 1::9] == inf).all()) and bool((c[:, 2::9] == inf).all())
    assert bool((c[:, 3::9] == 0).all()) and bool((c[:, 6::9] == 0).all()) and bool((c[:, 8::9] == 0).all())
    assert bool(torch.isnan(c[:, 5::9]).all())
    assert bool((c[:, 7::9] >= big * 0.99).all()) and not bool(torch.isnan(c[:, 7::9]).any())
    assert torch.equal(c[:, 0::9], plain[:, 0::9]) and torch.equal(c[:, 4::9], plain[:, 4::9])


def test_half_to_even_in_rows_near_the_end_of_bf16():
    """Every bf16 value in [2^120, 2^128) as a row's maximum, its half (63.5 steps, to 64) and its small parts: near the
    upper end a reciprocal of the maximum is no normal fp32 number."""
    import bbh

    bits = torch.arange(0x7B80, 0x7F80, device=DEV, dtype=torch.int32).to(torch.int16)
    top = bits.view(torch.bfloat16)
    assert top[0].item() == 2.0**120 and top[-1].item() == torch.finfo(torch.bfloat16).max
    x = torch.randn(top.numel(), 64, generator=gen("bf16 end"), device=DEV).clamp(-1, 1).bfloat16() * top[:, None]
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = top, top / 2, -top / 2, -top
    for k in range(4, 12):
        x[:, k] = top * 2.0 ** (2 - k)
    q, s = bbh.quantize_i8(x)
    want = torch.round(x.double() * 127 / top.double()[:, None])
    assert torch.equal(q.double(), want)
    assert bool(((s.double() * 127 / top.double() - 1).abs() <= U).all())
