"""Every kernel, tile and split of linear_i8, each by a size that bbh.linear_i8_plan says runs it."""
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
DEV = "cuda"

#: (tokens, outputs, inputs). Few tokens; split K: tokens a tile 16, 32, 64, 128 and 1, 2, 4, 8 CTAs for K; SM pairs
#: with 128, 192 and 256 columns, stored by TMA (outputs a multiple of 8) and row by row.
SIZES = [(1, 71, 30), (1, 73, 1066), (2, 70, 2114), (1, 4096, 4096), (11, 70, 31),
         (19, 71, 30), (283, 141, 1473), (143, 135, 936), (18, 75, 932),
         (1285, 135, 30), (646, 147, 2316), (615, 140, 2742), (284, 135, 1887), (272, 152, 2403), (117, 137, 3874),
         (122, 136, 4785),
         (2574, 135, 30), (1377, 144, 3139), (1312, 137, 3599), (622, 141, 3546), (693, 135, 4587), (289, 137, 8823),
         (270, 133, 10428), (296, 256, 8192),
         (68, 9877, 34), (2466, 140, 4946), (2616, 133, 5265), (1228, 138, 7369), (1286, 150, 9366), (177, 2048, 8192),
         (552, 135, 17184), (258, 596, 19973),
         (4971, 135, 33), (4971, 136, 33), (143, 10067, 30), (143, 10064, 30), (265, 7589, 30), (265, 7592, 30),
         (268, 14991, 1411), (268, 14992, 1411)]

EVERY = {("few", 1, 2), ("few", 1, 4), ("few", 1, 8), ("few", 2, 2), ("pair", 128, 64), ("pair", 192, 64),
         ("pair", 256, 128)} | {("split", t, s) for t in (16, 32, 64, 128) for s in (1, 2, 4, 8)}


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    import bbh

    assert bbh.linear_i8_device_error() == 0


def test_the_sizes_run_every_plan():
    import bbh

    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the sizes are for 148 SMs")
    ran = lambda gelu, sizes: {bbh.linear_i8_plan(*s, gelu=gelu) for s in sizes}
    assert ran(False, SIZES) == EVERY
    assert ran(True, SIZES) == EVERY | {("pair", 256, 64)}
    for gelu in (False, True):
        pairs = {p for p in ran(gelu, SIZES) if p[0] == "pair"}
        for some in ([s for s in SIZES if s[1] % 8 == 0], [s for s in SIZES if s[1] % 8]):
            assert {p for p in ran(gelu, some) if p[0] == "pair"} == pairs


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_plan(M, N, K, dtype):
    """Against 64 bits (the sum is exact; int -> fp32, * a_scale and * w_scale + bias are three roundings, the GELU's
    argument has a slope of 1.13 at most and its Phi is within 3e-6, and the output is rounded once), and bit for bit
    what a call with one token gives."""
    import bbh

    g = torch.Generator(device=DEV).manual_seed(zlib.crc32(repr((M, N, K)).encode()))
    ld = (K + 15) // 16 * 16
    rows = lambda n: torch.randint(-127, 128, (n, ld), generator=g, device=DEV, dtype=torch.int8)[:, :K]
    a, w = rows(M), rows(N)
    sa = torch.rand(M, generator=g, device=DEV) * 0.02 + 1e-4
    sw = (torch.rand(N, generator=g, device=DEV) + 0.1) / K**0.5
    b = torch.randn(N, generator=g, device=DEV).to(dtype)
    p = (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()
    z = p + b.double()
    off = U * (2 * p.abs() + z.abs())
    tail = 0.5 * torch.special.erfc(z.abs() / 2**0.5)
    for gelu in (False, True):
        c = bbh.linear_i8(a, sa, w, sw, b, gelu=gelu, dtype=dtype)
        want = z.clamp(min=0) - z.abs() * tail if gelu else z
        tol = (1.13 * off + 3e-6 * z.abs() * tail + U * want.abs() if gelu else off) + want.abs() * HALF[dtype] + TINY[dtype]
        err = (c.double() - want).abs()
        assert bool((err <= tol * (1 + 1e-6)).all()), (gelu, (err / tol).max().item())
        for i in {0, M // 2, M - 1}:
            one = bbh.linear_i8(a[i:i + 1], sa[i:i + 1], w, sw, b, gelu=gelu, dtype=dtype)
            assert torch.equal(one[0], c[i]), (gelu, i)
