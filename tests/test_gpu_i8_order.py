"""Launches of the 8-bit linear path that follow one another closely: every operand of a call written by the call in
front, into the memory that the calls before have read."""
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu

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


def c_quantize(x, q, s):
    """bbh.quantize_i8 into given tensors."""
    import bbh

    rc = bbh.lib().bbh_quantize_i8(x.data_ptr(), x.stride(0), q.data_ptr(), q.stride(0), s.data_ptr(), x.shape[0],
                                   x.shape[1], 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0


@pytest.mark.parametrize("what", ["activations", "weights", "both"])
@pytest.mark.parametrize("M,N,K", [(1, 1024, 2048), (4, 384, 384), (16, 1024, 1024), (24, 1024, 2048), (200, 1024, 2048),
                                   (1500, 768, 256)])
def test_operands_rewritten_between_calls(M, N, K, what):
    """The integers and scales of the activations, the weights or both quantised anew into the same tensors in front of
    each linear call: the results are those of calls that are waited for."""
    import bbh

    rounds = 40
    g = gen(M, N, K, what)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV).half()
    xs, ws = rand(rounds, M, K), rand(rounds, N, K)
    (q, s), (w, t) = bbh.quantize_i8(xs[0]), bbh.quantize_i8(ws[0])
    out = torch.empty(rounds, M, N, dtype=torch.float16, device=DEV)
    torch.cuda.synchronize()
    for i in range(rounds):
        if what != "weights":
            c_quantize(xs[i], q, s)
        if what != "activations":
            c_quantize(ws[i], w, t)
        bbh.linear_i8(q, s, w, t, out=out[i])
    torch.cuda.synchronize()
    for i in range(rounds):
        a = bbh.quantize_i8(xs[i] if what != "weights" else xs[0])
        b = bbh.quantize_i8(ws[i] if what != "activations" else ws[0])
        torch.cuda.synchronize()
        assert torch.equal(bbh.linear_i8(*a, *b), out[i]), i


@pytest.mark.parametrize("M", [1, 12, 60, 900])
def test_layers_that_share_buffers(M):
    """A stack of layers whose 8-bit activations all go through one pair of tensors, its outputs through two in turn."""
    import bbh

    D, depth = 512, 30
    g = gen("stack", M)
    layers = [bbh.quantize_i8((torch.randn(D, D, generator=g, device=DEV) / D**0.5).half()) for _ in range(depth)]
    x = torch.randn(M, D, generator=g, device=DEV).half()
    q, s = bbh.quantize_i8(x)
    two = [torch.empty_like(x), torch.empty_like(x)]
    h = x
    for i, (w, t) in enumerate(layers):
        c_quantize(h, q, s)
        h = bbh.linear_i8(q, s, w, t, gelu=i % 2 == 0, out=two[i % 2])
    got = h.clone()
    h = x
    for i, (w, t) in enumerate(layers):
        a = bbh.quantize_i8(h)
        torch.cuda.synchronize()
        h = bbh.linear_i8(*a, w, t, gelu=i % 2 == 0)
        torch.cuda.synchronize()
    assert torch.equal(got, h)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,D", [(1, 1), (3, 9), (40, 384), (1000, 1023), (2, 20000)])
def test_one_tensor_as_x_and_residual(M, D, dtype):
    """x + x, also with an output over both: the same bits as from two copies."""
    import bbh

    x = torch.randn(M, D, generator=gen("twice", M, D), device=DEV).to(dtype)
    y, v = bbh.rmsnorm(x, residual=x.clone())
    q, s, _ = bbh.rmsnorm_i8(x, residual=x.clone())
    for outputs in ("none", "y", "sum"):
        t = x.clone()
        out = {"none": {}, "y": {"out": t}, "sum": {"sum_out": t}}[outputs]
        a, b = bbh.rmsnorm(t, residual=t, **out)
        assert torch.equal(a, y) and torch.equal(b, v)
    t = x.clone()
    a, b, c = bbh.rmsnorm_i8(t, residual=t, sum_out=t)
    assert torch.equal(a, q) and torch.equal(b, s) and torch.equal(c, v)
    t = x.clone()
    with pytest.raises(bbh.BBHError, match="overlap"):
        bbh.rmsnorm(t, residual=t, out=t, sum_out=t)
