"""TreeLinear.fused: activation(x W^T + bias) + residual against the formula in 64 bits, over the GEMV, the tcgen05 kernel on single CTAs and on
CTA pairs, split and unsplit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh", "swiglu"]


def weights(M, N, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    W = torch.randn(M, N, device="cuda", generator=g) * 0.02
    W[:, torch.randperm(N, device="cuda", generator=g)[:max(1, N // 100)]] *= 8
    W[0, 0], W[-1, -1], W[M // 2, :8] = 0.0, 1e-9, 0.0                      # (escapes, also in the last record)
    return W.to(torch.bfloat16)


def layer(M, N, bias=True, seed=0):
    from statetree_b200 import TreeLinear
    W = weights(M, N, seed)
    b = torch.randn(M, device="cuda", generator=torch.Generator("cuda").manual_seed(seed + 1)).to(torch.bfloat16) if bias else None
    return TreeLinear.from_weight(W, b), W, b


def reference(x, W, b, act, res):
    """(result in 64 bits, bound).  The sum of N products in fp32: each of N additions is off by 2^-24 of the magnitudes so far at most
    (twice that where a matrix unit cuts off), so N 2^-23 sum |x w|; an activation passes it on with a slope of 1.13 at most and adds 2^-20
    of itself; SwiGLU passes gate's on times up and up's times the activated gate.  Then one rounding, half a step: 2^-8"""
    z = x.double() @ W.double().t()
    e = x.double().abs() @ W.double().abs().t() * (W.shape[1] * 2.0 ** -23)
    if b is not None:
        z, e = z + b.double(), e + 2.0 ** -24 * b.double().abs()
    silu = lambda t: t * torch.sigmoid(t)                                   # noqa: E731
    if act == "swiglu":
        z, e = z.view(z.shape[0], -1, 2, 16), e.view(z.shape[0], -1, 2, 16)
        g, u = z[:, :, 0], z[:, :, 1]
        y = (silu(g) * u).flatten(1)
        e = (1.13 * e[:, :, 0] * u.abs() + silu(g).abs() * e[:, :, 1] + 1.13 * e[:, :, 0] * e[:, :, 1]).flatten(1) + 2.0 ** -20 * y.abs()
    else:
        y = {None: lambda t: t, "relu": lambda t: t.clamp_min(0), "silu": silu, "gelu": lambda t: t * 0.5 * torch.erfc(-t / math.sqrt(2)),
             "gelu_tanh": lambda t: t * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3))}[act](z)
        e = 1.13 * e + (2.0 ** -20 * z.abs() if act else 0)
    if res is not None:
        y = y + res.double()
    return y, e + 2.0 ** -8 * y.abs() + 2.0 ** -134


def check(got, x, W, b, act, res=None):
    want, tol = reference(x.reshape(-1, W.shape[1]), W, b, act, None if res is None else res.reshape(-1, res.shape[-1]))
    off = (got.reshape(want.shape).double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    # as a whole: every rounding is within 2^-8 of its value, so their norm is within 2^-8 of the result's (an equality where one value is
    # nearly all of it: -40.86 of a norm of 45.54 rounded by 0.1104 of its half step of 0.125); what fp32 leaves has either sign, some
    # sqrt N 2^-24 of the norm of the terms: below 2^-13 of the result's where no sum cancels that far
    assert float(off.norm()) <= (2.0 ** -8 + 2.0 ** -13) * float(want.norm()) + 1e-30


def inputs(B, N, seed=5):
    return torch.randn(B, N, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(torch.bfloat16)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("B", [1, 3, 8, 9, 16, 17, 40, 128, 130, 300, 330, 700])
@pytest.mark.parametrize("M,N", [(256, 1024), (2048, 512), (128, 4096)])
def test_rows_and_activations(act, B, M, N):
    """every kernel and every split; with bias and residual, and with neither"""
    tl, W, b = layer(M, N)
    x = inputs(B, N)
    width = M // 2 if act == "swiglu" else M
    res = inputs(B, width, 6) * 3
    check(tl.fused(x, act, res), x, W, b, act, res)
    bare, W, _ = layer(M, N, bias=False, seed=3)
    y = bare.fused(x, act)
    assert y.shape == (B, width) and y.dtype == torch.bfloat16
    check(y, x, W, None, act)


@pytest.mark.parametrize("M,N", [(16, 64), (32, 192), (48, 64), (144, 1152), (4304, 1152), (1040, 4160), (160, 8192)])
@pytest.mark.parametrize("B", [1, 20, 150, 400])
def test_sizes_that_fill_no_tile(M, N, B):
    tl, W, b = layer(M, N)
    x, res = inputs(B, N), inputs(B, M, 6)
    for act in (None, "gelu"):
        check(tl.fused(x, act, res), x, W, b, act, res)
    if M % 32 == 0:
        check(tl.fused(x, "swiglu"), x, W, b, "swiglu")


@pytest.mark.parametrize("M,N,B", [(24576, 4096, 8), (24576, 4096, 300), (4096, 12288, 1), (4096, 12288, 2000), (6144, 4096, 513), (24576, 1024, 200)])
def test_large(M, N, B):
    tl, W, b = layer(M, N)
    x = inputs(B, N)
    act = "swiglu" if M == 24576 else None
    res = inputs(B, M // 2 if act else M, 6)
    check(tl.fused(x, act, res), x, W, b, act, res)


@pytest.mark.parametrize("B", [1, 12, 50, 200, 500])
@pytest.mark.parametrize("act", [None, "swiglu"])
def test_in_place_and_strided_residual(B, act):
    """the result over the residual; a residual that is part of wider rows, at an odd address; given outputs"""
    tl, W, b = layer(512, 768)
    width = 256 if act else 512
    x = inputs(B, 768)
    res = inputs(B, width, 6)
    want = tl.fused(x, act, res)
    check(want, x, W, b, act, res)
    stream = res.clone()
    assert tl.fused(x, act, stream, out=stream) is stream and torch.equal(stream, want)
    for shift, pad in ((0, 64), (4, 4), (1, 3), (2, 2)):
        wide = torch.zeros(B, width + pad + shift, dtype=torch.bfloat16, device="cuda")
        part = wide[:, shift:shift + width]
        part.copy_(res)
        assert torch.equal(tl.fused(x, act, part), want)
    out = torch.empty(B, width, dtype=torch.bfloat16, device="cuda")
    assert tl.fused(x, act, res, out=out) is out and torch.equal(out, want)
    assert torch.equal(tl.fused(x, act, res[:1].expand(B, width)), tl.fused(x, act, res[:1].repeat(B, 1)))


def test_shapes_types_and_empty_calls():
    tl, W, b = layer(256, 512)
    x = inputs(30, 512)
    want = tl.fused(x, "silu")
    y = tl.fused(x.view(2, 3, 5, 512), "silu", torch.zeros(2, 3, 5, 256, dtype=torch.bfloat16, device="cuda"))
    assert y.shape == (2, 3, 5, 256) and torch.equal(y.view(30, 256), want)
    f = tl.fused(x.float(), "silu")
    assert f.dtype == torch.float32 and torch.equal(f, want.float())
    assert torch.equal(tl.fused(x.cpu(), "silu"), want.cpu())
    assert torch.equal(tl.fused(x[0], "silu"), tl.fused(x[:1], "silu")[0])
    assert tl.fused(x[:0], "silu").shape == (0, 256) and tl.fused(x.view(30, 1, 512)[:, :0]).shape == (30, 0, 256)
    odd = torch.zeros(30, 513, dtype=torch.bfloat16, device="cuda")
    odd[:, 1:] = x
    assert torch.equal(tl.fused(odd[:, 1:], "silu"), want)


@pytest.mark.parametrize("B", [1, 64, 300])
def test_what_is_not_finite(B):
    """an infinite or NaN input reaches its own row alone; activations of values far out"""
    tl, W, b = layer(128, 256)
    x = inputs(B, 256)
    clean = tl.fused(x, "silu")
    x = x.clone()
    x[0, 3] = float("nan")
    y = tl.fused(x, "silu")
    assert bool(torch.isnan(y[0]).all()) and torch.equal(y[1:], clean[1:])
    for scale in (1e4, 1e18):
        for act in ("silu", "gelu", "gelu_tanh"):
            far = (inputs(B, 256).float() * scale).to(torch.bfloat16)
            z = far.double() @ W.double().t() + b.double()
            y = tl.fused(far, act).double()
            assert bool(torch.isfinite(y).all())
            sure = z.abs() > far.double().abs() @ W.double().abs().t() * 256 * 2.0 ** -23 + 100
            assert bool((y[sure & (z < 0)] == 0).all())
            up = sure & (z > 0)
            assert bool(((y - z).abs()[up] <= (2.0 ** -8 * z.abs() + far.double().abs() @ W.double().abs().t() * 256 * 2.0 ** -23)[up]).all())


@pytest.mark.parametrize("B", [1, 16, 100, 600])
def test_graph_and_streams(B):
    """captured, replayed over new inputs and residuals, beside calls on another stream; the plain forward keeps its results"""
    tl, W, b = layer(512, 2048)
    x, res = inputs(B, 2048), inputs(B, 512, 6)
    plain = tl(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tl.fused(x, "gelu", res)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = tl.fused(x, "gelu", res)
            z = tl.fused(x, None, y)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (8, 9):
        x.copy_(inputs(B, 2048, seed))
        res.copy_(inputs(B, 512, seed + 10))
        graph.replay()
        other = tl.fused(x, "gelu", res)
        assert torch.equal(other, y)
        check(y, x, W, b, "gelu", res)
        check(z, x, W, b, None, y)
    x.copy_(inputs(B, 2048))
    assert torch.equal(tl(x), plain)


def test_same_bits_every_time():
    tl, W, b = layer(1024, 8192)
    for B in (1, 30, 200, 400):
        x, res = inputs(B, 8192), inputs(B, 1024, 6)
        y = tl.fused(x, "silu", res)
        for _ in range(5):
            assert torch.equal(tl.fused(x, "silu", res), y)


def test_swiglu_agrees_with_the_separate_steps():
    """interleave_gate_up + fused against two layers and torch's silu, within the roundings of the separate steps"""
    from statetree_b200 import TreeLinear
    from statetree_b200.linear import interleave_gate_up
    g, u = weights(512, 1024, 1), weights(512, 1024, 2)
    both = TreeLinear.from_weight(interleave_gate_up(g, u))
    for B in (4, 33, 300):
        x = inputs(B, 1024)
        a, c = x.double() @ g.double().t(), x.double() @ u.double().t()
        want = torch.nn.functional.silu(a) * c
        y = both.fused(x, "swiglu")
        assert float((y.double() - want).norm() / want.norm()) < 2.0 ** -8


def test_refusals():
    tl, W, b = layer(144, 256)
    x, res = inputs(20, 256), inputs(20, 144, 6)
    for kw in (dict(activation="tanh"), dict(activation="swiglu")):                 # (144 rows: an odd number of tiles)
        with pytest.raises(ValueError):
            tl.fused(x, **kw)
    good = torch.empty(20, 144, dtype=torch.bfloat16, device="cuda")
    flat = torch.zeros(20 * 256 + 20 * 144, dtype=torch.bfloat16, device="cuda")
    for args, kw in (((x[:, :64],), {}), ((x[0, 0],), {}), ((x,), dict(residual=res.float())), ((x,), dict(residual=res[:19])), ((x,), dict(residual=res.cpu())),
                     ((x,), dict(residual=res.view(4, 5, 144))), ((x,), dict(out=good.float())), ((x,), dict(out=good[:, :143])),
                     ((x,), dict(out=torch.empty(144, 20, dtype=torch.bfloat16, device="cuda").t())), ((x,), dict(out=torch.empty(20, 145, dtype=torch.bfloat16, device="cuda")[:, :144])),
                     ((flat[:20 * 256].view(20, 256),), dict(out=flat[100:100 + 20 * 144].view(20, 144))),
                     ((x,), dict(out=flat[144:21 * 144].view(20, 144), residual=flat[:20 * 144].view(20, 144)))):
        with pytest.raises(RuntimeError):
            tl.fused(*args, **kw)
    check(tl.fused(x, None, res), x, W, b, None, res)
