"""TreeLinear.fused of layers whose bias is held in another type than BF16 (Module.half(), .float(), .double(), as a whole model is converted)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def layer(M, N):
    from statetree_b200 import TreeLinear
    g = torch.Generator("cuda").manual_seed(0)
    W = (torch.randn(M, N, device="cuda", generator=g) * 0.02).to(torch.bfloat16)
    return TreeLinear.from_weight(W, torch.randn(M, device="cuda", generator=g).to(torch.bfloat16))


@pytest.mark.parametrize("convert", ["half", "float", "double"])
@pytest.mark.parametrize("act", [None, "gelu", "swiglu"])
@pytest.mark.parametrize("B", [1, 40, 300])
def test_converted_layers(B, act, convert):
    """the values of a BF16 bias between 2^-14 and 2^16 are values of all three types, so that every bit is as before, on both host paths"""
    tl = layer(256, 512)
    tl.bias.copy_(torch.where(tl.bias.abs() < 2.0 ** -14, torch.ones_like(tl.bias), tl.bias))
    x = torch.randn(B, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    want = tl.fused(x, act)
    getattr(tl, convert)()
    assert tl.bias.dtype == dict(half=torch.float16, float=torch.float32, double=torch.float64)[convert]
    assert torch.equal(tl.fused(x, act), want)
    assert torch.equal(tl.fused(x, act, out=torch.empty_like(want)), want)
    res = torch.ones_like(want)
    assert torch.equal(tl.fused(x, act, res), tl.fused(x, act, res, out=torch.empty_like(want)))
    assert tl.fused(x.float(), act).dtype == torch.float32


def test_a_bias_beyond_bf16_is_rounded_first():
    tl = layer(256, 512)
    x = torch.randn(3, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    tl.float()
    tl.bias += 2.0 ** -12
    fine = tl.bias.clone()
    got = tl.fused(x)
    assert torch.equal(tl.bias, fine)                            # (the layer keeps what it was given)
    tl.bias = fine.to(torch.bfloat16)
    assert torch.equal(tl.fused(x), got)


def test_biases_that_are_refused():
    """another length, another device: either host path"""
    tl = layer(256, 512)
    x = torch.zeros(3, 512, dtype=torch.bfloat16, device="cuda")
    good = tl.bias
    for bad in (good[:240], good.cpu(), good.float().cpu(), good.view(16, 16), torch.stack([good, good], 1)[:, 0]):
        tl.bias = bad
        for kw in (dict(), dict(out=torch.empty(3, 256, dtype=torch.bfloat16, device="cuda"))):
            with pytest.raises(RuntimeError, match="bias"):
                tl.fused(x, **kw)
    tl.bias = good
    assert torch.equal(tl.fused(x), good.expand(3, 256))
