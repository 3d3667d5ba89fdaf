"""The activations of TreeLinear.fused where they are small: one product a sum, exact in fp32, so that the activation alone is compared, relative to
its own value, over every kernel and split."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def exact(z, act):
    """(value in 64 bits, relative error of the fp32 arithmetic).  exp is off by 2 + 1.18 |x| units of 2^-23, sums and quotients by 2^-24 each;
    tanh's exponent is formed in four roundings, each of which the exponential turns into |x| 2^-24.  Phi comes from a fit that is off by 2^-18.8,
    and an exponent of z^2 / 2 formed in three roundings, with the exponential's own two units"""
    if act == "silu":
        return z * torch.sigmoid(z), (2 + 1.18 * z.abs()) * 2.0 ** -23 + 2.0 ** -22
    if act == "gelu_tanh":
        u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        return z * torch.sigmoid(u), (2 + 1.18 * u.abs()) * 2.0 ** -23 + u.abs() * 2.0 ** -22 + 2.0 ** -22
    return 0.5 * z * torch.erfc(-z / math.sqrt(2)), 2.0 ** -18.8 + z * z * 2.0 ** -23 + 2.0 ** -21


@pytest.mark.parametrize("act,far", [("gelu", 12.5), ("silu", 80.0), ("gelu_tanh", 9.5)])
@pytest.mark.parametrize("B", [1, 8, 16, 40, 200, 330, 1500])
@pytest.mark.parametrize("M,N", [(128, 64), (256, 2048)])
def test_tails(M, N, B, act, far):
    """sums from 0 down to -far, and as far up"""
    from statetree_b200 import TreeLinear
    w = (1 + torch.arange(M, device="cuda") % 128 / 128).to(torch.bfloat16)                      # (every mantissa)
    tl = TreeLinear.from_weight(w[:, None].expand(M, N).contiguous())
    x = torch.zeros(B, N, dtype=torch.bfloat16, device="cuda")
    for side in (-1, 1):
        x[:, 7] = side * torch.linspace(far / 2, 0.01, B, device="cuda")
        z = x[:, 7:8].double() * w.double()
        want, rel = exact(z, act)
        off = (tl.fused(x, act).double() - want).abs()
        tol = (2.0 ** -8 + rel) * want.abs() + 2.0 ** -126       # (below it values are held in steps of 2^-133)
        assert bool((off <= tol).all()), (side, float((off / tol).max()), float(z.flatten()[(off / tol).argmax()]))


@pytest.mark.parametrize("B", [1, 40, 600])
def test_swiglu_tail(B):
    """the same of a gate, times an exact up"""
    from statetree_b200 import TreeLinear
    from statetree_b200.linear import interleave_gate_up
    w = (1 + torch.arange(128, device="cuda") / 128).to(torch.bfloat16)
    tl = TreeLinear.from_weight(interleave_gate_up(w[:, None].expand(128, 64).contiguous(), torch.full((128, 64), -4.0, dtype=torch.bfloat16, device="cuda")))
    x = torch.zeros(B, 64, dtype=torch.bfloat16, device="cuda")
    x[:, 63] = -torch.linspace(40.0, 0.01, B, device="cuda")
    z = x[:, 63:].double() * w.double()
    want, rel = exact(z, "silu")
    want = want * (x[:, 63:].double() * -4)
    off = (tl.fused(x, "swiglu").double() - want).abs()
    assert bool((off <= (2.0 ** -8 + rel + 2.0 ** -24) * want.abs() + 2.0 ** -126).all())
