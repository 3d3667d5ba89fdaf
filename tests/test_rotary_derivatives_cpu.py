"""Derivatives that the rotation does not give are refused, not left out (no GPU: before anything is launched)."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

CASES = ["q", "k", "cos", "sin", "q_norm", "k_norm"]


def arguments():
    z = lambda *shape: torch.ones(*shape)                                                     # noqa: E731
    return dict(q=z(2, 2, 64), k=z(2, 1, 64), positions=torch.zeros(2, dtype=torch.long), cos=z(4, 32), sin=z(4, 32), q_norm=z(64), k_norm=z(64))


@pytest.mark.parametrize("name", CASES)
def test_forward_mode(name):
    from statetree_b200.rotary import rotate
    with forward_ad.dual_level():
        args = arguments()
        args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            rotate(**args)
        with pytest.raises(RuntimeError, match="forward-mode"):
            rotate(**args, out=(torch.empty(2, 2, 64), torch.empty(2, 1, 64)))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            rotate(**args)
        with pytest.raises(RuntimeError, match="CUDA"):                                        # (an open level alone is no reason)
            rotate(**arguments())


def test_forward_mode_into_an_output():
    from statetree_b200.rotary import rotate
    with forward_ad.dual_level():
        out = forward_ad.make_dual(torch.ones(2, 2, 64), torch.ones(2, 2, 64))
        args = dict(arguments(), k=None, k_norm=None)
        with pytest.raises(RuntimeError, match="forward-mode"):
            rotate(**args, out=(out, None))


@pytest.mark.parametrize("name", ["cos", "sin", "q_norm", "k_norm", "out"])
def test_gradients_to_what_gives_none(name):
    """... whether q needs one or not; without gradients being recorded the call is one like any other"""
    from statetree_b200.rotary import rotate
    for q_too in (False, True):
        args = arguments()
        if name not in ("q_norm", "k_norm"):
            args.update(q_norm=None, k_norm=None)
        if name == "out":
            args["out"] = (torch.empty(2, 2, 64).requires_grad_(), torch.empty(2, 1, 64))
        else:
            args[name].requires_grad_()
        args["q"].requires_grad_(q_too)
        with pytest.raises(RuntimeError, match="gradients"):
            rotate(**args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            rotate(**args)
