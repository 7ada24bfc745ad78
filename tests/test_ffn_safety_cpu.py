"""The feed-forward block and the activation checkpoints on a host without a GPU: what
they refuse, what they ask for, and how their launches are dealt."""
import pytest
import torch
from torch.autograd import forward_ad

from morph_b200 import ffn
from morph_b200.precision import pack_activation

BF16 = torch.bfloat16


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("which", range(5))
def test_forward_mode_tangents_are_refused(which, grad_mode):
    """An output without a tangent would stand for a zero derivative, whether or not
    reverse mode records the call."""
    r = lambda *s: torch.randn(*s).to(BF16)  # noqa: E731
    args = [r(3, 64), r(96, 64), r(96, 64), r(64, 96), r(3, 64)]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        x, gate, up, down, dy = args
        calls = [lambda: ffn.feed_forward_backward(dy, x, gate, up, down)]
        if which < 4:
            calls.append(lambda: ffn.feed_forward(x, gate, up, down))
        if which < 3:
            calls += [lambda: ffn.gated_linear(x, gate, up),
                      lambda: ffn.gated_linear_backward(args[3].t(), x, gate, up)]
        if which == 0:
            calls.append(lambda: pack_activation(x))
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        module = ffn.GatedFeedForward(64, 96)
        if which == 0:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                module(x)
    with forward_ad.dual_level():  # without a tangent: the usual checks
        with pytest.raises(ValueError):
            pack_activation(torch.zeros(3, 64, dtype=BF16))
