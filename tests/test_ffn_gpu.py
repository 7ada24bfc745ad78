"""The gated feed-forward block on the GPU against its 64-bit form.

Tolerances (tests/_ffn_ref.py): half a step of the output's type, and eight
standard deviations of what the 16-bit intermediates' roundings and the FP32
sums add, element by element."""
import pytest
import torch

import _ffn_ref as ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(tokens, d, f, dtype, device, seed=0, grad="dy"):
    g = torch.Generator(device=device).manual_seed(seed + tokens * 7 + d * 3 + f)
    r = lambda *s, std=1.0: (torch.randn(*s, device=device, generator=g) * std).to(dtype)  # noqa: E731
    return dict(x=r(tokens, d), gate=r(f, d, std=d ** -0.5), up=r(f, d, std=d ** -0.5), down=r(d, f, std=f ** -0.5),
                grad=r(tokens, d if grad == "dy" else f, std=0.5))


# tokens cross the weight-streaming kernel's paddings (16) and limit (256) and the
# pair kernel's row tiles (256); widths end inside k-blocks (64), feature tiles
# (64, 128) and store chunks (64), and need not be multiples of 8
SHAPES = [(1, 64, 64), (1, 1024, 2816), (2, 8, 8), (5, 136, 200), (15, 256, 512), (16, 512, 264), (17, 320, 64),
          (33, 1000, 1111), (64, 256, 1024), (100, 72, 328), (129, 640, 384), (200, 512, 1000), (256, 256, 512),
          (257, 256, 512), (300, 200, 328), (513, 1024, 640), (777, 136, 1096), (1025, 64, 2048), (600, 333, 777)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,d,f", SHAPES)
def test_gated_linear(cuda, tokens, d, f, dtype):
    from morph_b200 import ffn
    for kind in ("silu", "gelu_tanh"):
        v = _inputs(tokens, d, f, dtype, cuda)
        h = ffn.gated_linear(v["x"], v["gate"], v["up"], kind)
        assert h.shape == (tokens, f) and h.dtype == dtype and h.is_contiguous()
        ref.assert_close(h, ref.forward(v["x"], v["gate"], v["up"], None, kind),
                         ref.forward_sigma(v["x"], v["gate"], v["up"], None, kind, torch.finfo(dtype).eps / 2), kind)
    ffn.check()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,d,f", SHAPES)
def test_feed_forward(cuda, tokens, d, f, dtype):
    from morph_b200 import ffn
    v = _inputs(tokens, d, f, dtype, cuda)
    y = ffn.feed_forward(v["x"], v["gate"], v["up"], v["down"])
    assert y.shape == (tokens, d) and y.dtype == dtype and y.is_contiguous()
    args = (v["x"], v["gate"], v["up"], v["down"], "silu")
    ref.assert_close(y, ref.forward(*args), ref.forward_sigma(*args, torch.finfo(dtype).eps / 2), "y")


def _check_grads(got, want, sigmas, dtype, names):
    for name, a, b, s in zip(names, got, want, sigmas(torch.finfo(dtype).eps / 2)):
        assert a.dtype == dtype and a.shape == b.shape and a.is_contiguous()
        ref.assert_close(a, b, s, name)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,d,f", SHAPES)
def test_feed_forward_backward(cuda, tokens, d, f, dtype):
    from morph_b200 import ffn
    for kind in ("silu", "gelu_tanh"):
        v = _inputs(tokens, d, f, dtype, cuda)
        got = ffn.feed_forward_backward(v["grad"], v["x"], v["gate"], v["up"], v["down"], kind)
        want, sigmas = ref.backward(v["grad"], v["x"], v["gate"], v["up"], v["down"], kind)
        _check_grads(got, want, sigmas, dtype, ("dx", "dgate", "dup", "ddown"))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,d,f", SHAPES)
def test_gated_linear_backward_from_the_checkpoint(cuda, tokens, d, f, dtype):
    """From (codes, scales): the gradients at the restored input, exactly as if it
    had been given."""
    from morph_b200 import ffn
    from morph_b200.precision import pack_activation, unpack_activation
    v = _inputs(tokens, d, f, dtype, cuda, grad="dh")
    saved = pack_activation(v["x"])
    restored = unpack_activation(*saved, dtype)
    got = ffn.gated_linear_backward(v["grad"], saved, v["gate"], v["up"])
    want, sigmas = ref.backward(v["grad"], restored, v["gate"], v["up"], None, "silu")
    _check_grads(got, want, sigmas, dtype, ("dx", "dgate", "dup"))
    same = ffn.gated_linear_backward(v["grad"], restored, v["gate"], v["up"])
    assert all(torch.equal(a, b) for a, b in zip(got, same))
