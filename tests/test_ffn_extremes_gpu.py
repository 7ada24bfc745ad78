"""The feed-forward block where its activation saturates, at odd widths with cut and
double tiles, and past 32-bit offsets in every pass."""
import math

import pytest
import torch

import _ffn_ref as ref
from test_ffn_gpu import _assert_same_sum, _check_grads, _inputs

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _saturated(tokens, d, f, dtype, device, top):
    """x[:, 0] = 1 and gate zero but for its column 0, so that g[t, j] = gate[j, 0] without
    any error: +-1e2 to +-top, all saturated (sigma is 0 or 1 to the last bit of FP32 from
    |g| = 89 on in SiLU, far below in GELU). u and the output's gradient are unit normals."""
    v = _inputs(tokens, d, f, dtype, device, grad="dh")
    x, gate = v["x"].clone(), torch.zeros_like(v["gate"])
    x[:, 0] = 1
    g = torch.logspace(2, math.log10(top), f, device=device, dtype=torch.float64)
    g = (g * torch.where(torch.arange(f, device=device) % 3 == 1, -1., 1.)).to(dtype)
    gate[:, 0] = g
    return x, gate, v["up"], v["down"], v["grad"], g.double()


# few tokens (with and without a split contraction), whole tiles, cut tiles and their join
@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype,top", [(BF16, 1e15), (FP16, 6e4)])
@pytest.mark.parametrize("tokens,d,f", [(3, 64, 96), (20, 1024, 704), (300, 136, 520), (256, 2048, 5504)])
def test_saturated_gates(cuda, tokens, d, f, dtype, top, kind):
    """act(g) = g or 0 and act'(g) = 1 or 0 for large gates of either sign, with no NaN
    from g^3 or from a zero times a slope, in both passes."""
    from morph_b200 import ffn
    x, gate, up, down, dh, g = _saturated(tokens, d, f, dtype, cuda, top)
    unit = torch.finfo(dtype).eps / 2
    on = (g > 0).double()
    xd, ud, dhd = x.double(), up.double(), dh.double()
    u = xd @ ud.t()
    acc = lambda a, b: math.sqrt(a.shape[1]) * 2.0 ** -23 * ((a * a) @ (b * b)).sqrt()  # noqa: E731
    eu = acc(xd, ud.t())
    a = g * on
    limit = torch.finfo(dtype).max
    h = ffn.gated_linear(x, gate, up, kind)
    want = a * u
    fits = want.abs() <= limit * (1 - 2.0 ** -7)  # FP16: past its range a product is infinite
    assert not torch.isnan(h).any()
    ref.assert_close(torch.where(fits, h, 0), torch.where(fits, want, 0), torch.where(fits, a.abs() * eu, 0) + 2.0 ** -20 * torch.where(fits, want.abs(), 0), "h")
    assert (h[:, g < 0] == 0).all()
    if dtype is FP16:  # a smaller output gradient, so that du stays in range
        dh, dhd = dh * 2.0 ** -6, dhd * 2.0 ** -6
    dx, dgate, dup = ffn.gated_linear_backward(dh, x, gate, up, kind)
    dg, du = dhd * u * on, dhd * a
    edg, edu = unit * dg.abs() + dhd.abs() * eu * on + 2.0 ** -20 * dg.abs(), (unit + 2.0 ** -20) * du.abs()
    sq = lambda p, q: (p * p) @ (q * q)  # noqa: E731
    assert not any(torch.isnan(t).any() for t in (dx, dgate, dup))
    ref.assert_close(dgate, dg.t() @ xd, (sq(edg.t(), xd) + acc(dg.t(), xd) ** 2).sqrt(), "dgate")
    want = du.t() @ xd
    fits = want.abs() <= limit * (1 - 2.0 ** -7)
    sigma = (sq(edu.t(), xd) + acc(du.t(), xd) ** 2).sqrt()
    ref.assert_close(torch.where(fits, dup, 0), torch.where(fits, want, 0), torch.where(fits, sigma, 0), "dup")
    gd = gate.double()
    want = dg @ gd + du @ ud
    fits = want.abs() <= limit * (1 - 2.0 ** -7)
    sigma = (sq(edg, gd) + sq(edu, ud) + acc(dg, gd) ** 2 + acc(du, ud) ** 2).sqrt()
    ref.assert_close(torch.where(fits, dx, 0), torch.where(fits, want, 0), torch.where(fits, sigma, 0), "dx")
    assert (dgate[g < 0] == 0).all() and (dup[g < 0] == 0).all()
    # the whole block (an FP32 dh inside): no NaN either
    if dtype is BF16:
        y = ffn.feed_forward(x, gate, up, down, kind)
        grads = ffn.feed_forward_backward(x, x, gate, up, down, kind)
        assert not torch.isnan(y).any() and not any(torch.isnan(t).any() for t in grads)
    ffn.check()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,d,f", [(129, 2047, 5503), (257, 1535, 4097), (2300, 4095, 8191), (900, 1023, 2815)])
def test_odd_widths_with_cut_and_double_tiles(cuda, tokens, d, f, dtype):
    from morph_b200 import ffn
    v = _inputs(tokens, d, f, dtype, cuda)
    args = (v["x"], v["gate"], v["up"], v["down"], "gelu_tanh")
    unit = torch.finfo(dtype).eps / 2
    ref.assert_close(ffn.feed_forward(*args), ref.forward(*args), ref.forward_sigma(*args, unit), "y")
    got = ffn.feed_forward_backward(v["grad"], *args)
    want, sigmas = ref.backward(v["grad"], *args)
    _check_grads(got, want, sigmas, dtype, ("dx", "dgate", "dup", "ddown"))
    ffn.check()


@pytest.mark.parametrize("f", [2048, 2047])
def test_every_pass_past_32_bit_offsets(cuda, f):
    """2.25e9 elements of h, dh, dg and du: the down projection and dx of repeated tokens
    are those of one period, the weight gradients a multiple of its own."""
    from morph_b200 import ffn
    d, period = 64, 64
    turns = 17188
    v = _inputs(period, d, f, BF16, cuda)
    weights = [v[n] for n in ("gate", "up", "down")]
    x, dy = v["x"].repeat(turns, 1), v["grad"].repeat(turns, 1)
    assert x.shape[0] * f > 2 ** 31
    one = ffn.feed_forward(v["x"], *weights)
    y = ffn.feed_forward(x, *weights).view(turns, period, d)
    for t in (0, 2 ** 31 // f // period, turns - 1):
        _assert_same_sum(y[t], one)
    # bit for bit alike where no tile is cut: of 4297 row tiles on 74 pairs (5 beyond full
    # rounds) the launch cuts the first 5 or 6, so the first 6 * 256 tokens (24 periods) are
    # sums in another order
    assert torch.equal(y[24:224], y[24:25].expand(200, -1, -1)) and torch.equal(y[-200:], y[24:25].expand(200, -1, -1))
    for t in range(1, 24):
        _assert_same_sum(y[t], one)
    del y
    part = ffn.feed_forward_backward(v["grad"], v["x"], *weights)
    got = ffn.feed_forward_backward(dy, x, *weights)
    dx = got[0].view(turns, period, d)
    for t in (0, 2 ** 31 // f // period, turns - 1):
        _assert_same_sum(dx[t], part[0])
    assert torch.equal(dx[-200:], dx[-1:].expand(200, -1, -1))
    want, sigmas = ref.backward(v["grad"], v["x"], *weights, "silu")
    for name, a, w, s in zip(("dgate", "dup", "ddown"), got[1:], want[1:], sigmas(2.0 ** -9)[1:]):
        # each period adds the same rounded terms, so the errors of one period grow with
        # their number, and an FP32 sum of turns * period terms in steps of 16 is off by at
        # most its length times 2^-23 of its largest partial sum
        steps = turns * period / 16 * 2.0 ** -23
        ref.assert_close(a, turns * w, turns * (s + steps / 8 * (w.abs() + 8 * w.std())), name)
    ffn.check()


@pytest.mark.parametrize("tokens", [4, 200])
def test_weights_past_32_bit_offsets(cuda, tokens):
    """2.16e9 elements in each weight and each weight gradient: y and dx over the whole
    contraction, the weight gradients at the first, the last and the middle features."""
    from morph_b200 import ffn
    d, f, parts = 2056, 1_050_000, 50
    assert d * f > 2 ** 31
    g = torch.Generator(device=cuda).manual_seed(tokens)
    r = lambda std, *s: torch.empty(*s, dtype=BF16, device=cuda).normal_(0, std, generator=g)  # noqa: E731
    x, dy = r(1.0, tokens, d), r(0.5, tokens, d)
    gate, up, down = r(d ** -0.5, f, d), r(d ** -0.5, f, d), r(f ** -0.5, d, f)
    y = ffn.feed_forward(x, gate, up, down)
    dx, dgate, dup, ddown = ffn.feed_forward_backward(dy, x, gate, up, down)
    unit = 2.0 ** -9
    want_y = sq_y = want_dx = sq_dx = 0
    step = f // parts
    for lo in range(0, f, step):
        w = gate[lo:lo + step], up[lo:lo + step], down[:, lo:lo + step]
        want_y = want_y + ref.forward(x, *w, "silu")
        sq_y = sq_y + ref.forward_sigma(x, *w, "silu", unit) ** 2
        want, sigmas = ref.backward(dy, x, *w, "silu")
        s = sigmas(unit)
        want_dx, sq_dx = want_dx + want[0], sq_dx + s[0] ** 2
        if lo // step in (0, parts // 2, parts - 1):
            ref.assert_close(dgate[lo:lo + step], want[1], s[1], "dgate")
            ref.assert_close(dup[lo:lo + step], want[2], s[2], "dup")
            ref.assert_close(ddown[:, lo:lo + step], want[3], s[3], "ddown")
    # a part's sigma counts an FP32 sum of its own length: the whole one's is at most
    # sqrt(parts) times the parts' together
    ref.assert_close(y, want_y, (parts * sq_y).sqrt(), "y")
    ref.assert_close(dx, want_dx, (parts * sq_dx).sqrt(), "dx")
    ffn.check()
