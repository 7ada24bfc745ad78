"""Plain 64-bit forms of the gated feed-forward block and of its 8-bit
activation checkpoints, with the error bounds their kernels are held to."""
import math

import torch

BLOCK = 128


def e4m3_table():
    return torch.tensor([(c & 7) * 2.0 ** -9 if c < 8 else (8 + (c & 7)) * 2.0 ** ((c >> 3) - 10) for c in range(127)],
                        dtype=torch.float64)


def pack(x):
    """(codes, scales) of a CPU tensor [rows, d] from the definition, block by block."""
    table = e4m3_table()
    rows, d = x.shape
    nb = -(-d // BLOCK)
    codes = torch.empty(rows, d, dtype=torch.uint8)
    scales = torch.empty(rows, nb, dtype=torch.uint8)
    for j in range(nb):
        v = x[:, j * BLOCK:(j + 1) * BLOCK].double()
        finite = torch.isfinite(v)
        amax = torch.where(finite, v.abs(), 0.).amax(1)
        s = torch.zeros(rows, dtype=torch.int64)
        for r in range(rows):
            a = amax[r].item()
            if a > 0:
                m, e = math.frexp(a)  # a = m 2^e, m in [0.5, 1)
                s[r] = max(-127, e - 9 if m <= 0.875 else e - 8)
        q = v * torch.exp2(-s.double())[:, None]
        mag = torch.where(finite, q.abs(), 0.)
        hi = torch.searchsorted(table, mag.contiguous()).clamp(max=126)
        lo = (hi - 1).clamp(min=0)
        down, up = mag - table[lo], table[hi] - mag
        code = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
        code = torch.where(finite, code + 128 * torch.signbit(q), 127)
        codes[:, j * BLOCK:(j + 1) * BLOCK] = code.to(torch.uint8)
        scales[:, j] = (s + 127).to(torch.uint8)
    return codes, scales


def unpack(codes, scales):
    table = torch.cat([e4m3_table(), torch.tensor([math.nan], dtype=torch.float64)])
    c = codes.long()
    v = table[c & 127] * torch.where(c >= 128, -1., 1.)
    return v * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def act(g, kind):
    """act(g) and its derivative."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g ** 3))
    return g * (1 + t) / 2, (1 + t) / 2 + g * (1 - t * t) / 2 * k * (1 + 3 * 0.044715 * g * g)


def forward(x, gate, up, down, kind):
    x, gate, up = x.double(), gate.double(), up.double()
    a, _ = act(x @ gate.T, kind)
    h = a * (x @ up.T)
    return h if down is None else h @ down.double().T


def _sq(a, b):
    return (a * a) @ (b * b)


def forward_sigma(x, gate, up, down, kind, unit):
    """One standard deviation (an upper bound of it) of y's error before its own
    rounding: every element of h carries an independent error of at most `unit`
    relative, and of FP32 accumulation order at most sqrt(K) 2^-23 of the root of
    the squares' sum."""
    x, gate, up = x.double(), gate.double(), up.double()
    acc = lambda a, b: math.sqrt(a.shape[1]) * 2.0 ** -23 * _sq(a, b).sqrt()  # noqa: E731
    g, u = x @ gate.T, x @ up.T
    a, da = act(g, kind)
    # the SFU's exp and reciprocal: 2^-20 relative over the arguments that matter
    eh = (da * u * acc(x, gate.T)).abs() + (a * acc(x, up.T)).abs() + 2.0 ** -20 * (a * u).abs()
    if down is None:
        return eh
    h, wd = a * u, down.double()
    eh = eh + unit * h.abs()
    return (_sq(eh, wd.T) + acc(h, wd.T) ** 2).sqrt()


def backward(dy, x, gate, up, down, kind):
    """Gradients, and one standard deviation of each one's error before its own
    rounding (the roundings of dg, du and h as independent errors of `unit`
    relative, passed on to first order)."""
    dy, x, gate, up = dy.double(), x.double(), gate.double(), up.double()
    g, u = x @ gate.T, x @ up.T
    a, da = act(g, kind)
    dh = dy if down is None else dy @ down.double()
    dg, du, h = dh * u * da, dh * a, a * u
    grads = [dg @ gate + du @ up, dg.T @ x, du.T @ x]
    if down is not None:
        grads.append(dy.T @ h)

    def sigmas(unit):
        f32 = lambda a, b: math.sqrt(a.shape[1]) * 2.0 ** -23 * _sq(a, b).sqrt()  # noqa: E731
        eg, eu = f32(x, gate.T), f32(x, up.T)
        # |act''| <= 1.2 for both activations (0.5 and 1.13 at 0)
        edh = 0 if down is None else f32(dy, down.double())  # dh stays in FP32
        edg = unit * dg.abs() + (u * da * edh).abs() + (dh * da * eu).abs() + 1.2 * (dh * u * eg).abs() \
            + 2.0 ** -18 * (dh * u).abs()
        edu = unit * du.abs() + (a * edh).abs() + (dh * da * eg).abs() + 2.0 ** -20 * du.abs()
        eh = unit * h.abs() + (da * u * eg).abs() + (a * eu).abs() + 2.0 ** -20 * h.abs()
        out = [(_sq(edg, gate) + _sq(edu, up) + f32(dg, gate) ** 2 + f32(du, up) ** 2).sqrt(),
               (_sq(edg.T, x) + f32(dg.T, x) ** 2).sqrt(), (_sq(edu.T, x) + f32(du.T, x) ** 2).sqrt()]
        if down is not None:
            out.append((_sq(dy.T, eh) + f32(dy.T, h) ** 2).sqrt())
        return out

    return grads, sigmas


def assert_close(got, want, sigma, what):
    """|got - want| within half a step of the output's type and eight standard
    deviations of the errors before it (plus half the smallest subnormal)."""
    t = torch.finfo(got.dtype)
    unit = t.eps / 2
    err = (got.double() - want).abs()
    sigma = sigma if isinstance(sigma, torch.Tensor) else torch.full_like(want, sigma)
    bound = unit * want.abs() + 8 * sigma * (1 + unit) + t.smallest_normal * t.eps / 2
    bad = ~(err <= bound)
    if bad.any():
        i = bad.nonzero()[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at {i}: "
                             f"{got[tuple(i)].item()} for {want[tuple(i)].item()}, bound {bound[tuple(i)].item()}")
