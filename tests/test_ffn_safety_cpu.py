"""The feed-forward block and the activation checkpoints on a host without a GPU: what
they refuse, what they ask for, and how their launches are dealt."""
import ctypes
import math
import os
import random
import subprocess

import pytest
import torch
from torch.autograd import forward_ad

from morph_b200 import _lib, ffn
from morph_b200.precision import pack_activation

BF16 = torch.bfloat16
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


def _launch(tokens, d, f, dx=True, weights=3, pairs=74):
    """The problems of a backward pass's last launch, as mb_feed_forward_backward orders
    them: (mt, nt, kb, nseg) by falling contraction."""
    t = lambda n, size: -(-n // size)  # noqa: E731
    w = [(t(f, 256), t(d, 256), t(tokens, 64), 1)] * min(weights, 2)
    w += [(t(d, 256), t(f, 256), t(tokens, 64), 1)] * (weights > 2)
    x = [(t(tokens, 256), t(d, 256), t(f, 64), 2)] if dx else []
    problems = w + x if x and 2 * t(f, 64) < t(tokens, 64) else x + w
    return " ".join(str(n) for n in [1, pairs, len(problems), *(n for p in problems for n in p)])


@pytest.fixture(scope="module")
def replay(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("deal") / "ffn_deal")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-x", "c++", "-I", os.path.join(REPO, "morph_b200", "csrc"),
                    os.path.join(REPO, "tests", "c", "ffn_deal.cpp"), "-o", exe], check=True)

    def run(lines):
        out = subprocess.run([exe], input="\n".join(lines), capture_output=True, text=True, check=True).stdout
        return [tuple(int(n) for n in line.split()) for line in out.splitlines()]
    return run


def test_every_tile_is_dealt_once(replay):
    """Random launches of one to four problems, single and double tiles, few and many
    pairs: each k-block of each tile once, pieces inside the workspace."""
    rng = random.Random(5)
    log = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))  # noqa: E731
    lines = []
    for _ in range(1500):
        lines.append(_launch(log(161, 60000), log(1, 9000), log(1, 12000), rng.random() < 0.7, rng.choice([1, 2, 3, 3, 3]),
                             rng.choice([1, 2, 30, 66, 72, 73, 74, 74, 96])))
        lines.append(f"{rng.randrange(2)} {rng.choice([7, 70, 74, 96])} 1 {log(1, 200)} {log(1, 100)} {log(1, 600)} "
                     f"{rng.choice([1, 2])}")
    got = replay(lines)
    assert len(got) == len(lines)
    bad = [line for line, (ok, *_) in zip(lines, got) if not ok]
    assert not bad, bad[:3]


@pytest.mark.parametrize("tokens,d,f,dx,most", [
    (8192, 512, 1024, True, 1.5), (8192, 512, 1024, False, 1.5), (32768, 512, 2048, True, 1.1),
    # 48 tiles of 512 k-blocks: two pieces of each would be 96, more than the 74 pairs, so
    # one pair has 512 + 6 against a share of 48 (512 + 6) / 74 = 336: 1.54
    (32768, 512, 2048, False, 1.55),
    # 6 tiles of 256 k-blocks in at most 4 pieces, 256 / 4 + 6 = 70, and 64 tiles of 16:
    # a share of (24 (64 + 6) + 64 (16 + 6)) / 74 = 41.7: 1.68
    (16384, 256, 512, True, 1.68), (65536, 1024, 1024, True, 1.1),
    (4096, 4096, 11008, True, 1.1), (2048, 2048, 5504, True, 1.2)])
def test_narrow_blocks_with_many_tokens_are_dealt_evenly(replay, tokens, d, f, dx, most):
    """Past 2 f tokens the weight gradients have the longer contraction: they go first,
    all three are cut where a tile is more than a pair's share, and the busiest pair ends
    within `most` of the even share (8192 tokens, d 512, f 1024, dealt with dx first: 2.2
    times, without dx 3.0)."""
    [(ok, busiest, share, _)] = replay([_launch(tokens, d, f, dx)])
    assert ok and busiest <= most * share, (busiest, share)


def _aligned(rows, cols, pitch=None, offset=0):
    """A 16-bit view whose storage starts on 16 bytes, `offset` elements in."""
    pitch = pitch or cols
    buf = torch.zeros(rows * pitch + offset + 16, dtype=BF16)
    skip = (-buf.data_ptr() % 16) // 2
    return buf[skip + offset:][:rows * pitch].view(rows, pitch)[:, :cols]


def test_only_unaligned_matrices_ask_for_room():
    """The workspace grows by the copies that the call makes, not by those of every
    matrix that a call may have."""
    tokens, d, f = 5, 64, 96
    area = lambda rows, cols: -(-rows * (-(-cols // 8) * 8) * 2 // 256) * 256  # noqa: E731
    good = [(tokens, d), (f, d), (f, d), (d, f)]

    def room(mats):
        return ffn._args(0, tokens, d, f, *mats)[2]
    assert room([_aligned(*s) for s in good]) == 0
    assert room([_aligned(*s, pitch=s[1] + 8) for s in good]) == 0
    for i, s in enumerate(good):
        for bad in (dict(offset=1), dict(pitch=s[1] + 3), dict(pitch=s[1] + 8, offset=4)):
            mats = [_aligned(*t, **(bad if i == j else {})) for j, t in enumerate(good)]
            assert room(mats) == area(*s)
    assert room([_aligned(*s, offset=1) for s in good]) == sum(area(*s) for s in good)
    # a single row has no pitch
    assert ffn._padding((4096, 67, 1, 67)) == 0 and ffn._padding((4098, 67, 1, 67)) == area(1, 67)
    assert ffn._padding((0, 67, 0, 67)) == 0
    odd = _aligned(f, 65), _aligned(f, 65)
    assert ffn._args(0, tokens, 65, f, _aligned(tokens, 65), *odd, _aligned(65, f))[2] == area(tokens, 65) + 2 * area(f, 65)


def test_too_long_contractions_are_refused_before_the_first_launch():
    """Past 2^21 blocks of 64: in the backward pass only the last launch contracts over
    tokens or over 2 f, and was refused after the others had run (without a device, a
    launch fails with another status)."""
    L = _lib.lib()
    long = (1 << 27) + 1

    def args(tokens, d, f):
        return _lib.FfnArgs(_lib.MB_BF16, 0, tokens, d, f, 4096, d, 4096, d, 4096, d, 4096, f)

    def forward(tokens, d, f):
        a = args(tokens, d, f)
        return (L.mb_feed_forward(ctypes.byref(a), 4096, d, 4096, 1 << 60, None),
                L.mb_gated_linear(ctypes.byref(a), 4096, f, 4096, 1 << 60, None))

    def backward(tokens, d, f, *wanted):
        at = {n: 4096 for n in wanted}
        r = _lib.FfnGrads(dy=4096, lddy=d, lddx=d, ld_dgate=d, ld_dup=d, ld_ddown=f, **at)
        return L.mb_feed_forward_backward(ctypes.byref(args(tokens, d, f)), ctypes.byref(r), 4096, 1 << 60, None)
    assert forward(300, long, 8) == (_lib.MB_ERR_TOO_LARGE,) * 2
    assert forward(300, 8, long)[0] == _lib.MB_ERR_TOO_LARGE
    assert backward(300, long, 8, "dx") == _lib.MB_ERR_TOO_LARGE
    assert backward(300, 8, (long + 1) // 2, "dx") == _lib.MB_ERR_TOO_LARGE
    for name in ("dgate", "dup", "ddown"):
        assert backward(long, 8, 8, name) == _lib.MB_ERR_TOO_LARGE
    assert backward(long, 8, 8) == _lib.MB_OK  # nothing asked
