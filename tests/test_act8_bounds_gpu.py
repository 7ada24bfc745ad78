"""Activation checkpoints: the documented error bound at its edges, and matrices that a
launch walks in more than one turn or past 32-bit offsets."""
import pytest
import torch

from _ffn_ref import pack, unpack

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [224.0, 225.0, 226.0, 255.0, 256.0, 447.0, 448.0])
def test_the_error_bound_holds_down_to_two_to_minus_13(cuda, top, dtype):
    """At s = 0 the largest is in (224, 448] and codes are normal from 2^-6 on; 2^-13 of
    the largest is at least 224 2^-13 = 1.75 2^-6, so such values have a normal code and
    an error of at most half a step, 2^-4 of them. 2^-14 of 225 has not: 7.5 2^-9 is
    2^-13.9 of it and rounds to 8 2^-9, 0.067 off."""
    from morph_b200.precision import pack_activation, unpack_activation
    lo = torch.tensor([top * 2.0 ** -13])
    v = torch.logspace(0, 13, 127, base=2.0, dtype=torch.float64) * lo.double()
    v = torch.cat([v, torch.tensor([top], dtype=torch.float64)])
    rows = torch.stack([v * 2.0 ** e * sign for e in (0, 5, -1) for sign in (1, -1)]).to(dtype)
    x = rows.to(cuda)
    codes, scales = pack_activation(x)
    got = unpack_activation(codes, scales, torch.float32).double().cpu()
    want = rows.double()
    inside = want.abs() >= want.abs().amax(1, keepdim=True) * 2.0 ** -13
    assert inside.any(1).all()
    assert ((got - want).abs() <= want.abs() * 2.0 ** -4)[inside].all()
    assert torch.equal(got, unpack(*pack(rows)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1024, 1000, 1001])
def test_more_blocks_than_a_launch_holds_at_once(cuda, d, dtype):
    """Gapless, row by row and element by element, over several turns of every CTA: rows
    repeat with a period that divides none of the launch's, each as in a small matrix."""
    from morph_b200.precision import pack_activation, unpack_activation
    period, turns = 37, 1500
    g = torch.Generator().manual_seed(d)
    small = (torch.randn(period, d, generator=g) * torch.exp2(torch.randint(-9, 9, (period, 1), generator=g).float())).to(dtype)
    want_codes, want_scales = pack(small)
    x = small.to(cuda).repeat(turns, 1)
    codes, scales = pack_activation(x)
    assert torch.equal(codes.view(turns, period, d), want_codes.to(cuda).expand(turns, -1, -1))
    assert torch.equal(scales.view(turns, period, -1), want_scales.to(cuda).expand(turns, -1, -1))
    got = unpack_activation(codes, scales, dtype)
    assert torch.equal(got.view(turns, period, d), unpack(want_codes, want_scales).to(dtype).to(cuda).expand(turns, -1, -1))


@pytest.mark.parametrize("d", [1024, 1000, 1001])
def test_offsets_past_32_bits(cuda, d):
    """2^31 elements and more, and rows that lie further apart than they are long."""
    from morph_b200.precision import pack_activation, unpack_activation
    period = 41
    turns = 2 ** 31 // (d * period) + 7
    g = torch.Generator().manual_seed(d)
    small = torch.randn(period, d, generator=g).to(torch.bfloat16)
    want_codes, want_scales = pack(small)
    value = unpack(want_codes, want_scales).to(torch.bfloat16).to(cuda)
    x = small.to(cuda).repeat(turns, 1)
    assert x.numel() > 2 ** 31
    codes, scales = pack_activation(x)
    del x
    assert torch.equal(codes.view(turns, period, d), want_codes.to(cuda).expand(turns, -1, -1))
    assert torch.equal(scales.view(turns, period, -1), want_scales.to(cuda).expand(turns, -1, -1))
    got = unpack_activation(codes, scales)
    del codes, scales
    assert torch.equal(got.view(turns, period, d), value.expand(turns, -1, -1))
    del got
    wide = torch.zeros(600, 2 ** 22, dtype=torch.bfloat16, device=cuda)  # 2.5e9 elements
    part = wide[:, :d]
    part.copy_(small.to(cuda).repeat(15, 1)[:600])
    codes, scales = pack_activation(part)
    assert torch.equal(codes, want_codes.to(cuda).repeat(15, 1)[:600])
    assert torch.equal(scales, want_scales.to(cuda).repeat(15, 1)[:600])
