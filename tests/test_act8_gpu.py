"""8-bit activation checkpoints against their definition: codes, scales and
restored values bit for bit."""
import pytest
import torch

from _ffn_ref import pack, unpack

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SHAPES = [(1, 1), (1, 7), (3, 8), (2, 127), (2, 128), (5, 129), (4, 1000), (37, 1024), (2, 1001), (700, 264)]


def _values(rows, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, d, generator=g) * torch.exp2(torch.randint(-12, 6, (rows, 1), generator=g).float())
    x[torch.rand(rows, d, generator=g) < 0.02] = 0
    return x.to(dtype)


def _check(x, codes, scales):
    want_c, want_s = pack(x.reshape(-1, x.shape[-1]).cpu())
    assert codes.shape == x.shape and codes.dtype == torch.uint8
    assert torch.equal(scales.cpu().reshape(want_s.shape), want_s)
    assert torch.equal(codes.cpu().reshape(want_c.shape), want_c)
    return want_c, want_s


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", SHAPES)
def test_codes_scales_and_values(cuda, rows, d, dtype):
    from morph_b200.precision import pack_activation, unpack_activation
    x = _values(rows, d, dtype, rows * 1000 + d)
    codes, scales = pack_activation(x.to(cuda))
    want = unpack(*_check(x, codes, scales))
    for out in DTYPES:
        got = unpack_activation(codes, scales, out).cpu()
        assert got.dtype == out and torch.equal(got, want.to(out))
    # the checkpoint's own error: half a step of a normal code, half the block's
    # smallest step below it (2^-10 of a unit whose largest code is at most 448)
    step = torch.exp2(scales.cpu().double() - 127).repeat_interleave(128, 1)[:, :d]
    err = (want - x.double()).abs()
    assert (err <= torch.maximum(x.double().abs() * 2.0 ** -4, step * 2.0 ** -10)).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_and_leading_dimensions(cuda, dtype):
    """Strided rows, a transposed view, an offset that breaks the alignment and
    more than two dimensions."""
    from morph_b200.precision import pack_activation
    base = _values(64, 512, dtype, 3).to(cuda)
    for x in (base[:, :256], base[:, 8:264], base[:, 1:201], base[::2, :128], base[:, ::2], base.t(),
              base.view(4, 16, 512), base.view(4, 16, 512)[:, 3:9], base[5], base[:1].expand(6, 512)):
        codes, scales = pack_activation(x)
        _check(x.contiguous().cpu().reshape(-1, x.shape[-1]), codes.reshape(-1, x.shape[-1]),
               scales.reshape(-1, scales.shape[-1]))
        assert codes.shape == x.shape and scales.shape[:-1] == x.shape[:-1]


@pytest.mark.parametrize("dtype", DTYPES)
def test_block_edges_nonfinite_values_and_extremes(cuda, dtype):
    from morph_b200.precision import pack_activation, unpack_activation
    t = torch.finfo(dtype)
    x = torch.zeros(12, 256, dtype=dtype)
    x[1, 5], x[1, 130] = float("inf"), 3.0
    x[2, 7], x[2, 8] = float("nan"), -2.5
    x[3] = float("-inf")
    x[4, :3] = torch.tensor([t.max, -t.max, t.max / 2], dtype=dtype)
    x[5, 0] = t.smallest_normal
    x[6, 0] = t.smallest_normal * t.eps  # the smallest subnormal
    x[7, :4] = torch.tensor([1.75, 1.0, -0.0, 0.875], dtype=dtype)       # 448 exactly, no larger scale
    x[8, :2] = torch.tensor([1.75 + 2 * 1.75 * t.eps, -1e-3], dtype=dtype)  # just past it
    x[9, :6] = torch.tensor([224., 232., 248., 240., 17., 19.], dtype=dtype)  # ties to even
    x[10] = 448.0
    x[11] = -0.0
    codes, scales = pack_activation(x.to(cuda))
    want = unpack(*_check(x, codes, scales))
    bad = ~torch.isfinite(x)
    for out in DTYPES:
        got = unpack_activation(codes, scales, out).cpu()
        limit = torch.finfo(out).max
        assert torch.equal(torch.isnan(got), bad)
        assert torch.equal(got[~bad], want[~bad].clamp(-limit, limit).to(out))


def test_empty_rows(cuda):
    from morph_b200.precision import pack_activation, unpack_activation
    codes, scales = pack_activation(torch.empty(0, 200, dtype=torch.bfloat16, device=cuda))
    assert codes.shape == (0, 200) and scales.shape == (0, 2)
    assert unpack_activation(codes, scales).shape == (0, 200)


def test_another_stream_and_graph_replay(cuda):
    from morph_b200.precision import pack_activation, unpack_activation
    x = _values(33, 520, torch.bfloat16, 1).to(cuda)
    want = unpack_activation(*pack_activation(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = unpack_activation(*pack_activation(x))
    y = _values(33, 520, torch.bfloat16, 2).to(cuda)
    x.copy_(y)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, unpack_activation(*pack_activation(y))) and not torch.equal(out, want)
