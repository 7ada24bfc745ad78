"""What the feed-forward block does where something else goes wrong or runs at the
same time: other tensor-core kernels on other streams, waits that expire, sizes past
32 bits, memory that a call holds.

Tolerances as in tests/test_ffn_gpu.py."""
import pytest
import torch

import _ffn_ref as ref
from test_ffn_gpu import _assert_same_sum, _check_grads, _inputs

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
NAMES = ("x", "gate", "up", "down")


@pytest.mark.parametrize("tokens", [4, 100, 160])
def test_few_tokens_beside_other_tensor_core_kernels(cuda, tokens):
    """The weight-streaming kernel's clusters share the SMs with torch's 16-bit products
    and with the Muon GEMM on other streams: all of them finish, each with its own
    result."""
    from morph_b200 import ffn
    from morph_b200.muon import gemm16
    v = _inputs(tokens, 1024, 2816, BF16, cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    a = torch.randn(1024, 512, device=cuda, generator=g).to(BF16)
    b = torch.randn(264, 512, device=cuda, generator=g).to(BF16)
    want = ffn.feed_forward(*(v[n] for n in NAMES)), gemm16(a, a)[0], b @ a.t()
    streams = [torch.cuda.Stream() for _ in want]
    torch.cuda.synchronize()
    got = [[], [], []]
    for _ in range(20):
        for s, call, out in zip(streams, (lambda: ffn.feed_forward(*(v[n] for n in NAMES)), lambda: gemm16(a, a)[0],
                                          lambda: b @ a.t()), got):
            with torch.cuda.stream(s):
                out.append(call())
    torch.cuda.synchronize()
    for out, w in zip(got, want):
        assert all(torch.equal(o, w) for o in out)
    ffn.check()


def _stale_memory(like):
    """Leave blocks of these tensors' sizes in the allocator that hold finite values."""
    junk = [torch.full_like(t, 7.0) for t in like] * 2
    del junk


# few tokens (split and unsplit contractions), whole tiles, cut tiles with a join, double
# tiles; the tile or CTA whose load is withheld
FAULTS = [(0, 1, 512, 1024), (3, 20, 512, 1024), (5, 120, 512, 6000), (0, 300, 512, 1024), (5, 700, 512, 1024),
          (2, 256, 2048, 5504), (7, 2500, 4096, 4096)]


def _assert_right_or_nan(got, want):
    lost = torch.isnan(got)
    assert torch.equal(torch.where(lost, want, got), want)
    return bool(lost.any())


@pytest.mark.parametrize("unit,tokens,d,f", FAULTS)
def test_an_expired_wait_leaves_nan_in_the_outputs(cuda, unit, tokens, d, f):
    """Every element of a call whose kernel gave up a wait is right or NaN, never what
    the memory held before."""
    from morph_b200 import _lib, ffn
    v = _inputs(tokens, d, f, BF16, cuda)
    args = [v[n] for n in NAMES]
    calls = [lambda: (ffn.gated_linear(*args[:3]),), lambda: (ffn.feed_forward(*args),),
             lambda: ffn.feed_forward_backward(v["grad"], *args)]
    ffn.check()
    for call in calls:
        want = call()
        _stale_memory(want)
        _lib.check(_lib.lib().mb_debug_arm_fault(_lib.MB_FAULT_FFN, unit, 5_000_000))
        got = call()
        with pytest.raises(TimeoutError):
            ffn.check()
        assert any([_assert_right_or_nan(a, b) for a, b in zip(got, want)])
        assert all(torch.equal(a, b) for a, b in zip(call(), want))
    ffn.check()


def test_an_optimizer_refuses_a_step_after_an_expired_wait(cuda):
    """Nobody calls ffn.check: the gradients' NaN make the gate refuse the step."""
    from morph_b200 import HybridMuonAdamW, _lib, ffn
    torch.manual_seed(1)
    stage = torch.nn.Module()
    stage.norm = torch.nn.LayerNorm(256, device=cuda)
    stage.ffn = ffn.GatedFeedForward(256, 704, device=cuda)
    x = torch.randn(300, 256, device=cuda)
    opt = HybridMuonAdamW(stage, lr=1e-3, muon_lr=1e-2)
    y = stage.ffn(stage.norm(x))
    _lib.check(_lib.lib().mb_debug_arm_fault(_lib.MB_FAULT_FFN, 0, 5_000_000))
    y.square().mean().backward()
    before = {n: p.detach().clone() for n, p in stage.named_parameters()}
    with pytest.raises(FloatingPointError):
        opt.step()
    assert all(torch.equal(before[n], p) for n, p in stage.named_parameters())
    with pytest.raises(TimeoutError):
        ffn.check()


@pytest.mark.parametrize("param_dtype", [torch.float32, BF16])
@pytest.mark.parametrize("checkpoint", ["x", "fp8"])
def test_the_module_keeps_its_parameters_and_its_input_only(cuda, checkpoint, param_dtype):
    """FP32 masters: no 16-bit copy of a weight lives from the forward to the backward
    pass, and the gradients are those of the block on the cast weights, bit for bit."""
    from morph_b200 import ffn
    from morph_b200.precision import pack_activation
    d, f, tokens = 512, 1408, 70
    torch.manual_seed(2)
    m = ffn.GatedFeedForward(d, f, checkpoint=checkpoint, device=cuda, param_dtype=param_dtype)
    x = torch.randn(2, tokens // 2, d, device=cuda, requires_grad=True)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t), t)[1], lambda t: t):
        y = m(x)
    params = {w.data_ptr() for w in m.parameters()}
    block = [t for t in kept if t.dtype != torch.float32 or t.data_ptr() in params]
    assert len(kept) == len(block)  # nothing of the casts around it
    own = [t for t in block if t.data_ptr() not in params]
    want = tokens * d * 2 if checkpoint == "x" else tokens * (d + d // 128)
    assert sum(t.numel() * t.element_size() for t in own) == want
    del kept, block, own
    torch.cuda.synchronize()
    y = m(x)
    del y
    base = torch.cuda.memory_allocated()
    y = m(x)
    held = torch.cuda.memory_allocated() - base
    assert held <= want + 2 * y.numel() * 4 + 16384  # the output, and its 16-bit form
    dy = torch.randn(2, tokens // 2, d, device=cuda)
    y.backward(dy)
    weights = [w.weight.detach().to(BF16) for w in (m.gate, m.up, m.down)]
    x16 = x.detach().to(BF16)
    saved = pack_activation(x16) if checkpoint == "fp8" else x16
    dx, *grads = ffn.feed_forward_backward(dy.to(BF16), saved, *weights)
    assert torch.equal(y, ffn.feed_forward(x16, *weights).float())
    assert x.grad.dtype == torch.float32 and torch.equal(x.grad, dx.float())
    for w, g in zip((m.gate, m.up, m.down), grads):
        assert w.weight.grad.dtype == param_dtype and torch.equal(w.weight.grad, g.to(param_dtype))


def test_a_module_with_frozen_parts(cuda):
    """Only the gradients asked for, with FP32 masters: input alone, one weight alone."""
    from morph_b200 import ffn
    torch.manual_seed(4)
    m = ffn.GatedFeedForward(128, 192, device=cuda)
    x = torch.randn(30, 128, device=cuda)
    m(x).sum().backward()
    full = {n: p.grad.clone() for n, p in m.named_parameters()}
    for keep in full:
        for n, p in m.named_parameters():
            p.grad = None
            p.requires_grad_(n == keep)
        m(x).sum().backward()
        for n, p in m.named_parameters():
            assert (p.grad is None) == (n != keep)
        got = dict(m.named_parameters())[keep].grad
        ref.assert_close(got.to(BF16), full[keep].double(), 1e-5 * full[keep].double().std(), keep)
    for p in m.parameters():
        p.requires_grad_(False)
    x.requires_grad_(True)
    m(x).sum().backward()
    assert x.grad.dtype == torch.float32 and torch.isfinite(x.grad).all() and (x.grad != 0).any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,d,f", [(8192, 512, 1024), (5000, 136, 200), (3000, 264, 88), (9000, 72, 1111), (16384, 256, 512)])
def test_narrow_blocks_with_many_tokens(cuda, tokens, d, f, dtype):
    """More tokens than 2 f: the weight gradients have the longest contraction, and the
    pieces of all three are joined into their own outputs."""
    from morph_b200 import ffn
    v = _inputs(tokens, d, f, dtype, cuda)
    args = [v[n] for n in NAMES]
    got = ffn.feed_forward_backward(v["grad"], *args)
    want, sigmas = ref.backward(v["grad"], *args, "silu")
    _check_grads(got, want, sigmas, dtype, ("dx", "dgate", "dup", "ddown"))
    for needs in ((False, True, True, True), (True, False, True, False), (False, False, True, True), (True, False, False, True)):
        for need, a, b in zip(needs, got, ffn.feed_forward_backward(v["grad"], *args, needs=needs)):
            assert (b is None) == (not need)
            if need:
                _assert_same_sum(b, a)
    ffn.check()


@pytest.mark.parametrize("tokens,d,f", [(3, 4096, 8192), (300, 1024, 2048)])
def test_one_unaligned_view_costs_its_own_copy(cuda, tokens, d, f):
    """An x one element off 16 bytes among large aligned weights: the call's peak memory
    is its outputs, its workspace and a copy of x."""
    from morph_b200 import _lib, ffn
    v = _inputs(tokens, d, f, BF16, cuda)
    args = [v[n] for n in NAMES]
    buf = torch.empty(tokens * d + 1, dtype=BF16, device=cuda)
    x = buf[1:].view(tokens, d)
    x.copy_(v["x"])
    L = _lib.lib()
    for call, out, ws in (
            (lambda x: (ffn.feed_forward(x, *args[1:]),), tokens * d, L.mb_feed_forward_workspace_bytes(tokens, f)),
            (lambda x: ffn.feed_forward_backward(v["grad"], x, *args[1:]), tokens * d + 3 * d * f,
             L.mb_feed_forward_backward_workspace_bytes(tokens, d, f, 0, 1))):
        want = call(v["x"])
        base = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        got = call(x)
        peak = torch.cuda.max_memory_allocated() - base
        assert peak <= 2 * out + ws + 2 * tokens * d + (2 << 20) * 6, (peak, out, ws)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
