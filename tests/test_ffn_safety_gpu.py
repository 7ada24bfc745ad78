"""What the feed-forward block does where something else goes wrong or runs at the
same time: other tensor-core kernels on other streams, waits that expire, sizes past
32 bits, memory that a call holds.

Tolerances as in tests/test_ffn_gpu.py."""
import pytest
import torch

import _ffn_ref as ref
from test_ffn_gpu import _inputs

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
