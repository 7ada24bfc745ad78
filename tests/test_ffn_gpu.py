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


# tokens cross the weight-streaming kernel's paddings (16) and limits (128, 160) and
# the pair kernel's row tiles (256); widths end inside k-blocks (64), feature tiles
# (64, 128) and store chunks (64), and need not be multiples of 8
SHAPES = [(1, 1, 1), (3, 1, 40), (200, 3, 1), (1, 64, 64), (1, 1024, 2816), (2, 8, 8), (5, 136, 200), (15, 256, 512), (16, 512, 264), (17, 320, 64),
          (33, 1000, 1111), (64, 256, 1024), (100, 72, 328), (128, 192, 456), (129, 640, 384), (160, 264, 512),
          (161, 512, 264), (150, 333, 777), (200, 512, 1000), (256, 256, 512),
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


@pytest.mark.parametrize("tokens,d,f", [(1, 4096, 11008), (128, 2048, 5504), (130, 4096, 11008), (1021, 2048, 5504),
                                        (2500, 1536, 4096), (2300, 4096, 8192), (2500, 4096, 8200)])
def test_served_and_trained_sizes(cuda, tokens, d, f):
    """The sizes of a 7B-shaped block and of smaller ones: every way a launch's last
    round is cut and joined, and double tiles over odd and even numbers of row tiles."""
    from morph_b200 import ffn
    v = _inputs(tokens, d, f, BF16, cuda)
    args = (v["x"], v["gate"], v["up"], v["down"], "silu")
    ref.assert_close(ffn.feed_forward(*args), ref.forward(*args), ref.forward_sigma(*args, torch.finfo(BF16).eps / 2), "y")
    got = ffn.feed_forward_backward(v["grad"], *args)
    want, sigmas = ref.backward(v["grad"], *args)
    _check_grads(got, want, sigmas, BF16, ("dx", "dgate", "dup", "ddown"))
    ffn.check()


@pytest.mark.parametrize("tokens", [3, 40, 300, 700])
def test_results_do_not_depend_on_the_run(cuda, tokens):
    """Bit for bit the same again, also while another stream keeps the GPU busy."""
    from morph_b200 import ffn
    v = _inputs(tokens, 1024, 2816, FP16, cuda)
    args = (v["x"], v["gate"], v["up"], v["down"])
    first = (ffn.feed_forward(*args),) + ffn.feed_forward_backward(v["grad"], *args)
    side = torch.cuda.Stream()
    a = torch.randn(2048, 2048, device=cuda)
    for _ in range(5):
        with torch.cuda.stream(side):
            a = (a @ a) * 1e-3
        again = (ffn.feed_forward(*args),) + ffn.feed_forward_backward(v["grad"], *args)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
    torch.cuda.synchronize()


def test_gradients_against_differences(cuda):
    """d/dt of L(theta + t v) at 0, with L's 64-bit form differenced centrally
    (error O(t^2), below 1e-6 of the value here), against the kernels' gradients
    contracted with v."""
    from morph_b200 import ffn
    for kind in ("silu", "gelu_tanh"):
        v = _inputs(50, 96, 160, FP16, cuda)
        names = ("x", "gate", "up", "down")
        grads = ffn.feed_forward_backward(v["grad"], *(v[n] for n in names), kind)
        _, sigmas = ref.backward(v["grad"], *(v[n] for n in names), kind)
        g = torch.Generator(device=cuda).manual_seed(9)
        unit = torch.finfo(FP16).eps / 2
        for name, grad, sigma in zip(names, grads, sigmas(unit)):
            d = torch.randn(v[name].shape, device=cuda, generator=g, dtype=torch.float64)
            d *= v[name].double().norm() / d.norm()

            def loss(t):
                args = [v[n].double() + (t * d if n == name else 0) for n in names]
                return (ref.forward(*args, kind) * v["grad"].double()).sum()
            h = 1e-4
            want = (8 * (loss(h) - loss(-h)) - (loss(2 * h) - loss(-2 * h))) / (12 * h)
            got = (grad.double() * d).sum()
            # independent errors: the output's rounding and what came before it
            err = ((unit * grad.double()) ** 2 + sigma ** 2).mul(d * d).sum().sqrt()
            assert abs(got - want) <= 8 * err + 1e-6 * abs(want), (name, kind)


def _assert_same_sum(got, want):
    """Equal but for the order of an FP32 sum (a launch cut another way): 2^-23 times
    the root of a few thousand terms, of values of the tensor's own size, then each
    side's rounding."""
    unit = torch.finfo(got.dtype).eps / 2
    ref.assert_close(got, want.double(), unit / 8 * want.double().abs() + 1e-5 * want.double().std(), "the same sum")


def _leaves(v, *names):
    return [v[n].clone().requires_grad_(True) for n in names]


@pytest.mark.parametrize("checkpoint", ["x", "fp8"])
@pytest.mark.parametrize("down", [False, True])
def test_autograd_equals_the_functions(cuda, down, checkpoint):
    from morph_b200 import ffn
    from morph_b200.precision import pack_activation
    v = _inputs(140, 264, 520, BF16, cuda, grad="dy" if down else "dh")
    names = ("x", "gate", "up", "down")[:4 if down else 3]
    leaves = _leaves(v, *names)
    f = ffn.feed_forward if down else ffn.gated_linear
    b = ffn.feed_forward_backward if down else ffn.gated_linear_backward
    x3 = leaves[0].view(2, 70, 264)
    y = f(x3, *leaves[1:], "gelu_tanh", checkpoint)
    assert y.shape == (2, 70, 264 if down else 520)
    with torch.no_grad():
        plain = f(v["x"], *(v[n] for n in names[1:]), "gelu_tanh")
    assert torch.equal(y.view(plain.shape), plain) and not plain.requires_grad
    y.backward(v["grad"].view(y.shape))
    saved = pack_activation(v["x"]) if checkpoint == "fp8" else v["x"]
    want = b(v["grad"], saved, *(v[n] for n in names[1:]), "gelu_tanh")
    for leaf, w in zip(leaves, want):
        assert torch.equal(leaf.grad, w)
    # accumulation into .grad, and a second backward pass is refused by autograd
    f(x3, *leaves[1:], "gelu_tanh", checkpoint).backward(v["grad"].view(y.shape))
    assert torch.equal(leaves[1].grad, want[1] + want[1])


def test_a_second_derivative_is_refused(cuda):
    from morph_b200 import ffn
    v = _inputs(10, 64, 96, BF16, cuda)
    leaves = _leaves(v, "x", "gate", "up", "down")
    y = ffn.feed_forward(*leaves)
    plain = torch.autograd.grad(y, leaves, v["grad"], retain_graph=True)
    grads = torch.autograd.grad(y, leaves, v["grad"], create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, grads))
    with pytest.raises(RuntimeError):
        grads[0].float().sum().backward()


@pytest.mark.parametrize("needs", [(True, False, False, False), (False, True, False, False), (False, False, True, False),
                                   (False, False, False, True), (False, True, True, True), (True, False, True, True),
                                   (False, False, False, False)])
@pytest.mark.parametrize("tokens", [20, 400])
def test_only_the_gradients_asked_for(cuda, tokens, needs):
    from morph_b200 import ffn
    v = _inputs(tokens, 320, 704, BF16, cuda)
    args = (v["grad"], v["x"], v["gate"], v["up"], v["down"])
    full = ffn.feed_forward_backward(*args)
    some = ffn.feed_forward_backward(*args, needs=needs)
    for need, a, b in zip(needs, full, some):
        assert (b is None) == (not need)
        if need:
            _assert_same_sum(b, a)
    leaves = _leaves(v, "x", "gate", "up", "down")
    for leaf, need in zip(leaves, needs):
        leaf.requires_grad_(need)
    y = ffn.feed_forward(*leaves)
    assert y.requires_grad == any(needs)
    if any(needs):
        y.backward(v["grad"])
        for leaf, need, b in zip(leaves, needs, some):
            assert (leaf.grad is None) == (not need) and (not need or torch.equal(leaf.grad, b))


@pytest.mark.parametrize("tokens", [33, 300])
def test_views_offsets_and_odd_pitches(cuda, tokens):
    """Weights sliced from one fused matrix, rows of a wider buffer, transposed
    storage, an offset off 16 bytes, rows broadcast: each as its contiguous copy."""
    from morph_b200 import ffn
    v = _inputs(tokens, 136, 264, BF16, cuda)
    args = [v["grad"], v["x"], v["gate"], v["up"], v["down"]]
    want_y = ffn.feed_forward(*args[1:])
    want = ffn.feed_forward_backward(*args)
    fused = torch.cat([v["gate"], v["up"]])

    def wide(t):  # rows of a wider buffer, 16-byte aligned
        buf = torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=t.dtype, device=cuda)
        buf[:, 8:8 + t.shape[1]] = t
        return buf[:, 8:8 + t.shape[1]]

    def odd(t):  # an odd pitch and offset
        buf = torch.full((t.shape[0], t.shape[1] + 3), float("nan"), dtype=t.dtype, device=cuda)
        buf[:, 1:1 + t.shape[1]] = t
        return buf[:, 1:1 + t.shape[1]]

    forms = [[v["grad"], v["x"], fused[:264], fused[264:], v["down"]], [wide(t) for t in args], [odd(t) for t in args],
             [t.t().contiguous().t() for t in args]]
    for form in forms:
        assert torch.equal(ffn.feed_forward(*form[1:]), want_y)
        assert all(torch.equal(a, b) for a, b in zip(ffn.feed_forward_backward(*form), want))
    row = v["x"][:1].expand(tokens, -1)
    assert torch.equal(ffn.feed_forward(row, *args[2:]), ffn.feed_forward(row.contiguous(), *args[2:]))


def test_shared_weights_and_the_same_tensor_twice(cuda):
    """gate and up may be one tensor, dy may be x: nothing is keyed by address."""
    from morph_b200 import ffn
    v = _inputs(300, 256, 512, FP16, cuda)
    got = ffn.feed_forward_backward(v["x"], v["x"], v["gate"], v["gate"], v["down"])
    want, sigmas = ref.backward(v["x"], v["x"], v["gate"], v["gate"], v["down"], "silu")
    _check_grads(got, want, sigmas, FP16, ("dx", "dgate", "dup", "ddown"))
    w = v["gate"].clone().requires_grad_(True)
    h = ffn.gated_linear(v["x"], w, w)
    (g,) = torch.autograd.grad(h, w, torch.ones_like(h))
    parts = ffn.gated_linear_backward(torch.ones_like(h), v["x"], v["gate"], v["gate"])
    assert torch.equal(g, parts[1] + parts[2])


@pytest.mark.parametrize("tokens", [7, 500])
def test_nothing_outside_the_outputs_is_written(cuda, tokens):
    """The C entries on buffers with guard rows and columns (pitch past the last
    column, rows behind the last token)."""
    import ctypes

    from morph_b200 import _lib
    d, f = 136, 200
    v = _inputs(tokens, d, f, BF16, cuda)
    L = _lib.lib()

    def guarded(rows, cols):
        return torch.full((rows + 9, cols + 24), 7.0, dtype=BF16, device=cuda)

    outs = dict(y=guarded(tokens, d), dx=guarded(tokens, d), dgate=guarded(f, d), dup=guarded(f, d), ddown=guarded(d, f))
    a = _lib.FfnArgs(_lib.MB_BF16, 0, tokens, d, f, v["x"].data_ptr(), d, v["gate"].data_ptr(), d, v["up"].data_ptr(), d,
                     v["down"].data_ptr(), f)
    n = L.mb_feed_forward_workspace_bytes(tokens, f)
    ws = torch.full((n + 256,), 99, dtype=torch.uint8, device=cuda)
    _lib.check(L.mb_feed_forward(ctypes.byref(a), outs["y"].data_ptr(), d + 24, ws.data_ptr(), n, _lib.stream_handle()))
    assert (ws[n:] == 99).all()
    r = _lib.FfnGrads(None, None, v["grad"].data_ptr(), d, outs["dx"].data_ptr(), d + 24, outs["dgate"].data_ptr(), d + 24,
                      outs["dup"].data_ptr(), d + 24, outs["ddown"].data_ptr(), f + 24)
    n = L.mb_feed_forward_backward_workspace_bytes(tokens, d, f, 0, 1)
    ws = torch.full((n + 256,), 99, dtype=torch.uint8, device=cuda)
    _lib.check(L.mb_feed_forward_backward(ctypes.byref(a), ctypes.byref(r), ws.data_ptr(), n, _lib.stream_handle()))
    assert (ws[n:] == 99).all()
    from morph_b200 import ffn
    names = ("x", "gate", "up", "down")
    want = (ffn.feed_forward(*(v[k] for k in names)),) + ffn.feed_forward_backward(v["grad"], *(v[k] for k in names))
    for (name, buf), w in zip(outs.items(), want):
        rows, cols = w.shape
        assert torch.equal(buf[:rows, :cols], w), name
        assert (buf[rows:] == 7).all() and (buf[:, cols:] == 7).all(), name


def test_no_tokens(cuda):
    from morph_b200 import ffn
    v = _inputs(4, 64, 96, BF16, cuda)
    x = v["x"][:0].view(2, 0, 64)
    y = ffn.feed_forward(x, v["gate"], v["up"], v["down"])
    assert y.shape == (2, 0, 64)
    assert ffn.gated_linear(x, v["gate"], v["up"]).shape == (2, 0, 96)
    dx, *grads = ffn.feed_forward_backward(y, x, v["gate"], v["up"], v["down"])
    assert dx.shape == (2, 0, 64) and all((g == 0).all() for g in grads)


@pytest.mark.parametrize("tokens", [20, 300])
def test_nonfinite_values_stay_in_their_rows(cuda, tokens):
    """A NaN or an infinity in one token reaches that token's outputs and the weight
    gradients, no other token's outputs."""
    from morph_b200 import ffn
    from morph_b200.precision import pack_activation
    v = _inputs(tokens, 128, 384, BF16, cuda)
    clean = ffn.feed_forward(v["x"], v["gate"], v["up"], v["down"])
    x = v["x"].clone()
    x[3, 5], x[11, 0] = float("nan"), float("inf")
    y = ffn.feed_forward(x, v["gate"], v["up"], v["down"])
    keep = torch.ones(tokens, dtype=torch.bool, device=cuda)
    keep[3] = keep[11] = False
    assert torch.equal(y[keep], clean[keep])
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[11]).any()
    for saved in (x, pack_activation(x)):
        dx, dgate, dup, ddown = ffn.feed_forward_backward(v["grad"], saved, v["gate"], v["up"], v["down"])
        assert torch.isfinite(dx[keep]).all() and torch.isnan(dx[3]).all()
        assert torch.isnan(dgate).all() and torch.isnan(ddown).all()
    big = v["x"].clone()
    big[0] = 3e38  # g and u overflow where their rows add up
    assert torch.equal(ffn.feed_forward(big, v["gate"], v["up"], v["down"])[1:], clean[1:])


@pytest.mark.parametrize("tokens", [12, 300])
def test_streams_graphs_and_overlapping_calls(cuda, tokens):
    """Calls on two streams at once, and two captured graphs replayed at once, each
    with its own workspace."""
    from morph_b200 import ffn
    names = ("x", "gate", "up", "down")
    vs = [_inputs(tokens, 512, 1400, BF16, cuda, seed=s) for s in (1, 2)]

    def step(v):
        return (ffn.feed_forward(*(v[n] for n in names)),) + ffn.feed_forward_backward(v["grad"], *(v[n] for n in names))
    want = [step(v) for v in vs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(vs[i])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))
    graphs, outs = [], []
    for v in vs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(v))
        graphs.append(graph)
    fresh = [_inputs(tokens, 512, 1400, BF16, cuda, seed=s) for s in (3, 4)]
    for v, n in zip(vs, fresh):
        for k in v:
            v[k].copy_(n[k])
    torch.cuda.synchronize()
    for _ in range(4):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for v, o in zip(vs, outs):
        assert all(torch.equal(a, b) for a, b in zip(o, step(v)))
    ffn.check()


def test_a_captured_training_step(cuda):
    """Forward and backward through autograd in one graph, replayed on other data."""
    from morph_b200 import ffn
    from morph_b200.precision import pack_activation
    names = ("x", "gate", "up", "down")
    v, w = (_inputs(300, 256, 512, BF16, cuda, seed=s) for s in (5, 6))
    leaves = _leaves(v, *names)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ffn.feed_forward(*leaves, checkpoint="fp8")
        grads = torch.autograd.grad(y, leaves, v["grad"])
    with torch.no_grad():
        for leaf, n in zip(leaves, names):
            leaf.copy_(w[n])
        v["grad"].copy_(w["grad"])
    graph.replay()
    assert torch.equal(y, ffn.feed_forward(*(w[n] for n in names)))
    want = ffn.feed_forward_backward(w["grad"], pack_activation(w["x"]), *(w[n] for n in names[1:]))
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


FIRST_CALL_IN_A_CAPTURE = """
import torch
from morph_b200 import ffn, precision
r = lambda *s: torch.randn(*s, device="cuda").bfloat16()
for tokens in (300, 3):
    x, gate, up, down, dy = r(tokens, 256), r(512, 256), r(512, 256), r(256, 512), r(tokens, 256)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ffn.feed_forward(x, gate, up, down)
        grads = ffn.feed_forward_backward(dy, precision.pack_activation(x), gate, up, down)
    graph.replay()
    want = ffn.feed_forward_backward(dy, precision.pack_activation(x), gate, up, down)
    assert torch.equal(y, ffn.feed_forward(x, gate, up, down))
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
print("captured")
"""


def test_the_first_call_of_a_process_may_be_captured(cuda):
    import os
    import subprocess
    import sys
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_CAPTURE], cwd=repo, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr


def test_a_thread_without_a_context(cuda):
    """The first CUDA call of a fresh thread may be the block's."""
    import threading

    from morph_b200 import ffn
    v = _inputs(200, 128, 256, BF16, cuda)
    want = ffn.gated_linear(v["x"], v["gate"], v["up"])
    got = []
    t = threading.Thread(target=lambda: got.append(ffn.gated_linear(v["x"], v["gate"], v["up"])))
    t.start()
    t.join()
    assert len(got) == 1 and torch.equal(got[0], want)


def test_rows_past_32_bit_offsets(cuda):
    """2.2e9 elements of x (4.4 GB) and of h: the last tokens' outputs."""
    from morph_b200 import ffn
    d, f, tokens = 64, 2048, 1_100_000
    v = _inputs(64, d, f, BF16, cuda)
    x = v["x"].repeat(tokens // 64 + 1, 1)[:tokens]
    h = ffn.gated_linear(x, v["gate"], v["up"])
    assert h.numel() > 2 ** 31
    want = ffn.gated_linear(v["x"], v["gate"], v["up"])
    for lo in (0, 2 ** 31 // f // 64 * 64, (tokens - 64) // 64 * 64):
        _assert_same_sum(h[lo:lo + 64], want)
    del h


@pytest.mark.parametrize("unit,tokens", [(0, 20), (3, 20), (0, 300), (5, 700)])
def test_an_expired_wait_is_reported(cuda, unit, tokens):
    """A withheld load: the bounded waits end, ffn.check raises once, and the next
    call is right."""
    from morph_b200 import _lib, ffn
    v = _inputs(tokens, 512, 1024, BF16, cuda)
    want = ffn.gated_linear(v["x"], v["gate"], v["up"])
    ffn.check()
    _lib.check(_lib.lib().mb_debug_arm_fault(_lib.MB_FAULT_FFN, unit, 5_000_000))
    ffn.gated_linear(v["x"], v["gate"], v["up"])
    with pytest.raises(TimeoutError):
        ffn.check()
    ffn.check()
    assert torch.equal(ffn.gated_linear(v["x"], v["gate"], v["up"]), want)
    ffn.check()


def test_a_training_step_through_the_block(cuda):
    """The module with 8-bit checkpoints under HybridMuonAdamW: its three weights go to
    Muon by the reference's names, their gradients are the block's at the restored
    input, and the step moves them."""
    from morph_b200 import HybridMuonAdamW, fp8_eligible, partition
    from morph_b200.ffn import GatedFeedForward
    from morph_b200.precision import pack_activation, unpack_activation

    class Stage(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = torch.nn.LayerNorm(256, device=cuda)
            self.ffn = GatedFeedForward(256, 704, checkpoint="fp8", device=cuda)

        def forward(self, x):
            return x + self.ffn(self.norm(x))

    torch.manual_seed(3)
    stage = Stage()
    muon, adam = partition(stage)
    named = dict(stage.named_parameters())
    assert {n for n in named if fp8_eligible(n)} == {"ffn.gate.weight", "ffn.up.weight", "ffn.down.weight"}
    assert {id(p) for p in muon} == {id(named[n]) for n in named if n.startswith("ffn.")}
    x = torch.randn(3, 67, 256, device=cuda)
    target = torch.randn(3, 67, 256, device=cuda)
    opt = HybridMuonAdamW(stage, lr=1e-3, muon_lr=1e-2)
    before = {n: p.detach().clone() for n, p in named.items()}
    for _ in range(2):
        opt.zero_grad()
        out = stage(x)
        loss = (out - target).square().mean()
        loss.backward()
        normed = stage.norm(x).to(BF16)
        restored = unpack_activation(*pack_activation(normed), BF16).view(-1, 256)
        dy = (2 * (out.detach() - target) / out.numel()).to(BF16).view(-1, 256)
        want, sigmas = ref.backward(dy, restored, *(w.detach().to(BF16) for w in (
            stage.ffn.gate.weight, stage.ffn.up.weight, stage.ffn.down.weight)), "silu")
        for name, w, s in zip(("gate", "up", "down"), want[1:], sigmas(torch.finfo(BF16).eps / 2)[1:]):
            got = getattr(stage.ffn, name).weight.grad
            assert got.dtype == torch.float32
            ref.assert_close(got.to(BF16), w, s, name)
        opt.step()
    assert all(not torch.equal(before[n], p) for n, p in named.items() if n.startswith("ffn."))


def test_refusals_on_the_gpu(cuda):
    """Shapes, types and devices that do not fit raise ValueError and launch nothing."""
    from morph_b200 import ffn
    from morph_b200.precision import pack_activation, unpack_activation
    v = _inputs(4, 64, 96, BF16, cuda)
    x, gate, up, down, dy = (v[k] for k in ("x", "gate", "up", "down", "grad"))
    codes, scales = pack_activation(x)
    bad = [lambda: ffn.feed_forward(x, gate[:, :56], up, down), lambda: ffn.feed_forward(x, gate, up[:90], down),
           lambda: ffn.feed_forward(x, gate, up, down.t()), lambda: ffn.feed_forward(x, gate, up, down.half()),
           lambda: ffn.feed_forward(x.half(), gate, up, down), lambda: ffn.feed_forward(x.cpu(), gate, up, down),
           lambda: ffn.feed_forward(x, gate.cpu(), up, down), lambda: ffn.feed_forward(x[0, 0], gate, up, down),
           lambda: ffn.gated_linear(x.float(), gate.float(), up.float()), lambda: ffn.gated_linear(x[:, :0], gate[:, :0], up[:, :0]),
           lambda: ffn.gated_linear(x, gate[:0], up[:0]), lambda: ffn.gated_linear(x, gate.view(2, 48, 64), up),
           lambda: ffn.feed_forward_backward(dy[:2], x, gate, up, down),
           lambda: ffn.feed_forward_backward(dy.half(), x, gate, up, down),
           lambda: ffn.feed_forward_backward(dy, (codes, scales[:2]), gate, up, down),
           lambda: ffn.feed_forward_backward(dy, (codes.float(), scales), gate, up, down),
           lambda: ffn.feed_forward_backward(dy, (codes[:, :56], scales), gate, up, down),
           lambda: ffn.feed_forward_backward(dy, x, gate, up, down, needs=(True,)),
           lambda: ffn.gated_linear_backward(dy, x, gate, up), lambda: pack_activation(x.double()),
           lambda: pack_activation(x[:, :0]), lambda: pack_activation(x[0, 0]),
           lambda: unpack_activation(codes, scales, torch.float64), lambda: unpack_activation(codes.cpu(), scales)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()
