"""The gated feed-forward block (SwiGLU / GEGLU) on the sm_100a tensor cores,
forward and backward, with 8-bit activation checkpoints.

    h = act(x gate^T) * (x up^T)        gated_linear
    y = h down^T                        feed_forward

``x`` is [..., d]; ``gate`` and ``up`` are [f, d] and ``down`` [d, f], as
``nn.Linear`` keeps the ``ffn.gate`` / ``ffn.up`` / ``ffn.down`` weights of
morph/model/morph_model.py:23-28. Everything is bfloat16, or everything is
float16; products accumulate in FP32, and h and the gradients of the two
projections' outputs are rounded to 16 bits once each, as the next product's
operand.

Both functions are differentiable, once and in reverse mode (a tensor with a
forward-mode tangent is refused). What they keep for the backward pass is the
block's input only, as it is (``checkpoint="x"``) or in 8 bits
(``checkpoint="fp8"``, ``precision.pack_activation``: 1 + 1/128 bytes per
element); the projections are recomputed from it. The ``*_backward`` functions
are the same backward pass for engines that replay stages themselves
(streamtrain/engine.py:165-211): they take x or its ``(codes, scales)``.

Calls run on the current stream of the tensors' device, allocate their outputs
and workspace from torch's caching allocator and never synchronise, so they can
be captured in a CUDA graph (a captured autograd backward pass, as with any torch
operator, must find no eager graph of the same leaves alive). Matrices whose rows
do not start on 16 bytes (d or f not a multiple of 8, odd views) are copied to
padded rows of the workspace by one launch before and, for outputs, one after;
transposed and broadcast ones by torch.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .precision import check_activation, pack_activation, refuse_tangents

ACTIVATIONS = {"silu": _lib.MB_ACT_SILU, "gelu_tanh": _lib.MB_ACT_GELU_TANH}
CHECKPOINTS = ("x", "fp8")
DTYPES = {torch.bfloat16: _lib.MB_BF16, torch.float16: _lib.MB_F16}
GRADS = ("dx", "dgate", "dup", "ddown")
PITCHES = ("lddx", "ld_dgate", "ld_dup", "ld_ddown")


def _activation_code(activation) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, not {activation!r}")
    return ACTIVATIONS[activation]


def _check(tensor, what, shape, like) -> None:
    if not isinstance(tensor, torch.Tensor) or tensor.shape != shape:
        raise ValueError(f"{what} must be a tensor of shape {list(shape)}")
    if tensor.dtype is not like.dtype or tensor.get_device() != like.get_device():
        raise ValueError(f"{what} is {tensor.dtype} on {tensor.device}, expected {like.dtype} on {like.device}")


def _check_weights(gate, up, down, d):
    if not isinstance(gate, torch.Tensor) or gate.dim() != 2 or not gate.is_cuda:
        raise ValueError("gate must be [f, d] on a CUDA device")
    if gate.dtype not in DTYPES:
        raise ValueError(f"the block computes in bfloat16 or float16, not {gate.dtype}")
    shape = gate.shape
    f, width = shape
    if f == 0 or d == 0:
        raise ValueError("d and f must be at least 1")
    if width != d:
        raise ValueError(f"gate must be a tensor of shape {[f, d]}")
    _check(up, "up", shape, gate)
    if down is not None:
        _check(down, "down", (d, f), gate)
    return f


def _rows(t, rows, cols):
    """(tensor, address, pitch) of a [rows, cols] tensor whose rows are contiguous and
    apart: itself, or a copy. The pitch of a single row is its length."""
    if t.is_contiguous():
        return t, t.data_ptr(), cols
    ld, inner = t.stride()
    if (inner == 1 or cols == 1) and (ld >= cols or rows <= 1):
        return t, t.data_ptr(), ld if rows > 1 else cols
    t = t.detach().contiguous()
    return t, t.data_ptr(), cols


def _workspace(nbytes, like):
    """(tensor, address): a buffer from the caching allocator, which a captured
    graph keeps for itself; none for an empty one."""
    if nbytes == 0:
        return None, None
    ws = like.new_empty(nbytes, dtype=torch.uint8)
    return ws, ws.data_ptr()


def _two_d(t):
    return t if t.dim() == 2 else t.detach().reshape(-1, t.shape[-1])


def _padding(*mats):
    """Workspace bytes for the padded copies that the library makes of the matrices
    (address, pitch, rows, columns) whose rows TMA cannot take (Padding of mb_ffn.cu)."""
    return sum((rows * (-(-cols // 8) * 8) * 2 + 255) // 256 * 256 for at, ld, rows, cols in mats
               if at and rows and (at % 16 or rows > 1 and ld % 8))


def _args(code, tokens, d, f, x, gate, up, down):
    """The C arguments, the tensors they point into, and the workspace for copies of them."""
    dtype = DTYPES[gate.dtype]
    gate, at_gate, ld_gate = _rows(gate, f, d)
    up, at_up, ld_up = _rows(up, f, d)
    at_x, ldx, at_down, ld_down = 0, 0, 0, 0
    if x is not None:
        x, at_x, ldx = _rows(x, tokens, d)
    if down is not None:
        down, at_down, ld_down = _rows(down, d, f)
    pad = 0
    if (at_gate | at_up | at_x | at_down) % 16 or (ld_gate | ld_up | ldx | ld_down) % 8:
        pad = _padding((at_x, ldx, tokens, d), (at_gate, ld_gate, f, d), (at_up, ld_up, f, d), (at_down, ld_down, d, f))
    return (_lib.FfnArgs(dtype, code, tokens, d, f, at_x, ldx, at_gate, ld_gate, at_up, ld_up, at_down, ld_down),
            (x, gate, up, down), pad)


def _input(x, gate):
    if not isinstance(x, torch.Tensor) or x.dim() == 0:
        raise ValueError("x must be a tensor [..., d]")
    if not isinstance(gate, torch.Tensor) or x.dtype is not gate.dtype or x.get_device() != gate.get_device():
        raise ValueError("x and the weights must have one dtype and one device")
    return x.shape[-1]


def _forward(x, gate, up, down, code):
    d = _input(x, gate)
    f = _check_weights(gate, up, down, d)
    index = x.get_device()
    stream = _lib.raw_stream(index)
    if stream is None:
        with torch.cuda.device(index):
            return _forward(x, gate, up, down, code)
    x2 = _two_d(x)
    tokens = x2.shape[0]
    width = f if down is None else d
    a, keep, pad = _args(code, tokens, d, f, x2, gate, up, down)
    out = x.new_empty((tokens, width))
    L = _lib.lib()
    if down is None:
        name, run, nbytes = "gated_linear", L.mb_gated_linear, L.mb_gated_linear_workspace_bytes(tokens)
    else:
        name, run, nbytes = "feed_forward", L.mb_feed_forward, L.mb_feed_forward_workspace_bytes(tokens, f)
    if width % 8:
        pad += _padding((out.data_ptr(), width, tokens, width))
    nbytes += pad
    ws, address = _workspace(nbytes, x)
    rc = run(ctypes.byref(a), out.data_ptr(), width, address, nbytes, stream)
    if rc:
        _lib.check(rc, name)
    del keep, ws
    return out if x.dim() == 2 else out.view(x.shape[:-1] + (width,))


def _backward(grad, saved, gate, up, down, code, needs):
    refuse_tangents(grad, saved, gate, up, down)
    if isinstance(saved, torch.Tensor):
        d, like, codes = _input(saved, gate), saved, None
    else:
        codes, scales = saved
        check_activation(codes, scales)
        d, like = codes.shape[-1], codes
    f = _check_weights(gate, up, down, d)
    if gate.get_device() != like.get_device():
        raise ValueError("the checkpoint and the weights are on different devices")
    _check(grad, "the output's gradient", like.shape[:-1] + (f if down is None else d,), gate)
    if len(needs) != (3 if down is None else 4):
        raise ValueError("needs names one truth value for x and each weight")
    index = gate.get_device()
    stream = _lib.raw_stream(index)
    if stream is None:
        with torch.cuda.device(index):
            return _backward(grad, saved, gate, up, down, code, needs)
    g2 = _two_d(grad)
    tokens = g2.shape[0]
    a, keep, pad = _args(code, tokens, d, f, None if codes is not None else _two_d(saved), gate, up, down)
    r = _lib.FfnGrads()
    if codes is not None:
        r.codes, r.scales = codes.data_ptr(), scales.data_ptr()
    g2, r.dy, r.lddy = _rows(g2, tokens, f if down is None else d)
    mats = [(r.dy or 0, r.lddy, *g2.shape)]  # beside those of _args
    grads = [None] * len(needs)
    for i, (need, rows, cols) in enumerate(zip(needs, (tokens, f, f, d), (d, d, d, f))):
        if need:
            grads[i] = buf = gate.new_empty((rows, cols))
            setattr(r, GRADS[i], buf.data_ptr())
            setattr(r, PITCHES[i], cols)
            mats.append((buf.data_ptr(), cols, rows, cols))
    L = _lib.lib()
    nbytes = L.mb_feed_forward_backward_workspace_bytes(tokens, d, f, codes is not None, down is not None)
    if (d | f | r.lddy) % 8 or (r.dy or 0) % 16:
        pad += _padding(*mats)
    nbytes += pad
    ws, address = _workspace(nbytes, gate)
    rc = L.mb_feed_forward_backward(ctypes.byref(a), ctypes.byref(r), address, nbytes, stream)
    if rc:
        _lib.check(rc, "feed_forward_backward")
    del keep, ws
    if grads[0] is not None and like.dim() != 2:
        grads[0] = grads[0].view(like.shape)
    return tuple(grads)


def _cast(t, dtype):
    return t if dtype is None or t is None or t.dtype is dtype else t.to(dtype)


def _block_grads(ctx, grad):
    kept = ctx.saved_tensors
    weights, rest = (kept[:3], kept[3:]) if ctx.has_down else (kept[:2], kept[2:])
    saved = rest if ctx.checkpoint == "fp8" else rest[0]
    gate, up, down = (*(_cast(w, ctx.dtype) for w in weights), None)[:3]
    grads = _backward(grad, saved, gate, up, down, ctx.code, ctx.needs_input_grad[:1 + len(weights)])
    if ctx.dtype is not None:
        types = (ctx.x_dtype, *(w.dtype for w in weights))
        grads = tuple(_cast(g, t) for g, t in zip(grads, types))
    return (*grads, *([None] * (3 if ctx.has_down else 4)))


_block_grads_once = once_differentiable(_block_grads)


class _Block(torch.autograd.Function):
    """``dtype`` is the type to compute in where the leaves have another (FP32 masters).
    What is saved of the weights is the leaves themselves: they are cast again in the
    backward pass, so that no 16-bit copy of them lives between the two."""

    @staticmethod
    def forward(ctx, x, gate, up, down, code, checkpoint, dtype):
        ctx.code, ctx.checkpoint, ctx.has_down, ctx.dtype = code, checkpoint, down is not None, dtype
        ctx.x_dtype = x.dtype
        x = _cast(x, dtype)
        y = _forward(x, *(_cast(w, dtype) for w in (gate, up, down)), code)
        kept = pack_activation(x) if checkpoint == "fp8" else (x,)
        ctx.save_for_backward(gate, up, *((down,) if ctx.has_down else ()), *kept)
        return y

    @staticmethod
    def backward(ctx, grad):
        # the wrapper that refuses a second derivative costs 30 us; only a backward pass
        # that records a graph (create_graph=True) needs it
        return _block_grads_once(ctx, grad) if torch.is_grad_enabled() else _block_grads(ctx, grad)


def _block(x, gate, up, down, activation, checkpoint, dtype=None):
    code = _activation_code(activation)
    if checkpoint not in CHECKPOINTS:
        raise ValueError(f"checkpoint must be one of {list(CHECKPOINTS)}, not {checkpoint!r}")
    leaves = (x, gate, up) if down is None else (x, gate, up, down)
    if not all([isinstance(t, torch.Tensor) for t in leaves]):
        raise ValueError("x and the weights must be tensors")
    refuse_tangents(*leaves)
    if torch.is_grad_enabled() and any([t.requires_grad for t in leaves]):
        return _Block.apply(x, gate, up, down, code, checkpoint, dtype)
    return _forward(*(_cast(t, dtype) for t in (x, gate, up, down)), code)


def gated_linear(x, gate, up, activation="silu", checkpoint="x"):
    """h = act(x gate^T) * (x up^T), [..., f], in one kernel. Differentiable;
    ``checkpoint`` says what is kept of x for the backward pass."""
    return _block(x, gate, up, None, activation, checkpoint)


def gated_linear_backward(dh, x, gate, up, activation="silu", needs=(True, True, True)):
    """(dx, dgate, dup) of ``gated_linear`` from its output's gradient ``dh``
    [..., f]. ``x`` is the input, or the ``(codes, scales)`` of its 8-bit
    checkpoint. An entry of ``needs`` that is false gives None."""
    return _backward(dh, x, gate, up, None, _activation_code(activation), needs)


def feed_forward(x, gate, up, down, activation="silu", checkpoint="x"):
    """y = (act(x gate^T) * (x up^T)) down^T, [..., d]. Differentiable;
    ``checkpoint`` says what is kept of x for the backward pass."""
    if down is None:
        raise ValueError("down must be a tensor")
    return _block(x, gate, up, down, activation, checkpoint)


def feed_forward_backward(dy, x, gate, up, down, activation="silu", needs=(True, True, True, True)):
    """(dx, dgate, dup, ddown) of ``feed_forward`` from its output's gradient
    ``dy`` [..., d]. ``x`` is the input, or the ``(codes, scales)`` of its 8-bit
    checkpoint. An entry of ``needs`` that is false gives None."""
    if down is None:
        raise ValueError("down must be a tensor")
    return _backward(dy, x, gate, up, down, _activation_code(activation), needs)


def check(device=None) -> None:
    """Wait for ``device`` (default: the current one) and raise TimeoutError if a
    block kernel there gave up a bounded wait since the last check. The results that
    it does not have are NaN, and so are the outputs made from them: an optimizer's
    finiteness gate refuses such gradients without this call."""
    with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
        _lib.check(_lib.lib().mb_ffn_status(), "feed_forward")


class GatedFeedForward(torch.nn.Module):
    """The block as a module, with the reference's parameter names (``gate.weight``,
    ``up.weight``, ``down.weight``: bias-free ``nn.Linear``, so ``muon.partition``
    gives them to Muon and ``fp8_eligible`` admits them). It computes in ``dtype``;
    FP32 masters are cast to it on the way, with gradients cast back; the backward pass
    casts them again (at d 4096, f 11008: 0.8 GB of traffic) instead of keeping 2 bytes per weight
    of each block since the forward pass."""

    def __init__(self, d, f, activation="silu", checkpoint="x", dtype=torch.bfloat16, device=None,
                 param_dtype=torch.float32):
        super().__init__()
        _activation_code(activation)
        if checkpoint not in CHECKPOINTS:
            raise ValueError(f"checkpoint must be one of {list(CHECKPOINTS)}, not {checkpoint!r}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"the block computes in bfloat16 or float16, not {dtype}")
        make = lambda i, o: torch.nn.Linear(i, o, bias=False, device=device, dtype=param_dtype)  # noqa: E731
        self.gate, self.up, self.down = make(d, f), make(d, f), make(f, d)
        self.activation, self.checkpoint, self.dtype = activation, checkpoint, dtype

    def forward(self, x):
        y = _block(x, self.gate.weight, self.up.weight, self.down.weight, self.activation, self.checkpoint, self.dtype)
        return _cast(y, x.dtype)
