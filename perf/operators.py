"""Measured cases of the gated feed-forward block and its 8-bit activation checkpoints.

Four operators:

* ``checkpoint``: an activation saved in 8 bits and restored (E4M3 codes, one
  power-of-two scale per 128 features of a row);
* ``gated``: h = act(x gate^T) * (x up^T);
* ``forward``: the whole block, y = h down^T, from one token to long batches;
* ``backward``: the block's gradients from the 8-bit checkpoint (or from x
  itself), alone as a layer-replaying engine runs it, or with the forward pass
  before it as one autograd training step (``step``).

``run`` computes the plain form in 32 bits where ``own`` is false and makes the
framework's calls where it is true; ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

BLOCK = 128  # features per checkpoint scale
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

# The cost of the largest listed case (feed-forward work, tokens * d * f * 16)
# and the widest checkpoint (elements): no drawn case goes beyond them.
MAX_TDF = 4096 * 4096 * 11008 * 16
MAX_ELEMENTS = 32768 * 4096


def listed():
    return [
        # a decode batch's residual rows, odd row count: launch latency counts
        dict(name="checkpoint-37x1024-fp16", op="checkpoint", tokens=37, d=1024, dtype="fp16"),
        # an FP32 stage boundary whose width is no multiple of the scale block
        dict(name="checkpoint-8191x1000-fp32", op="checkpoint", tokens=8191, d=1000, dtype="fp32"),
        # one layer boundary of a long training batch
        dict(name="checkpoint-32768x4096-bf16", op="checkpoint", tokens=32768, d=4096, dtype="bf16"),
        # the fused projections alone, as a caller with its own output projection uses them
        dict(name="gated-5x2048x5504-bf16", op="gated", tokens=5, d=2048, f=5504, dtype="bf16", act="silu"),
        dict(name="gated-1021x2048x5504-fp16-gelu", op="gated", tokens=1021, d=2048, f=5504, dtype="fp16",
             act="gelu_tanh"),
        # generation, one token through the 7B-shaped block: weight streaming
        dict(name="forward-1x4096x11008-bf16", op="forward", tokens=1, d=4096, f=11008, dtype="bf16", act="silu"),
        # a small model's decode batch: the weights fit the L2 cache
        dict(name="forward-16x1024x2816-fp16", op="forward", tokens=16, d=1024, f=2816, dtype="fp16", act="silu"),
        # a short prompt, ragged, between weight-bound and compute-bound
        dict(name="forward-130x4096x11008-bf16", op="forward", tokens=130, d=4096, f=11008, dtype="bf16",
             act="silu"),
        # a training microbatch's forward pass
        dict(name="forward-8192x4096x11008-bf16", op="forward", tokens=8192, d=4096, f=11008, dtype="bf16",
             act="silu"),
        # replay of one stage of a small model from x itself
        dict(name="backward-777x1024x2816-fp16", op="backward", tokens=777, d=1024, f=2816, dtype="fp16",
             act="gelu_tanh", saved="x", step=False),
        # replay of one 7B-shaped stage from its 8-bit boundary
        dict(name="backward-4096x4096x11008-bf16-fp8", op="backward", tokens=4096, d=4096, f=11008, dtype="bf16",
             act="silu", saved="fp8", step=False),
        # one autograd training step with the checkpoint kept in 8 bits
        dict(name="step-2048x2048x5504-bf16-fp8", op="backward", tokens=2048, d=2048, f=5504, dtype="bf16",
             act="silu", saved="fp8", step=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A feature width: a multiple of 8 mostly, now and then any number."""
    w = _log_int(rng, lo, hi)
    return w if rng.random() < 0.2 else max(8, w // 8 * 8)


def draw(rng):
    op = rng.choice(["checkpoint", "gated", "forward", "forward", "backward", "backward"])
    if op == "checkpoint":
        d = _width(rng, 256, 4096)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        top = MAX_ELEMENTS * 2 // BYTES[dtype] // d
        return dict(op=op, tokens=_log_int(rng, 32, min(32768, top)), d=d, dtype=dtype)
    d = _width(rng, 512, 4096)
    f = _width(rng, 1024, 11008)
    step = op == "backward" and rng.random() < 0.5
    per_token = d * f * (22 if step else {"gated": 4, "forward": 6, "backward": 16}[op])
    top = min(8192, MAX_TDF // per_token)
    case = dict(op=op, tokens=_log_int(rng, 1, top), d=d, f=f, dtype=rng.choice(["bf16", "fp16"]),
                act=rng.choice(["silu", "silu", "gelu_tanh"]))
    if op == "backward":
        case.update(saved=rng.choice(["fp8", "fp8", "x"]), step=step)
    return case


# ------------------------------------------------------------- inputs --

def _randn(gen, shape, std, dtype):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _activation(gen, tokens, d, dtype):
    """Residual-stream values: unit scale, with a few channels far above it."""
    channel = torch.ones(d, device="cuda")
    channel[torch.randint(0, d, (max(1, d // 256),), generator=gen, device="cuda")] = 12.0
    return (torch.randn((tokens, d), generator=gen, device="cuda") * channel).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    tokens, d = case["tokens"], case["d"]
    state = dict(case=case, x=_activation(gen, tokens, d, dtype))
    if case["op"] == "checkpoint":
        return state
    f = case["f"]
    state["gate"] = _randn(gen, (f, d), d ** -0.5, dtype)
    state["up"] = _randn(gen, (f, d), d ** -0.5, dtype)
    if case["op"] == "gated":
        return state
    state["down"] = _randn(gen, (d, f), f ** -0.5, dtype)
    if case["op"] == "forward":
        return state
    state["dy"] = _randn(gen, (tokens, d), 0.25, dtype)
    if case["step"]:
        for name in ("x", "gate", "up", "down"):
            state[name].requires_grad_(True)
    elif case["saved"] == "fp8":
        # the forward pass left the 8-bit checkpoint behind; x itself is gone
        state["codes"], state["scales"] = _encode_table(state.pop("x"))
    return state


# ------------------------------------- the checkpoint's bytes, for `prepare` --

def _e4m3_magnitudes(device):
    """The 127 finite magnitudes of E4M3FN in code order: code = 8 e + m."""
    values = []
    for code in range(127):
        e, m = code >> 3, code & 7
        values.append(m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return torch.tensor(values, dtype=torch.float64, device=device)


def _encode_table(x):
    """Codes (uint8) and biased block exponents (uint8) of finite rows x, by
    search in the table of E4M3 values."""
    tokens, d = x.shape
    blocks = -(-d // BLOCK)
    table = _e4m3_magnitudes(x.device)
    codes = torch.empty((tokens, d), dtype=torch.uint8, device=x.device)
    scales = torch.empty((tokens, blocks), dtype=torch.uint8, device=x.device)
    for lo in range(0, tokens, 4096):  # bounds the 64-bit temporaries
        part = x[lo:lo + 4096].detach().double()
        padded = torch.zeros((part.shape[0], blocks * BLOCK), dtype=torch.float64, device=x.device)
        padded[:, :d] = part
        v = padded.view(-1, blocks, BLOCK)
        amax = v.abs().amax(-1)
        s = torch.floor(torch.log2(amax.clamp_min(1e-300))) - 8
        s = torch.where(amax * torch.exp2(-s) < 256, s - 1, s)   # log2 rounded up at a power of two
        s = torch.where(amax * torch.exp2(-s) > 448, s + 1, s)
        s = torch.where(amax == 0, torch.zeros_like(s), s).clamp(-127, 127)
        q = (v * torch.exp2(-s)[..., None]).reshape(part.shape[0], -1)[:, :d].contiguous()
        mag = q.abs()
        hi = torch.searchsorted(table, mag).clamp(max=126)
        low = (hi - 1).clamp_min(0)
        below, above = mag - table[low], table[hi] - mag
        pick_low = (below < above) | ((below == above) & (low % 2 == 0))
        code = torch.where(pick_low, low, hi)
        codes[lo:lo + 4096] = (code + 128 * torch.signbit(q)).to(torch.uint8)
        scales[lo:lo + 4096] = (s + 127).to(torch.uint8)
    return codes, scales


def _decode(codes, scales, dtype):
    """The values that codes and block exponents stand for, in `dtype`."""
    table = _e4m3_magnitudes(codes.device).to(dtype)
    table = torch.cat([table, table.new_full((1,), math.nan)])
    c = codes.int()
    value = table[c & 127] * (1 - 2 * (c >> 7)).to(dtype)
    scale = torch.exp2((scales.int() - 127).to(dtype)).repeat_interleave(BLOCK, dim=1)[:, :codes.shape[1]]
    return value * scale


# --------------------------------------------------------- plain form, 32 bits --

def _plain_roundtrip(x):
    """x quantised and restored, in FP32, by arithmetic on its exponents."""
    v = x.detach().float()
    tokens, d = v.shape
    blocks = -(-d // BLOCK)
    pad = blocks * BLOCK - d
    if pad:
        v = torch.cat([v, v.new_zeros(tokens, pad)], dim=1)
    v = v.view(tokens, blocks, BLOCK)
    mant, expo = torch.frexp(v.abs().amax(-1, keepdim=True))      # mant in [0.5, 1)
    s = torch.where(mant <= 0.875, expo - 9, expo - 8)
    s = torch.where(mant == 0, torch.zeros_like(s), s).clamp(-127, 127)
    q = torch.ldexp(v, -s)
    step = torch.ldexp(torch.ones_like(q), (torch.frexp(q)[1] - 1).clamp_min(-6) - 3)
    q = torch.round(q / step) * step                              # half to even
    return torch.ldexp(q, s).view(tokens, -1)[:, :d]


def _plain_z(g, act):
    """act(g) = g * sigmoid(z): z and dz/dg."""
    if act == "silu":
        return g, torch.ones_like(g)
    c = 2.0 * math.sqrt(2.0 / math.pi)
    return c * (g + 0.044715 * g * g * g), c * (1.0 + 3 * 0.044715 * g * g)


def _plain_gated(x, gate, up, act):
    g, u = x @ gate.t(), x @ up.t()
    z, _ = _plain_z(g, act)
    return g / (1.0 + torch.exp(-z)) * u


def _plain_backward(dy, x, gate, up, down, act):
    g, u = x @ gate.t(), x @ up.t()
    z, dz = _plain_z(g, act)
    s = 1.0 / (1.0 + torch.exp(-z))
    a = g * s
    dh = dy @ down
    dg = dh * u * (s + a * (1.0 - s) * dz)
    du = dh * a
    return dg @ gate + du @ up, dg.t() @ x, du.t() @ x, dy.t() @ (a * u)


def _run_plain(state):
    case = state["case"]
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "checkpoint":
        return _plain_roundtrip(state["x"]).to(dtype)
    gate, up = state["gate"].detach().float(), state["up"].detach().float()
    if op == "gated":
        return _plain_gated(state["x"].float(), gate, up, case["act"]).to(dtype)
    down = state["down"].detach().float()
    if op == "forward":
        return (_plain_gated(state["x"].float(), gate, up, case["act"]) @ down.t()).to(dtype)
    if not case["step"]:
        saved = _decode(state["codes"], state["scales"], torch.float32) if case["saved"] == "fp8" else state["x"].float()
        return tuple(t.to(dtype) for t in _plain_backward(state["dy"].float(), saved, gate, up, down, case["act"]))
    x = state["x"].detach()
    y = (_plain_gated(x.float(), gate, up, case["act"]) @ down.t()).to(dtype)
    saved = _plain_roundtrip(x) if case["saved"] == "fp8" else x.float()
    return (y,) + tuple(t.to(dtype) for t in _plain_backward(state["dy"].float(), saved, gate, up, down, case["act"]))


# ------------------------------------------------------- the framework's calls --

def _run_own(state):
    from morph_b200 import ffn, precision
    case = state["case"]
    op = case["op"]
    if op == "checkpoint":
        codes, scales = precision.pack_activation(state["x"])
        return precision.unpack_activation(codes, scales, state["x"].dtype)
    if op == "gated":
        return ffn.gated_linear(state["x"], state["gate"], state["up"], activation=case["act"])
    if op == "forward":
        return ffn.feed_forward(state["x"], state["gate"], state["up"], state["down"], activation=case["act"])
    if not case["step"]:
        saved = (state["codes"], state["scales"]) if case["saved"] == "fp8" else state["x"]
        return ffn.feed_forward_backward(state["dy"], saved, state["gate"], state["up"], state["down"],
                                         activation=case["act"])
    leaves = (state["x"], state["gate"], state["up"], state["down"])
    y = ffn.feed_forward(*leaves, activation=case["act"], checkpoint=case["saved"])
    return (y.detach(),) + tuple(torch.autograd.grad(y, leaves, state["dy"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------- work --

def work(case):
    tokens, d, op = case["tokens"], case["d"], case["op"]
    size = BYTES[case["dtype"]]
    blocks = -(-d // BLOCK)
    packed = tokens * (d + blocks)
    if op == "checkpoint":
        # save: read x, write the checkpoint; restore: read it, write the values
        return {"bytes": 2 * (tokens * d * size + packed), "flops": 4 * tokens * d}
    f = case["f"]
    if op == "gated":
        return {"bytes": size * (tokens * d + 2 * d * f + tokens * f), "flops": 4 * tokens * d * f}
    if op == "forward":
        return {"bytes": size * (2 * tokens * d + 3 * d * f), "flops": 6 * tokens * d * f}
    saved = packed if case["saved"] == "fp8" else tokens * d * size
    backward = saved + size * (2 * tokens * d + 6 * d * f)
    if not case["step"]:
        return {"bytes": backward, "flops": 16 * tokens * d * f}
    # step: x in, y out, the checkpoint written and read, then the gradients
    written = saved if case["saved"] == "fp8" else 0
    return {"bytes": backward + written + size * 2 * tokens * d, "flops": 22 * tokens * d * f}


# ------------------------------------------------------- definition, 64 bits --

def _exact_act(g, act):
    """act(g) and act'(g), each from the activation's own definition."""
    if act == "silu":
        sig = torch.sigmoid(g)
        return g * sig, sig * (1 + g * (1 - sig))
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g ** 2)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "checkpoint":
        return _decode(*_encode_table(state["x"]), torch.float64)
    gate, up = state["gate"].detach().double(), state["up"].detach().double()
    y, saved = None, None
    if "x" in state:
        saved = state["x"].detach().double()
        value, _ = _exact_act(torch.matmul(saved, gate.T), case["act"])
        value *= torch.matmul(saved, up.T)
        if op == "gated":
            return value
        y = torch.matmul(value, state["down"].detach().double().T)
        if op == "forward":
            return y
    if case["saved"] == "fp8":
        pair = _encode_table(state["x"]) if case["step"] else (state["codes"], state["scales"])
        saved = _decode(*pair, torch.float64)
    down, dy = state["down"].detach().double(), state["dy"].double()
    g, u = torch.matmul(saved, gate.T), torch.matmul(saved, up.T)
    value, slope = _exact_act(g, case["act"])
    ddown = torch.matmul(dy.T, value * u)
    dh = torch.matmul(dy, down)
    dgate_in, dup_in = dh * u * slope, dh * value
    grads = (torch.matmul(dgate_in, gate) + torch.matmul(dup_in, up), torch.matmul(dgate_in.T, saved),
             torch.matmul(dup_in.T, saved), ddown)
    return (y,) + grads if case["step"] else grads
