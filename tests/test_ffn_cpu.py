"""The feed-forward block and the activation checkpoints on a host without a GPU:
argument checks, workspace sizes, argument layouts, and the module's parameters."""
import ctypes

import pytest
import torch

from morph_b200 import _lib, ffn, partition
from morph_b200.precision import check_activation, fp8_eligible, pack_activation, unpack_activation

BF16 = torch.bfloat16


def test_argument_layouts():
    assert ctypes.sizeof(_lib.FfnArgs) == 96 and _lib.FfnArgs.x.offset == 32 and _lib.FfnArgs.ld_down.offset == 88
    assert ctypes.sizeof(_lib.FfnGrads) == 96 and _lib.FfnGrads.dx.offset == 32


def test_workspace_sizes():
    L = _lib.lib()
    assert L.mb_feed_forward_workspace_bytes(0, 64) == 0 == L.mb_gated_linear_workspace_bytes(0)
    assert L.mb_gated_linear_workspace_bytes(-1) == 0
    assert L.mb_feed_forward_workspace_bytes(3, 65) >= 3 * 72 * 2
    for tokens in (1, 100, 5000, 1 << 20):
        n = L.mb_feed_forward_backward_workspace_bytes(tokens, 4096, 11008, 0, 1)
        m = L.mb_feed_forward_backward_workspace_bytes(tokens, 4096, 11008, 1, 1)
        assert n >= tokens * 11008 * 10 and m - n >= tokens * 4096 * 2
    assert L.mb_feed_forward_backward_workspace_bytes(1 << 31, 1, 1, 0, 0) == 0
    # x, dy, dx; gate, up, down and their gradients; h
    assert L.mb_ffn_padding_bytes(5, 33, 65) >= 2 * (3 * 5 * 40 + 5 * 72 + 4 * 65 * 40 + 2 * 33 * 72)
    assert L.mb_ffn_padding_bytes(0, 33, 65) == 0


def _args(**over):
    a = dict(dtype=_lib.MB_BF16, activation=0, tokens=4, d=64, f=96, x=4096, ldx=64, gate=4096, ld_gate=64, up=4096,
             ld_up=64, down=4096, ld_down=96)
    a.update(over)
    return _lib.FfnArgs(**a)


# Refused before anything reaches a device: the pointers are never followed.
@pytest.mark.parametrize("over,status", [
    (dict(dtype=_lib.MB_F32), _lib.MB_ERR_ARG), (dict(activation=2), _lib.MB_ERR_ARG), (dict(tokens=-1), _lib.MB_ERR_ARG),
    (dict(d=0), _lib.MB_ERR_ARG), (dict(f=0), _lib.MB_ERR_ARG), (dict(tokens=1 << 31), _lib.MB_ERR_TOO_LARGE),
    (dict(x=None), _lib.MB_ERR_ARG), (dict(gate=None), _lib.MB_ERR_ARG), (dict(up=None), _lib.MB_ERR_ARG),
    (dict(ldx=56), _lib.MB_ERR_ARG), (dict(ldx=65), _lib.MB_ERR_ALIGN), (dict(ld_gate=68), _lib.MB_ERR_ALIGN),
    (dict(x=4098), _lib.MB_ERR_ALIGN), (dict(down=4104), _lib.MB_ERR_ALIGN), (dict(ld_down=88), _lib.MB_ERR_ARG)])
def test_c_entries_refuse_bad_arguments(over, status):
    L = _lib.lib()
    a = _args(**over)  # workspaces without room for padded copies: unaligned rows are refused
    need = L.mb_feed_forward_workspace_bytes(4, 96)
    assert L.mb_feed_forward(ctypes.byref(a), 4096, 64, 4096, need, None) == status
    r = _lib.FfnGrads(dy=4096, lddy=64, dx=4096, lddx=64)
    if "down" not in over and "ld_down" not in over:
        assert L.mb_gated_linear(ctypes.byref(a), 4096, 96, None, 0, None) == status
    need = L.mb_feed_forward_backward_workspace_bytes(4, 64, 96, 0, 1)
    assert L.mb_feed_forward_backward(ctypes.byref(a), ctypes.byref(r), 4096, need, None) == status


def test_c_entries_refuse_bad_outputs_and_workspaces():
    L = _lib.lib()
    a = _args()
    assert L.mb_feed_forward(None, 4096, 64, 4096, 1 << 40, None) == _lib.MB_ERR_ARG
    assert L.mb_feed_forward(ctypes.byref(a), None, 64, 4096, 1 << 40, None) == _lib.MB_ERR_ARG
    assert L.mb_feed_forward(ctypes.byref(a), 4096, 60, 4096, 1 << 40, None) == _lib.MB_ERR_ARG
    need = L.mb_feed_forward_workspace_bytes(4, 96)
    assert L.mb_feed_forward(ctypes.byref(a), 4096, 68, 4096, need, None) == _lib.MB_ERR_ALIGN
    assert L.mb_feed_forward(ctypes.byref(a), 4097, 64, 4096, 1 << 40, None) == _lib.MB_ERR_ALIGN
    assert L.mb_feed_forward(ctypes.byref(a), 4096, 64, None, 1 << 40, None) == _lib.MB_ERR_ARG
    assert L.mb_feed_forward(ctypes.byref(a), 4096, 64, 4096, need - 1, None) == _lib.MB_ERR_ARG
    assert L.mb_feed_forward(ctypes.byref(a), 4096, 64, 4096 + 16, 1 << 40, None) == _lib.MB_ERR_ALIGN
    none = _lib.FfnGrads(dy=4096, lddy=64)
    assert L.mb_feed_forward_backward(ctypes.byref(a), ctypes.byref(none), None, 0, None) == _lib.MB_OK  # nothing asked
    assert L.mb_feed_forward_backward(ctypes.byref(a), None, 4096, 1 << 40, None) == _lib.MB_ERR_ARG
    for bad in (dict(dy=None), dict(lddy=56), dict(dx=4100), dict(ld_dgate=1, dgate=4096), dict(codes=4096, scales=None)):
        r = _lib.FfnGrads(**{**dict(dy=4096, lddy=64, dx=4096, lddx=64), **bad})
        need = L.mb_feed_forward_backward_workspace_bytes(4, 64, 96, "codes" in bad, 1)
        assert L.mb_feed_forward_backward(ctypes.byref(a), ctypes.byref(r), 4096, need, None) in (
            _lib.MB_ERR_ARG, _lib.MB_ERR_ALIGN)
    r = _lib.FfnGrads(dy=4096, lddy=96, ddown=4096, ld_ddown=96)  # ddown of a block without down
    b = _args(down=None)
    assert L.mb_feed_forward_backward(ctypes.byref(b), ctypes.byref(r), 4096, 1 << 40, None) == _lib.MB_ERR_ARG
    empty = _args(tokens=0, x=None)
    assert L.mb_feed_forward(ctypes.byref(empty), None, 64, None, 0, None) == _lib.MB_OK


def test_checkpoint_entries_refuse_bad_arguments():
    L = _lib.lib()
    assert L.mb_act_pack(4096, _lib.MB_BF16, 0, 64, 64, None, None, None) == _lib.MB_OK
    for args in ((4096, 3, 2, 64, 64, 4096, 4096), (None, 2, 2, 64, 64, 4096, 4096), (4096, 2, -1, 64, 64, 4096, 4096),
                 (4096, 2, 2, 0, 64, 4096, 4096), (4096, 2, 2, 64, 63, 4096, 4096), (4096, 2, 2, 64, 64, None, 4096),
                 (4096, 2, 2, 64, 64, 4096, None)):
        assert L.mb_act_pack(*args, None) == _lib.MB_ERR_ARG
    assert L.mb_act_unpack(4096, 4096, 2, 64, 4096, 3, 64, None) == _lib.MB_ERR_ARG
    assert L.mb_act_unpack(4096, None, 2, 64, 4096, 2, 64, None) == _lib.MB_ERR_ARG


def test_python_refuses_what_is_not_on_a_gpu_or_does_not_fit():
    x = torch.zeros(3, 64, dtype=BF16)
    w = torch.zeros(96, 64, dtype=BF16)
    dn = torch.zeros(64, 96, dtype=BF16)
    for call in (lambda: ffn.feed_forward(x, w, w, dn), lambda: ffn.gated_linear(x, w, w),
                 lambda: ffn.feed_forward_backward(x, x, w, w, dn), lambda: pack_activation(x),
                 lambda: ffn.feed_forward(x, w, w, None), lambda: ffn.feed_forward(None, w, w, dn),
                 lambda: ffn.gated_linear(x.float(), w, w), lambda: ffn.gated_linear(x, w, w, activation="relu"),
                 lambda: ffn.gated_linear(x, w, w, checkpoint="fp4"), lambda: unpack_activation(x, x),
                 lambda: ffn.GatedFeedForward(8, 16, activation="tanh"),
                 lambda: ffn.GatedFeedForward(8, 16, checkpoint=None),
                 lambda: ffn.GatedFeedForward(8, 16, dtype=torch.float32)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        check_activation(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8))


def test_module_parameters():
    m = torch.nn.Module()
    m.ffn = ffn.GatedFeedForward(64, 96)
    names = dict(m.named_parameters())
    assert set(names) == {"ffn.gate.weight", "ffn.up.weight", "ffn.down.weight"}
    assert names["ffn.gate.weight"].shape == (96, 64) and names["ffn.down.weight"].shape == (64, 96)
    assert all(fp8_eligible(n) and p.dtype == torch.float32 for n, p in names.items())
    muon, adam = partition(m)
    assert len(muon) == 3 and not adam


def test_raw_stream_only_for_the_current_device(monkeypatch):
    """Another current device gives None: the callers then switch to the tensors' one."""
    monkeypatch.setattr(_lib, "_CUDA", (lambda: 1, lambda index: 70 + index))
    assert _lib.raw_stream(1) == 71 and _lib.raw_stream(0) is None
    monkeypatch.setattr(_lib, "_CUDA", (lambda: 0, lambda index: 0))
    assert _lib.raw_stream(0) == 0  # the legacy stream's handle
