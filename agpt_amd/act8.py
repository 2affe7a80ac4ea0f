"""8-bit activation checkpoints, and the weight gradients formed from them
(include/agpt_act8.h has the format). Torch CUDA tensors, current stream; no
CPU fallback.

    kept = act8.pack(x)                   # forward: a quarter of x's fp32 bytes
    dw, db = act8.wgrad(dy, kept)         # backward of a linear layer whose input was x
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _native
from .block import _check_apart, _check_cuda, _dtype, _launch, _ptr, _rows

BLOCK = 32  # columns of a row under one scale


@dataclass
class Act8:
    """A checkpoint of [T, W] activations: opaque code and scale bytes."""
    codes: torch.Tensor
    scales: torch.Tensor
    T: int
    W: int
    relu: bool

    def __post_init__(self):
        n, device = -(-self.T // 8) * 8 * self.W, self.codes.device
        for name, t, want in (("codes", self.codes, n), ("scales", self.scales, n // BLOCK)):
            if t.dtype != torch.uint8 or t.numel() != want or not t.is_contiguous() or t.device != device:
                raise ValueError(f"{name} must be {want} contiguous bytes on the codes' device")

    @property
    def device(self):
        return self.codes.device


def pack(x, relu: bool = False) -> Act8:
    """Keeps x [T, W] (fp32 or bf16, W a multiple of 32, rows may be strided)
    in 8 bits: each block of 32 columns of a row under a power-of-two scale,
    values off by at most half a step of 1/127 .. 2/127 of the block's largest.
    relu: x is a ReLU's output (what is not above zero is kept as zero, what is
    stays above it; steps of 1/255 .. 2/255)."""
    _check_cuda("x", x)
    dt, ld = _dtype("x", x), _rows("x", x)
    T, W = x.shape
    if W < BLOCK or W % BLOCK:
        raise ValueError("the width must be a multiple of 32")
    lib = _native.attn_lib()
    codes = torch.empty(lib.agpt_act8_code_bytes(T, W), device=x.device, dtype=torch.uint8)
    scales = torch.empty(lib.agpt_act8_scale_bytes(T, W), device=x.device, dtype=torch.uint8)
    _launch(x.device, lib.agpt_act8_pack, _ptr(x), ld, dt, int(relu), _ptr(codes), _ptr(scales), T, W)
    return Act8(codes, scales, T, W, bool(relu))


def unpack(kept: Act8, dtype=torch.float32, out=None):
    """The values [T, W] that a checkpoint stands for, exactly, in fp32 or bf16."""
    if out is None:
        out = torch.empty(kept.T, kept.W, device=kept.device, dtype=dtype)
    else:
        _check_cuda("out", out, kept.device)
        if out.shape != (kept.T, kept.W):
            raise ValueError("out must be shaped as the checkpoint")
        _check_apart("out", out, kept.codes, kept.scales)
    dt, ld = _dtype("out", out), _rows("out", out)
    lib = _native.attn_lib()
    _launch(kept.device, lib.agpt_act8_unpack, _ptr(kept.codes), _ptr(kept.scales), int(kept.relu), _ptr(out), ld, dt, kept.T,
            kept.W)
    return out


def _grads(dy, kept, bias):
    _check_cuda("dy", dy, kept.device)
    dt, ld = _dtype("dy", dy), _rows("dy", dy)
    T, out = dy.shape
    if T != kept.T or out < 1:
        raise ValueError("dy must have the checkpoint's rows, at least one wide")
    lib = _native.attn_lib()
    n = lib.agpt_act8_wgrad_workspace_floats(T, out, kept.W)
    ws = torch.empty(n, device=dy.device, dtype=torch.float32)
    dw = torch.empty(out, kept.W, device=dy.device, dtype=torch.float32)
    db = torch.empty(out, device=dy.device, dtype=torch.float32) if bias else None
    return lib, dt, ld, T, out, ws, n, dw, db


def wgrad(dy, kept: Act8, bias: bool = True):
    """(dw [out, in], db [out] or None), fp32: the gradients of a linear layer's
    weight and bias from dy [T, out] (fp32 or bf16, rows may be strided) and its
    checkpointed input."""
    lib, dt, ld, T, out, ws, n, dw, db = _grads(dy, kept, bias)
    _launch(dy.device, lib.agpt_act8_wgrad, _ptr(dy), ld, dt, _ptr(kept.codes), _ptr(kept.scales), int(kept.relu), _ptr(dw),
            _ptr(db), _ptr(ws), n, T, out, kept.W)
    return dw, db


def relu_wgrad(dh, h: Act8, kept: Act8, bias: bool = True):
    """The backward between a ReLU's output and the input of the linear layer in
    front of it, in one pass: (dh masked where the checkpointed output h is zero,
    dw, db). dh [T, out] is the gradient at the ReLU's output, kept the linear
    layer's checkpointed input."""
    if not h.relu or h.T != kept.T or h.device != kept.device:
        raise ValueError("h must be a checkpoint of a ReLU's outputs (relu=True) with the input's rows, on its device")
    if dh.dim() != 2 or dh.shape[1] != h.W:
        raise ValueError("dh must be shaped as h")
    lib, dt, ld, T, out, ws, n, dw, db = _grads(dh, kept, bias)
    masked = torch.empty(T, out, device=dh.device, dtype=dh.dtype)
    _launch(dh.device, lib.agpt_act8_relu_wgrad, _ptr(dh), ld, dt, _ptr(h.codes), _ptr(masked), _ptr(kept.codes),
            _ptr(kept.scales), int(kept.relu), _ptr(dw), _ptr(db), _ptr(ws), n, T, out, kept.W)
    return masked, dw, db
