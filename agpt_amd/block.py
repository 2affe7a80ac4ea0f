"""Kernels around the trie-attention path in a training step
(include/agpt_block.h): the projection epilogue (bias + RoPE, in place or with
the split, with or without a norm of queries and keys), the row norms and the
RMSProp update. Torch CUDA tensors, current stream; no CPU
fallback."""
from __future__ import annotations

import ctypes as C

import torch

from . import _native


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(t) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


# The current stream's handle and the current device by themselves: torch.cuda's
# own calls build objects around them, 3 us of a 10 us lookup of one token.
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _launch(device, fn, *args) -> None:
    """Calls fn(*args, the device's current stream) with `device` (a tensor's)
    current, and raises on its status."""
    i = device.index
    if i == _current_device():
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(i))
    if rc:
        _native.check(rc)


def _check_cuda(name: str, t, device=None) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}")


_DTYPES = {torch.float32: _native.AGPT_DTYPE_F32, torch.bfloat16: _native.AGPT_DTYPE_BF16}


def _dtype(name: str, t) -> int:
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise ValueError(f"{name} must be float32 or bfloat16")
    return dt


def _check_f32(name: str, t, n: int, device) -> None:
    if t.dtype != torch.float32 or t.numel() != n or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous float32 with {n} elements on {device}")


def _check_apart(name: str, out, *inputs) -> None:
    """Refuses an output that shares memory with an input."""
    def span(t):  # bytes from its first to behind its last element
        n = sum((s - 1) * d for s, d in zip(t.shape, t.stride())) + 1 if t.numel() else 0
        return t.data_ptr(), t.data_ptr() + n * t.element_size()
    a, b = span(out)
    for t in inputs:
        c, d = span(t)
        if a < d and c < b:
            raise ValueError(f"{name} must not overlap an input")


_MAX_WIDTH = 2**31 - 1


def _rows(name: str, t) -> int:
    """The row stride, in elements, of a 2-D tensor whose rows are contiguous
    (and whose width is an int of the C entry points)."""
    if t.dim() == 2 and t.shape[1] > _MAX_WIDTH:
        raise ValueError(f"{name} is wider than 2^31 - 1")
    if t.dim() == 2 and t.numel() == 0:
        return max(1, t.shape[1])
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{name} must be 2-D with contiguous rows that do not overlap")
    return t.stride(0) if t.shape[0] > 1 else max(1, t.shape[1])


def bias_rope_(x, bias=None, positions=None, cos_t=None, sin_t=None, n_heads: int = 1):
    """In place on x [T, D] fp32: x += bias, then (cos_t given) RoPE of each
    head at row position positions[t] (int32 [T]). Returns x."""
    if not x.is_cuda or not x.is_contiguous() or x.dim() != 2:
        raise ValueError("x must be a contiguous CUDA [T, D] tensor")
    T, D = x.shape
    if D % n_heads:
        raise ValueError("D must be a multiple of n_heads")
    seq = 0 if cos_t is None else cos_t.shape[0]
    _native.check(_native.attn_lib().agpt_bias_rope(
        _ptr(x), _ptr(bias), _ptr(positions), _ptr(cos_t), _ptr(sin_t), seq, T, n_heads, D // n_heads,
        _stream(x)))
    return x


def bias_rope_split(qkv, bias=None, positions=None, cos_t=None, sin_t=None, n_heads: int = 1):
    """qkv [T, 3D] -> contiguous (q, k, v) [T, D]: bias on all, RoPE on q, k."""
    if not qkv.is_cuda or not qkv.is_contiguous() or qkv.dim() != 2 or qkv.shape[1] % 3:
        raise ValueError("qkv must be a contiguous CUDA [T, 3D] tensor")
    T, D3 = qkv.shape
    D = D3 // 3
    if D % n_heads:
        raise ValueError("D must be a multiple of n_heads")
    q, k, v = (torch.empty(T, D, device=qkv.device, dtype=qkv.dtype) for _ in range(3))
    seq = 0 if cos_t is None else cos_t.shape[0]
    _native.check(_native.attn_lib().agpt_bias_rope_split(
        _ptr(qkv), _ptr(bias), _ptr(positions), _ptr(cos_t), _ptr(sin_t), seq, T, n_heads, D // n_heads,
        _ptr(q), _ptr(k), _ptr(v), _stream(qkv)))
    return q, k, v


def _qk_args(qkv, wq, wk, bias, positions, cos_t, sin_t, n_heads, n_kv_heads):
    """Checks what the norm's two directions share; the row's head counts and sizes."""
    _check_cuda("qkv", qkv)
    dt, ld = _dtype("qkv", qkv), _rows("qkv", qkv)
    Hk = n_heads if n_kv_heads is None else n_kv_heads
    if n_heads < 1 or Hk < 1:
        raise ValueError("n_heads and n_kv_heads must be at least 1")
    T, width = qkv.shape
    if width < 1 or width % (n_heads + 2 * Hk):
        raise ValueError("qkv's width must be a multiple of n_heads + 2 n_kv_heads")
    hd = width // (n_heads + 2 * Hk)
    device, seq = qkv.device, 0
    _check_f32("wq", wq, hd, device)
    _check_f32("wk", wk, hd, device)
    if bias is not None:
        _check_f32("bias", bias, width, device)
    if cos_t is not None:
        if sin_t is None or positions is None:
            raise ValueError("the rotation needs cos_t, sin_t and positions")
        seq = cos_t.shape[0]
        _check_f32("cos_t", cos_t, seq * hd, device)
        _check_f32("sin_t", sin_t, seq * hd, device)
        if (positions.dtype != torch.int32 or positions.shape != (T,) or positions.device != device
                or not positions.is_contiguous()):
            raise ValueError(f"positions must be a contiguous int32 [T] tensor on {device}")
    return dt, ld, T, hd, Hk, seq


def qk_norm_rope_split(qkv, wq, wk, bias=None, positions=None, cos_t=None, sin_t=None, n_heads: int = 1,
                       n_kv_heads: int | None = None, eps: float = 1e-5):
    """bias_rope_split with an RMSNorm of every query and key head in front of
    the rotation: qkv [T, (n_heads + 2 n_kv_heads) hd] (fp32 or bf16, rows may
    be strided) -> contiguous q [T, n_heads hd], k and v [T, n_kv_heads hd].
    wq, wk [hd] and bias are fp32; n_kv_heads None: as many as n_heads."""
    dt, ld, T, hd, Hk, seq = _qk_args(qkv, wq, wk, bias, positions, cos_t, sin_t, n_heads, n_kv_heads)
    q = torch.empty(T, n_heads * hd, device=qkv.device, dtype=qkv.dtype)
    k = torch.empty(T, Hk * hd, device=qkv.device, dtype=qkv.dtype)
    v = torch.empty_like(k)
    _launch(qkv.device, _native.attn_lib().agpt_qk_norm_rope_split, _ptr(qkv), ld, _ptr(bias), _ptr(wq), _ptr(wk),
            _ptr(positions), _ptr(cos_t), _ptr(sin_t), seq, T, n_heads, Hk, hd, eps, dt, _ptr(q), _ptr(k), _ptr(v))
    return q, k, v


def qk_norm_rope_split_bwd(dq, dk, dv, qkv, wq, wk, bias=None, positions=None, cos_t=None, sin_t=None,
                           n_heads: int = 1, n_kv_heads: int | None = None, eps: float = 1e-5, out=None):
    """(dqkv, dwq, dwk, dbias or None) of qk_norm_rope_split from the gradients
    of its outputs; weights' and bias' gradients are fp32 sums in a fixed order.
    cos_t None: dq and dk are gradients in front of the rotation already (as
    TrieAttention.backward returns them when it is given the tables)."""
    dt, ld, T, hd, Hk, seq = _qk_args(qkv, wq, wk, bias, positions, cos_t, sin_t, n_heads, n_kv_heads)
    for name, t, h in (("dq", dq, n_heads), ("dk", dk, Hk), ("dv", dv, Hk)):
        _check_cuda(name, t, qkv.device)
        if t.shape != (T, h * hd) or t.dtype != qkv.dtype or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [T, {h * hd}] tensor of qkv's type")
    if out is None:
        out = torch.empty(T, qkv.shape[1], device=qkv.device, dtype=qkv.dtype)
    else:
        _check_cuda("out", out, qkv.device)
        if out.shape != qkv.shape or out.dtype != qkv.dtype:
            raise ValueError("out must be shaped as qkv and of its type")
        _check_apart("out", out, dq, dk, dv, qkv)
    ld_out = _rows("out", out)
    lib = _native.attn_lib()
    n = lib.agpt_qk_norm_workspace_floats(n_heads, Hk, hd)
    ws = torch.empty(n, device=qkv.device, dtype=torch.float32)
    dwq, dwk = (torch.empty(hd, device=qkv.device, dtype=torch.float32) for _ in range(2))
    db = torch.empty(qkv.shape[1], device=qkv.device, dtype=torch.float32) if bias is not None else None
    _launch(qkv.device, lib.agpt_qk_norm_rope_split_bwd, _ptr(dq), _ptr(dk), _ptr(dv), _ptr(qkv), ld, _ptr(bias),
            _ptr(wq), _ptr(wk), _ptr(positions), _ptr(cos_t), _ptr(sin_t), seq, T, n_heads, Hk, hd, eps, dt, _ptr(out),
            ld_out, _ptr(dwq), _ptr(dwk), _ptr(db), _ptr(ws), n)
    return out, dwq, dwk, db


def rmsprop_(params, grads, sq_avg, lr: float, beta: float, eps: float = 1e-8):
    """In place: sq_avg = beta sq_avg + (1-beta) g^2; params -= lr g / (sqrt(sq_avg) + eps)."""
    for t in (params, grads, sq_avg):
        if not t.is_cuda or not t.is_contiguous():
            raise ValueError("params, grads and sq_avg must be contiguous CUDA tensors")
    n = params.numel()
    if grads.numel() != n or sq_avg.numel() != n:
        raise ValueError("params, grads and sq_avg must have the same size")
    _native.check(_native.attn_lib().agpt_rmsprop(
        _ptr(params), _ptr(grads), _ptr(sq_avg), C.c_float(lr), C.c_float(beta), C.c_float(eps), n,
        _stream(params)))


def relu_bwd(dy, h):
    """Returns (dh, db): dh = dy where h > 0 else 0 ([T, width]), db = its
    column sum [width] (fixed order), in one pass."""
    for t in (dy, h):
        if not t.is_cuda or not t.is_contiguous() or t.dim() != 2 or t.dtype != torch.float32:
            raise ValueError("dy and h must be contiguous float32 CUDA [T, width] tensors")
    if dy.shape != h.shape:
        raise ValueError("dy and h must have the same shape")
    T, W = dy.shape
    lib = _native.attn_lib()
    ws = torch.empty(lib.agpt_norm_workspace_floats(W), device=dy.device, dtype=torch.float32)
    dh = torch.empty_like(dy)
    db = torch.empty(W, device=dy.device, dtype=torch.float32)
    _native.check(lib.agpt_relu_bwd(_ptr(dy), _ptr(h), _ptr(dh), _ptr(db), _ptr(ws), ws.numel(), T, W,
                                    _stream(dy)))
    return dh, db


def norm_fwd(x, w, b=None, eps: float = 1e-5):
    """LayerNorm (b given) or RMSNorm of the rows of x [T, D]; returns
    (y, mean or None, rstd)."""
    T, D = x.shape
    y = torch.empty_like(x)
    rstd = torch.empty(T, device=x.device, dtype=torch.float32)
    mean = torch.empty(T, device=x.device, dtype=torch.float32) if b is not None else None
    _native.check(_native.attn_lib().agpt_norm_fwd(
        _ptr(x), _ptr(w), _ptr(b), _ptr(y), _ptr(mean), _ptr(rstd), T, D, C.c_float(eps), _stream(x)))
    return y, mean, rstd


def norm_bwd(dy, x, w, mean, rstd, layer: bool, dres=None):
    """Returns (dx, dw, db or None) of norm_fwd; dres [T, D] (a residual
    stream's gradient at x) is added into dx in the same pass."""
    T, D = x.shape
    if dres is not None and (not dres.is_cuda or not dres.is_contiguous() or dres.shape != x.shape):
        raise ValueError("dres must be a contiguous CUDA tensor shaped as x")
    lib = _native.attn_lib()
    ws = torch.empty(lib.agpt_norm_workspace_floats(D), device=x.device, dtype=torch.float32)
    dx = torch.empty_like(x)
    dw = torch.empty(D, device=x.device, dtype=torch.float32)
    db = torch.empty(D, device=x.device, dtype=torch.float32) if layer else None
    _native.check(lib.agpt_norm_bwd(_ptr(dy), _ptr(dres), _ptr(x), _ptr(w), _ptr(mean), _ptr(rstd), _ptr(dx), _ptr(dw),
                                    _ptr(db), _ptr(ws), ws.numel(), T, D, _stream(x)))
    return dx, dw, db
