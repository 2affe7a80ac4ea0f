"""Token embedding with scaling, and its gradient by sorted tokens
(include/agpt_embed.h). Torch CUDA tensors, current stream; no CPU fallback.

Tokens are int32 or int64; a token outside [0, vocab) is padding: its row of x
is zero and its row of dx counts nowhere. Sums run in a fixed order: two calls
give the same bytes.
"""
from __future__ import annotations

import torch

from . import _native
from .block import _MAX_WIDTH, _check_apart, _check_cuda, _dtype, _launch, _ptr, _rows

_BITS = {torch.int32: 32, torch.int64: 64}


def _tokens(tokens) -> int:
    _check_cuda("tokens", tokens)
    if tokens.dtype not in _BITS or tokens.dim() != 1 or not tokens.is_contiguous():
        raise ValueError("tokens must be a contiguous 1-D int32 or int64 tensor")
    return _BITS[tokens.dtype]


def embed_fwd(tokens, table, scale: float = 1.0, out=None):
    """x [T, D] = scale * table[tokens], table [V, D] fp32 or bf16 (formed in
    fp32, rounded once to the table's type)."""
    bits = _tokens(tokens)
    _check_cuda("table", table, tokens.device)
    dt = _dtype("table", table)
    if table.dim() != 2 or not table.is_contiguous():
        raise ValueError("table must be a contiguous [V, D] tensor")
    T, (V, D) = tokens.shape[0], table.shape
    if V < 1 or not 1 <= D <= _MAX_WIDTH:
        raise ValueError("the table's V and D must be at least 1, D below 2^31")
    if out is None:
        out = torch.empty(T, D, device=table.device, dtype=table.dtype)
    else:
        _check_cuda("out", out, table.device)
        if out.shape != (T, D) or out.dtype != table.dtype or not out.is_contiguous():
            raise ValueError("out must be a contiguous [T, D] tensor of the table's type")
        _check_apart("out", out, table, tokens)
    _launch(table.device, _native.attn_lib().agpt_embed_fwd, _ptr(table), _ptr(tokens), bits, scale, _ptr(out), T, V, D, dt)
    return out


class EmbedPlan:
    """The rows of a batch sorted by token, for the gradient of every pass over
    it: hold one where the tokens stay the same from step to step (the batches
    of a trie), as TrieAttention.plan is held."""

    def __init__(self, tokens, vocab: int):
        bits = _tokens(tokens)
        self.T, self.vocab, self.device = tokens.shape[0], int(vocab), tokens.device
        lib = _native.attn_lib()
        if self.vocab < 1:
            raise ValueError("vocab must be at least 1")
        self.rows = torch.empty(lib.agpt_embed_plan_ints(self.T, self.vocab), device=self.device, dtype=torch.int32)
        n = lib.agpt_embed_plan_workspace_bytes(self.T, self.vocab)
        ws = torch.empty(n, device=self.device, dtype=torch.uint8)
        _launch(self.device, lib.agpt_embed_plan, _ptr(tokens), bits, self.T, self.vocab, _ptr(self.rows), _ptr(ws), n)


def embed_bwd(dx, tokens, vocab: int | None = None, scale: float = 1.0, out=None):
    """d_table [V, D] fp32 = scale * the sum of dx's rows by token. tokens: the
    batch's tokens (sorted in this call; vocab needed) or its EmbedPlan. dx
    [T, D] fp32 or bf16; rows may be strided."""
    plan = tokens if isinstance(tokens, EmbedPlan) else None
    if plan is None:
        bits = _tokens(tokens)
        if vocab is None or vocab < 1:
            raise ValueError("vocab, at least 1, is needed with tokens that are not planned")
        n_rows, device = tokens.shape[0], tokens.device
    else:
        if vocab is not None and vocab != plan.vocab:
            raise ValueError("the plan has another vocabulary")
        vocab, n_rows, device = plan.vocab, plan.T, plan.device
    _check_cuda("dx", dx, device)
    dt, ld = _dtype("dx", dx), _rows("dx", dx)
    T, D = dx.shape
    if T != n_rows or D < 1:
        raise ValueError("dx must have one row per token, at least one wide")
    if out is None:
        out = torch.empty(vocab, D, device=device, dtype=torch.float32)
    else:
        _check_cuda("out", out, device)
        if out.shape != (vocab, D) or out.dtype != torch.float32 or not out.is_contiguous():
            raise ValueError("out must be a contiguous float32 [vocab, D] tensor")
        _check_apart("out", out, dx, plan.rows if plan is not None else tokens)
    lib = _native.attn_lib()
    if plan is None:
        n = lib.agpt_embed_bwd_tokens_workspace_bytes(T, vocab, D)
        ws = torch.empty(n, device=device, dtype=torch.uint8)
        _launch(device, lib.agpt_embed_bwd_tokens, _ptr(dx), ld, _ptr(tokens), bits, scale, _ptr(out), _ptr(ws), n, T, vocab,
                D, dt)
        return out
    n = lib.agpt_embed_bwd_workspace_floats(T, D)
    ws = torch.empty(n, device=device, dtype=torch.float32)
    _launch(device, lib.agpt_embed_bwd, _ptr(dx), ld, _ptr(plan.rows), scale, _ptr(out), _ptr(ws), n, T, vocab, D, dt)
    return out
