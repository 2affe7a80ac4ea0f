"""GPU: the training step with the embedding by lookup, the norms of queries and
keys and the 8-bit checkpoints, one by one and together, against a float64 model
on the CPU (attention as in c3_reference, torch autograd; a checkpointed layer's
weight gradient from the values that its input is kept as).

Bars: loss 1e-4 relative, gradients 2e-4 of a tensor's largest |value| (fp32
through two layers against float64, the bar of the plain step's test). With
checkpoints 1e-3: an activation's fp32 error, at most 1e-5 of its block's
largest, moves at most 1e-5 * 127 of the values over a rounding border, each by
at most 2/127 of the largest; over the rows of a sum that is sqrt(1.3e-3) * 2/127
= 6e-4 of a typical entry, on top of 2e-4."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from agpt_amd import model, trie
from c3_reference import _rope, ancestor_mask
from oracle import oracle as ORC
from test_gpu_act8 import kept

pytestmark = pytest.mark.gpu


class _Keep(torch.autograd.Function):
    """x·wᵀ in float64; dw from the values that an 8-bit checkpoint of x holds."""

    @staticmethod
    def forward(ctx, x, w, relu):
        ctx.save_for_backward(x, w)
        ctx.relu = relu
        return x @ w.T

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        v = torch.from_numpy(kept(x.numpy().astype(np.float32).astype(np.float64), ctx.relu))
        return dy @ w, dy.T @ v, None


def _step_f64(cfg, flat, tr, mass, relu_masks):
    fl = torch.tensor(flat, dtype=torch.float64, requires_grad=True)
    P, off = {}, 0
    for name, shape in model.param_shapes(cfg):
        n = int(np.prod(shape))
        P[name] = fl[off:off + n].view(shape)
        off += n
    T, H, D = tr.n_nodes, cfg.n_heads, cfg.d_model
    hd = D // H
    cos_t, sin_t = (torch.tensor(t, dtype=torch.float64) for t in ORC.rope_table(cfg.max_depth, hd))
    pos = torch.from_numpy((tr.depth - 1).astype(np.int64))
    mask = ancestor_mask(tr.parent)

    def rms(x, w):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + cfg.eps) * w

    def lin(x, w, relu=False):
        return _Keep.apply(x, w, relu) if cfg.act8 else x @ w.T

    def head(x, w):
        x = x.view(T, H, hd)
        x = rms(x, w) if w is not None else x
        return _rope(x.reshape(T, D), pos, cos_t, sin_t, H, hd).reshape(T, H, hd)
    x = P["tok_emb"][torch.from_numpy(tr.token.astype(np.int64))] * cfg.emb_scale
    for l in range(cfg.n_layers):
        n1 = rms(x, P[f"n1_w{l}"])
        q = head(lin(n1, P[f"wq{l}"]) + P[f"bq{l}"], P.get(f"qn_w{l}"))
        k = head(lin(n1, P[f"wk{l}"]) + P[f"bk{l}"], P.get(f"kn_w{l}"))
        v = (lin(n1, P[f"wv{l}"]) + P[f"bv{l}"]).reshape(T, H, hd)
        s = (torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(hd)).masked_fill(~mask[None], float("-inf"))
        o = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(T, D)
        x = x + o @ P[f"wo{l}"].T + P[f"bo{l}"]
        pre = lin(rms(x, P[f"n2_w{l}"]), P[f"w1{l}"]) + P[f"b1{l}"]
        act = torch.where(relu_masks[l], pre, torch.zeros((), dtype=torch.float64))
        x = x + lin(act, P[f"w2{l}"], True) + P[f"b2{l}"]
    logp = torch.log_softmax(lin(rms(x, P["nf_w"]), P["w_out"]) + P["b_out"], -1)
    ends = np.append(np.flatnonzero(tr.radix_head)[1:], T) - 1
    tgt = torch.zeros(T, cfg.vocab, dtype=torch.float64)
    is_end = np.zeros(T, bool)
    is_end[ends] = True
    for i in range(T):
        if is_end[i]:
            a, b = tr.next_offsets[i], tr.next_offsets[i + 1]
            c = tr.next_val[a:b].astype(np.float64)
            if c.size:
                tgt[i, torch.from_numpy(tr.next_tok[a:b].astype(np.int64))] += torch.from_numpy(c / c.sum())
        else:
            tgt[i, int(tr.token[i + 1])] = 1.0
    loss = -(torch.tensor(mass, dtype=torch.float64)[:, None] * tgt * torch.log(logp.exp() + 1e-10)).sum()
    loss.backward()
    return float(loss.detach()), fl.grad.numpy()


@pytest.mark.parametrize("opts", [
    dict(embed="lookup", emb_scale=8.0), dict(qk_norm=True), dict(act8=True), dict(qk_norm=True, act8=True),
    dict(embed="lookup", emb_scale=11.5, qk_norm=True, act8=True)],
    ids=["lookup", "qk_norm", "act8", "qk_norm-act8", "all"])
def test_step_matches_float64(gpu, opts):
    tok = trie.markov_corpus(260, 2, 7, 1.1, seed=5)
    tr = trie.build_trie(tok, 10, counts=True)
    cfg = model.ModelConfig(vocab=7, d_model=64, n_heads=4, n_layers=2, d_ff=128, max_depth=10, **opts)
    m = model.TrieGPT(cfg, device=gpu, seed=3)
    if cfg.qk_norm:  # weights away from one
        P = m.params()
        with torch.no_grad():
            for l in range(cfg.n_layers):
                P[f"qn_w{l}"].mul_(torch.linspace(0.5, 1.5, 16, device=gpu))
                P[f"kn_w{l}"].mul_(torch.linspace(1.4, 0.7, 16, device=gpu))
    m.plan(tr, max_rows=400)
    assert len(m.groups) > 1
    masks = {l: [] for l in range(cfg.n_layers)}
    m.relu_hook = lambda l, h: masks[l].append((h > 0).cpu())
    flat0 = m.flat.detach().cpu().numpy().copy()
    loss = float(m.step())
    grad = m.flat.grad.detach().cpu().numpy()
    mass = np.concatenate([b.mass.cpu().numpy() for _, b in m.groups])
    want_loss, want = _step_f64(cfg, flat0, tr, mass, [torch.cat(masks[l]) for l in range(cfg.n_layers)])
    assert abs(loss - want_loss) <= 1e-4 * abs(want_loss)
    off = 0
    for name, shape in model.param_shapes(cfg):
        n = int(np.prod(shape))
        g, w = grad[off:off + n], want[off:off + n]
        off += n
        bar = 1e-3 if cfg.act8 else 2e-4
        assert np.abs(g - w).max() <= bar * max(np.abs(w).max(), 1e-6), (name, np.abs(g - w).max(), np.abs(w).max())
    # the same step again from the same weights: the same bytes
    with torch.no_grad():
        m.flat.copy_(torch.from_numpy(flat0))
    m.sq_avg.zero_()
    m.relu_hook = None
    assert float(m.step()) == loss
    m.close()


def test_checkpoints_hold_less_memory(gpu):
    """What a step keeps between forward and backward: with 8-bit checkpoints at
    least the feed-forward activations' three quarters less (T x 512 fp32 per
    layer of a 4-layer, 128-wide model)."""
    tr = trie.config_trie("C1", scale=0.002, counts=True)
    held = {}
    for bits8 in (False, True):
        m = model.TrieGPT(model.ModelConfig(act8=bits8), device=gpu, seed=1)
        m.plan(tr)
        m.step()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        lv = m.loss(m.groups[0])
        held[bits8] = torch.cuda.memory_allocated() - before
        del lv
        m.close()
    assert held[False] - held[True] >= 0.7 * 4 * 4 * 512 * tr.n_nodes


def test_mgpt_files_refuse_what_they_cannot_hold(gpu, tmp_path):
    for opts in (dict(qk_norm=True), dict(embed="lookup", emb_scale=2.0)):
        m = model.TrieGPT(model.ModelConfig(vocab=7, d_model=64, n_heads=4, n_layers=1, d_ff=64, **opts), device=gpu)
        with pytest.raises(ValueError):
            m.save(str(tmp_path / "m.mgpt"))
        with pytest.raises(ValueError):
            m.load(str(tmp_path / "m.mgpt"))
    a, b = (model.TrieGPT(model.ModelConfig(vocab=7, d_model=64, n_heads=4, n_layers=1, d_ff=64, embed=e, act8=e != "onehot"),
                          device=gpu, seed=s) for e, s in (("lookup", 1), ("onehot", 2)))
    a.save(str(tmp_path / "a.mgpt"))
    b.load(str(tmp_path / "a.mgpt"))
    assert torch.equal(a.flat, b.flat)


def test_options_refused():
    for opts in (dict(embed="table"), dict(emb_scale=2.0)):
        with pytest.raises(ValueError):
            model.TrieGPT(model.ModelConfig(**opts), device="cpu")
