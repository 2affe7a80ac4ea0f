"""Operators of the training step that are timed against their plain forms.

Kinds of case, each one pass through the public entry points:
  embed_fwd   rows of the embedding table for a batch of tokens, scaled
  embed_bwd   the table's gradient: each token's rows summed
  qk_fwd      projection epilogue: bias, norm of every query and key head, position rotation, split
  qk_bwd      its gradient, with those of the norm weights and the bias
  act8_round  activations into an 8-bit checkpoint and back
  act8_linear a linear layer's input kept in 8 bits, and the weight and bias gradient from it
  act8_ffn    the two linear layers of a feed-forward block kept in 8 bits, and their backward's
              weight gradients with the ReLU's mask

An 8-bit checkpoint holds blocks of 32 consecutive values of a row under one scale that is a power of
two. A signed block has the smallest scale s with max |x| <= 127 s and codes 128 + rint(x / s); a block
of a ReLU's outputs has the smallest s with max x <= 255 s and codes that are 0 exactly where x <= 0.

Sizes are the character model's (vocabulary 65, d_model 128 as 8 heads x 16, feed-forward 512, depth 32,
batches of 2^20 node-tokens) and generic ones: a vocabulary of 50,000, grouped heads of 128, widths to 1024.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
DEV = "cuda"
EPS = 1e-5
GROUP = 32


def listed() -> list[dict]:
    return [
        # One token of the character model: latency of a lookup.
        dict(name="embed_fwd_token", op="embed_fwd", T=1, V=65, D=128, dtype="f32", pad=False, scale=11.0),
        # A long batch over a word vocabulary, bf16 table, rows of padding (-1) among the tokens.
        dict(name="embed_fwd_words", op="embed_fwd", T=65_537, V=50_000, D=1024, dtype="bf16", pad=True, scale=32.0),
        # The character model's full batch: 65 tokens, each with thousands of rows.
        dict(name="embed_bwd_chars", op="embed_bwd", T=1 << 20, V=65, D=128, dtype="f32", pad=False, scale=11.0),
        # A batch over a word vocabulary: most rows of the gradient are zero or one row's.
        dict(name="embed_bwd_words", op="embed_bwd", T=16_384, V=50_000, D=1024, dtype="bf16", pad=True, scale=32.0),
        # One token through the epilogue.
        dict(name="qk_fwd_token", op="qk_fwd", T=1, H=8, Hk=8, hd=16, seq=32, dtype="f32", bias=True),
        # The character model's full batch, both directions.
        dict(name="qk_fwd_chars", op="qk_fwd", T=1 << 20, H=8, Hk=8, hd=16, seq=32, dtype="f32", bias=True),
        dict(name="qk_bwd_chars", op="qk_bwd", T=1 << 20, H=8, Hk=8, hd=16, seq=32, dtype="f32", bias=True),
        # Grouped heads of 128 in bf16, an odd number of rows, no bias.
        dict(name="qk_bwd_grouped", op="qk_bwd", T=32_769, H=32, Hk=8, hd=128, seq=4096, dtype="bf16", bias=False),
        # Feed-forward activations into a checkpoint and back.
        dict(name="act8_round_ffn", op="act8_round", T=300_001, I=512, dtype="f32", relu=True),
        # One small subtree's rows through a square projection: latency.
        dict(name="act8_linear_subtree", op="act8_linear", T=181, I=128, O=128, dtype="f32", relu=False),
        # A wide layer in bf16, odd sizes.
        dict(name="act8_linear_wide", op="act8_linear", T=65_537, I=1024, O=1000, dtype="bf16", relu=True),
        # The character model's feed-forward block over its full batch.
        dict(name="act8_ffn_chars", op="act8_ffn", T=1 << 20, I=128, F=512, dtype="f32"),
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng) -> dict:
    op = rng.choice(["embed_fwd", "embed_bwd", "qk_fwd", "qk_bwd", "act8_round", "act8_linear", "act8_ffn"])
    dtype = rng.choice(["f32", "bf16"])
    if op.startswith("embed"):
        D = _log(rng, 16, 1024)
        if rng.random() < 0.6:
            D = max(16, D // 16 * 16)
        V = _log(rng, 30, 50_000)
        T = _log(rng, 1, min(1 << 20, (1 << 27) // D))
        return dict(op=op, T=T, V=V, D=D, dtype=dtype, pad=rng.random() < 0.3, scale=round(math.sqrt(D), 2))
    if op.startswith("qk"):
        hd = rng.choice([16, 32, 64, 128, 24, 80, 96, 256])
        Hk = rng.choice([1, 2, 3, 4, 8])
        H = Hk * rng.choice([1, 1, 2, 4])
        T = _log(rng, 1, min(1 << 20, (1 << 20) * 384 // ((H + 2 * Hk) * hd)))
        return dict(op=op, T=T, H=H, Hk=Hk, hd=hd, seq=_log(rng, 16, 4096), dtype=dtype, bias=rng.random() < 0.5)
    I = GROUP * _log(rng, 1, 32)
    if op == "act8_round":
        return dict(op=op, T=_log(rng, 1, min(1 << 20, (1 << 28) // I)), I=I, dtype=dtype, relu=rng.random() < 0.5)
    if op == "act8_linear":
        O = _log(rng, 17, 1024)
        if rng.random() < 0.6:
            O = max(32, O // 32 * 32)
        T = _log(rng, 1, min(1 << 20, (1 << 36) // (I * O)))
        return dict(op=op, T=T, I=I, O=O, dtype=dtype, relu=rng.random() < 0.5)
    I = GROUP * _log(rng, 1, 16)
    F = 4 * I if I <= 128 else 2 * I
    return dict(op=op, T=_log(rng, 1, min(1 << 20, (1 << 35) // (I * F))), I=I, F=F, dtype=dtype)


# ---- inputs ----------------------------------------------------------------

def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def _tokens(gen, case):
    """Token ids with frequencies falling as 1 / (rank + 2), ranks scattered over the ids; -1 where padded."""
    T, V = case["T"], case["V"]
    w = 1.0 / (torch.arange(V, device=DEV, dtype=torch.float64) + 2.0)
    w = w[torch.randperm(V, generator=gen, device=DEV)]
    u = torch.rand(T, generator=gen, device=DEV, dtype=torch.float64) * w.sum()
    tok = torch.searchsorted(torch.cumsum(w, 0), u).clamp_(max=V - 1)
    if case["pad"]:
        tok[torch.rand(T, generator=gen, device=DEV) < 0.05] = -1
    return tok


def _tables(seq, hd):
    """cos and sin of pos / 10000^(2i/hd), each in columns 2i and 2i+1."""
    pos = torch.arange(seq, device=DEV, dtype=torch.float64)[:, None]
    inv = 10000.0 ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
    a = (pos * inv).repeat_interleave(2, dim=1)
    return a.cos().float(), a.sin().float()


def _activations(gen, T, W, dtype, relu):
    """Rows of a norm's output, with a few columns larger than the others; clipped at zero for a ReLU's."""
    big = 1.0 + 4.0 * (torch.rand(W, generator=gen, device=DEV) < 0.05)
    x = torch.randn(T, W, generator=gen, device=DEV) * big
    return (x.clamp_(min=0) if relu else x).to(dtype)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt, T = DTYPES[case["dtype"]], case["T"]
    s = dict(case)
    if case["op"].startswith("embed"):
        s["tokens"] = _tokens(gen, case)
        if case["op"] == "embed_fwd":
            s["table"] = _normal(gen, (case["V"], case["D"]), dt, 0.02)
        else:
            s["dx"] = _normal(gen, (T, case["D"]), dt, 1e-3)
    elif case["op"].startswith("qk"):
        H, Hk, hd = case["H"], case["Hk"], case["hd"]
        C = (H + 2 * Hk) * hd
        s["qkv"] = _normal(gen, (T, C), dt)
        s["b"] = _normal(gen, (C,), torch.float32, 0.1) if case["bias"] else None
        s["wq"], s["wk"] = (1.0 + _normal(gen, (hd,), torch.float32, 0.1) for _ in range(2))
        s["pos"] = torch.randint(0, case["seq"], (T,), generator=gen, device=DEV, dtype=torch.int32)
        s["cos"], s["sin"] = _tables(case["seq"], hd)
        if case["op"] == "qk_bwd":
            s["dq"] = _normal(gen, (T, H * hd), dt, 1e-2)
            s["dk"], s["dv"] = (_normal(gen, (T, Hk * hd), dt, 1e-2) for _ in range(2))
    elif case["op"] == "act8_ffn":
        s["x"] = _activations(gen, T, case["I"], dt, False)
        s["h"] = _activations(gen, T, case["F"], dt, True)
        s["dy"] = _normal(gen, (T, case["I"]), dt, 1e-3)
        s["dh"] = _normal(gen, (T, case["F"]), dt, 1e-3)
    else:
        s["x"] = _activations(gen, T, case["I"], dt, case["relu"])
        if case["op"] == "act8_linear":
            s["dy"] = _normal(gen, (T, case["O"]), dt, 1e-3)
    return s


# ---- the plain forms: elementary operations in 32 bits, rounded once --------

def _embed_fwd(s):
    tok, E = s["tokens"], s["table"].float()
    x = E[tok.clamp(0, s["V"] - 1)] * s["scale"]
    return (x * ((tok >= 0) & (tok < s["V"]))[:, None]).to(s["table"].dtype)


def _embed_bwd(s):
    tok, V, dx = s["tokens"], s["V"], s["dx"]
    if V > 1024:
        # 64 bits: a frequent token's sum runs over many thousands of rows
        dE = torch.zeros(V + 1, s["D"], device=DEV, dtype=torch.float64)
        dE.index_add_(0, torch.where((tok >= 0) & (tok < V), tok, V), dx.double())
        return (dE[:V] * s["scale"]).float()
    # few tokens with many rows each: a product with the comparison's zeros and ones, in 64 parts of the rows
    hot = (tok[:, None] == torch.arange(V, device=DEV)).float()
    n = tok.shape[0] // 64 * 64
    x = dx.float()
    dE = hot[n:].t() @ x[n:]
    if n:
        dE = dE + torch.bmm(hot[:n].view(64, n // 64, V).transpose(1, 2), x[:n].view(64, n // 64, -1)).sum(0)
    return dE * s["scale"]


def _rotate(y, c, s):
    y0, y1 = y[..., 0::2], y[..., 1::2]
    return torch.stack((y0 * c - y1 * s, y0 * s + y1 * c), dim=-1).flatten(-2)


def _qk_parts(s):
    """u [T, heads, hd] with the bias, the norms' weights by head, cos and sin [T, 1, hd / 2]."""
    T, H, Hk, hd = s["T"], s["H"], s["Hk"], s["hd"]
    u = s["qkv"].float()
    if s["b"] is not None:
        u = u + s["b"]
    u = u.view(T, H + 2 * Hk, hd)
    w = torch.cat((s["wq"].expand(H, hd), s["wk"].expand(Hk, hd)))
    p = s["pos"].long()
    return u, w, s["cos"][p][:, None, 0::2], s["sin"][p][:, None, 0::2]


def _qk_fwd(s):
    T, H, Hk, dt = s["T"], s["H"], s["Hk"], s["qkv"].dtype
    u, w, c, sn = _qk_parts(s)
    n = u[:, :H + Hk]
    r = 1.0 / torch.sqrt((n * n).mean(-1, keepdim=True) + EPS)
    z = _rotate(n * r * w, c, sn)
    return [t.reshape(T, -1).to(dt) for t in (z[:, :H], z[:, H:], u[:, H + Hk:])]


def _qk_bwd(s):
    T, H, Hk, hd, dt = s["T"], s["H"], s["Hk"], s["hd"], s["qkv"].dtype
    u, w, c, sn = _qk_parts(s)
    n = u[:, :H + Hk]
    g = torch.cat((s["dq"].float().view(T, H, hd), s["dk"].float().view(T, Hk, hd)), dim=1)
    g = _rotate(g, c, -sn)
    r = 1.0 / torch.sqrt((n * n).mean(-1, keepdim=True) + EPS)
    y = n * r
    gy = g * y
    h = g * w
    d = r * (h - y * (h * y).mean(-1, keepdim=True))
    d = torch.cat((d, s["dv"].float().view(T, Hk, hd)), dim=1).view(T, -1)
    out = [d.to(dt), gy[:, :H].sum((0, 1)), gy[:, H:].sum((0, 1))]
    return out + [d.sum(0)] if s["b"] is not None else out


def _kept(x, relu):
    """The values that an 8-bit checkpoint of x stands for."""
    top = 255.0 if relu else 127.0
    g = x.float().view(x.shape[0], -1, GROUP)
    m, e = torch.frexp((g.clamp(min=0.0) if relu else g.abs()).amax(-1, keepdim=True))  # amax = m 2^e, m in [0.5, 1)
    bits = 8 if relu else 7
    e = (e - bits + (m > top / 2 ** bits)).clamp(min=-126)
    s = torch.ldexp(torch.ones_like(m), e)
    c = torch.round(g / s)  # g / s is exact
    c = torch.where(g > 0, c.clamp(1.0, 255.0), torch.zeros_like(c)) if relu else c
    return (c * s).view(x.shape)


def _act8_linear(s):
    dy = s["dy"].float()
    return [dy.t() @ _kept(s["x"], s["relu"]), dy.sum(0)]


def _act8_ffn(s):
    h = _kept(s["h"], True)
    dy = s["dy"].float()
    dh = torch.where(h > 0, s["dh"].float(), 0.0)
    return [dy.t() @ h, dy.sum(0), dh.to(s["dh"].dtype), dh.t() @ _kept(s["x"], False), dh.sum(0)]


def run(state: dict):
    op = state["op"]
    if own:
        return _own(state)
    if op == "embed_fwd":
        return _embed_fwd(state)
    if op == "embed_bwd":
        return _embed_bwd(state)
    if op == "qk_fwd":
        return _qk_fwd(state)
    if op == "qk_bwd":
        return _qk_bwd(state)
    if op == "act8_round":
        return _kept(state["x"], state["relu"]).to(state["x"].dtype)
    return _act8_linear(state) if op == "act8_linear" else _act8_ffn(state)


def _own(s):
    """The same passes by the framework's entry points."""
    from agpt_amd import act8, block, embed

    op = s["op"]
    if op == "embed_fwd":
        return embed.embed_fwd(s["tokens"], s["table"], s["scale"])
    if op == "embed_bwd":
        return embed.embed_bwd(s["dx"], s["tokens"], s["V"], s["scale"])
    if op == "qk_fwd":
        return list(block.qk_norm_rope_split(s["qkv"], s["wq"], s["wk"], s["b"], s["pos"], s["cos"], s["sin"],
                                             n_heads=s["H"], n_kv_heads=s["Hk"], eps=EPS))
    if op == "qk_bwd":
        out = block.qk_norm_rope_split_bwd(s["dq"], s["dk"], s["dv"], s["qkv"], s["wq"], s["wk"], s["b"], s["pos"],
                                           s["cos"], s["sin"], n_heads=s["H"], n_kv_heads=s["Hk"], eps=EPS)
        return list(out) if s["b"] is not None else list(out[:3])
    if op == "act8_round":
        return act8.unpack(act8.pack(s["x"], relu=s["relu"]), s["x"].dtype)
    if op == "act8_linear":
        return list(act8.wgrad(s["dy"], act8.pack(s["x"], relu=s["relu"])))
    kx, kh = act8.pack(s["x"]), act8.pack(s["h"], relu=True)
    dw2, db2 = act8.wgrad(s["dy"], kh)
    dh, dw1, db1 = act8.relu_wgrad(s["dh"], kh, kx)
    return [dw2, db2, dh, dw1, db1]


# ---- what a pass cannot do without ------------------------------------------

def work(case: dict) -> dict:
    op, T = case["op"], case["T"]
    es = 4 if case["dtype"] == "f32" else 2
    if op.startswith("embed"):
        V, D = case["V"], case["D"]
        if op == "embed_fwd":
            return dict(bytes=8 * T + (min(T, V) + T) * D * es, flops=T * D)
        return dict(bytes=8 * T + T * D * es + V * D * 4, flops=T * D)
    if op.startswith("qk"):
        C = (case["H"] + 2 * case["Hk"]) * case["hd"]
        tabs = 4 * T + 8 * min(T, case["seq"]) * case["hd"] + (4 * C if case["bias"] else 0) + 8 * case["hd"]
        if op == "qk_fwd":
            return dict(bytes=2 * T * C * es + tabs, flops=8 * T * C)
        return dict(bytes=3 * T * C * es + tabs + (4 * C if case["bias"] else 0) + 8 * case["hd"], flops=16 * T * C)
    I = case["I"]
    if op == "act8_round":
        return dict(bytes=2 * T * I * es, flops=4 * T * I)
    if op == "act8_linear":
        O = case["O"]
        return dict(bytes=T * (I + O) * es + 4 * O * (I + 1), flops=2 * T * I * O)
    F = case["F"]
    return dict(bytes=T * (2 * I + 3 * F) * es + 4 * (2 * I * F + I + F), flops=4 * T * I * F)


# ---- the definitions in 64 bits ----------------------------------------------

def _f64_kept(x, relu):
    top = 255.0 if relu else 127.0
    v = x.double().unflatten(1, (-1, GROUP))
    need = (v.clamp(min=0.0) if relu else v.abs()).max(-1, keepdim=True).values / top
    m, e = torch.frexp(need)
    k = torch.where(m == 0.5, e - 1, e)  # smallest k with need <= 2^k
    k = torch.maximum(k, torch.full_like(k, -126)).double()
    unit = torch.exp2(k)
    n = torch.round(v / unit)
    if relu:
        n = torch.where(v > 0, n.clamp(min=1.0, max=255.0), 0.0)
    return (n * unit).flatten(1)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    op, T = case["op"], case["T"]
    if op == "embed_fwd":
        out = torch.zeros(T, case["D"], device=DEV, dtype=torch.float64)
        for a in range(0, T, 1 << 16):
            t = s["tokens"][a:a + (1 << 16)]
            ok = (t >= 0) & (t < case["V"])
            out[a:a + (1 << 16)][ok] = s["table"].double()[t[ok]] * case["scale"]
        return out
    if op == "embed_bwd":
        # by order of tokens: running sums in 64 bits, their differences at the tokens' borders
        tok = s["tokens"]
        order = torch.argsort(tok, stable=True)
        ends = torch.searchsorted(tok[order], torch.arange(case["V"] + 1, device=DEV))
        out = torch.empty(case["V"], case["D"], device=DEV, dtype=torch.float64)
        for a in range(0, case["D"], 32):
            run_ = torch.cumsum(s["dx"][:, a:a + 32].double()[order], 0)
            run_ = torch.cat((torch.zeros_like(run_[:1]), run_))
            out[:, a:a + 32] = (run_[ends[1:]] - run_[ends[:-1]]) * case["scale"]
        return out
    if op.startswith("qk"):
        H, Hk, hd = case["H"], case["Hk"], case["hd"]
        u = s["qkv"].double() + (s["b"].double() if s["b"] is not None else 0.0)
        u = u.unflatten(1, (H + 2 * Hk, hd))
        p = s["pos"].long()
        turn = torch.complex(s["cos"].double()[p][:, 0::2], s["sin"].double()[p][:, 0::2])[:, None]
        outs = []
        grads, dws = [], []
        for a, b, w in ((0, H, "wq"), (H, H + Hk, "wk")):
            part, w = u[:, a:b], s[w].double()
            root = torch.sqrt(part.square().mean(-1, keepdim=True) + EPS)
            unit = part / root
            if op == "qk_fwd":
                z = torch.view_as_complex((unit * w).unflatten(-1, (hd // 2, 2))) * turn
                outs.append(torch.view_as_real(z).reshape(T, -1))
                continue
            g = s["dq" if a == 0 else "dk"].double().unflatten(1, (b - a, hd // 2, 2))
            g = torch.view_as_real(torch.view_as_complex(g) * turn.conj()).flatten(-2)
            dws.append((g * unit).sum((0, 1)))
            gw = g * w
            grads.append(((gw - unit * (gw * unit).mean(-1, keepdim=True)) / root).flatten(1))
        if op == "qk_fwd":
            return outs + [u[:, H + Hk:].reshape(T, -1)]
        d = torch.cat(grads + [s["dv"].double()], dim=1)
        return [d, *dws] + ([d.sum(0)] if s["b"] is not None else [])
    if op == "act8_round":
        return _f64_kept(s["x"], case["relu"])
    dy = s["dy"].double()
    if op == "act8_linear":
        return [_f64_kept(s["x"], case["relu"]).t().mm(dy).t(), dy.sum(0)]
    h = _f64_kept(s["h"], True)
    first = [h.t().mm(dy).t(), dy.sum(0)]
    dh = s["dh"].double() * (s["h"] > 0)
    return first + [dh, _f64_kept(s["x"], False).t().mm(dh).t(), dh.sum(0)]
