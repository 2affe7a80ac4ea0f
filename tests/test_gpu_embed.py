"""GPU: the embedding and its gradient against 64-bit sums.

Forward: one fp32 product, off by at most 2^-24 of it, and for bf16 one more
rounding of at most 2^-8. Backward: a row passes at most `depth` fp32 additions
(sorted first: 64 in a slot, the slots of a workgroup, a piece per span of 64
rows; in one launch: an eighth of a token's rows, the lane groups and the
waves), each off by at most 2^-24 of a partial sum no larger than the sum of
magnitudes, and the scale's product once."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from agpt_amd import embed

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _tokens(rng, T, V, kind):
    if kind == "one":      # every row the same token
        return np.full(T, V // 2)
    if kind == "each":     # every token at most once, in falling order
        return (np.arange(T)[::-1] % V).copy()
    if kind == "pad":      # padding of both sorts among skewed tokens
        t = np.minimum((V * rng.random(T) ** 3).astype(np.int64), V - 1)
        t[rng.random(T) < 0.2] = -1
        t[rng.random(T) < 0.1] = V + 7
        return t
    if kind == "none":     # padding only
        return np.full(T, -1)
    return np.minimum((V * rng.random(T) ** 3).astype(np.int64), V - 1)


def _check_bwd(got, dx, tok, V, scale):
    """got [V, D] against float64 sums of the dx values."""
    x = dx.double().cpu()
    t = torch.from_numpy(np.asarray(tok))
    ok = (t >= 0) & (t < V)
    want = torch.zeros(V, x.shape[1], dtype=torch.float64).index_add_(0, t[ok], x[ok]) * scale
    size = torch.zeros(V, x.shape[1], dtype=torch.float64).index_add_(0, t[ok], x[ok].abs()) * abs(scale)
    depth = 330 + len(tok) // 8
    got = got.double().cpu()
    assert bool((got[~torch.isin(torch.arange(V), t[ok])] == 0).all())
    assert bool(((got - want).abs() <= depth * 2.0 ** -24 * size).all()), float(((got - want).abs() - depth * 2.0 ** -24 * size).max())


@pytest.mark.parametrize("T,V,D,dtype,bits,kind", [
    (1, 65, 128, "f32", 64, "skew"), (0, 65, 128, "f32", 64, "skew"), (777, 65, 128, "f32", 64, "pad"),
    (1000, 50_000, 1024, "bf16", 32, "pad"), (513, 300, 100, "bf16", 64, "skew"), (513, 300, 33, "f32", 32, "skew"),
    (300, 1, 1, "f32", 32, "pad"), (65, 7, 2050, "bf16", 32, "none"), (100, 40, 1500, "f32", 64, "each")])
def test_embed_fwd(gpu, T, V, D, dtype, bits, kind):
    rng = np.random.default_rng(T + V + D)
    tok = _tokens(rng, T, V, kind)
    E = torch.from_numpy(rng.standard_normal((V, D)).astype(np.float32)).to(DT[dtype])
    scale = float(np.float32(11.3))
    t = torch.from_numpy(tok.astype(np.int64 if bits == 64 else np.int32)).to(gpu)
    got = embed.embed_fwd(t, E.to(gpu), scale).double().cpu()
    ok = torch.from_numpy((tok >= 0) & (tok < V))
    want = E.double()[torch.from_numpy(np.clip(tok, 0, V - 1))] * scale * ok[:, None]
    u = 2.0 ** -24 + (2.0 ** -8 * (1 + 2.0 ** -24) if dtype == "bf16" else 0.0)
    assert got.shape == (T, D) and bool(((got - want).abs() <= u * want.abs()).all())


@pytest.mark.parametrize("T,V,D,dtype,bits,kind", [
    (1, 65, 128, "f32", 64, "skew"), (0, 65, 128, "f32", 64, "skew"), (64, 65, 128, "f32", 32, "one"),
    (65, 65, 128, "f32", 64, "one"), (777, 65, 128, "f32", 64, "pad"), (5000, 255, 64, "f32", 32, "skew"),
    (5000, 256, 64, "bf16", 64, "pad"), (9001, 50_000, 256, "bf16", 32, "pad"), (4096, 70_000, 32, "f32", 64, "skew"),
    (8193, 300, 100, "bf16", 64, "skew"), (513, 300, 33, "f32", 32, "skew"), (3000, 1, 1, "f32", 32, "pad"),
    (700, 7, 2050, "bf16", 32, "one"), (65, 7, 40, "f32", 32, "none"), (10_000, 20_000, 64, "f32", 64, "each"),
    (20_000, 3, 1500, "f32", 64, "skew"), (16_385, 1024, 96, "f32", 32, "skew"),
    (16_384, 1024, 96, "f32", 32, "skew"), (16_384, 5, 40, "bf16", 64, "one"), (2048, 300, 520, "f32", 64, "pad"),
    (2049, 300, 1040, "bf16", 32, "skew"), (300, 131_072, 8, "f32", 64, "skew"), (40, 1_000_000, 16, "f32", 64, "pad"),
    (65_536, 400, 24, "bf16", 32, "skew"), (65_537, 400, 24, "f32", 64, "pad"), (40_001, 70_000, 16, "f32", 64, "pad"),
    (30_000, 65, 64, "f32", 32, "one"), (70_001, 131, 36, "f32", 32, "pad"), (16_384, 400_000, 8, "f32", 64, "pad"), (511, 129, 3, "f32", 32, "skew")])
def test_embed_bwd(gpu, T, V, D, dtype, bits, kind):
    rng = np.random.default_rng(7 * T + V + D)
    tok = _tokens(rng, T, V, kind)
    dx = torch.from_numpy(rng.standard_normal((T, D)).astype(np.float32)).to(DT[dtype]).to(gpu)
    t = torch.from_numpy(tok.astype(np.int64 if bits == 64 else np.int32)).to(gpu)
    scale = float(np.float32(0.7))
    got = embed.embed_bwd(dx, t, V, scale)
    _check_bwd(got, dx, tok, V, scale)
    plan = embed.EmbedPlan(t, V)
    order, keys, off = plan.rows[:T].cpu().numpy(), plan.rows[T:2 * T].cpu().numpy(), plan.rows[2 * T:].cpu().numpy()
    k = np.where((tok >= 0) & (tok < V), tok, V)
    want = np.argsort(k, kind="stable")
    assert np.array_equal(order, want) and np.array_equal(keys, k[want])
    assert np.array_equal(off, np.searchsorted(k[want], np.arange(V + 1)))
    # the plan's sums may be another variant's: each within the bar, and each the same bytes every time
    again = embed.embed_bwd(dx, plan, scale=scale)
    _check_bwd(again, dx, tok, V, scale)
    assert torch.equal(again, embed.embed_bwd(dx, plan, V, scale=scale))
    assert torch.equal(got, embed.embed_bwd(dx, t, V, scale))


def test_embed_bwd_large_batch(gpu):
    """A training batch of 300,001 rows over 65 tokens, one of them a third of them."""
    rng = np.random.default_rng(5)
    T, V, D = 300_001, 65, 128
    tok = _tokens(rng, T, V, "skew")
    dx = torch.from_numpy(rng.standard_normal((T, D)).astype(np.float32)).to(gpu)
    _check_bwd(embed.embed_bwd(dx, torch.from_numpy(tok).to(gpu), V, 2.0), dx, tok, V, 2.0)


@pytest.mark.parametrize("dtype,ld,shift", [("f32", 160, 0), ("f32", 131, 0), ("f32", 128, 1), ("bf16", 136, 0),
                                            ("bf16", 130, 2)])
def test_embed_bwd_strides(gpu, dtype, ld, shift):
    rng = np.random.default_rng(ld)
    T, V, D = 1111, 50, 128
    tok = _tokens(rng, T, V, "pad")
    flat = torch.from_numpy(rng.standard_normal(T * ld + 8).astype(np.float32)).to(DT[dtype]).to(gpu)
    dx = torch.as_strided(flat, (T, D), (ld, 1), shift)
    got = embed.embed_bwd(dx, torch.from_numpy(tok).to(gpu), V, 1.0)
    _check_bwd(got, dx, tok, V, 1.0)


def test_embed_not_finite_rows_stay_apart(gpu):
    """A row that is not finite reaches its own token only; padding's reaches none."""
    tok = torch.tensor([3, -1, 5, 3, 9], device=gpu)
    dx = torch.ones(5, 16, device=gpu)
    dx[1], dx[2] = float("nan"), float("inf")
    got = embed.embed_bwd(dx, tok, 8).cpu()
    want = torch.zeros(8, 16)
    want[3], want[5] = 2.0, float("inf")
    assert torch.equal(got, want)


def test_embed_graph_and_stream(gpu):
    """Captured and replayed over new inputs, beside the eager call, on a stream of its own."""
    rng = np.random.default_rng(1)
    T, V, D = 5001, 65, 64
    E = torch.from_numpy(rng.standard_normal((V, D)).astype(np.float32)).to(gpu)
    toks = [torch.from_numpy(_tokens(rng, T, V, "pad")).to(gpu) for _ in range(3)]
    dxs = [torch.from_numpy(rng.standard_normal((T, D)).astype(np.float32)).to(gpu) for _ in range(3)]
    tok, dx = toks[0].clone(), dxs[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        embed.embed_fwd(tok, E, 2.0)
        embed.embed_bwd(dx, tok, V, 2.0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            x, dE = embed.embed_fwd(tok, E, 2.0), embed.embed_bwd(dx, tok, V, 2.0)
    torch.cuda.synchronize()
    for t, d in zip(toks * 2, dxs * 2):
        tok.copy_(t)
        dx.copy_(d)
        g.replay()
        want = embed.embed_fwd(t, E, 2.0), embed.embed_bwd(d, t, V, 2.0)
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(dE, want[1])


def test_embed_refuses(gpu):
    t = torch.zeros(4, dtype=torch.int64, device=gpu)
    E, dx = torch.zeros(5, 8, device=gpu), torch.zeros(4, 8, device=gpu)
    for call in (lambda: embed.embed_fwd(t.float(), E), lambda: embed.embed_fwd(t, E.half()), lambda: embed.embed_fwd(t, E.t()),
                 lambda: embed.embed_fwd(t[None], E), lambda: embed.embed_fwd(t, E.cpu()),
                 lambda: embed.embed_fwd(t, E, out=torch.zeros(4, 7, device=gpu)), lambda: embed.embed_bwd(dx[:3], t, 5),
                 lambda: embed.embed_bwd(dx, t), lambda: embed.embed_bwd(dx, t, 0), lambda: embed.embed_bwd(dx.t(), t, 5),
                 lambda: embed.embed_bwd(dx, embed.EmbedPlan(t, 5), 6), lambda: embed.embed_bwd(dx.expand(4, 8)[:, :0], t, 5),
                 lambda: embed.embed_bwd(dx, t, 5, out=torch.zeros(5, 8, device=gpu, dtype=torch.bfloat16)),
                 lambda: embed.embed_bwd(dx[:1].expand(4, 8), t, 5),
                 lambda: embed.embed_fwd(t, E, out=E[:4]), lambda: embed.embed_bwd(dx, t, 4, out=dx)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("T,V,D", [(90, 7, 12), (3000, 7, 12)])
def test_embed_gradient_by_differences(gpu, T, V, D):
    """<dx, x(E)> is linear in E: with small whole numbers every sum is exact and
    a difference over a step of 1 is the gradient itself."""
    g = torch.Generator().manual_seed(T)
    tok = torch.randint(-1, V + 1, (T,), generator=g).to(gpu)
    E = torch.randint(-4, 5, (V, D), generator=g).float().to(gpu)
    dx = torch.randint(-4, 5, (T, D), generator=g).float().to(gpu)
    got = embed.embed_bwd(dx, tok, V, 2.0)

    def f(table):
        return float((embed.embed_fwd(tok, table, 2.0).double() * dx.double()).sum())
    for v in range(V):
        for c in range(0, D, 5):
            up, down = E.clone(), E.clone()
            up[v, c] += 1
            down[v, c] -= 1
            assert float(got[v, c]) == (f(up) - f(down)) / 2
