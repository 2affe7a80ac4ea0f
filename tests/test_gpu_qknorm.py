"""GPU: the projection epilogue with the norm of query and key heads, and its
gradient, against the formulas in float64.

Bars, in units of u = 2^-24, each a sum of the roundings on the way (u: bias
sum 1; r: the sum of squares' tree of at most 8 + 6 additions, its squares, and
through the square root half of them, mean, eps, root and quotient; y two
products; the rotation two products and a sum): 24 u of |y0 c| + |y1 s|
forward. Backward, with h = g w: 48 u of r (|h| + |y| mean |h y|), magnitudes
taken before the rotation's difference. Sums over rows: 200 u of the sum of
magnitudes (the terms' own roundings, and at most 150 additions on a row's way
at these sizes). A bf16 result adds one rounding, 2^-8 of the value."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from agpt_amd import block
from agpt_amd.attention import rope_tables

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def _inputs(T, H, Hk, hd, dtype, bias, seq, dev, seed, ld=0):
    rng = np.random.default_rng(seed)
    C = (H + 2 * Hk) * hd

    def rnd(*shape, std=1.0):
        return torch.from_numpy((std * rng.standard_normal(shape)).astype(np.float32))
    flat = rnd(T, max(ld, C)).to(DT[dtype]).to(dev)
    s = dict(qkv=flat[:, :C], wq=(1 + rnd(hd, std=0.2)).to(dev), wk=(1 + rnd(hd, std=0.2)).to(dev),
             bias=rnd(C).to(dev) if bias else None,
             positions=torch.from_numpy(rng.integers(-2, seq + 3, T).astype(np.int32)).to(dev) if seq else None)
    s["cos_t"], s["sin_t"] = rope_tables(seq, hd, device=dev) if seq else (None, None)
    d = [rnd(T, h * hd).to(DT[dtype]).to(dev) for h in (H, Hk, Hk)]
    return s, d


def _tables(s, T, hd):
    if s["cos_t"] is None:
        return torch.ones(T, 1, hd // 2, dtype=torch.float64), torch.zeros(T, 1, hd // 2, dtype=torch.float64)
    p = s["positions"].cpu().long().clamp(0, s["cos_t"].shape[0] - 1)
    return (t.double().cpu()[p][:, None, 0::2] for t in (s["cos_t"], s["sin_t"]))


def _turn(y, c, s):
    a, b = y[..., 0::2], y[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _turn_size(y, c, s):
    a, b = y[..., 0::2].abs(), y[..., 1::2].abs()
    return torch.stack((a * c.abs() + b * s.abs(), a * s.abs() + b * c.abs()), -1).flatten(-2)


def _check(s, d, H, Hk, hd, dtype):
    """Both directions of one call against float64."""
    T = s["qkv"].shape[0]
    heads = dict(n_heads=H, n_kv_heads=Hk, eps=EPS)
    got = [t.double().cpu() for t in block.qk_norm_rope_split(**s, **heads)]
    raw = block.qk_norm_rope_split_bwd(*d, **s, **heads)
    again = block.qk_norm_rope_split_bwd(*d, **s, **heads)
    for a, b in zip(raw, again):
        assert (a is None and b is None) or torch.equal(a, b)
    u = s["qkv"].double().cpu().reshape(T, H + 2 * Hk, hd)
    if s["bias"] is not None:
        u = u + s["bias"].double().cpu().view(H + 2 * Hk, hd)
    c, sn = _tables(s, T, hd)
    w = torch.cat((s["wq"].double().cpu().expand(H, hd), s["wk"].double().cpu().expand(Hk, hd)))
    n = u[:, :H + Hk]
    r = 1 / torch.sqrt((n * n).mean(-1, keepdim=True) + EPS)
    y = n * r
    half = 2.0 ** -8 if dtype == "bf16" else 0.0
    z, zs = _turn(y * w, c, sn), _turn_size(y * w, c, sn)
    want = [z[:, :H].flatten(1), z[:, H:].flatten(1), u[:, H + Hk:].flatten(1)]
    size = [zs[:, :H].flatten(1), zs[:, H:].flatten(1), u[:, H + Hk:].flatten(1).abs()]
    for name, a, b, m in zip("qkv", got, want, size):
        assert a.shape == b.shape and bool(((a - b).abs() <= 24 * U * m + half * (b.abs() + 24 * U * m)).all()), name
    dz = [x.double().cpu().view(T, x.shape[1] // hd, hd) for x in d]
    g0 = torch.cat(dz[:2], 1)
    g, gs = _turn(g0, c, -sn), _turn_size(g0, c, sn)
    h, hs = g * w, gs * w.abs()
    du = r * (h - y * (h * y).mean(-1, keepdim=True))
    ds = r * (hs + y.abs() * (hs * y.abs()).mean(-1, keepdim=True))
    du, ds = torch.cat((du, dz[2]), 1).flatten(1), torch.cat((ds, dz[2].abs()), 1).flatten(1)
    dx = raw[0].double().cpu()
    assert bool(((dx - du).abs() <= 48 * U * ds + half * (du.abs() + 48 * U * ds)).all())
    for name, a, lo, hi in (("dwq", raw[1], 0, H), ("dwk", raw[2], H, H + Hk)):
        b, m = (g * y)[:, lo:hi].sum((0, 1)), (gs * y.abs())[:, lo:hi].sum((0, 1))
        assert bool(((a.double().cpu() - b).abs() <= 200 * U * m).all()), name
    assert (raw[3] is None) == (s["bias"] is None)
    if raw[3] is not None:
        assert bool(((raw[3].double().cpu() - du.sum(0)).abs() <= 200 * U * ds.sum(0)).all())


@pytest.mark.parametrize("T,H,Hk,hd,dtype,bias,seq", [
    (1, 8, 8, 16, "f32", True, 32), (0, 8, 8, 16, "f32", True, 32), (1037, 8, 8, 16, "f32", True, 32),
    (515, 4, 4, 32, "f32", False, 24), (301, 2, 2, 64, "bf16", True, 128), (130, 32, 8, 128, "bf16", False, 4096),
    (77, 16, 2, 128, "f32", True, 100), (33, 3, 1, 4, "f32", True, 5), (33, 3, 1, 8, "bf16", True, 5),
    (50, 5, 1, 20, "bf16", True, 9), (64, 6, 3, 24, "f32", True, 17), (41, 4, 2, 80, "bf16", False, 50),
    (29, 4, 1, 256, "f32", True, 300), (29, 2, 1, 252, "bf16", True, 300), (19, 3, 3, 256, "bf16", False, 64),
    (100, 8, 8, 16, "f32", True, 0), (60, 64, 8, 96, "bf16", True, 33), (5, 100, 50, 256, "f32", True, 7),
    (4099, 1, 1, 4, "f32", True, 3), (2500, 1, 1, 64, "bf16", True, 40)])
def test_qk_norm(gpu, T, H, Hk, hd, dtype, bias, seq):
    s, d = _inputs(T, H, Hk, hd, dtype, bias, seq, gpu, T + 31 * H + hd)
    _check(s, d, H, Hk, hd, dtype)


@pytest.mark.parametrize("H,Hk,hd,dtype,ld", [(8, 8, 16, "f32", 400), (4, 2, 64, "bf16", 520), (3, 1, 20, "bf16", 108)])
def test_qk_norm_strided_rows(gpu, H, Hk, hd, dtype, ld):
    s, d = _inputs(333, H, Hk, hd, dtype, True, 16, gpu, ld, ld=ld)
    assert s["qkv"].stride(0) == ld
    _check(s, d, H, Hk, hd, dtype)
    # into a strided output too: the columns past the row stay as they were
    C = (H + 2 * Hk) * hd
    buf = torch.full((333, ld), 7.0, device=gpu, dtype=DT[dtype])
    heads = dict(n_heads=H, n_kv_heads=Hk)
    want = block.qk_norm_rope_split_bwd(*d, **s, **heads)[0]
    got = block.qk_norm_rope_split_bwd(*d, **s, **heads, out=buf[:, :C])[0]
    assert torch.equal(got, want) and bool((buf[:, C:] == 7.0).all())


def test_qk_norm_gradient_by_differences(gpu):
    """The gradient against central differences of the formulas in float64
    (step 1e-5 on values near 1: truncation 1e-10, far below the fp32 bar of
    1e-4 of the largest gradient)."""
    T, H, Hk, hd = 3, 2, 1, 8
    s, d = _inputs(T, H, Hk, hd, "f32", True, 11, gpu, 3)
    dx, dwq, dwk, db = block.qk_norm_rope_split_bwd(*d, **s, n_heads=H, n_kv_heads=Hk, eps=EPS)
    c, sn = _tables(s, T, hd)
    dz = torch.cat([x.double().cpu().view(T, x.shape[1] // hd, hd) for x in d], 1)

    def loss(x, wq, wk, b):
        u = (x + b).view(T, H + 2 * Hk, hd)
        n = u[:, :H + Hk]
        y = n / torch.sqrt((n * n).mean(-1, keepdim=True) + EPS) * torch.cat((wq.expand(H, hd), wk.expand(Hk, hd)))
        return (torch.cat((_turn(y, c, sn), u[:, H + Hk:]), 1) * dz).sum()
    at = [s[k].double().cpu().contiguous() for k in ("qkv", "wq", "wk", "bias")]
    for i, got in enumerate((dx, dwq, dwk, db)):
        got = got.double().cpu().reshape(-1)
        want = torch.empty_like(got)
        for j in range(got.numel()):
            v = []
            for e in (1e-5, -1e-5):
                a = [t.clone() for t in at]
                a[i].view(-1)[j] += e
                v.append(loss(*a))
            want[j] = (v[0] - v[1]) / 2e-5
        assert float((got - want).abs().max()) <= 1e-4 * float(want.abs().max())


def test_qk_norm_extremes(gpu):
    """A head of zeros, one of tiny and one of large values, and a row that is
    not finite: zeros stay zeros (eps holds the root up), the others follow the
    formula, the bad row stays its own."""
    s, _ = _inputs(4, 1, 1, 16, "f32", False, 0, gpu, 1)
    s["qkv"][0, :16] = 0.0
    s["qkv"][1] *= 1e-12
    s["qkv"][2] *= 1e15
    s["qkv"][3, 3] = float("inf")
    q, k, v = (t.double().cpu() for t in block.qk_norm_rope_split(**s, n_heads=1, eps=EPS))
    assert bool((q[0] == 0).all())
    x = s["qkv"].double().cpu()[:3, :16]
    want = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * s["wq"].double().cpu()
    assert bool(((q[:3] - want).abs() <= 24 * U * want.abs()).all())
    assert not bool(torch.isfinite(q[3, 3])) and bool(torch.isfinite(k).all())
    assert torch.equal(v, s["qkv"].double().cpu()[:, 32:])


def test_qk_norm_graph_and_stream(gpu):
    s, d = _inputs(2000, 8, 8, 16, "f32", True, 32, gpu, 9)
    others = [_inputs(2000, 8, 8, 16, "f32", True, 32, gpu, 10 + i) for i in range(2)]
    heads = dict(n_heads=8)

    def both(s, d):
        return [*block.qk_norm_rope_split(**s, **heads), *block.qk_norm_rope_split_bwd(*d, **s, **heads)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        both(s, d)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = both(s, d)
    torch.cuda.synchronize()
    for s2, d2 in others * 2:
        for k in s:
            s[k].copy_(s2[k])
        for a, b in zip(d, d2):
            a.copy_(b)
        g.replay()
        want = both(s2, d2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_qk_norm_refuses(gpu):
    s, d = _inputs(5, 2, 1, 16, "f32", True, 8, gpu, 1)
    bad = [dict(qkv=s["qkv"].half()), dict(qkv=s["qkv"][:, :60]), dict(qkv=s["qkv"].t()), dict(wq=s["wq"][:8]),
           dict(wk=s["wk"].double()), dict(bias=s["bias"][:5]), dict(positions=s["positions"].long()),
           dict(positions=s["positions"][:3]), dict(sin_t=None), dict(sin_t=s["sin_t"][:3]), dict(wq=s["wq"].cpu())]
    for kw in bad:
        a = dict(s, **kw)
        with pytest.raises(ValueError):
            block.qk_norm_rope_split(**a, n_heads=2, n_kv_heads=1)
        with pytest.raises(ValueError):
            block.qk_norm_rope_split_bwd(*d, **a, n_heads=2, n_kv_heads=1)
    for dd in ([d[0][:, :16], d[1], d[2]], [d[0], d[1].bfloat16(), d[2]], [d[0], d[1], d[2].cpu()]):
        with pytest.raises(ValueError):
            block.qk_norm_rope_split_bwd(*dd, **s, n_heads=2, n_kv_heads=1)
    with pytest.raises(ValueError):
        block.qk_norm_rope_split(**s, n_heads=0)
    for out in (s["qkv"], torch.empty(4, 64, device=gpu), torch.empty(5, 64, device=gpu).bfloat16()):  # overlaps; shape; type
        with pytest.raises(ValueError):
            block.qk_norm_rope_split_bwd(*d, **s, n_heads=2, n_kv_heads=1, out=out)
    buf = torch.zeros(5 * 96, device=gpu)  # an output that begins inside dq
    with pytest.raises(ValueError):
        block.qk_norm_rope_split_bwd(buf[:160].view(5, 32), d[1], d[2], **s, n_heads=2, n_kv_heads=1,
                                     out=buf[100:420].view(5, 64))
