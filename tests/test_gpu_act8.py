"""GPU: 8-bit activation checkpoints against their definition, and the weight
gradients against 64-bit products of the values that they stand for.

Codes and values are compared exactly (x / s is exact for a power-of-two s, so
the definition has one answer). Weight gradients: the parts of dy and the
values multiply exactly; each of the additions on the way is taken as off by at
most 2^-23 of the sum of magnitudes (a matrix unit may truncate), of which a
chunk of c rows has 3 c / 16 steps of 16 products, and chunks are then added:
the bar counts 3 rows + 64 additions. Bias gradients likewise, 2^-24 each."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from agpt_amd import act8

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def kept(x, relu):
    """The values of a checkpoint of x (float64 [T, W]), from the definition."""
    top = 255.0 if relu else 127.0
    g = x.reshape(x.shape[0], x.shape[1] // 32, 32)
    big = np.where(g > 0, g, 0.0) if relu else np.abs(g)
    bad = ~np.isfinite(g).all(-1, keepdims=True) | (big.max(-1, keepdims=True) > top * 2.0 ** 120)
    need = np.where(bad, 1.0, big.max(-1, keepdims=True)) / top
    m, e = np.frexp(need)
    e = np.maximum(np.where(m == 0.5, e - 1, e), -126)
    e = np.where(need == 0, -126, e)
    s = np.ldexp(1.0, e)
    with np.errstate(invalid="ignore"):
        c = np.rint(g / s)
        if relu:
            c = np.where(g > 0, np.clip(c, 1, 255), 0.0)
    return np.where(bad, np.nan, c * s).reshape(x.shape)


def _x(rng, T, W, dtype, relu, std=1.0):
    x = (std * rng.standard_normal((T, W))).astype(np.float32)
    if relu:
        x = np.maximum(x, 0)
    return torch.from_numpy(x).to(DT[dtype])


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("T,W,dtype", [(1, 32, "f32"), (0, 64, "f32"), (7, 128, "f32"), (8, 96, "bf16"), (9, 512, "f32"),
                                       (1037, 128, "bf16"), (333, 1056, "f32")])
def test_pack_unpack(gpu, T, W, dtype, relu):
    rng = np.random.default_rng(T + W)
    x = _x(rng, T, W, dtype, relu, std=3.0)
    k = act8.pack(x.to(gpu), relu=relu)
    want = kept(x.double().numpy(), relu)
    for out in (torch.float32, torch.bfloat16):
        assert np.array_equal(act8.unpack(k, out).double().cpu().numpy(), want)
    # the promised distance: half a step, less than a whole one for a small ReLU output. The smallest
    # power of two s with big <= top s has big > top s / 2: s < 2 big / top
    step = 2 / 255 if relu else 2 / 127
    big = np.abs(x.double().numpy().reshape(T, W // 32, 32)).max(-1, keepdims=True)
    off = np.abs(want - x.double().numpy()).reshape(T, W // 32, 32)
    assert (off <= big * step * (1.0 if relu else 0.5)).all()
    if relu:
        assert np.array_equal(want > 0, x.double().numpy() > 0)


def test_pack_borders(gpu):
    """Scales and codes at their borders: the largest value exactly on, one step
    below and above the top code at several exponents, ties, denormals, zeros,
    negative inputs of a ReLU block, the largest finite values."""
    rows = []
    for e in (-140, -126, -100, -1, 0, 1, 60, 120):
        for top in (127.0, 255.0):
            for v in (top, np.nextafter(np.float32(top), np.float32(0)), np.nextafter(np.float32(top), np.float32(1e9))):
                r = np.zeros(32, np.float32)
                r[0] = np.ldexp(np.float32(v), e)
                r[1:9] = np.ldexp(np.float32([0.5, 1.5, 2.5, -0.5, -1.5, 0.49, 126.5, -126.5]), e)
                rows.append(r)
    rows.append(np.zeros(32, np.float32))
    rows.append(np.full(32, -0.0, np.float32))
    rows.append(np.full(32, 1e-45, np.float32))
    rows.append(np.full(32, -3.0, np.float32))
    rows.append(np.full(32, np.finfo(np.float32).max, np.float32))
    x = np.stack(rows)
    for relu in (False, True):
        got = act8.unpack(act8.pack(torch.from_numpy(x).to(gpu), relu=relu)).cpu().numpy().astype(np.float64)
        assert np.array_equal(got, kept(x.astype(np.float64), relu), equal_nan=True)


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_not_finite_blocks(gpu, relu, bad):
    """A block with an infinity or a NaN reads as NaN, its neighbours as they are;
    the weight gradient is NaN in that block's columns only."""
    rng = np.random.default_rng(2)
    x = _x(rng, 20, 128, "f32", relu)
    x[13, 40] = float(bad)
    k = act8.pack(x.to(gpu), relu=relu)
    got = act8.unpack(k).cpu().numpy()
    want = kept(x.double().numpy(), relu)
    assert np.array_equal(got.astype(np.float64), want, equal_nan=True)
    assert np.isnan(got[13, 32:64]).all() and np.isfinite(np.delete(got, 13, 0)).all()
    dw, _ = act8.wgrad(torch.ones(20, 64, device=gpu), k)
    nan = torch.isnan(dw).cpu()
    assert bool(nan[:, 32:64].all()) and not bool(nan[:, :32].any()) and not bool(nan[:, 64:].any())


@pytest.mark.parametrize("dtype,ld,shift", [("f32", 131, 0), ("f32", 136, 4), ("f32", 128, 1), ("bf16", 130, 0), ("bf16", 144, 2)])
def test_strided_rows(gpu, dtype, ld, shift):
    rng = np.random.default_rng(ld)
    T, W = 203, 128
    flat = _x(rng, 1, T * ld + 8, dtype, False)[0].to(gpu)
    x = torch.as_strided(flat, (T, W), (ld, 1), shift)
    k = act8.pack(x)
    want = kept(x.double().cpu().numpy(), False)
    buf = torch.full((T, ld), 7.0, device=gpu, dtype=DT[dtype])
    act8.unpack(k, out=buf[:, :W])
    assert np.array_equal(buf[:, :W].double().cpu().numpy(), want) and bool((buf[:, W:] == 7.0).all())
    _check_wgrad(x, k, want)


def _check_wgrad(dy, k, val, bias=True):
    T = dy.shape[0]
    dw, db = act8.wgrad(dy, k, bias=bias)
    again = act8.wgrad(dy, k, bias=bias)
    d = dy.double().cpu().numpy()
    assert np.all(np.abs(dw.double().cpu().numpy() - d.T @ val) <= (3 * T + 64) * 2.0 ** -23 * (np.abs(d).T @ np.abs(val)))
    assert torch.equal(dw, again[0])
    if bias:
        assert np.all(np.abs(db.double().cpu().numpy() - d.sum(0)) <= (T + 64) * 2.0 ** -24 * np.abs(d).sum(0))
        assert torch.equal(db, again[1])
    else:
        assert db is None


@pytest.mark.parametrize("T,out,W,dtype,relu", [
    (1, 128, 128, "f32", False), (0, 128, 64, "f32", False), (181, 128, 128, "f32", False), (181, 128, 512, "f32", True),
    (1037, 512, 128, "f32", False), (65, 65, 128, "f32", False), (300, 1, 32, "f32", True), (77, 33, 160, "f32", False),
    (130, 64, 96, "bf16", False), (257, 1000, 1024, "bf16", True), (500, 17, 32, "bf16", False), (15, 200, 288, "bf16", True),
    (16, 64, 128, "f32", True), (17, 66, 64, "f32", False), (4100, 130, 256, "f32", False), (33, 7, 2048, "f32", False),
    (70, 201, 160, "f32", False), (95, 333, 288, "bf16", True), (64, 127, 192, "bf16", False), (31, 128, 160, "f32", True),
    (33, 600, 1312, "f32", False), (3000, 128, 256, "bf16", False), (600, 520, 512, "f32", False),
    (700, 1023, 288, "bf16", True)])
def test_wgrad(gpu, T, out, W, dtype, relu):
    rng = np.random.default_rng(T + 3 * out + W)
    k = act8.pack(_x(rng, T, W, "f32", relu).to(gpu), relu=relu)
    val = act8.unpack(k).double().cpu().numpy()
    dy = _x(rng, T, out, dtype, False, std=1e-3).to(gpu)
    _check_wgrad(dy, k, val, bias=out != 33)


@pytest.mark.parametrize("T,out,W,dtype,ld,shift", [
    (70, 67, 480, "f32", 67, 0), (333, 120, 512, "bf16", 131, 3), (95, 190, 224, "bf16", 191, 1), (601, 129, 256, "f32", 133, 2),
    (47, 255, 416, "f32", 256, 0), (1025, 300, 256, "bf16", 301, 5), (513, 97, 224, "f32", 99, 1)])
def test_wgrad_partly_filled_tiles(gpu, T, out, W, dtype, ld, shift):
    """Widths on both sides of the rule that shares operands between waves, under
    odd strides and shifts; what stands around the rows does not enter."""
    rng = np.random.default_rng(T + out)
    k = act8.pack(_x(rng, T, W, "f32", False).to(gpu))
    val = act8.unpack(k).double().cpu().numpy()
    flat = torch.full((T * ld + shift + 8,), float("nan"), dtype=DT[dtype])
    torch.as_strided(flat, (T, out), (ld, 1), shift).copy_(_x(rng, T, out, dtype, False))
    _check_wgrad(torch.as_strided(flat.to(gpu), (T, out), (ld, 1), shift), k, val)


def test_two_streams_at_once(gpu):
    """Calls that overlap on two streams have workspaces of their own."""
    rng = np.random.default_rng(12)
    T, out, W = 20000, 200, 256
    ks = [act8.pack(_x(rng, T, W, "f32", False).to(gpu)) for _ in range(2)]
    dys = [_x(rng, T, out, "f32", False).to(gpu) for _ in range(2)]
    want = [act8.wgrad(d, k) for d, k in zip(dys, ks)]
    streams = [torch.cuda.Stream(gpu) for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(act8.wgrad(dys[i], ks[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for dw, db in got[i]:
            assert torch.equal(dw, want[i][0]) and torch.equal(db, want[i][1])


def test_wgrad_keeps_all_of_fp32(gpu):
    """Every bit of an fp32 dy enters: against 1 + k 2^-23 in one row, whose
    products with small whole values are exact in fp32."""
    T, out = 1, 128
    dy = torch.from_numpy((1 + np.arange(out) * 2.0 ** -23).astype(np.float32))[None].to(gpu)
    x = torch.zeros(T, 32, device=gpu)
    x[0, 0], x[0, 1], x[0, 2] = 64.0, 1.0, -2.0  # s = 1: kept as they are
    dw, db = act8.wgrad(dy, act8.pack(x))
    assert torch.equal(dw[:, 0], 64 * dy[0]) and torch.equal(dw[:, 1], dy[0]) and torch.equal(dw[:, 2], -2 * dy[0])
    assert torch.equal(db, dy[0]) and bool((dw[:, 3:] == 0).all())


@pytest.mark.parametrize("T,out,W,dtype,relu", [
    (1, 128, 128, "f32", False), (0, 64, 64, "f32", False), (181, 512, 128, "f32", False), (1037, 512, 128, "f32", False),
    (77, 96, 160, "f32", True), (130, 64, 96, "bf16", False), (257, 992, 544, "bf16", True), (9, 32, 32, "f32", False),
    (130, 256, 288, "f32", False), (77, 128, 160, "bf16", True), (2049, 160, 1024, "f32", False)])
def test_relu_wgrad(gpu, T, out, W, dtype, relu):
    rng = np.random.default_rng(T + 5 * out + W)
    x = act8.pack(_x(rng, T, W, "f32", relu).to(gpu), relu=relu)
    h0 = _x(rng, T, out, "f32", True)
    h0[:, ::7] *= 1e-6  # far below a block's step, and still above zero
    h = act8.pack(h0.to(gpu), relu=True)
    dy = _x(rng, T, out, dtype, False, std=1e-3)
    dy[(h0 <= 0) & torch.from_numpy(rng.random((T, out)) < 0.1)] = float("nan")  # where the ReLU is shut nothing counts
    got, dw, db = act8.relu_wgrad(dy.to(gpu), h, x)
    want = torch.where(h0 > 0, dy, torch.zeros((), dtype=dy.dtype))
    assert got.dtype == dy.dtype and torch.equal(got.cpu(), want)
    val, d = act8.unpack(x).double().cpu().numpy(), want.double().numpy()
    assert np.all(np.abs(dw.double().cpu().numpy() - d.T @ val) <= (3 * T + 64) * 2.0 ** -23 * (np.abs(d).T @ np.abs(val)))
    assert np.all(np.abs(db.double().cpu().numpy() - d.sum(0)) <= (T + 64) * 2.0 ** -24 * np.abs(d).sum(0))
    again = act8.relu_wgrad(dy.to(gpu), h, x, bias=False)
    assert torch.equal(again[0], got) and torch.equal(again[1], dw) and again[2] is None


def test_wgrad_large_batch(gpu):
    """A training batch of 100,003 rows (chunks of many steps) against float64."""
    rng = np.random.default_rng(4)
    T = 100_003
    x = _x(rng, T, 128, "f32", False).to(gpu)
    dy = _x(rng, T, 192, "f32", False).to(gpu)
    k = act8.pack(x)
    dw, db = act8.wgrad(dy, k)
    val, d = act8.unpack(k).double(), dy.double()
    want = d.t() @ val
    # T / 16 steps of 3 in at most 16 chunks' worth of rows: errors of either sign, far inside a
    # bar of sqrt(additions) of the root of the sum of squares
    bar = 16 * 2.0 ** -23 * (d.square().t() @ val.square()).sqrt() * (3 * T / 16) ** 0.5
    assert bool(((dw.double() - want).abs() <= bar).all())
    assert bool(((db.double() - d.sum(0)).abs() <= 16 * 2.0 ** -24 * d.square().sum(0).sqrt() * T ** 0.5).all())


def test_graph_and_stream(gpu):
    rng = np.random.default_rng(8)
    T, W, F = 1500, 128, 256
    ins = [[_x(rng, T, w, "f32", r).to(gpu) for w, r in ((W, False), (F, True), (W, False), (F, False))] for _ in range(3)]

    def step(x, h, dy, dh):
        kx, kh = act8.pack(x), act8.pack(h, relu=True)
        return [*act8.wgrad(dy, kh), *act8.relu_wgrad(dh, kh, kx), act8.unpack(kx)]
    buf = [t.clone() for t in ins[0]]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(*buf)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = step(*buf)
    torch.cuda.synchronize()
    for new in ins * 2:
        for a, b in zip(buf, new):
            a.copy_(b)
        g.replay()
        want = step(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refuses(gpu):
    x = torch.zeros(4, 64, device=gpu)
    k, h = act8.pack(x), act8.pack(x, relu=True)
    for call in (lambda: act8.pack(x[:, :40]), lambda: act8.pack(x.half()), lambda: act8.pack(x[0]), lambda: act8.pack(x.t()),
                 lambda: act8.pack(x[:1].expand(4, 64)), lambda: act8.unpack(k, torch.float16),
                 lambda: act8.unpack(k, out=x[:3]),
                 lambda: act8.unpack(k, out=k.codes[:256].view(torch.float32).view(1, 64).expand(4, 64)), lambda: act8.wgrad(x[:3], k), lambda: act8.wgrad(x.double(), k),
                 lambda: act8.wgrad(x.cpu(), k), lambda: act8.wgrad(x[:, :0], k), lambda: act8.relu_wgrad(x, k, k),
                 lambda: act8.relu_wgrad(x[:, :32], h, k), lambda: act8.relu_wgrad(x, h, act8.pack(x[:3]))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("T,out,W", [(50, 6, 32), (300, 70, 160)])
def test_wgrad_by_differences(gpu, T, out, W):
    """<dy, val·Wᵀ> is linear in W: with whole numbers that the checkpoint holds as
    they are, every sum is exact and a difference over a step of 1 is the gradient."""
    g = torch.Generator().manual_seed(T)
    x = torch.randint(-8, 9, (T, W), generator=g).float()
    x[:, ::32] = 64.0  # every block's scale is 1
    dy = torch.randint(-4, 5, (T, out), generator=g).float()
    k = act8.pack(x.to(gpu))
    val = act8.unpack(k).double().cpu()
    assert torch.equal(val, x.double())
    dw, db = (t.double().cpu() for t in act8.wgrad(dy.to(gpu), k))
    weight = torch.randint(-3, 4, (out, W), generator=g).double()

    def f(w):
        return float((dy.double() * (val @ w.T)).sum())
    for o in range(0, out, 7):
        for i in range(0, W, 13):
            up, down = weight.clone(), weight.clone()
            up[o, i] += 1
            down[o, i] -= 1
            assert float(dw[o, i]) == (f(up) - f(down)) / 2
    assert torch.equal(db, dy.double().sum(0))
