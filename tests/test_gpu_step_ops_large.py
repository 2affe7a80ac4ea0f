"""GPU: offsets past 2^31 elements and 2^32 bytes. Only the last rows differ from
zero (or from a constant), so the right answer is the same call on those rows
alone: rows that do not depend on others equal it bit by bit, sums over rows up
to the order of `TAIL` additions, each off by at most 2^-24 of the magnitudes
(the zeros in between add nothing)."""
from __future__ import annotations

import pytest
import torch

from agpt_amd import act8, block, embed

pytestmark = pytest.mark.gpu

TAIL = 1000


@pytest.fixture(autouse=True)
def _free(gpu):
    yield
    torch.cuda.empty_cache()


def _tail(T, W, gpu, g, fill=0.0):
    x = torch.full((T, W), fill, device=gpu)
    x[-TAIL:] = torch.randn(TAIL, W, generator=g, device=gpu)
    return x


def _close(got, want, size, n=TAIL):
    assert bool(((got - want).abs() <= 2 * n * 2.0 ** -24 * size).all())


def test_embedding_rows(gpu):
    T, V, D = 2**21 + 3, 300, 1024
    g = torch.Generator(gpu).manual_seed(0)
    tok = torch.randint(-1, V, (T,), generator=g, device=gpu)
    table = torch.randn(V, D, generator=g, device=gpu)
    x = embed.embed_fwd(tok, table, 0.5)
    assert torch.equal(x[-TAIL:], embed.embed_fwd(tok[-TAIL:].clone(), table, 0.5))
    assert torch.equal(x[T // 2:T // 2 + TAIL], embed.embed_fwd(tok[T // 2:T // 2 + TAIL].clone(), table, 0.5))
    del x
    dx = _tail(T, D, gpu, g)
    got = embed.embed_bwd(dx, tok, V, 0.5)
    want = embed.embed_bwd(dx[-TAIL:], tok[-TAIL:].clone(), V, 0.5)
    _close(got, want, embed.embed_bwd(dx[-TAIL:].abs(), tok[-TAIL:].clone(), V, 0.5))
    assert torch.equal(got, embed.embed_bwd(dx, embed.EmbedPlan(tok, V), scale=0.5))


@pytest.mark.parametrize("n", [100, TAIL, 5000])
def test_embedding_table(gpu, n):
    """A table of more than 2^31 entries: by the one launch and by a plan."""
    V, D = 2**21 + 5, 1024
    g = torch.Generator(gpu).manual_seed(1)
    tok = V - 1 - torch.randperm(2 * n, generator=g, device=gpu)[:n]
    dx = torch.randn(n, D, generator=g, device=gpu)
    for plan in (tok, embed.EmbedPlan(tok, V)):
        got = embed.embed_bwd(dx, plan, V, out=torch.full((V, D), 7.0, device=gpu))
        assert torch.equal(got[tok], dx)
        got[tok] = 0
        assert not bool(got.any())
    got[tok] = dx
    assert torch.equal(embed.embed_fwd(tok, got), dx)


def test_query_key_norms(gpu):
    H, Hk, hd = 4, 2, 64
    T, C = 2**22 + 7, (H + 2 * Hk) * hd
    g = torch.Generator(gpu).manual_seed(2)
    qkv = _tail(T, C, gpu, g, fill=1.0)
    w = [1 + 0.1 * torch.randn(hd, generator=g, device=gpu) for _ in range(2)]
    bias = torch.randn(C, generator=g, device=gpu)
    pos = torch.randint(0, 32, (T,), generator=g, device=gpu, dtype=torch.int32)
    ang = torch.rand(32, hd, generator=g, device=gpu)
    kw = dict(bias=bias, cos_t=ang.cos(), sin_t=ang.sin(), n_heads=H, n_kv_heads=Hk)
    end = pos[-TAIL:].clone()
    outs = block.qk_norm_rope_split(qkv, *w, positions=pos, **kw)
    for a, b in zip(outs, block.qk_norm_rope_split(qkv[-TAIL:], *w, positions=end, **kw)):
        assert torch.equal(a[-TAIL:], b)
    del outs
    d = [_tail(T, h * hd, gpu, g) for h in (H, Hk, Hk)]
    short = [t[-TAIL:] for t in d]
    got = block.qk_norm_rope_split_bwd(*d, qkv, *w, positions=pos, **kw)
    want = block.qk_norm_rope_split_bwd(*short, qkv[-TAIL:], *w, positions=end, **kw)
    assert torch.equal(got[0][-TAIL:], want[0]) and not bool(got[0][:-TAIL].any())
    # |dq| summed bounds what the bias' sums add up; a weight's terms are |dq||y| with |y| <= sqrt(hd), and two heads' more
    _close(got[3], want[3], want[0].abs().sum(0))
    rows = sum(t.abs().sum() for t in short[:2])
    for i in (1, 2):
        _close(got[i], want[i], rows * hd ** 0.5)


def test_checkpoints(gpu):
    T, W = 2**22 + 9, 512
    g = torch.Generator(gpu).manual_seed(3)
    x = _tail(T, W, gpu, g)
    for relu in (False, True):
        k, ke = act8.pack(x, relu=relu), act8.pack(x[-TAIL:], relu=relu)
        back = act8.unpack(k)
        assert torch.equal(back[-TAIL:], act8.unpack(ke)) and not bool(back[:-TAIL].any())
        del back
    h, he = k, ke
    for out in (512, 128, 65):  # shared operands, and a wave alone where the input is narrow
        W_in = 512 if out != 128 else 64
        xin = x[:, :W_in]
        k, ke = act8.pack(xin), act8.pack(xin[-TAIL:])
        dy = _tail(T, 512, gpu, g)[:, :out]
        val = act8.unpack(ke)
        size = dy[-TAIL:].abs().t().double() @ val.abs().double()
        dw, db = act8.wgrad(dy, k)
        we, be = act8.wgrad(dy[-TAIL:], ke)
        _close(dw.double(), we.double(), size, 3 * TAIL)
        _close(db, be, dy[-TAIL:].abs().sum(0))
        del dy
    dh = _tail(T, W, gpu, g, fill=1.0)  # behind a shut ReLU
    k, ke = act8.pack(x[:, :128]), act8.pack(x[-TAIL:, :128])
    got, want = act8.relu_wgrad(dh, h, k), act8.relu_wgrad(dh[-TAIL:], he, ke)
    assert torch.equal(got[0][-TAIL:], want[0]) and not bool(got[0][:-TAIL].any())
    size = want[0].abs().t().double() @ act8.unpack(ke).abs().double()
    _close(got[1].double(), want[1].double(), size, 3 * TAIL)
    _close(got[2], want[2], want[0].abs().sum(0))
