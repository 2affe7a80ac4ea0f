"""CPU: what the embedding, the query / key norm and the 8-bit checkpoints
refuse, at the C ABI (nothing is launched) and in the Python mirror, and the
symbols of their headers."""
from __future__ import annotations

import ctypes as C
import re

import pytest
import torch

from agpt_amd import _native, act8, block, embed
from conftest import ROOT

P = 1 << 20  # a non-null, 16-byte aligned address that no refused call reads
BAD = _native.AGPT_ERR_INVALID_ARG
UNS = _native.AGPT_ERR_UNSUPPORTED


@pytest.mark.parametrize("header,table", [("agpt_embed.h", _native.EMBED_SYMBOLS), ("agpt_act8.h", _native.ACT8_SYMBOLS)])
def test_header_symbols_are_bound(header, table):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / header).read_text(), flags=re.S)
    names = set(re.findall(r"\b(agpt_\w+)\s*\(", text))
    assert names == set(table)
    lib = _native.attn_lib()
    assert all(hasattr(lib, n) for n in names)


def _refuses(rc, code, part):
    msg = _native.attn_lib().agpt_last_error().decode()
    assert rc == code and part in msg, (rc, msg)


@pytest.mark.parametrize("kw,part", [
    (dict(T=-1), "T < 0"), (dict(V=0), "V < 1"), (dict(D=0), "D < 1"), (dict(bits=16), "token_bits"),
    (dict(D=2**30 + 1), "2^30"), (dict(dtype=7), "dtype"), (dict(table=None), "null"), (dict(tokens=None), "null"), (dict(x=None), "null"),
    (dict(tokens=P + 4, bits=64), "aligned")])
def test_embed_fwd_refuses(kw, part):
    a = dict(table=P, tokens=P, bits=32, x=P, T=3, V=5, D=8, dtype=0)
    a.update(kw)
    _refuses(_native.attn_lib().agpt_embed_fwd(a["table"], a["tokens"], a["bits"], C.c_float(1), a["x"], a["T"], a["V"],
                                               a["D"], a["dtype"], None), BAD, part)


@pytest.mark.parametrize("kw,part", [
    (dict(T=-1), "T < 0"), (dict(V=0), "V < 1"), (dict(V=2**31 - 1), "2^31"), (dict(T=2**31), "2^31"),
    (dict(bits=8), "token_bits"), (dict(plan=None), "null"), (dict(tokens=None), "null"), (dict(ws=None), "null"),
    (dict(n=100), "workspace")])
def test_embed_plan_refuses(kw, part):
    a = dict(tokens=P, bits=32, T=300, V=5, plan=P, ws=P, n=1 << 40)
    a.update(kw)
    _refuses(_native.attn_lib().agpt_embed_plan(a["tokens"], a["bits"], a["T"], a["V"], a["plan"], a["ws"], a["n"], None),
             BAD, part)


@pytest.mark.parametrize("kw,part", [
    (dict(T=-1), "T < 0"), (dict(V=0), "V < 1"), (dict(D=0), "D < 1"), (dict(ld=7), "row stride"),
    (dict(D=2**30 + 8, ld=2**31), "2^30"), (dict(dtype=2), "dtype"), (dict(dx=None), "null"), (dict(plan=None), "null"), (dict(dE=None), "null"),
    (dict(ws=None), "null"), (dict(n=3), "workspace"), (dict(dx=P + 2), "aligned")])
def test_embed_bwd_refuses(kw, part):
    a = dict(dx=P, ld=8, plan=P, dE=P, ws=P, n=1 << 20, T=300, V=5, D=8, dtype=0)
    a.update(kw)
    _refuses(_native.attn_lib().agpt_embed_bwd(a["dx"], a["ld"], a["plan"], C.c_float(1), a["dE"], a["ws"], a["n"], a["T"],
                                               a["V"], a["D"], a["dtype"], None), BAD, part)


@pytest.mark.parametrize("kw,part", [
    (dict(T=-1), "T < 0"), (dict(V=0), "V < 1"), (dict(V=2**31 - 1), "2^31"), (dict(D=0), "D < 1"),
    (dict(D=2**30 + 8, ld=2**31), "2^30"), (dict(ld=7), "row stride"), (dict(bits=8), "token_bits"), (dict(dtype=2), "dtype"), (dict(dx=None), "null"),
    (dict(tokens=None), "null"), (dict(dE=None), "null"), (dict(ws=None), "null"), (dict(n=3), "workspace"),
    (dict(dx=P + 2), "aligned"), (dict(tokens=P + 2), "aligned")])
def test_embed_bwd_tokens_refuses(kw, part):
    a = dict(dx=P, ld=8, tokens=P, bits=32, dE=P, ws=P, n=1 << 30, T=300, V=5, D=8, dtype=0)
    a.update(kw)
    _refuses(_native.attn_lib().agpt_embed_bwd_tokens(a["dx"], a["ld"], a["tokens"], a["bits"], C.c_float(1), a["dE"],
                                                      a["ws"], a["n"], a["T"], a["V"], a["D"], a["dtype"], None), BAD, part)


QK = dict(eps=1e-5, qkv=P, ld=192, bias=P, wq=P, wk=P, pos=P, cos=P, sin=P, seq=32, T=3, H=2, Hk=1, hd=48, dtype=0, q=P, k=P, v=P)


@pytest.mark.parametrize("kw,code,part", [
    (dict(T=-1), BAD, "T < 0"), (dict(H=0), BAD, "n_heads"), (dict(Hk=0), BAD, "n_kv_heads"),
    (dict(hd=6), UNS, "head_dim"), (dict(hd=260), UNS, "head_dim"), (dict(hd=0), UNS, "head_dim"),
    (dict(H=5000), BAD, "65536"), (dict(dtype=3), BAD, "dtype"), (dict(ld=188), BAD, "row stride"),
    (dict(ld=194), BAD, "multiple of 4"), (dict(ld=196, dtype=1), BAD, "of 8"), (dict(seq=0), BAD, "rope_seq_len"),
    (dict(qkv=None), BAD, "null"), (dict(wq=None), BAD, "null"), (dict(v=None), BAD, "null"),
    (dict(sin=None), BAD, "null"), (dict(pos=None), BAD, "null"), (dict(qkv=P + 8), BAD, "16-byte"),
    (dict(bias=P + 4), BAD, "16-byte"), (dict(eps=-1e-5), BAD, "eps"), (dict(eps=float("nan")), BAD, "eps")])
def test_qk_norm_refuses(kw, code, part):
    a = dict(QK, **kw)
    lib = _native.attn_lib()
    _refuses(lib.agpt_qk_norm_rope_split(a["qkv"], a["ld"], a["bias"], a["wq"], a["wk"], a["pos"], a["cos"], a["sin"],
                                         a["seq"], a["T"], a["H"], a["Hk"], a["hd"], C.c_float(a["eps"]), a["dtype"], a["q"],
                                         a["k"], a["v"], None), code, part)
    n = lib.agpt_qk_norm_workspace_floats(2, 1, 48) + 10**9
    _refuses(lib.agpt_qk_norm_rope_split_bwd(a["q"], a["k"], a["v"], a["qkv"], a["ld"], a["bias"], a["wq"], a["wk"],
                                             a["pos"], a["cos"], a["sin"], a["seq"], a["T"], a["H"], a["Hk"], a["hd"],
                                             C.c_float(a["eps"]), a["dtype"], P, a["ld"], P, P, P, P, n, None), code, part)


@pytest.mark.parametrize("kw,part", [(dict(ldd=100), "row stride"), (dict(n=10), "workspace"), (dict(ws=None), "null"),
                                     (dict(dwq=None), "null"), (dict(dx=None), "null"), (dict(dx=P + 4), "16-byte")])
def test_qk_norm_bwd_refuses(kw, part):
    a = dict(QK, ldd=192, dx=P, dwq=P, ws=P, n=1 << 30)
    a.update(kw)
    _refuses(_native.attn_lib().agpt_qk_norm_rope_split_bwd(
        P, P, P, a["qkv"], a["ld"], a["bias"], a["wq"], a["wk"], a["pos"], a["cos"], a["sin"], a["seq"], a["T"], a["H"],
        a["Hk"], a["hd"], C.c_float(a["eps"]), a["dtype"], a["dx"], a["ldd"], a["dwq"], P, P, a["ws"], a["n"], None), BAD, part)


@pytest.mark.parametrize("kw,code,part", [
    (dict(T=-1), BAD, "T < 0"), (dict(W=0), BAD, "width"), (dict(W=48), BAD, "multiple of 32"),
    (dict(W=1 << 17), UNS, "32768"), (dict(ld=63), BAD, "row stride"), (dict(dtype=5), BAD, "dtype"),
    (dict(x=None), BAD, "null"), (dict(codes=None), BAD, "null"), (dict(scales=None), BAD, "null"),
    (dict(codes=P + 8), BAD, "16-byte"), (dict(x=P + 2), BAD, "aligned")])
def test_act8_pack_and_unpack_refuse(kw, code, part):
    a = dict(x=P, ld=64, dtype=0, codes=P, scales=P, T=3, W=64)
    a.update(kw)
    if a["W"] > 64:
        a["ld"] = a["W"]
    lib = _native.attn_lib()
    _refuses(lib.agpt_act8_pack(a["x"], a["ld"], a["dtype"], 0, a["codes"], a["scales"], a["T"], a["W"], None), code, part)
    _refuses(lib.agpt_act8_unpack(a["codes"], a["scales"], 0, a["x"], a["ld"], a["dtype"], a["T"], a["W"], None), code, part)


@pytest.mark.parametrize("kw,code,part", [
    (dict(T=-1), BAD, "T < 0"), (dict(out=0), BAD, "width"), (dict(W=40), BAD, "multiple of 32"),
    (dict(out=40000), UNS, "32768"), (dict(ld=31), BAD, "row stride"), (dict(dtype=5), BAD, "dtype"),
    (dict(dy=None), BAD, "null"), (dict(codes=None), BAD, "null"), (dict(dw=None), BAD, "null"),
    (dict(ws=None), BAD, "null"), (dict(n=10), BAD, "workspace"), (dict(dw=P + 4), BAD, "16-byte")])
def test_act8_wgrad_refuses(kw, code, part):
    a = dict(dy=P, ld=64, dtype=0, codes=P, scales=P, dw=P, db=P, ws=P, n=1 << 40, T=300, out=64, W=64)
    a.update(kw)
    if a["out"] > 64:
        a["ld"] = a["out"]
    lib = _native.attn_lib()
    _refuses(lib.agpt_act8_wgrad(a["dy"], a["ld"], a["dtype"], a["codes"], a["scales"], 0, a["dw"], a["db"], a["ws"],
                                 a["n"], a["T"], a["out"], a["W"], None), code, part)
    _refuses(lib.agpt_act8_relu_wgrad(a["dy"], a["ld"], a["dtype"], P, P + (1 << 30), a["codes"], a["scales"], 0, a["dw"],
                                      a["db"], a["ws"], a["n"], a["T"], a["out"], a["W"], None), code,
             "" if part == "width" else part)


@pytest.mark.parametrize("ld", [2**25 + 4, 2**26, 2**32 + 64])
def test_act8_wgrad_refuses_strides_past_its_offsets(ld):
    """24 rows of 2^25 fp32 columns are 3.2e9 bytes; from 2^26 on they pass 32 bits."""
    lib = _native.attn_lib()
    for out, W in ((200, 256), (128, 128)):
        _refuses(lib.agpt_act8_wgrad(P, ld, 0, P, P, 0, P, P, P, 1 << 40, 300, out, W, None), UNS, "2^25")
    _refuses(lib.agpt_act8_relu_wgrad(P, ld, 0, P, P + (1 << 40), P, P, 0, P, P, P, 1 << 40, 1, 128, 64, None), UNS, "2^25")


@pytest.mark.parametrize("kw,part", [(dict(out=66), "multiple of 32"), (dict(ld=66), "16-byte"), (dict(dy=P + 8), "16-byte"),
                                     (dict(hc=None), "null"), (dict(dh=None), "null"), (dict(dh=P), "overlap"),
                                     (dict(hc=P + 8), "16-byte")])
def test_act8_relu_wgrad_refuses(kw, part):
    a = dict(dy=P, ld=64, hc=P, dh=P + (1 << 30), out=64)
    a.update(kw)
    a["ld"] = max(a["ld"], a["out"])
    _refuses(_native.attn_lib().agpt_act8_relu_wgrad(a["dy"], a["ld"], 0, a["hc"], a["dh"], P, P, 0, P, P, P, 1 << 40, 300,
                                                     a["out"], 64, None), BAD, part)


def test_sizes():
    lib = _native.attn_lib()
    assert lib.agpt_act8_code_bytes(9, 64) == 16 * 64 and lib.agpt_act8_scale_bytes(9, 64) == 16 * 2
    assert lib.agpt_act8_code_bytes(0, 64) == 0 and lib.agpt_act8_code_bytes(-1, 64) == 0
    assert lib.agpt_embed_plan_ints(10, 65) == 20 + 66
    T = 2**31 - 5000  # sizes past 32 bits
    assert lib.agpt_embed_plan_workspace_bytes(T, 65) > 8 * T
    assert lib.agpt_act8_code_bytes(1 << 32, 512) == 1 << 41


def test_checkpoint_of_other_sizes_is_refused():
    """Act8 is public: bytes that do not fit its sizes never reach a kernel."""
    codes, scales = torch.zeros(16 * 64, dtype=torch.uint8), torch.zeros(32, dtype=torch.uint8)
    assert act8.Act8(codes, scales, 9, 64, False).device.type == "cpu"
    for args in ((codes[:-1], scales, 9, 64), (codes, scales[:-1], 9, 64), (codes, scales, 17, 64), (codes, scales, 9, 96),
                 (codes.int(), scales, 9, 64), (torch.zeros(2048, dtype=torch.uint8)[::2], scales, 9, 64),
                 (codes, scales.to("meta"), 9, 64)):
        with pytest.raises(ValueError):
            act8.Act8(*args, False)


def test_widths_past_an_int_are_refused():
    """Before they are cut to the C entry points' 32 bits."""
    with pytest.raises(ValueError, match="wider"):
        block._rows("x", torch.empty(1, 2**32 + 64, device="meta"))


def test_python_mirror_needs_a_gpu():
    x = torch.zeros(4, 64)
    tok = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: embed.embed_fwd(tok, x), lambda: embed.EmbedPlan(tok, 4), lambda: embed.embed_bwd(x, tok, 4),
                 lambda: embed.embed_bwd(x, tok), lambda: act8.pack(x),
                 lambda: block.qk_norm_rope_split(x, x[0], x[0]), lambda: block.qk_norm_rope_split_bwd(x, x, x, x, x, x)):
        with pytest.raises(ValueError):
            call()
