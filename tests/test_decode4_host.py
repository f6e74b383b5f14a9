"""The 4-bit decode operators without a GPU: the C structs' layouts, every refusal of the entry points (each
before any CUDA call), the Python wrappers' refusals, and the float64 oracle's own format."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from nanosaur2_web_b200 import _lib, ops
from oracle import decode4 as O4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD, UNSUP, OK = _lib.NSA_ERR_INVALID_ARGUMENT, _lib.NSA_ERR_UNSUPPORTED, _lib.NSA_OK
FAKE = 1 << 32   # never dereferenced: validation fails first


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layouts_match_c(tmp_path):
    structs = {"nsa_weight4": _lib.Weight4Desc, "nsa_linear4_desc": _lib.Linear4Desc, "nsa_kv4_cache": _lib.Kv4CacheDesc,
               "nsa_kv4_batch": _lib.Kv4Batch, "nsa_kv4_append_desc": _lib.Kv4AppendDesc,
               "nsa_kv4_attention_desc": _lib.Kv4AttentionDesc}
    lines, want = [], []
    for c, py in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        want.append(ctypes.sizeof(py))
        for name, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof({c}, {name}));')
            want.append(getattr(py, name).offset)
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "nsattn.h"\nint main(){' + "".join(lines) + "return 0;}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    assert [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()] == want


def test_weight_refusals():
    L = _lib.lib()
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    assert L.nsa_weight4_sizes(17, 129, 64, ctypes.byref(a), ctypes.byref(b)) == OK
    assert (a.value, b.value) == (32 * 2 * 64, 32 * 2 * 2 * 2)
    for n, k, g in ((0, 8, 32), (8, 0, 32), (8, 8, 16), (8, 8, 0)):
        assert L.nsa_weight4_sizes(n, k, g, None, None) == BAD

    def quant(codes=FAKE, scales=FAKE, W=FAKE, dtype=0, ld=0, group=32):
        w = _lib.Weight4Desc(40, 72, group, codes, scales)
        return L.nsa_quantize4(ctypes.byref(w), W, dtype, ld, None)
    assert L.nsa_quantize4(None, FAKE, 0, 0, None) == BAD
    for kw in (dict(codes=None), dict(scales=None), dict(codes=FAKE + 8), dict(W=None), dict(W=FAKE + 2), dict(dtype=2),
               dict(ld=71), dict(ld=-72), dict(group=48)):
        assert quant(**kw) == BAD, kw
    w = _lib.Weight4Desc(40, 72, 32, FAKE, FAKE)
    assert L.nsa_expand4(ctypes.byref(w), None, 0, None) == BAD
    assert L.nsa_expand4(ctypes.byref(w), FAKE + 1, 0, None) == BAD
    assert L.nsa_expand4(ctypes.byref(w), FAKE, 70, None) == BAD

    def lin(M=2, lda=0, ldc=0, resid=0, out=0, K=72, A=FAKE, C=FAKE + (1 << 20), bias=None):
        w = _lib.Weight4Desc(40, K, 32, FAKE, FAKE)
        d = _lib.Linear4Desc(M, lda, ldc, resid, out)
        return L.nsa_linear4(ctypes.byref(d), ctypes.byref(w), A, bias, C, None)
    for kw in (dict(M=-1), dict(K=76), dict(lda=64), dict(lda=76), dict(ldc=39), dict(out=3), dict(resid=1, out=1),
               dict(A=None), dict(A=FAKE + 8), dict(C=None), dict(C=FAKE + (1 << 20) + 2), dict(bias=FAKE + 2),
               dict(C=FAKE + 128)):
        assert lin(**kw) == BAD, kw
    assert b"overlap" in L.nsa_last_error()
    assert lin(M=0, A=None, C=None) == OK
    assert lin(K=98312) == UNSUP
    assert L.nsa_linear4(None, ctypes.byref(w), FAKE, None, FAKE, None) == BAD


CACHE = dict(n_pages=8, P=16, Hkv=2, D=128, codes=FAKE, scales=FAKE)
BATCH = dict(B=2, L=3, max_pages=4, table_ld=0, table=FAKE, start=FAKE, count=None)
OUT = FAKE + (1 << 24)


def cache_of(**kw):
    return _lib.Kv4CacheDesc(**{**CACHE, **{k: v for k, v in kw.items() if k in CACHE}})


def batch_of(**kw):
    return _lib.Kv4Batch(**{**BATCH, **{k: v for k, v in kw.items() if k in BATCH}})


COMMON = [(dict(D=96), UNSUP), (dict(D=512), UNSUP), (dict(P=8), BAD), (dict(P=24), BAD), (dict(P=2048), BAD),
          (dict(n_pages=-1), BAD), (dict(n_pages=1 << 30), UNSUP), (dict(Hkv=0), BAD), (dict(B=-1), BAD), (dict(L=-1), BAD), (dict(max_pages=-1), BAD),
          (dict(max_pages=1 << 27), BAD), (dict(table_ld=3), BAD), (dict(table=None), BAD), (dict(start=None), BAD),
          (dict(start=FAKE + 2), BAD), (dict(count=FAKE + 1), BAD), (dict(codes=FAKE + 4), BAD), (dict(scales=None), BAD)]


@pytest.mark.parametrize("kw,want", COMMON)
def test_cache_refusals(kw, want):
    L = _lib.lib()
    c, b = cache_of(**kw), batch_of(**kw)
    a = _lib.Kv4AppendDesc(Hq=4, in_dtype=0, ld=1024, bstride=3 * 1024, qOff=0, kOff=512, vOff=768, qo_ld=512, qo_bstride=1536, eps=1e-6)
    assert L.nsa_kv4_append(ctypes.byref(a), ctypes.byref(c), ctypes.byref(b), FAKE, FAKE, FAKE, None, OUT, None) == want
    assert L.nsa_kv4_read(ctypes.byref(c), ctypes.byref(b), OUT, 512, 1536, None) == want
    t = _lib.Kv4AttentionDesc(4, 512, 1536, 512, 1536, 0, 0, 0)
    assert L.nsa_kv4_attention(ctypes.byref(t), ctypes.byref(c), ctypes.byref(b), FAKE, OUT, FAKE, 1 << 40, None) == want
    assert L.nsa_kv4_attention(ctypes.byref(t), None, ctypes.byref(b), FAKE, OUT, FAKE, 1 << 40, None) == BAD
    assert L.nsa_kv4_read(ctypes.byref(c), None, OUT, 512, 1536, None) == BAD


def test_append_refusals():
    L = _lib.lib()
    base = dict(Hq=4, in_dtype=0, ld=1024, bstride=3 * 1024, qOff=0, kOff=512, vOff=768, qo_ld=512, qo_bstride=1536,
                sinOff=0, rope_rows=0, eps=1e-6)

    def call(qkv=FAKE, qw=FAKE, kw=FAKE, cs=None, out=OUT, batch={}, **d):
        desc = _lib.Kv4AppendDesc(**{**base, **d})
        return L.nsa_kv4_append(ctypes.byref(desc), ctypes.byref(cache_of()), ctypes.byref(batch_of(**batch)), qkv, qw, kw, cs,
                                out, None)
    for kw in (dict(Hq=3), dict(Hq=0), dict(in_dtype=5), dict(ld=1022), dict(ld=-1024), dict(bstride=2), dict(qOff=-4), dict(kOff=514),
               dict(vOff=1), dict(eps=-1.0), dict(eps=float("nan")), dict(qkv=None), dict(qkv=FAKE + 4), dict(qw=None),
               dict(kw=FAKE + 8), dict(cs=FAKE, rope_rows=0), dict(cs=FAKE, rope_rows=4, sinOff=-4),
               dict(cs=FAKE, rope_rows=4, sinOff=6), dict(cs=FAKE + 4, rope_rows=4), dict(out=None), dict(out=OUT + 8),
               dict(qo_ld=516), dict(qo_ld=504), dict(qo_bstride=1024), dict(out=FAKE + 64)):
        assert call(**kw) == BAD, kw
    assert b"overlap" in L.nsa_last_error()
    assert call(qkv=None, out=None, batch=dict(B=0)) == OK and call(qkv=None, out=None, batch=dict(L=0)) == OK
    assert L.nsa_kv4_append(None, ctypes.byref(cache_of()), ctypes.byref(batch_of()), FAKE, FAKE, FAKE, None, OUT, None) == BAD


def test_read_and_attention_refusals():
    L = _lib.lib()
    c, b = cache_of(), batch_of()
    for out, ld, bs in ((None, 512, 1536), (OUT + 2, 512, 1536), (OUT, 508, 1536), (OUT, 504, 1536), (OUT, 512, 1024)):
        assert L.nsa_kv4_read(ctypes.byref(c), ctypes.byref(b), out, ld, bs, None) == BAD
    base = dict(Hq=4, q_ld=512, q_bstride=1536, o_ld=512, o_bstride=1536, window=0, sinks=0, scale=0.0)

    def call(q=FAKE, out=OUT, ws=None, nbytes=0, batch={}, **d):
        desc = _lib.Kv4AttentionDesc(**{**base, **d})
        return L.nsa_kv4_attention(ctypes.byref(desc), ctypes.byref(c), ctypes.byref(batch_of(**batch)), q, out, ws, nbytes, None)
    for kw in (dict(Hq=5), dict(Hq=-4), dict(window=-1), dict(sinks=-1), dict(sinks=4), dict(scale=-1.0), dict(scale=float("inf")),
               dict(scale=float("nan")), dict(q_ld=508), dict(q_bstride=-8), dict(o_ld=504), dict(o_bstride=1024), dict(q=None),
               dict(q=FAKE + 8), dict(out=None), dict(out=FAKE + 64)):
        assert call(**kw) == BAD, kw
    assert b"overlap" in L.nsa_last_error()
    assert call(q=None, out=None, batch=dict(B=0)) == OK
    assert call(batch=dict(B=1 << 20, L=64, max_pages=1 << 26), q_bstride=512 * 64, o_bstride=512 * 64) == UNSUP   # too many blocks
    # a workspace where keys are split over CTAs: none for few short sequences, an error names the size otherwise
    d = _lib.Kv4AttentionDesc(**base)
    assert L.nsa_kv4_attention_workspace_size(ctypes.byref(d), ctypes.byref(c), ctypes.byref(b)) == 0
    big = batch_of(max_pages=4096)
    need = L.nsa_kv4_attention_workspace_size(ctypes.byref(d), ctypes.byref(c), ctypes.byref(big))
    assert need > 0
    for ws, n in ((None, 0), (FAKE, need - 1), (FAKE + 8, need)):
        assert call(ws=ws, nbytes=n, batch=dict(max_pages=4096)) == _lib.NSA_ERR_WORKSPACE
    assert str(need).encode() in L.nsa_last_error()
    d = _lib.Kv4AttentionDesc(**{**base, "Hq": 5})
    assert L.nsa_kv4_attention_workspace_size(ctypes.byref(d), ctypes.byref(c), ctypes.byref(b)) == 0


def test_wrappers_refuse_host_tensors_and_wrong_shapes():
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    W = ops.Weight4(torch.zeros((1, 1, 16, 64), dtype=torch.uint8), torch.zeros((1, 1, 16, 4), dtype=torch.bfloat16), 16, 64, 32)
    cache = ops.Kv4Cache(torch.zeros((2, 2, 1, 16, 32), dtype=torch.uint8), torch.zeros((2, 2, 1, 16, 2), dtype=torch.bfloat16))
    assert (cache.page, cache.Hkv, cache.D) == (16, 1, 64)
    table, start = torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    w = torch.ones(64)
    for call in (lambda: ops.linear4(x, W), lambda: ops.quantize4(x), lambda: ops.expand4(W),
                 lambda: ops.kv4_attention(q, cache, table, start), lambda: ops.kv4_read(cache, table, start, 1),
                 lambda: ops.kv4_append(torch.zeros((1, 1, 192)), cache, table, start, Hq=1, q_norm=w, k_norm=w, cs=None)):
        with pytest.raises(ops.NsaError, match="CUDA"):
            call()
    with pytest.raises(ops.NsaError, match="non-empty"):
        ops.quantize4(torch.zeros((0, 4)))
    with pytest.raises(ops.NsaError, match="head dims"):
        ops.kv4_cache(4, 1, 96)
    with pytest.raises(ops.NsaError, match="multiple of 16"):
        ops.kv4_cache(4, 1, 64, page=20)


def test_linear4_refuses_rows_that_fit_no_cluster():
    """K = 98304 leaves room for 2^19 outputs, not for 2^22: refused before anything is launched."""
    w = _lib.Weight4Desc(1 << 22, 98304, 32, FAKE, FAKE)
    d = _lib.Linear4Desc(1, 0, 0, 0, 0)
    assert _lib.lib().nsa_linear4(ctypes.byref(d), ctypes.byref(w), FAKE, None, FAKE + (1 << 30), None) == UNSUP
    assert b"shared memories" in _lib.lib().nsa_last_error()


def test_oracle_format():
    """Scales have five significant bits, are the smallest that reach the largest value, and every value of the
    format is a bf16 number within half a step of the input."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 64)) * np.exp(4 * rng.standard_normal((50, 1)))
    c, s = O4.quantise(x, 32)
    m, e = np.frexp(s)
    assert (m * 32 == np.rint(m * 32)).all() and (np.abs(c) <= 7).all()
    amax = np.abs(x).reshape(50, 2, 32).max(-1)
    assert (7 * s >= amax).all() and (7 * np.ldexp(m - 1 / 32, e) < amax).all()
    v = O4.values(c, s)
    assert (np.abs(v - x) <= s.repeat(32, -1) / 2).all()
    assert (torch.from_numpy(v).bfloat16().double().numpy() == v).all()


def test_batch_positions():
    """`positions` is refused below 0; the workspace's size does not depend on it."""
    L = _lib.lib()
    c, bad = cache_of(), _lib.Kv4Batch(**BATCH, positions=-1)
    t = _lib.Kv4AttentionDesc(4, 512, 1536, 512, 1536, 0, 0, 0)
    a = _lib.Kv4AppendDesc(Hq=4, in_dtype=0, ld=1024, bstride=3 * 1024, qOff=0, kOff=512, vOff=768, qo_ld=512, qo_bstride=1536, eps=1e-6)
    assert L.nsa_kv4_append(ctypes.byref(a), ctypes.byref(c), ctypes.byref(bad), FAKE, FAKE, FAKE, None, OUT, None) == BAD
    assert L.nsa_kv4_read(ctypes.byref(c), ctypes.byref(bad), OUT, 512, 1536, None) == BAD
    assert L.nsa_kv4_attention(ctypes.byref(t), ctypes.byref(c), ctypes.byref(bad), FAKE, OUT, FAKE, 1 << 40, None) == BAD
    assert b"positions" in L.nsa_last_error()
    size = lambda n: L.nsa_kv4_attention_workspace_size(ctypes.byref(t), ctypes.byref(c), ctypes.byref(_lib.Kv4Batch(**{**BATCH, "max_pages": 4096}, positions=n)))
    assert size(0) == size(50) == size(4096 * 16) == size(1 << 30) > 0


@pytest.mark.parametrize("sinks", [2 ** 31 - 1, 2 ** 31 - 15, 2 ** 31 - 16, 1 << 20])
def test_attention_plan_of_any_number_of_sinks(sinks):
    """Sinks that cover the whole table: planned like a call without a window."""
    L = _lib.lib()
    c, b = cache_of(), batch_of(max_pages=4096)
    size = lambda window, n: L.nsa_kv4_attention_workspace_size(
        ctypes.byref(_lib.Kv4AttentionDesc(4, 512, 1536, 512, 1536, window, n, 0)), ctypes.byref(c), ctypes.byref(b))
    assert size(16, sinks) == size(0, 0) > 0


def test_gemma_layer_decode_refuses_buffers_and_weights_of_other_sizes():
    """`linear`, which takes bf16 weights, works on pointers and pitches: with h_ready, buffers of more rows than x would
    have made it write past their qkv."""
    from nanosaur2_web_b200 import blocks
    bf, hid, inter = torch.bfloat16, 64, 48
    w = lambda *s: torch.zeros(s, dtype=bf)
    attn = dict(in_norm=torch.ones(hid), w_qkv=w(1536, hid), q_norm=torch.ones(256), k_norm=torch.ones(256), w_o=w(hid, 1024),
                post_norm=torch.ones(hid))
    mlp = dict(pre_norm=torch.ones(hid), w_gate_up=w(2 * inter, hid), w_down=w(hid, inter), post_norm=torch.ones(hid))
    cache = ops.Kv4Cache(torch.zeros((2, 2, 1, 16, 128), dtype=torch.uint8), w(2, 2, 1, 16, 8))
    make = lambda B, L, i=inter, dev="cpu": blocks.gemma_decode_buffers(B, L, hid, i, dev)

    def call(attn=attn, mlp=mlp, **kw):
        blocks.gemma_layer_decode(torch.zeros((1, 2, hid)), attn=attn, mlp=mlp, cs=None, cache=cache, h_ready="buffers" in kw,
                                  table=torch.zeros((1, 2), dtype=torch.int32), start=torch.zeros(1, dtype=torch.int32), **kw)
    good = make(1, 2)
    bad = [dict(buffers=make(1, 4)), dict(buffers=make(2, 2)), dict(buffers=make(2, 1)), dict(buffers=make(1, 1)), dict(buffers=make(1, 2, inter + 8)),
           dict(buffers={k: v for k, v in good.items() if k != "a"}), dict(buffers={**good, "gu": good["gu"].bfloat16()}),
           dict(buffers={**good, "o": torch.zeros((hid, 2)).T})]
    for kw in bad:
        with pytest.raises(ops.NsaError, match="the buffers are not"):
            call(**kw)
    for name, W in (("w_qkv", w(1536, hid - 8)), ("w_qkv", w(1280, hid)), ("w_o", w(hid, 512)), ("w_o", w(8, 1024))):
        with pytest.raises(ops.NsaError, match=name):
            call(attn={**attn, name: W})
    for name, W in (("w_gate_up", w(2 * inter, 8)), ("w_down", w(hid, inter + 8)), ("w_down", w(8, inter)), ("w_gate_up", w(95, hid))):
        with pytest.raises(ops.NsaError, match=name):
            call(mlp={**mlp, name: W})
    q4 = ops.Weight4(torch.zeros((4, 1, 16, 64), dtype=torch.uint8), torch.zeros((4, 1, 16, 4), dtype=bf), hid, 40, 32)
    with pytest.raises(ops.NsaError, match="w_down"):
        call(mlp={**mlp, "w_down": q4})
    for kw in (dict(buffers=make(1, 2, dev="meta")), dict(attn={**attn, "in_norm": torch.ones(hid, device="meta")})):
        with pytest.raises(ops.NsaError, match="x's device"):
            call(**kw)
    with pytest.raises(ops.NsaError, match="CUDA"):   # the sizes are right: on to the calls
        call(buffers=good)


@pytest.mark.parametrize("B,L", [(0, 1), (0, 3), (2, 0), (0, 0)])
def test_gemma_layer_decode_of_no_sequences_or_no_tokens(B, L):
    from nanosaur2_web_b200 import blocks
    bf, hid, inter = torch.bfloat16, 64, 48
    w = lambda *s: torch.zeros(s, dtype=bf)
    one = torch.ones(hid)
    attn = dict(in_norm=one, w_qkv=w(1536, hid), q_norm=torch.ones(256), k_norm=torch.ones(256), w_o=w(hid, 1024), post_norm=one)
    mlp = dict(pre_norm=one, w_gate_up=w(2 * inter, hid), w_down=w(hid, inter), post_norm=one)
    cache = ops.Kv4Cache(torch.zeros((2, 2, 1, 16, 128), dtype=torch.uint8), w(2, 2, 1, 16, 8))
    x = torch.zeros((B, L, hid))
    for buffers in (None, blocks.gemma_decode_buffers(B, L, hid, inter, "cpu")):
        assert blocks.gemma_layer_decode(x, attn=attn, mlp=mlp, cs=None, cache=cache, table=torch.zeros((B, 2), dtype=torch.int32),
                                         start=torch.zeros(B, dtype=torch.int32), buffers=buffers) is x
