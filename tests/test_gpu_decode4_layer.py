"""blocks.gemma_layer_decode: the 4-bit decode operators as they are used, one Gemma layer over a cache.

Against the layer in float64 (oracle/decode4.py's cache step and attention) on the same 4-bit weights, with the
operands that the path rounds to bf16 (h, q', a, h2, g) rounded there too: without that, h's rounding alone (2^-9 of a
value on average) would move 1 to 2% of the cached codes across a border, each by a whole step s of about 0.3, which is
4% of a first token's update.  What is left is fp32 against float64: a rounding to bf16 that falls on the other side moves
an operand by 2^-8 in about 1 of 10^4 cases, and one of 10^4 codes with it.  One value code off by s = 0.3 changes a by
0.3 in one of 256 dims, o (weights of 1 / 32 rms) by 0.01 of its unit scale, an update (norm weights of about 1.2) by 0.04 at
most over 640 columns, and the MLP half passes on as much: 0.1 max-abs and cosine >= 0.999 of the updates."""

import numpy as np
import pytest
import torch

from oracle import decode4 as O4
from tests._helpers import bf16_round

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
HID, INTER, H, D = 640, 2048, 4, 256


@pytest.fixture(scope="module", autouse=True)
def _lib_loaded():
    torch.cuda.set_device(DEV)
    from nanosaur2_web_b200 import _lib
    _lib.lib()
    yield
    torch.cuda.synchronize()


def t(x, dtype=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(device=DEV, dtype=dtype)


def n64(x):
    return x.double().cpu().numpy()


def layer_weights(rng, four=True):
    from nanosaur2_web_b200 import ops

    def lin(n, k):
        W = t(rng.standard_normal((n, k)) / np.sqrt(k))
        q = ops.quantize4(W, 32)
        return (q if four else ops.expand4(q)), n64(ops.expand4(q))

    def norm(n):
        return t(1 + 0.2 * rng.standard_normal(n))
    w = {k: lin(*s) for k, s in dict(qkv=(6 * D, HID), o=(HID, H * D), gu=(2 * INTER, HID), down=(HID, INTER)).items()}
    attn = {"in_norm": norm(HID), "w_qkv": w["qkv"][0], "q_norm": norm(D), "k_norm": norm(D), "w_o": w["o"][0], "post_norm": norm(HID)}
    mlp = {"pre_norm": norm(HID), "w_gate_up": w["gu"][0], "w_down": w["down"][0], "post_norm": norm(HID)}
    return attn, mlp, {k: v[1] for k, v in w.items()}


def bf16(x):
    return bf16_round(x.astype(np.float32)).astype(np.float64)


class Oracle:
    """The layer over its own cache of quantised keys and values, token by token, in float64."""

    def __init__(self, attn, mlp, w, cs, window, sinks):
        self.a, self.m = {k: n64(v) for k, v in attn.items() if "w_" not in k}, {k: n64(v) for k, v in mlp.items() if "w_" not in k}
        self.w, self.window, self.sinks, self.k, self.v = w, window, sinks, [], []
        L = cs.L
        self.cos, self.sin = n64(cs.buf[:cs.sinOff]).reshape(L, D // 2), n64(cs.buf[cs.sinOff:]).reshape(L, D // 2)

    def rms(self, x, w):
        return x / np.sqrt((x * x).mean() + 1e-6) * w

    def token(self, x):
        pos = len(self.k)
        qkv = self.w["qkv"] @ bf16(self.rms(x, self.a["in_norm"]))
        q = bf16(O4.norm_rope(qkv[:H * D].reshape(H, D), self.a["q_norm"], self.cos[pos], self.sin[pos], 1e-6))
        k = O4.norm_rope(qkv[H * D:(H + 1) * D], self.a["k_norm"], self.cos[pos], self.sin[pos], 1e-6)
        self.k.append(O4.values(*O4.quantise(k, 32)))
        self.v.append(O4.values(*O4.quantise(qkv[(H + 1) * D:], 32)))
        k, v = np.array(self.k), np.array(self.v)
        a = np.concatenate([O4.attention(q[h], k, v, pos, self.window, self.sinks, 1 / 16)[0] for h in range(H)])
        x = x + self.rms(self.w["o"] @ bf16(a), self.a["post_norm"])
        gu = self.w["gu"] @ bf16(self.rms(x, self.m["pre_norm"]))
        g, u = gu[:INTER], gu[INTER:]
        g = 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)))
        return x + self.rms(self.w["down"] @ bf16(g * u), self.m["post_norm"])


def close(got, want, base, what):
    err = np.abs(got - want).max()
    a, b = (got - base).ravel(), (want - base).ravel()
    cos = a @ b / np.linalg.norm(a) / np.linalg.norm(b)
    assert err <= 0.1 and cos >= 0.999, (what, err, cos)


@pytest.mark.parametrize("four,window,sinks", [(True, 0, 0), (True, 12, 3), (False, 12, 0)])
def test_layer_prompt_then_tokens(four, window, sinks):
    """Prompts of different lengths enter in one padded call, then tokens one by one and a few at once, each step
    captured once and replayed; pages are given out step by step."""
    from nanosaur2_web_b200 import ops
    from nanosaur2_web_b200.blocks import gemma_decode_buffers, gemma_layer_decode
    rng = np.random.default_rng(3 + window)
    attn, mlp, w = layer_weights(rng, four)
    cs = ops.ropeTable(64, D, 1e4, DEV)
    B, lens = 3, np.array([21, 5, 14])
    cache = ops.kv4_cache(B * 4, 1, D, 16, DEV)
    cache.codes.fill_(0xF0)
    cache.scales.fill_(float("nan"))
    table = t(rng.permutation(B * 4).reshape(B, 4), torch.int32)
    oracles = [Oracle(attn, mlp, w, cs, window, sinks) for _ in range(B)]
    kw = dict(attn=attn, mlp=mlp, cs=cs, cache=cache, table=table, window=window, sinks=sinks)
    # the prompts
    x = rng.standard_normal((B, 21, HID)).astype(np.float32)
    got = t(x)
    start = torch.zeros(B, dtype=torch.int32, device=DEV)
    gemma_layer_decode(got, start=start, count=t(lens, torch.int32), **kw)
    ops.check_device(DEV)
    for b in range(B):
        want = np.array([oracles[b].token(x[b, i].astype(np.float64)) for i in range(lens[b])])
        close(n64(got[b, :lens[b]]), want, x[b, :lens[b]], f"prompt {b}")
    start += t(lens, torch.int32)
    # tokens: one at a time, then three
    for L, steps in ((1, 4), (3, 2)):
        buf = gemma_decode_buffers(B, L, HID, INTER, DEV)
        xin = torch.zeros((B, L, HID), device=DEV)
        side = torch.cuda.Stream(DEV)
        side.wait_stream(torch.cuda.current_stream(DEV))
        with torch.cuda.stream(side):
            gemma_layer_decode(xin, start=start, buffers=buf, **kw)   # warm-up; the step itself writes the slots again
        torch.cuda.current_stream(DEV).wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gemma_layer_decode(xin, start=start, buffers=buf, **kw)
        for step in range(steps):
            x = rng.standard_normal((B, L, HID)).astype(np.float32)
            xin.copy_(t(x))
            g.replay()
            ops.check_device(DEV)
            for b in range(B):
                want = np.array([oracles[b].token(x[b, i].astype(np.float64)) for i in range(L)])
                close(n64(xin[b]), want, x[b], f"step {step} of {L}, sequence {b}")
            start += L


def test_layers_chain_their_norms_and_refuse():
    from nanosaur2_web_b200 import ops
    from nanosaur2_web_b200.blocks import gemma_decode_buffers, gemma_layer_decode
    rng = np.random.default_rng(8)
    layers = [layer_weights(rng)[:2] for _ in range(2)]
    cs = ops.ropeTable(32, D, 1e4, DEV)
    table, start = t([[0, 1]], torch.int32), t([0], torch.int32)
    x0 = t(rng.standard_normal((1, 4, HID)))
    outs = []
    for chained in (False, True):
        x, buf = x0.clone(), gemma_decode_buffers(1, 4, HID, INTER, DEV)
        caches = [ops.kv4_cache(2, 1, D, 16, DEV) for _ in layers]
        for i, (attn, mlp) in enumerate(layers):
            nxt = layers[i + 1][0]["in_norm"] if chained and i == 0 else None
            gemma_layer_decode(x, attn=attn, mlp=mlp, cs=cs, cache=caches[i], table=table, start=start, buffers=buf,
                               h_ready=chained and i == 1, next_norm=nxt)
        outs.append(x)
    ops.check_device(DEV)
    assert torch.equal(outs[0], outs[1])
    attn, mlp = layers[0]
    kw = dict(attn=attn, mlp=mlp, cs=cs, table=table, start=start)
    with pytest.raises(ops.NsaError, match="contiguous float32"):
        gemma_layer_decode(x0.bfloat16(), cache=caches[0], **kw)
    with pytest.raises(ops.NsaError, match="cache must hold"):
        gemma_layer_decode(x0, cache=ops.kv4_cache(2, 1, 128, 16, DEV), **kw)
    with pytest.raises(ops.NsaError, match="h_ready"):
        gemma_layer_decode(x0, cache=caches[0], h_ready=True, **kw)


def test_prompt_through_the_bf16_layer_and_its_cache_agree():
    """The same prompt through gemma_layer (bf16 weights expanded from the 4-bit ones, attention over exact keys) and
    through gemma_layer_decode: the difference is the cache's four bits, whose relative error per value is at most
    s / 2 of a group's largest 7 s."""
    from nanosaur2_web_b200 import ops
    from nanosaur2_web_b200.blocks import gemma_layer, gemma_layer_decode
    rng = np.random.default_rng(9)
    attn, mlp, _ = layer_weights(rng)
    L = 48
    cs = ops.ropeTable(L, D, 1e4, DEV)
    x0 = t(rng.standard_normal((2, L, HID)))
    exp = ops.expand4
    a16 = dict(attn, w_qkv=exp(attn["w_qkv"]), w_o=exp(attn["w_o"]))
    m16 = dict(mlp, w_gate_up=exp(mlp["w_gate_up"]), w_down=exp(mlp["w_down"]))
    x1, x2 = x0.clone(), x0.clone()
    gemma_layer(x1, attn=a16, mlp=m16, cs=cs)
    cache = ops.kv4_cache(2 * 3, 1, D, 16, DEV)
    gemma_layer_decode(x2, attn=attn, mlp=mlp, cs=cs, cache=cache, table=t([[0, 1, 2], [3, 4, 5]], torch.int32),
                       start=torch.zeros(2, dtype=torch.int32, device=DEV))
    ops.check_device(DEV)
    a, b = n64(x1 - x0), n64(x2 - x0)
    rel = np.linalg.norm(a - b) / np.linalg.norm(a)
    # a code is off by s / 2 at most, uniformly: s / sqrt(12) against values of rms about 7 s / 2: 0.08 of v, averaged
    # over keys or not; scores move alike; two halves of the layer pass it on
    assert rel <= 0.25, rel
