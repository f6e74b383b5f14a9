"""Measured cases of the token-by-token operators of a transformer layer: the linear with 4-bit weights and
group scales, the quantiser that makes those weights, the step that normalises, rotates and stores new
tokens in a paged 4-bit key/value cache, and the attention that reads that cache.

``run`` computes each operator in its plain form (elementary torch operations in fp32, or fp64 where a
value decides between two codes), or with ``own`` through the framework's entry points.

The 4-bit format, shared by weights and cache.  A group of consecutive values has one scale s, the smallest
number with five significant bits that is >= (largest magnitude of the group) / 7, and codes
c = round(x / s), ties to even, -7 <= c <= 7, stored as c + 8.  Groups whose largest magnitude is below
2^-110 have s = 0 and c = 0.  s has five significant bits and c three, so s * c is a bf16 number exactly.

* Weights [N, K], groups of G = 32, 64 or 128 along K, rows padded to 16 and K to 128 with zeros:
  codes uint8 [N/16, K/128, 16, 64]; of the 128 values of a row's chunk, the 32-bit word at byte 16 c + 4 i
  holds values 32 i + 8 c + e, e = 0..7, e even in nibble e / 2 and e odd in nibble 4 + (e - 1) / 2.
  scales bf16 [N/16, K/128, 16, 128/G].
* Cache pages of P tokens: codes uint8 [pages, 2, Hkv, P, D/2] (keys, then values; value 2 j in the low
  and 2 j + 1 in the high nibble of byte j), scales bf16 [pages, 2, Hkv, P, D/32] (groups of 32 along D).
"""

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
THETA = 1e4


# ------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one new token through the Gemma text encoder's output projection: latency
        dict(name="linear_1_row_640x1024", op="linear4", M=1, N=640, K=1024, G=32, bias=False, out="f32"),
        # a handful of sequences through the same model's gate|up projection, bf16 operand for the next step
        dict(name="linear_5_rows_4096x640", op="linear4", M=5, N=4096, K=640, G=64, bias=False, out="bf16"),
        # one token of a wide model: the weights' bytes are everything
        dict(name="linear_1_row_16384x8192", op="linear4", M=1, N=16384, K=8192, G=128, bias=False, out="f32"),
        # a batch of sequences decoding together, with a bias
        dict(name="linear_24_rows_8200x4096", op="linear4", M=24, N=8200, K=4096, G=32, bias=True, out="f32"),
        # loading the Gemma q|k|v projection
        dict(name="quantize_1536x640", op="quantize4", N=1536, K=640, G=32, dtype="bf16"),
        # loading a wide fp32 weight whose width is no multiple of the group
        dict(name="quantize_8192x8200", op="quantize4", N=8192, K=8200, G=64, dtype="f32"),
        # one new token of one sequence, Gemma heads
        dict(name="append_1_token", op="kv4_append", B=1, L=1, Hq=4, Hkv=1, D=256, P=16, T=777, ragged=False,
             dtype="f32"),
        # a batch of prompts of different lengths entering the cache, grouped heads of 128
        dict(name="append_16x500_tokens", op="kv4_append", B=16, L=500, Hq=32, Hkv=8, D=128, P=64, T=2000,
             ragged=True, dtype="bf16"),
        # one token of one sequence over a thousand cached ones, Gemma's global layer: latency
        dict(name="attend_1_over_1024", op="kv4_attention", B=1, L=1, Hq=4, Hkv=1, D=256, P=16, T=1024,
             ragged=False, window=0, sinks=0),
        # Gemma's local layer: a window of 512 and four first tokens, sequences of different lengths
        dict(name="attend_16_window_512", op="kv4_attention", B=16, L=1, Hq=4, Hkv=1, D=256, P=64, T=4096,
             ragged=True, window=512, sinks=4),
        # a serving batch, grouped heads of 128, sequences of different lengths
        dict(name="attend_40_over_8192", op="kv4_attention", B=40, L=1, Hq=32, Hkv=8, D=128, P=64, T=8192,
             ragged=True, window=0, sinks=0),
        # four draft tokens checked against one long sequence
        dict(name="attend_4_tokens_131071", op="kv4_attention", B=1, L=4, Hq=32, Hkv=8, D=128, P=128, T=131071,
             ragged=False, window=0, sinks=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear4", "linear4", "quantize4", "kv4_append", "kv4_attention", "kv4_attention"])
    if op == "linear4":
        K = 8 * _log(rng, 8, 1500)
        N = min(_log(rng, 40, 20000), 100_000_000 // K)
        return dict(op=op, M=_log(rng, 1, 40), N=N, K=K, G=rng.choice([32, 64, 128]), bias=rng.random() < 0.5,
                    out=rng.choice(["f32", "bf16"]))
    if op == "quantize4":
        K = _log(rng, 60, 9000)
        return dict(op=op, N=min(_log(rng, 30, 12000), 60_000_000 // K), K=K, G=rng.choice([32, 64, 128]),
                    dtype=rng.choice(["f32", "bf16"]))
    D, group = rng.choice([64, 128, 256]), rng.choice([1, 2, 3, 4, 5, 8])
    Hkv = rng.choice([1, 2, 4, 8])
    P = rng.choice([16, 32, 64, 128])
    if op == "kv4_append":
        L = _log(rng, 1, 1500)
        B = min(_log(rng, 1, 24), max(1, 30_000_000 // (L * D * Hkv * (group + 2))))
        return dict(op=op, B=B, L=L, Hq=Hkv * group, Hkv=Hkv, D=D, P=P, T=L + rng.randrange(0, 2000),
                    ragged=rng.random() < 0.5, dtype=rng.choice(["f32", "bf16"]))
    L = _log(rng, 1, 12)
    T = L + _log(rng, 1, 60000)
    B = min(_log(rng, 1, 48), max(1, 150_000_000 // (T * D * Hkv)))
    window = 0 if rng.random() < 0.5 else _log(rng, 16, 4096)
    return dict(op=op, B=B, L=L, Hq=Hkv * group, Hkv=Hkv, D=D, P=P, T=T, ragged=rng.random() < 0.7, window=window,
                sinks=rng.choice([0, 1, 4, 64]) if window else 0)


def _lengths(case):
    """Tokens of each sequence after the step (the new ones among them)."""
    B, T, L = case["B"], case["T"], case["L"]
    if not case["ragged"]:
        return [T] * B
    return [max(L, T - (b * 37 % 64) * T // 100) for b in range(B)]


def _counts(case):
    """New tokens of each sequence (of the L rows it has in the batch)."""
    B, L = case["B"], case["L"]
    return [L - (b * 29 % 50) * L // 100 for b in range(B)] if case["ragged"] else [L] * B


def _visible(n, L, window, sinks):
    """(query, key) pairs and distinct keys that L queries, the last of them at position n - 1, see."""
    if not window:
        return sum(range(n - L + 1, n + 1)), n
    pairs = sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(n - L, n))
    lo = max(0, n - L + 1 - window)
    return pairs, n - lo + min(sinks, lo)


def work(case):
    op = case["op"]
    if op == "linear4":
        M, N, K = case["M"], case["N"], case["K"]
        groups = -(-K // case["G"])
        return {"bytes": N * K / 2 + 2 * N * groups + 2 * M * K + (4 * N if case["bias"] else 0) +
                (4 if case["out"] == "f32" else 2) * M * N, "flops": 2 * M * N * K}
    if op == "quantize4":
        N, K = case["N"], case["K"]
        # the weight in, codes and scales out, and the values that they stand for out once (they are returned)
        return {"bytes": N * K * ((4 if case["dtype"] == "f32" else 2) + 0.5 + 2) + 2 * N * -(-K // case["G"]),
                "flops": 4 * N * K}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if op == "kv4_append":
        n = sum(_counts(case))
        esz = 4 if case["dtype"] == "f32" else 2
        # q|k|v in, q' out, codes and scales out, and the cached values out once (they are returned)
        return {"bytes": n * (D * (Hq + 2 * Hkv) * esz + 2 * D * Hq + 2 * Hkv * (D // 2 + D // 16) + 4 * Hkv * D +
                              4 * D), "flops": n * D * (8 * Hq + 16 * Hkv)}
    seen = [_visible(n, case["L"], case["window"], case["sinks"]) for n in _lengths(case)]
    return {"bytes": sum(k for _, k in seen) * 2 * Hkv * (D // 2 + D // 16) + 4 * case["B"] * case["L"] * Hq * D,
            "flops": 4 * Hq * D * sum(p for p, _ in seen)}


# ------------------------------------------------------------------------------ the format, in plain torch

def _scale(amax):
    """The smallest five-bit number >= amax / 7 (fp64), 0 below 2^-110 * (1 / 7)."""
    m, e = torch.frexp(amax / 7)
    s = torch.ldexp(torch.ceil(m * 32) / 32, e)
    return torch.where(amax < 2.0 ** -110, torch.zeros_like(s), s)


def _quantise(x, group):
    """x [..., n * group] -> integer codes in -7..7 and fp64 scales [..., n]."""
    x = x.double().unflatten(-1, (-1, group))
    s = _scale(x.abs().amax(-1))
    c = torch.round(x / torch.where(s > 0, s, torch.ones_like(s))[..., None])
    return torch.where(s[..., None] > 0, c, torch.zeros_like(c)).flatten(-2), s


def _pack_weight(c, s, N, K, G):
    """Codes and scales of the padded weight (multiples of 16 and 128) in the tiled order."""
    Np, Kp = c.shape
    n = (c + 8).to(torch.uint8).view(Np // 16, 16, Kp // 128, 4, 4, 2, 2, 2)      # tile, row, chunk, i, c, lb, h, hb
    n = n.permute(0, 2, 1, 4, 3, 7, 5, 6)                                          # tile, chunk, row, c, i, hb, lb, h
    codes = (n[..., 0] | (n[..., 1] << 4)).reshape(Np // 16, Kp // 128, 16, 64).contiguous()
    scales = s.to(torch.bfloat16).view(Np // 16, 16, Kp // 128, 128 // G).permute(0, 2, 1, 3).contiguous()
    return codes, scales


def _unpack_weight(codes, scales, N, K):
    """The fp32 weight [N, K] that codes and scales stand for."""
    T, C = codes.shape[:2]
    n = torch.stack([codes & 15, codes >> 4], -1).view(T, C, 16, 4, 4, 2, 2, 2)    # tile, chunk, row, c, i, hb, lb, h
    n = n.permute(0, 2, 1, 4, 3, 6, 7, 5).reshape(T * 16, C * 128).float() - 8
    s = scales.float().permute(0, 2, 1, 3).reshape(T * 16, -1)
    return (n.view(T * 16, s.shape[1], -1) * s[..., None]).view(T * 16, C * 128)[:N, :K]


def _pad_weight(W):
    N, K = W.shape
    return torch.nn.functional.pad(W, (0, -K % 128, 0, -N % 16))


# ------------------------------------------------------------------------------------------------ the state

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _table(case, g):
    """A page table with the sequences' pages scattered over the pool."""
    mp = -(-case["T"] // case["P"])
    return torch.randperm(case["B"] * mp, device=DEV, generator=g).to(torch.int32).view(case["B"], mp)


def _dtype(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case=case)
    if case["op"] == "linear4":
        M, N, K, G = case["M"], case["N"], case["K"], case["G"]
        W = _randn(g, N, K) / math.sqrt(K)
        codes, scales = _pack_weight(*_quantise(_pad_weight(W), G), N, K, G)
        st.update(codes=codes, scales=scales, x=_randn(g, M, K).bfloat16(),
                  bias=0.1 * _randn(g, N) if case["bias"] else None)
    elif case["op"] == "quantize4":
        N, K = case["N"], case["K"]
        # rows and columns of different sizes, as trained weights have
        W = _randn(g, N, K) * (1 + 0.5 * _randn(g, N, 1).abs()) * (0.3 + _randn(g, 1, K).abs()) / math.sqrt(K)
        st.update(W=W.to(_dtype(case["dtype"])))
    elif case["op"] == "kv4_append":
        B, L, Hq, Hkv, D, P = (case[k] for k in ("B", "L", "Hq", "Hkv", "D", "P"))
        start = torch.tensor(_lengths(case), dtype=torch.int32) - L
        qkv = _randn(g, B, L, (Hq + 2 * Hkv) * D) * (0.5 + _randn(g, (Hq + 2 * Hkv) * D).abs())
        pos = torch.arange(case["T"], device=DEV, dtype=torch.float64)
        a = pos[:, None] * (THETA ** (-torch.arange(D // 2, device=DEV, dtype=torch.float64) / (D // 2)))
        table = _table(case, g)
        pages = table.numel()
        st.update(qkv=qkv.to(_dtype(case["dtype"])), start=start.to(DEV), table=table,
                  count=torch.tensor(_counts(case), dtype=torch.int32, device=DEV),
                  q_norm=1 + 0.2 * _randn(g, D), k_norm=1 + 0.2 * _randn(g, D),
                  cs=torch.cat([a.cos().flatten(), a.sin().flatten()]).float(),
                  codes=torch.full((pages, 2, Hkv, P, D // 2), 0x88, dtype=torch.uint8, device=DEV),
                  scales=torch.zeros((pages, 2, Hkv, P, D // 32), dtype=torch.bfloat16, device=DEV),
                  q=torch.zeros((B, L, Hq * D), dtype=torch.bfloat16, device=DEV),
                  kv=torch.zeros((B, L, 2 * Hkv * D), dtype=torch.bfloat16, device=DEV))
    else:
        B, L, Hq, Hkv, D, P = (case[k] for k in ("B", "L", "Hq", "Hkv", "D", "P"))
        table = _table(case, g)
        # keys after their norm (a few large channels), values of about unit size
        x = _randn(g, table.numel(), 2, Hkv, P, D)
        x[:, 0] *= 0.6 + 0.4 * _randn(g, D).abs()
        c, s = _quantise(x, 32)
        del x
        n = (c + 8).to(torch.uint8)
        del c
        st.update(codes=n[..., 0::2] | (n[..., 1::2] << 4), scales=s.to(torch.bfloat16), table=table,
                  start=(torch.tensor(_lengths(case), dtype=torch.int32) - L).to(DEV),
                  q=(1.5 * _randn(g, B, L, Hq * D)).bfloat16())
    return st


# ------------------------------------------------------------------------------------------ the plain forms

def _plain_linear(st):
    case = st["case"]
    y = st["x"].float() @ _unpack_weight(st["codes"], st["scales"], case["N"], case["K"]).T
    if st["bias"] is not None:
        y = y + st["bias"]
    return {"y": y.to(_dtype(case["out"]))}


def _plain_quantize(st):
    case = st["case"]
    c, s = _quantise(_pad_weight(st["W"]), case["G"])
    v = c.unflatten(-1, (-1, case["G"])) * s[..., None]
    return {"values": v.flatten(-2)[:case["N"], :case["K"]].bfloat16()}


def _norm_rope(x, w, cos, sin):
    """x [B, L, H, D]: per-head RMSNorm times w, then the rotation of pairs (i, i + D/2)."""
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    a, b = y.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(st):
    case = st["case"]
    B, L, Hq, Hkv, D = (case[k] for k in ("B", "L", "Hq", "Hkv", "D"))
    q, k, v = st["qkv"].split([Hq * D, Hkv * D, Hkv * D], -1)
    cos, sin = st["cs"].view(2, case["T"], D // 2)
    i = torch.arange(L, device=DEV)
    pos = (st["start"].long()[:, None] + i).clamp(max=case["T"] - 1)
    live = (i < st["count"][:, None])[..., None]
    cos, sin = cos[pos][:, :, None], sin[pos][:, :, None]
    qn = _norm_rope(q.float().unflatten(-1, (Hq, D)), st["q_norm"], cos, sin)
    # the keys in fp64: a value next to the border of two codes decides by the last bits
    kn = _norm_rope(k.double().unflatten(-1, (Hkv, D)), st["k_norm"].double(), cos.double(), sin.double())
    c, s = _quantise(torch.cat([kn.flatten(-2), v.double()], -1), 32)
    kv = (c.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)
    return {"q": torch.where(live, qn.flatten(-2).bfloat16(), st["q"]), "kv": torch.where(live, kv.bfloat16(), st["kv"])}


def _cached(st, which):
    """The cached keys (0) or values (1) of every sequence, fp32 [B, Hkv, tokens, D]."""
    t = st["table"].long()
    n = st["codes"][:, which][t]                                                   # [B, pages, Hkv, P, D/2]
    s = st["scales"][:, which][t].float()
    x = torch.stack([n & 15, n >> 4], -1).flatten(-2).float() - 8
    x = x.unflatten(-1, (-1, 32)) * s[..., None]
    return x.flatten(-2).permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_attention(st):
    case = st["case"]
    B, L, Hq, Hkv, D = (case[k] for k in ("B", "L", "Hq", "Hkv", "D"))
    q = st["q"].float().view(B, L, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    s = q @ _cached(st, 0).transpose(-1, -2) / math.sqrt(D)
    j = torch.arange(s.shape[-1], device=DEV)
    p = (st["start"][:, None] + torch.arange(L, device=DEV)).repeat_interleave(Hq // Hkv, 1)[:, None, :, None]
    see = j <= p
    if case["window"]:
        see = see & ((j > p - case["window"]) | (j < case["sinks"]))
    s = s.masked_fill(~see, float("-inf"))
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = (e / e.sum(-1, keepdim=True)) @ _cached(st, 1)
    return {"out": o.view(B, Hkv, L, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, L, Hq * D).bfloat16()}


# --------------------------------------------------------------------------------- the framework's operators

def _own(st):
    from nanosaur2_web_b200 import ops
    case = st["case"]
    if case["op"] == "linear4":
        W = ops.Weight4(st["codes"], st["scales"], case["N"], case["K"], case["G"])
        return {"y": ops.linear4(st["x"], W, bias=st["bias"], out_dtype=_dtype(case["out"]))}
    if case["op"] == "quantize4":
        return {"values": ops.expand4(ops.quantize4(st["W"], case["G"]))}
    cache = ops.Kv4Cache(st["codes"], st["scales"])
    if case["op"] == "kv4_append":
        cs = ops.RopeTable(st["cs"], case["T"] * (case["D"] // 2), case["T"], case["D"])
        ops.kv4_append(st["qkv"], cache, st["table"], st["start"], count=st["count"], Hq=case["Hq"],
                       q_norm=st["q_norm"], k_norm=st["k_norm"], cs=cs, eps=EPS, out=st["q"])
        ops.kv4_read(cache, st["table"], st["start"], case["L"], count=st["count"], out=st["kv"])
        return {"q": st["q"], "kv": st["kv"]}
    return {"out": ops.kv4_attention(st["q"], cache, st["table"], st["start"], window=case["window"],
                                     sinks=case["sinks"])}


def run(state):
    if own:
        return _own(state)
    return {"linear4": _plain_linear, "quantize4": _plain_quantize, "kv4_append": _plain_append,
            "kv4_attention": _plain_attention}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------- in 64 bits

def _exact_scale(amax):
    """The five-bit scale by search: candidates (16 + i) / 16 * 2^e around amax / 7, the smallest that is enough."""
    e = torch.floor(torch.log2((amax / 7).clamp(min=2.0 ** -200))) - 1
    s = torch.full_like(amax, float("inf"))
    for de in range(3):
        for i in range(16):
            cand = (16 + i) / 16 * torch.exp2(e + de)
            s = torch.where((7 * cand >= amax) & (cand < s), cand, s)
    return torch.where(amax < 2.0 ** -110, torch.zeros_like(s), s)


def _exact_values(x, group):
    """The values that the format keeps of x [rows, n] (fp64), n padded to the group with zeros."""
    n = x.shape[1]
    x = torch.nn.functional.pad(x, (0, -n % group)).view(x.shape[0], -1, group)
    s = _exact_scale(x.abs().max(-1, keepdim=True).values)
    t = x.abs() / s.clamp(min=2.0 ** -300)
    lo = torch.floor(t)
    up = (t - lo > 0.5) | ((t - lo == 0.5) & (lo % 2 == 1))
    return (torch.sign(x) * (lo + up) * s).view(x.shape[0], -1)[:, :n]


def _exact_weight(st):
    """fp64 [N, K] by looking each value's word, nibble and group up."""
    case = st["case"]
    N, K, G = case["N"], case["K"], case["G"]
    n, k = torch.arange(N, device=DEV)[:, None], torch.arange(K, device=DEV)
    r, e = k % 128, k % 8
    word = 4 * ((r // 8) % 4) + r // 32
    nib = torch.where(e % 2 == 0, e // 2, 4 + e // 2)
    at = 4 * word + nib // 2
    w = torch.empty((N, K), dtype=torch.float64, device=DEV)
    step = max(1, (1 << 25) // K)
    for a in range(0, N, step):
        m = n[a:a + step]
        byte = st["codes"][m // 16, k // 128, m % 16, at].int()
        c = ((byte >> (4 * (nib % 2))) & 15) - 8
        w[a:a + step] = c.double() * st["scales"][m // 16, k // 128, m % 16, r // G].double()
    return w


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear4":
        y = torch.einsum("mk,nk->mn", st["x"].double(), _exact_weight(st))
        return {"y": y if st["bias"] is None else y + st["bias"].double()}
    if case["op"] == "quantize4":
        return {"values": _exact_values(st["W"].double(), case["G"])}
    B, L, Hq, Hkv, D, P = (case[k] for k in ("B", "L", "Hq", "Hkv", "D", "P"))
    if case["op"] == "kv4_append":
        out = {"q": st["q"].double(), "kv": st["kv"].double()}
        x = st["qkv"].double()
        half = D // 2
        cs = st["cs"].double()
        for b, (n, m) in enumerate(zip(_lengths(case), _counts(case))):
            pos = torch.arange(n - L, n - L + m, device=DEV)
            z = x[b, :m].view(m, Hq + 2 * Hkv, D)
            qk = z[:, :Hq + Hkv] / (z[:, :Hq + Hkv].pow(2).sum(-1, keepdim=True) / D + EPS).sqrt()
            qk = torch.cat([qk[:, :Hq] * st["q_norm"].double(), qk[:, Hq:] * st["k_norm"].double()], 1)
            i = torch.arange(half, device=DEV)
            c = cs[pos[:, None] * half + i][:, None]
            s = cs[case["T"] * half + pos[:, None] * half + i][:, None]
            rot = torch.empty_like(qk)
            rot[..., :half] = qk[..., :half] * c - qk[..., half:] * s
            rot[..., half:] = qk[..., half:] * c + qk[..., :half] * s
            out["q"][b, :m] = rot[:, :Hq].reshape(m, -1)
            out["kv"][b, :m] = _exact_values(torch.cat([rot[:, Hq:], z[:, Hq + Hkv:]], 1).reshape(m, -1), 32)
        return out
    out = torch.zeros((B, L, Hq * D), dtype=torch.float64, device=DEV)
    G = Hq // Hkv
    for b, n in enumerate(_lengths(case)):
        j = torch.arange(n, device=DEV)
        page, slot = st["table"][b, j // P].long(), j % P
        kv = []
        for which in (0, 1):
            byte = st["codes"][page, which, :, slot]                                # [n, Hkv, D/2]
            x = torch.empty((n, Hkv, D), dtype=torch.float64, device=DEV)
            x[..., 0::2] = (byte % 16).double() - 8
            x[..., 1::2] = (byte // 16).double() - 8
            sc = st["scales"][page, which, :, slot].double()
            kv.append((x * sc.repeat_interleave(32, -1)).transpose(0, 1))
        q = st["q"][b].double().view(L, Hkv, G, D)
        for i in range(L):
            p = n - L + i
            ok = j <= p
            if case["window"]:
                ok &= (j > p - case["window"]) | (j < case["sinks"])
            w = torch.softmax((q[i] @ kv[0].transpose(1, 2) / D ** 0.5).masked_fill(~ok, float("-inf")), -1)
            out[b, i] = (w @ kv[1]).reshape(-1)
    return {"out": out}
