"""The 4-bit decode operators on the GPU (quantize4 / expand4 / linear4, kv4_append / kv4_read /
kv4_attention and blocks.gemma_layer_decode) against float64 (oracle/decode4.py).

Tolerances.  Codes and scales are decided exactly, so quantised weights, cached keys and values and their
bf16 read-backs are compared for equality.  linear4: exact products summed in fp32, within a group and then
over the groups; a chain of n additions errs by at most n 2^-23 sum |s c x| (2^-23: a sum may truncate), n =
group + K / group + 16 for the joins.  kv4_append's q': fp32 arithmetic, about 20 roundings of 2^-24 on
|y1| + |y2| of a rotated pair, then one bf16 rounding (2^-8).  kv4_attention: scores are fp32 sums of D exact
products (D 2^-23 sum |q k| scale, entering the weights by exp), the weights carry at least 15 bits more
than the exp's own 2^-21, so a weight errs by eps = 2 (D 2^-23 max sum |q k| scale + 2^-15) relative, the
output by eps sum p |v|, then one bf16 rounding."""

import numpy as np
import pytest
import torch

from oracle import decode4 as O4

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
BF = torch.bfloat16


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


def check_device():
    from nanosaur2_web_b200.ops import check_device as chk
    chk(DEV)


# ------------------------------------------------------------------------------------------- weights

def weights(rng, N, K, special=True):
    W = (rng.standard_normal((N, K)) * np.exp(rng.standard_normal((N, 1)))).astype(np.float32)
    if special:
        W[0] = 0
        W[min(1, N - 1), :] = np.round(W[min(1, N - 1), :] * 4) / 4 * 1.75   # multiples of a scale and its ties
        W[min(2, N - 1), ::3] *= 1e-37                                        # below 2^-110 and subnormal next to ordinary
        W[min(3, N - 1), :] = np.float32(2.0 ** -112)                         # a row that is stored as zeros
        W[min(4, N - 1), ::5] *= np.float32(3e36)                             # saturates at 2^120
    return W


@pytest.mark.parametrize("N,K,group,dtype", [(1, 1, 32, "f32"), (16, 128, 32, "bf16"), (17, 129, 64, "f32"),
                                             (40, 72, 128, "bf16"), (33, 640, 32, "f32"), (5, 1000, 64, "bf16")])
def test_quantize4_codes_scales_and_expansion(N, K, group, dtype):
    from nanosaur2_web_b200.ops import expand4, quantize4
    rng = np.random.default_rng(N * 1000 + K)
    Wt = t(weights(rng, N, K), BF if dtype == "bf16" else torch.float32)
    wide = torch.full((N, K + 5), float("nan"), device=DEV, dtype=Wt.dtype)   # the columns past K are never read
    wide[:, :K] = Wt
    q = quantize4(wide[:, :K], group)
    y = expand4(q)
    pad = torch.full((N, K + 3), 7.0, device=DEV, dtype=BF)
    expand4(q, pad[:, :K])
    check_device()
    W = np.zeros((N, -(-K // 128) * 128))
    W[:, :K] = n64(Wt)
    c, s = O4.quantise(W, group)
    codes, scales = O4.pack_weight(c, s, group)
    np.testing.assert_array_equal(q.codes.cpu().numpy(), codes)
    np.testing.assert_array_equal(n64(q.scales), scales)
    np.testing.assert_array_equal(n64(y), O4.values(c, s)[:, :K])
    np.testing.assert_array_equal(n64(pad)[:, :K], n64(y))
    assert (pad[:, K:] == 7).all()


def test_quantize4_ties_go_to_even_and_nonfinite_groups_read_nan():
    from nanosaur2_web_b200.ops import expand4, quantize4
    W = np.zeros((3, 64), np.float32)
    W[0, :16] = np.arange(-7.5, 8.5, 1.0)          # scale 8 / 7 rounded up would break the ties: pin the group at 7 s
    W[0, 15] = 7.0
    W[0, 0] = -7.0
    W[1, 3], W[1, 40] = np.inf, 2.0
    W[2, 5], W[2, 33] = np.nan, -3.0
    y = n64(expand4(quantize4(t(W), 32)))
    check_device()
    np.testing.assert_array_equal(y[0, 1:15], [-6, -6, -4, -4, -2, -2, 0, 0, 2, 2, 4, 4, 6, 6])
    assert np.isnan(y[1, :32]).all() and np.isnan(y[2, :32]).all()
    c, s = O4.quantise(W[1:, 32:], 32)
    np.testing.assert_array_equal(y[1:, 32:], O4.values(c, s))


def linear_case(rng, M, N, K, group, special=False):
    from nanosaur2_web_b200.ops import expand4, quantize4
    q = quantize4(t(weights(rng, N, K, special)), group)
    return q, n64(expand4(q)), t(rng.standard_normal((M, K)), BF)


def linear_tol(x, W, group):
    K = x.shape[1]
    return (group + K / group + 16) * 2.0 ** -23 * (np.abs(x) @ np.abs(W).T)


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 31, 33, 70])
@pytest.mark.parametrize("N,K,group", [(16, 128, 32), (40, 72, 128), (333, 1032, 64)])
def test_linear4_rows(M, N, K, group):
    from nanosaur2_web_b200.ops import linear4
    rng = np.random.default_rng(M * 7 + N)
    W, Wv, x = linear_case(rng, M, N, K, group)
    bias = t(rng.standard_normal(N))
    want = n64(x) @ Wv.T
    tol = linear_tol(n64(x), Wv, group) + 1e-30
    got = linear4(x, W)
    assert (np.abs(n64(got) - want) <= tol).all()
    with_bias = want + n64(bias)
    tol = tol + 2.0 ** -22 * np.abs(with_bias)
    assert (np.abs(n64(linear4(x, W, bias=bias)) - with_bias) <= tol).all()
    got = linear4(x, W, bias=bias, out_dtype=BF)
    assert got.dtype == BF and (np.abs(n64(got) - with_bias) <= tol + 2.0 ** -8 * np.abs(with_bias)).all()
    # pitched operands: other columns stay as they are, NaN past the rows of x is not read
    xw = torch.full((M, K + 8), float("nan"), dtype=BF, device=DEV)
    xw[:, :K] = x
    base = t(rng.standard_normal((M, N + 3)))
    ow = base.clone()
    linear4(xw[:, :K], W, bias=bias, out=ow[:, 1:N + 1], resid=True)
    check_device()
    assert (np.abs(n64(ow[:, 1:N + 1]) - (n64(base[:, 1:N + 1]) + with_bias)) <= tol + 2.0 ** -22 * np.abs(n64(base[:, 1:N + 1]))).all()
    assert torch.equal(ow[:, :1], base[:, :1]) and torch.equal(ow[:, N + 1:], base[:, N + 1:])


@pytest.mark.parametrize("M,N,K,group", [(1, 640, 1024, 32), (3, 4096, 640, 64), (20, 640, 2048, 128), (1, 20000, 4096, 128),
                                         (5, 16, 20000, 32), (2, 1, 8, 32), (33, 1536, 640, 32),
                                         (1, 5, 98304, 128), (2, 24, 60000, 64), (30, 4800, 256, 32)])
def test_linear4_shapes(M, N, K, group):
    from nanosaur2_web_b200.ops import linear4
    rng = np.random.default_rng(M + N + K)
    W, Wv, x = linear_case(rng, M, N, K, group)
    y = linear4(x, W)
    again = linear4(x, W)
    check_device()
    assert torch.equal(y, again)
    assert (np.abs(n64(y) - n64(x) @ Wv.T) <= linear_tol(n64(x), Wv, group) + 1e-30).all()


def test_linear4_takes_any_bf16_scales_and_propagates_nonfinite_rows():
    from nanosaur2_web_b200.ops import Weight4, linear4, quantize4
    rng = np.random.default_rng(5)
    W, Wv, x = linear_case(rng, 3, 48, 256, 32)
    s = t(np.abs(rng.standard_normal(W.scales.shape)) + 0.1, BF)      # eight significant bits
    W2 = Weight4(W.codes, s, 48, 256, 32)
    c = Wv.reshape(48, -1, 32) / np.where(n64(W.scales) == 0, 1, n64(W.scales)).transpose(0, 2, 1, 3).reshape(-1, 8, 1)[:48]
    s2 = n64(s).transpose(0, 2, 1, 3).reshape(-1, 8, 1)[:48]
    W2v = (np.rint(c) * s2).reshape(48, 256)
    assert (np.abs(n64(linear4(x, W2)) - n64(x) @ W2v.T) <= linear_tol(n64(x), W2v, 32)).all()
    # an infinity and a NaN of one row of x reach that row's outputs and no other's
    xi = x.clone()
    xi[1, 7] = float("nan")
    y, yi = linear4(x, W), linear4(xi, W)
    check_device()
    assert torch.isnan(yi[1]).all() and torch.equal(yi[0], y[0]) and torch.equal(yi[2], y[2])


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5])
def test_linear4_rows_of_wide_range_and_infinities(M):
    """Rows whose values span the whole of bf16 zero and subnormal
    groups, the largest finite values; infinities, which reach their row as the formula has it."""
    from nanosaur2_web_b200.ops import linear4
    rng = np.random.default_rng(M)
    W, Wv, _ = linear_case(rng, 1, 100, 640, 32)
    x = rng.standard_normal((M, 640)) * np.exp2(rng.integers(-30, 30, (M, 640)))
    x[0, :32] = 0
    x[0, 32:64] *= 2.0 ** -100
    x[M - 1, 64:96] = rng.standard_normal(32) * 2.0 ** -131          # subnormal in bf16
    x[0, 96:128] *= 2.0 ** 60
    x = t(x, BF)
    y = n64(linear4(x, W))
    want = n64(x) @ Wv.T
    assert (np.abs(y - want) <= linear_tol(n64(x), Wv, 32) + 1e-37).all()
    big = t(rng.choice([-1.0, 1.0], (M, 640)) * 3.0e38 * (rng.random((M, 640)) < 0.002), BF)
    with np.errstate(over="ignore", invalid="ignore"):
        want = n64(big) @ Wv.T
    y = n64(linear4(big, W))
    fine = np.abs(n64(big)) @ np.abs(Wv).T < 3e38      # else a sum of fp32 products overflows in one order or another
    assert (np.abs(y - want)[fine] <= (linear_tol(n64(big), Wv, 32) + 1e-30)[fine]).all()
    xi = x.clone()
    xi[0, 201], xi[M - 1, 500] = float("inf"), float("-inf")
    with np.errstate(invalid="ignore"):
        want = (n64(xi)[:, None, :] * Wv[None]).sum(-1)
    y = n64(linear4(xi, W))
    check_device()
    assert np.array_equal(np.isnan(y), np.isnan(want)) and np.array_equal(np.isinf(y), np.isinf(want))
    assert (np.sign(y[np.isinf(y)]) == np.sign(want[np.isinf(want)])).all()


def test_linear4_more_rows_than_one_grid_takes():
    """65535 passes of 32 rows are one launch; the rows behind them are another, with the same sums."""
    from nanosaur2_web_b200.ops import linear4
    rng = np.random.default_rng(5)
    W, Wv, _ = linear_case(rng, 1, 9, 8, 32)
    M = 32 * 65535 + 5
    x = torch.randint(-8, 9, (M, 8), device="cuda").to(BF)
    out = torch.zeros((M + 1, 9), device="cuda")
    linear4(x, W, out=out[:M])
    check_device()
    want = x.double() @ t(Wv, torch.float64).T
    tol = (32 + 1 + 16) * 2.0 ** -23 * (x.double().abs() @ t(np.abs(Wv), torch.float64).T)   # linear_tol's factor
    assert ((out[:M].double() - want).abs() <= tol + 1e-37).all() and (out[M] == 0).all()


def test_linear4_empty_and_other_stream():
    from nanosaur2_web_b200.ops import linear4
    rng = np.random.default_rng(9)
    W, Wv, x = linear_case(rng, 4, 64, 128, 32)
    assert linear4(x[:0], W).shape == (0, 64)
    s = torch.cuda.Stream(DEV)
    s.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(s):
        y = linear4(x, W)
    torch.cuda.current_stream(DEV).wait_stream(s)
    assert torch.equal(y, linear4(x, W))


def test_weight_wrappers_refuse_and_reuse():
    from nanosaur2_web_b200 import ops
    W = torch.randn((20, 96), device=DEV)
    q = ops.quantize4(W, 64)
    again = ops.quantize4(W.bfloat16(), 64, out=q)
    assert again is q and torch.equal(ops.expand4(q), ops.expand4(ops.quantize4(W.bfloat16(), 64)))
    x = torch.randn((3, 96), device=DEV).bfloat16()
    calls = [(lambda: ops.quantize4(W, 48), "group"), (lambda: ops.quantize4(W.T), "unit inner stride"),
             (lambda: ops.quantize4(W[:1].expand(4, 96)), "overlap"), (lambda: ops.quantize4(W, 32, out=q), "groups of"),
             (lambda: ops.quantize4(W.half()), "float32 or bfloat16"),
             (lambda: ops.expand4(q, torch.empty((20, 96), device=DEV)), "bfloat16"),
             (lambda: ops.linear4(x.float(), q), "bf16"), (lambda: ops.linear4(x[:, :88], q), "unit inner stride"),
             (lambda: ops.linear4(x, q, bias=torch.zeros(19, device=DEV)), "bias"),
             (lambda: ops.linear4(x, q, resid=True), "resid needs out"),
             (lambda: ops.linear4(x, q, out=torch.zeros((3, 20), device=DEV, dtype=BF), resid=True), "resid"),
             (lambda: ops.linear4(x, q, out=torch.zeros((1, 20), device=DEV).expand(3, 20)), "overlap"),
             (lambda: ops.linear4(x, q, out_dtype=torch.float16), "float32 or bfloat16"),
             (lambda: ops.linear4(x, ops.Weight4(q.codes, q.scales, 20, 200, 64)), "contiguous codes"),
             (lambda: ops.linear4(x, ops.Weight4(q.codes, q.scales.float(), 20, 96, 64)), "contiguous codes"),
             (lambda: ops.linear4(x.cpu(), q), "CUDA")]
    for call, match in calls:
        with pytest.raises(ops.NsaError, match=match):
            call()


def test_cache_wrappers_refuse():
    from nanosaur2_web_b200 import ops
    c = ops.kv4_cache(4, 2, 64, 16, DEV)
    table, start = t([[0, 1], [2, 3]], torch.int32), t([3, 5], torch.int32)
    q = torch.zeros((2, 1, 4 * 64), dtype=BF, device=DEV)
    x, w = torch.zeros((2, 1, 8 * 64), device=DEV), torch.ones(64, device=DEV)
    cs = ops.ropeTable(32, 64, 1e4, DEV)

    def append(**kw):
        a = dict(qkv=x, cache=c, table=table, start=start, Hq=4, q_norm=w, k_norm=w, cs=cs)
        a.update(kw)
        return ops.kv4_append(a.pop("qkv"), a.pop("cache"), a.pop("table"), a.pop("start"), **a)
    append()
    calls = [(lambda: ops.kv4_attention(q.float(), c, table, start), "bfloat16"),
             (lambda: ops.kv4_attention(q[:, :, :100], c, table, start), "whole heads"),
             (lambda: ops.kv4_attention(q[:, :, :64], c, table, start), "multiple of Hkv"),
             (lambda: ops.kv4_attention(q, c, table.long(), start), "int32"),
             (lambda: ops.kv4_attention(q, c, table[:1], start), "table"),
             (lambda: ops.kv4_attention(q, c, table, start[:1]), "start"),
             (lambda: ops.kv4_attention(q, c, table, start, count=start.long()), "count"),
             (lambda: ops.kv4_attention(q, c, table, start, sinks=4), "window"),
             (lambda: ops.kv4_attention(q, c, table, start, window=-1), "window"),
             (lambda: ops.kv4_attention(q, c, table, start, scale=float("nan")), "scale"),
             (lambda: ops.kv4_attention(q, c, table, start, out=q), "overlap"),
             (lambda: ops.kv4_attention(q, c, table, start, workspace=torch.zeros(4, device=DEV)), "uint8"),
             (lambda: ops.kv4_attention(q, ops.Kv4Cache(c.codes, c.scales[:, :1]), table, start), "contiguous codes"),
             (lambda: ops.kv4_read(c, table, start, -1), "L >= 0"),
             (lambda: ops.kv4_read(c, table, start, 1, out=torch.zeros((2, 1, 128), dtype=BF, device=DEV)), "bfloat16"),
             (lambda: append(Hq=3), "multiple of Hkv"), (lambda: append(Hq=8), "inside"), (lambda: append(vOff=480), "inside"),
             (lambda: append(qkv=x.half()), "float32 or bfloat16"), (lambda: append(q_norm=w[:32]), "float32 .64."),
             (lambda: append(cs=ops.ropeTable(32, 128, 1e4, DEV)), "head dim"),
             (lambda: append(cs=ops.RopeTable(cs.buf, cs.sinOff, 33, 64)), "head dim"), (lambda: append(eps=-1.0), "eps"),
             (lambda: append(out=torch.zeros((2, 1, 512), dtype=BF, device=DEV)), "bfloat16"),
             (lambda: append(start=start.cpu()), "CUDA")]
    for call, match in calls:
        with pytest.raises(ops.NsaError, match=match):
            call()
    # a table that broadcasts one row, and a workspace that is too small for a call that needs one
    same = table[:1].expand(2, 2)
    assert torch.equal(ops.kv4_read(c, same, start, 2), ops.kv4_read(c, same.contiguous(), start, 2))
    big = torch.zeros((2, 1024), dtype=torch.int32, device=DEV)
    with pytest.raises(ops.NsaError, match="workspace of"):
        ops.kv4_attention(q, c, big, start, workspace=torch.zeros(16, dtype=torch.uint8, device=DEV))
    check_device()


# --------------------------------------------------------------------------------------------- cache

class Cached:
    """A cache filled through kv4_append with known rows, and its values in float64."""

    def __init__(self, rng, B, T, Hkv, D, P, spare=3, garbage=True):
        from nanosaur2_web_b200 import ops
        self.P, self.D, self.Hkv = P, D, Hkv
        mp = -(-T // P)
        n = B * mp + spare
        self.cache = ops.kv4_cache(n, Hkv, D, P, DEV)
        if garbage:   # slots that nothing wrote: NaN scales
            self.cache.codes.fill_(0xFF)
            self.cache.scales.fill_(float("nan"))
        self.table = t(rng.permutation(n)[:B * mp].reshape(B, mp), torch.int32)
        # large channels among the keys; D values of unit scale
        k = rng.standard_normal((B, T, Hkv, D)) * (0.5 + np.abs(rng.standard_normal(D)))
        v = rng.standard_normal((B, T, Hkv, D))
        self.fill(k, v)

    def fill(self, k, v):
        """Codes written by index arithmetic on the host, independent of kv4_append."""
        B, T, Hkv, D = k.shape
        codes, scales = self.cache.codes.cpu().numpy(), self.cache.scales.float().cpu().numpy()
        tab = self.table.cpu().numpy()
        out = []
        for which, x in ((0, k), (1, v)):
            c, s = O4.quantise(x, 32)
            out.append(O4.values(c, s))
            for b in range(B):
                for pos in range(T):
                    page, slot = tab[b, pos // self.P], pos % self.P
                    nib = (c[b, pos] + 8).astype(np.uint8)
                    codes[page, which, :, slot] = nib[:, 0::2] | (nib[:, 1::2] << 4)
                    scales[page, which, :, slot] = s[b, pos]
        self.cache.codes.copy_(torch.from_numpy(codes))
        self.cache.scales.copy_(torch.from_numpy(scales))
        self.k, self.v = out


def attend_oracle(cd, q, start, count, window, sinks, scale, masked=None):
    """Rows, their bounds and which rows are written."""
    B, L, HD = q.shape
    D, H = cd.D, HD // cd.D
    out, tol = np.zeros((B, L, HD)), np.zeros((B, L, HD))
    for b in range(B):
        keep = np.ones(cd.k.shape[1], bool) if masked is None else ~masked[b]
        for i in range(min(L, count[b])):
            pos = start[b] + i
            for h in range(H):
                hk = h // (H // cd.Hkv)
                sl = slice(h * D, (h + 1) * D)
                j = np.arange(pos + 1)
                see = keep[:pos + 1].copy()
                if window:
                    see &= (j > pos - window) | (j < sinks)
                o, ov, sab = O4.attention(q[b, i, sl], cd.k[b, :pos + 1, hk][see], cd.v[b, :pos + 1, hk][see], see.sum(), 0, 0, scale)
                out[b, i, sl] = o
                tol[b, i, sl] = 2.0 ** -8 * np.abs(o) + 2 * (D * 2.0 ** -23 * sab + 2.0 ** -15) * ov + 1e-30
    return out, tol


CASES = [
    # B, L, Hq, Hkv, D, P, T, window, sinks
    (1, 1, 4, 1, 256, 16, 1, 0, 0), (1, 1, 4, 1, 256, 16, 16, 0, 0), (2, 1, 4, 1, 256, 16, 17, 0, 0),
    (3, 1, 4, 1, 256, 64, 200, 0, 0), (2, 1, 1, 1, 64, 32, 63, 0, 0), (2, 1, 8, 8, 64, 16, 100, 0, 0),
    (2, 2, 6, 2, 128, 48, 131, 0, 0), (1, 5, 16, 2, 128, 16, 77, 0, 0), (2, 3, 20, 2, 64, 16, 50, 0, 0),
    (1, 12, 12, 1, 256, 16, 40, 0, 0), (1, 1, 40, 1, 64, 1024, 300, 0, 0), (1, 40, 4, 1, 128, 32, 40, 0, 0),
    (2, 1, 4, 1, 256, 16, 150, 32, 0), (2, 1, 4, 1, 256, 16, 150, 1, 0), (2, 3, 4, 1, 256, 32, 150, 33, 4),
    (2, 4, 8, 2, 128, 16, 90, 7, 1), (1, 4, 8, 2, 64, 16, 300, 16, 17), (1, 2, 4, 2, 128, 16, 60, 1000, 4),
    (1, 2, 4, 2, 128, 16, 60, 16, 100), (1, 9, 4, 2, 64, 16, 60, 3, 2), (3, 1, 2, 1, 64, 16, 700, 100, 4),
]


@pytest.mark.parametrize("B,L,Hq,Hkv,D,P,T,window,sinks", CASES)
def test_kv4_attention(B, L, Hq, Hkv, D, P, T, window, sinks):
    from nanosaur2_web_b200.ops import kv4_attention
    rng = np.random.default_rng(B + 10 * L + 100 * Hq + T + window + D)
    cd = Cached(rng, B, T, Hkv, D, P)
    q = t(1.5 * rng.standard_normal((B, L, Hq * D)), BF)
    # sequences of different lengths; the longest ends at the table's last written token
    start = np.array([max(0, T - L - 13 * b) for b in range(B)], np.int32)
    got = kv4_attention(q, cd.cache, cd.table, t(start, torch.int32), window=window, sinks=sinks)
    again = kv4_attention(q, cd.cache, cd.table, t(start, torch.int32), window=window, sinks=sinks)
    check_device()
    assert torch.equal(got, again)
    want, tol = attend_oracle(cd, n64(q), start, [L] * B, window, sinks, 1 / np.sqrt(D))
    assert (np.abs(n64(got) - want) <= tol).all(), float((np.abs(n64(got) - want) / tol).max())


@pytest.mark.parametrize("D,Hkv,P,T", [(128, 1, 64, 5000), (64, 2, 16, 3001), (256, 1, 32, 2500), (256, 1, 16, 4500),
                                      (64, 1, 48, 9000)])
def test_kv4_attention_long_and_split(D, Hkv, P, T):
    """One sequence, long enough that its keys are shared out and joined; a scale of the caller's; large scores."""
    from nanosaur2_web_b200.ops import kv4_attention
    rng = np.random.default_rng(T)
    cd = Cached(rng, 1, T, Hkv, D, P)
    q = t(4 * rng.standard_normal((1, 2, 3 * Hkv * D)), BF)
    start = np.array([T - 2], np.int32)
    got = kv4_attention(q, cd.cache, cd.table, t(start, torch.int32), scale=0.2)
    check_device()
    want, tol = attend_oracle(cd, n64(q), start, [2], 0, 0, np.float32(0.2))
    assert (np.abs(n64(got) - want) <= tol).all(), float((np.abs(n64(got) - want) / tol).max())


@pytest.mark.parametrize("D,group,L", [(64, 4, 1), (128, 2, 2), (256, 1, 1), (128, 1, 4), (256, 3, 1), (64, 5, 1)])
def test_kv4_attention_few_rows_of_long_sequences(D, group, L):
    """Up to four rows per kv head share one tile's columns with their low parts; five do not.  Long sequences of other
    lengths, so that units are shared out and joined; a token whose values are infinite counts for the rows that see it."""
    from nanosaur2_web_b200.ops import kv4_attention
    rng = np.random.default_rng(D + group)
    B, Hkv, P, T = 2, 2, 32, 4600
    cd = Cached(rng, B, T, Hkv, D, P)
    q = t(2 * rng.standard_normal((B, L, group * Hkv * D)), BF)
    start = np.array([T - L, 4200], np.int32)
    run = lambda: n64(kv4_attention(q, cd.cache, cd.table, t(start, torch.int32)))
    got = run()
    want, tol = attend_oracle(cd, n64(q), start, [L] * B, 0, 0, 1 / np.sqrt(D))
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())
    k, v = cd.k.copy(), cd.v.copy()
    v[0, T - 1] = np.inf                                              # seen by the last new token of sequence 0 alone
    cd.fill(k, v)
    again = run()
    check_device()
    assert np.isnan(again[0, L - 1]).all()
    got[0, L - 1] = again[0, L - 1] = 0
    assert (np.abs(again - want)[:, :max(L - 1, 0)] <= tol[:, :max(L - 1, 0)]).all() and np.array_equal(again[1], got[1])


@pytest.mark.parametrize("B,L,Hq,Hkv,D,P,T,window,sinks", [(90, 1, 4, 2, 64, 16, 60, 0, 0), (70, 3, 6, 1, 128, 16, 45, 0, 0),
                                                           (37, 2, 4, 4, 256, 16, 40, 9, 3), (100, 1, 1, 1, 64, 16, 300, 33, 0),
                                                           (3, 70, 3, 3, 64, 16, 90, 0, 0)])
def test_kv4_attention_many_units(B, L, Hq, Hkv, D, P, T, window, sinks):
    """More sequences, heads and rows than one wave takes, of very different lengths, some without new tokens: CTAs
    hold ends, wholes and beginnings of units."""
    from nanosaur2_web_b200.ops import kv4_attention
    rng = np.random.default_rng(B)
    cd = Cached(rng, B, T, Hkv, D, P)
    q = t(1.5 * rng.standard_normal((B, L, Hq * D)), BF)
    start = np.array([(37 * b * b) % (T - L + 1) for b in range(B)], np.int32)
    count = np.array([L if b % 5 else b % 3 * L // 2 for b in range(B)], np.int32)
    out = torch.full((B, L, Hq * D), 9.0, dtype=BF, device=DEV)
    for _ in range(2):
        kv4_attention(q, cd.cache, cd.table, t(start, torch.int32), count=t(count, torch.int32), window=window, sinks=sinks, out=out)
    check_device()
    want, tol = attend_oracle(cd, n64(q), start, count, window, sinks, 1 / np.sqrt(D))
    got = n64(out)
    for b in range(B):
        assert (np.abs(got[b, :count[b]] - want[b, :count[b]]) <= tol[b, :count[b]]).all(), b
        assert (got[b, count[b]:] == 9).all()


def test_kv4_attention_counts_strides_and_rows_left_alone():
    from nanosaur2_web_b200.ops import kv4_attention
    rng = np.random.default_rng(3)
    B, L, Hq, Hkv, D, P, T = 4, 6, 4, 2, 128, 16, 60
    cd = Cached(rng, B, T, Hkv, D, P)
    big = t(rng.standard_normal((L, B, Hq * D + 16)), BF)
    q = big.transpose(0, 1)[:, :, 8:Hq * D + 8]                       # [B, L, Hq*D] with other strides
    start, count = np.array([10, 0, 54, 33], np.int32), np.array([6, 1, 0, 99], np.int32)
    wide = torch.zeros((B, cd.table.shape[1] + 3), dtype=torch.int32, device=DEV) - 5
    wide[:, :cd.table.shape[1]] = cd.table
    out = torch.full((L, B, Hq * D), 9.0, dtype=BF, device=DEV).transpose(0, 1)
    kv4_attention(q, cd.cache, wide[:, :cd.table.shape[1]], t(start, torch.int32), count=t(count, torch.int32), out=out)
    check_device()
    want, tol = attend_oracle(cd, n64(q), start, count, 0, 0, 1 / np.sqrt(D))
    for b in range(B):
        n = min(L, count[b])
        assert (np.abs(n64(out[b, :n]) - want[b, :n]) <= tol[b, :n]).all()
        assert (out[b, n:] == 9).all()


def test_kv4_attention_nonfinite_tokens_count_only_where_they_are_seen():
    from nanosaur2_web_b200.ops import kv4_attention
    rng = np.random.default_rng(4)
    B, L, Hq, Hkv, D, P, T = 1, 2, 4, 1, 128, 16, 100
    cd = Cached(rng, B, T, Hkv, D, P)
    clean = kv4_attention(t(rng.standard_normal((1, L, Hq * D)), BF), cd.cache, cd.table, t([98], torch.int32), window=40, sinks=4)
    rng = np.random.default_rng(4)
    cd = Cached(rng, B, T, Hkv, D, P)
    q = t(rng.standard_normal((1, L, Hq * D)), BF)
    k, v = cd.k.copy(), cd.v.copy()
    k[0, 4:59], v[0, 4:59] = np.nan, np.inf      # outside window and sinks of both queries
    cd.fill(k, v)
    got = kv4_attention(q, cd.cache, cd.table, t([98], torch.int32), window=40, sinks=4)
    assert torch.equal(got, clean)
    k[0, 59] = np.nan                            # seen by the first query only
    cd.fill(k, v)
    got = kv4_attention(q, cd.cache, cd.table, t([98], torch.int32), window=40, sinks=4)
    check_device()
    assert torch.isnan(got[0, 0]).all() and torch.equal(got[0, 1], clean[0, 1])


def test_kv4_bad_pages_and_positions_are_masked_and_reported():
    from nanosaur2_web_b200 import ops
    rng = np.random.default_rng(6)
    B, L, Hq, Hkv, D, P, T = 2, 1, 4, 1, 128, 16, 90
    cd = Cached(rng, B, T, Hkv, D, P)
    q = t(rng.standard_normal((B, L, Hq * D)), BF)
    table = cd.table.clone()
    table[0, 2], table[1, 0] = -1, cd.cache.codes.shape[0]
    masked = np.zeros((B, T), bool)
    masked[0, 32:48] = masked[1, :16] = True
    start = np.array([T - 1, T - 3], np.int32)
    got = ops.kv4_attention(q, cd.cache, table, t(start, torch.int32))
    with pytest.raises(ops.NsaError, match="page table entry"):
        check_device()
    check_device()                               # read and cleared
    want, tol = attend_oracle(cd, n64(q), start, [L] * B, 0, 0, 1 / np.sqrt(D), masked)
    assert (np.abs(n64(got) - want) <= tol).all()
    # nothing left to see: zeros
    table[:] = -7
    got = ops.kv4_attention(q, cd.cache, table, t(start, torch.int32))
    with pytest.raises(ops.NsaError):
        check_device()
    assert (got == 0).all()
    # positions outside the table
    before = cd.cache.codes.clone()
    qkv = t(rng.standard_normal((B, L, (Hq + 2 * Hkv) * D)))
    w = torch.ones(D, device=DEV)
    for bad in ([-1, -5], [96, 2 ** 31 - 1]):
        got = ops.kv4_attention(q, cd.cache, cd.table, t(bad, torch.int32))
        with pytest.raises(ops.NsaError, match="position"):
            check_device()
        assert (got == 0).all()
        ops.kv4_append(qkv, cd.cache, cd.table, t(bad, torch.int32), Hq=Hq, q_norm=w, k_norm=w, cs=None)
        with pytest.raises(ops.NsaError, match="position"):
            check_device()
        ops.kv4_read(cd.cache, cd.table, t(bad, torch.int32), 1)
        with pytest.raises(ops.NsaError, match="position"):
            check_device()
    # ... and past the RoPE table
    ops.kv4_append(qkv, cd.cache, cd.table, t([50, 60], torch.int32), Hq=Hq, q_norm=w, k_norm=w, cs=ops.ropeTable(50, D, 1e4, DEV))
    with pytest.raises(ops.NsaError, match="position"):
        check_device()
    assert torch.equal(cd.cache.codes, before)


@pytest.mark.parametrize("D,Hq,Hkv,dtype", [(64, 2, 1, "f32"), (64, 3, 3, "bf16"), (128, 8, 2, "f32"), (128, 4, 4, "bf16"),
                                            (256, 4, 1, "f32"), (256, 4, 1, "bf16")])
@pytest.mark.parametrize("rope", [True, False])
def test_kv4_append_and_read(D, Hq, Hkv, dtype, rope):
    from nanosaur2_web_b200 import ops
    rng = np.random.default_rng(D + Hq)
    B, L, P, T = 4, 7, 16, 60
    cache = ops.kv4_cache(B * 4 + 2, Hkv, D, P, DEV)
    cache.codes.fill_(0x5A)
    cache.scales.fill_(2.0)
    codes0, scales0 = cache.codes.clone(), cache.scales.clone()
    table = t(rng.permutation(B * 4 + 2)[:B * 4].reshape(B, 4), torch.int32)
    start, count = np.array([0, 15, 30, 53], np.int32), np.array([7, 3, 0, 7], np.int32)
    cols = (Hq + 2 * Hkv) * D + 12
    x = rng.standard_normal((B, L, cols)) * (0.2 + np.abs(rng.standard_normal(cols)))
    x[0, 0, :] = 0                                                       # a token of zeros
    x[1, 1, 4:4 + Hkv * D] *= 1e-30                                      # v heads come first: a tiny value vector
    qkv = t(x, BF if dtype == "bf16" else torch.float32)
    vOff, qOff, kOff = 4, 4 + Hkv * D, 8 + (Hq + Hkv) * D
    qw, kw = t(1 + 0.2 * rng.standard_normal(D)), t(1 + 0.2 * rng.standard_normal(D))
    cs = ops.ropeTable(T, D, 1e4, DEV) if rope else None
    out = torch.full((B, L, Hq * D), 9.0, dtype=BF, device=DEV)
    ops.kv4_append(qkv, cache, table, t(start, torch.int32), count=t(count, torch.int32), Hq=Hq, q_norm=qw, k_norm=kw,
                   cs=cs, eps=1e-6, qOff=qOff, kOff=kOff, vOff=vOff, out=out)
    kv = torch.full((B, L, 2 * Hkv * D + 8), 5.0, dtype=BF, device=DEV)
    ops.kv4_read(cache, table, t(start, torch.int32), L, count=t(count, torch.int32), out=kv[:, :, :2 * Hkv * D])
    check_device()
    x = n64(qkv)
    written = np.zeros(codes0.shape[:1] + (P,), bool)
    cos = sin = None
    for b in range(B):
        for i in range(L):
            if i >= count[b]:
                assert (out[b, i] == 9).all() and (kv[b, i] == 5).all()
                continue
            pos = start[b] + i
            written[int(table[b, pos // P]), pos % P] = True
            if rope:
                cos = n64(cs.buf[pos * (D // 2):(pos + 1) * (D // 2)])
                sin = n64(cs.buf[cs.sinOff + pos * (D // 2):cs.sinOff + (pos + 1) * (D // 2)])
            q = O4.norm_rope(x[b, i, qOff:qOff + Hq * D].reshape(Hq, D), n64(qw), cos, sin, np.float64(np.float32(1e-6)))
            plain = np.abs(O4.norm_rope(x[b, i, qOff:qOff + Hq * D].reshape(Hq, D), n64(qw), None, None, 1e-6))
            pair = plain + np.roll(plain, D // 2, -1)
            err = np.abs(n64(out[b, i]).reshape(Hq, D) - q)
            assert (err <= 2.0 ** -8 * np.abs(q) + 20 * 2.0 ** -24 * pair + 1e-30).all()
            k = O4.norm_rope(x[b, i, kOff:kOff + Hkv * D].reshape(Hkv, D), n64(kw), cos, sin, np.float64(np.float32(1e-6)))
            v = x[b, i, vOff:vOff + Hkv * D].reshape(Hkv, D)
            want = O4.values(*O4.quantise(np.concatenate([k, v]).reshape(-1), 32))
            np.testing.assert_array_equal(n64(kv[b, i, :2 * Hkv * D]), want)
            assert (kv[b, i, 2 * Hkv * D:] == 5).all()
    keep = torch.from_numpy(~written).to(DEV)
    for now, old in ((cache.codes, codes0), (cache.scales, scales0)):
        now, old = now.permute(0, 3, 1, 2, 4)[keep], old.permute(0, 3, 1, 2, 4)[keep]
        assert torch.equal(now, old)                                     # no other slot was touched
    assert ops.kv4_read(cache, table, t(start, torch.int32), 0).shape == (B, 0, 2 * Hkv * D)


def test_kv4_append_nonfinite_groups_read_nan():
    from nanosaur2_web_b200 import ops
    D = 128
    cache = ops.kv4_cache(1, 1, D, 16, DEV)
    table, start = t([[0]], torch.int32), t([0], torch.int32)
    x = torch.randn((1, 1, 3 * D), device=DEV)
    x[0, 0, 2 * D + 40] = float("inf")
    x[0, 0, 2 * D + 100] = float("nan")
    w = torch.ones(D, device=DEV)
    ops.kv4_append(x, cache, table, start, Hq=1, q_norm=w, k_norm=w, cs=None)
    v = ops.kv4_read(cache, table, start, 1)[0, 0, D:].float()
    check_device()
    nan = torch.isnan(v)
    assert nan[32:64].all() and nan[96:].all() and not nan[:32].any() and not nan[64:96].any()


def test_kv4_pool_past_4_gib():
    """Pages whose byte offsets need more than 32 bits."""
    from nanosaur2_web_b200 import ops
    Hkv, D, P, n = 8, 256, 64, 34000                 # 128 KiB of codes a page: 4.5 GB
    cache = ops.kv4_cache(n, Hkv, D, P, DEV)
    rng = np.random.default_rng(8)
    B, T = 1, 70
    table = t([[n - 1, n - 2]], torch.int32)
    qkv = t(rng.standard_normal((B, T, 3 * Hkv * D)), BF)
    w = torch.ones(D, device=DEV)
    q = ops.kv4_append(qkv, cache, table, t([0], torch.int32), Hq=Hkv, q_norm=w, k_norm=w, cs=None)
    kv = n64(ops.kv4_read(cache, table, t([0], torch.int32), T)).reshape(B, T, 2, Hkv, D)
    want = O4.values(*O4.quantise(n64(qkv[:, :, 2 * Hkv * D:]), 32)).reshape(B, T, Hkv, D)
    np.testing.assert_array_equal(kv[:, :, 1], want)

    class Known:
        pass
    cd = Known()
    cd.k, cd.v, cd.D, cd.Hkv = kv[:, :, 0], kv[:, :, 1], D, Hkv
    got = ops.kv4_attention(q[:, -2:].contiguous(), cache, table, t([T - 2], torch.int32))
    check_device()
    want, tol = attend_oracle(cd, n64(q[:, -2:]), [T - 2], [2], 0, 0, 1 / 16)
    assert (np.abs(n64(got) - want) <= tol).all()


def test_kv4_step_captured_and_replayed():
    """A captured append + attention over several steps, start advanced on the device, against the eager calls;
    two graphs, each with its own workspace from its pool, replayed in turn."""
    from nanosaur2_web_b200 import ops
    rng = np.random.default_rng(10)
    B, Hq, Hkv, D, P, steps = 3, 4, 1, 256, 16, 20
    w = torch.ones(D, device=DEV)
    cs = ops.ropeTable(64, D, 1e4, DEV)
    table = t(rng.permutation(B * 4).reshape(B, 4), torch.int32)
    rows = t(rng.standard_normal((steps, B, 1, (Hq + 2 * Hkv) * D)))

    def step(x, cache, start, out):
        q = ops.kv4_append(x, cache, table, start, Hq=Hq, q_norm=w, k_norm=w, cs=cs)
        ops.kv4_attention(q, cache, table, start, window=12, sinks=2, out=out)
        start += 1

    def fresh():
        return (ops.kv4_cache(B * 4, Hkv, D, P, DEV), t([0, 3, 7], torch.int32), torch.zeros((B, 1, Hq * D), dtype=BF, device=DEV))

    def zero(cache):
        cache.codes.fill_(0x88)
        cache.scales.zero_()
    eager = []
    cache, start, out = fresh()
    zero(cache)
    for i in range(steps):
        step(rows[i], cache, start, out)
        eager.append(out.clone())
    graphs = []
    for _ in range(2):
        cache, start, out = fresh()
        zero(cache)
        x = rows[0].clone()
        side = torch.cuda.Stream(DEV)
        side.wait_stream(torch.cuda.current_stream(DEV))
        with torch.cuda.stream(side):
            step(x, cache, start, out)           # warm-up: loads the kernels
        torch.cuda.current_stream(DEV).wait_stream(side)
        start -= 1
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(x, cache, start, out)
        graphs.append((g, x, start, out))
    for i in range(steps):
        for g, x, start, out in graphs:
            x.copy_(rows[i])
            g.replay()
            assert torch.equal(out, eager[i])
    check_device()


def test_kv4_append_and_read_of_many_tokens_exactly():
    """Enough tokens that fp32 leaves some keys undecided (outlying channels, cancelling rotations, exact borders):
    every cached value equals the fp64 definition."""
    from nanosaur2_web_b200 import ops
    rng = np.random.default_rng(12)
    for D, Hkv, dtype in ((128, 2, BF), (64, 3, torch.float32), (256, 1, BF)):
        B, L, P = 3, 500, 32
        x = rng.standard_normal((B, L, (2 + 2) * Hkv * D)) * np.exp(1.5 * rng.standard_normal((4 * Hkv * D)))
        x[:, ::7, 2 * Hkv * D:3 * Hkv * D] = np.round(x[:, ::7, 2 * Hkv * D:3 * Hkv * D])     # many equal and zero keys
        x[0, 5:9, 2 * Hkv * D:3 * Hkv * D] *= 1e-25
        x[1, 5:9, 2 * Hkv * D:3 * Hkv * D] *= 1e15
        qkv = t(x, dtype)
        w = 1 + 0.3 * rng.standard_normal(D)
        w[::9] *= 300
        w[1::9] *= 1e-4
        kw = t(w)
        cs = ops.ropeTable(L, D, 1e4, DEV)
        mp = -(-L // P)
        cache, table = ops.kv4_cache(B * mp, Hkv, D, P, DEV), t(rng.permutation(B * mp).reshape(B, mp), torch.int32)
        start = torch.zeros(B, dtype=torch.int32, device=DEV)
        ops.kv4_append(qkv, cache, table, start, Hq=2 * Hkv, q_norm=kw, k_norm=kw, cs=cs)
        kv = ops.kv4_read(cache, table, start, L)
        check_device()
        cos, sin = n64(cs.buf[:cs.sinOff]).reshape(L, 1, D // 2), n64(cs.buf[cs.sinOff:]).reshape(L, 1, D // 2)
        xk, xv = n64(qkv[:, :, 2 * Hkv * D:3 * Hkv * D]).reshape(B, L, Hkv, D), n64(qkv[:, :, 3 * Hkv * D:])
        k = O4.norm_rope(xk, n64(kw), cos, sin, np.float64(np.float32(1e-6)))
        want = np.concatenate([O4.values(*O4.quantise(k.reshape(B, L, -1), 32)), O4.values(*O4.quantise(xv, 32))], -1)
        np.testing.assert_array_equal(n64(kv), want)


def test_kv4_attention_of_long_sequences_captured_and_on_two_streams():
    """Keys split over CTAs and joined by the second kernel: replayed at several positions, and two calls at once."""
    from nanosaur2_web_b200 import ops
    rng = np.random.default_rng(20)
    cd = Cached(rng, 1, 5200, 1, 64, 32)
    q = t(rng.standard_normal((1, 2, 4 * 64)), BF)
    start, out = t([5000], torch.int32), torch.zeros((1, 2, 4 * 64), dtype=BF, device=DEV)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        ops.kv4_attention(q, cd.cache, cd.table, start, out=out)
    torch.cuda.current_stream(DEV).wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv4_attention(q, cd.cache, cd.table, start, out=out)
    for at in (5198, 0, 17, 4090):
        start.fill_(at)
        g.replay()
        want, tol = attend_oracle(cd, n64(q), [at], [2], 0, 0, 1 / 8)
        assert (np.abs(n64(out) - want) <= tol).all(), at
    streams, outs = [torch.cuda.Stream(DEV) for _ in range(2)], []
    starts = [t([a], torch.int32) for a in (5198, 3000)]
    ref = [ops.kv4_attention(q, cd.cache, cd.table, s) for s in starts]
    torch.cuda.synchronize()
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ops.kv4_attention(q, cd.cache, cd.table, starts[i % 2]))
    torch.cuda.synchronize()
    check_device()
    assert all(torch.equal(o, ref[i % 2]) for i, o in enumerate(outs))


def test_kv4_empty_batches_and_pools():
    from nanosaur2_web_b200 import ops
    c = ops.kv4_cache(2, 1, 64, 16, DEV)
    e = torch.zeros((0, 2), dtype=torch.int32, device=DEV)
    s0 = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert ops.kv4_attention(torch.zeros((0, 1, 64), dtype=BF, device=DEV), c, e, s0).shape == (0, 1, 64)
    table, start = t([[0, 1]], torch.int32), t([3], torch.int32)
    assert ops.kv4_attention(torch.zeros((1, 0, 64), dtype=BF, device=DEV), c, table, start).shape == (1, 0, 64)
    w = torch.ones(64, device=DEV)
    assert ops.kv4_append(torch.zeros((0, 1, 192), device=DEV), c, e, s0, Hq=1, q_norm=w, k_norm=w, cs=None).shape == (0, 1, 64)
    check_device()
    # a pool or a table without a page: every key is missing, zeros and a report
    q = torch.ones((1, 1, 64), dtype=BF, device=DEV)
    for cache, tab, match in ((ops.kv4_cache(0, 1, 64, 16, DEV), table, "page table entry"), (c, table[:, :0], "position")):
        assert (ops.kv4_attention(q, cache, tab, start) == 0).all()
        with pytest.raises(ops.NsaError, match=match):
            check_device()


def test_kv4_tokens_past_the_rope_table_are_masked_in_every_later_call():
    """60 rows of RoPE over 4 pages of 16: tokens 60 .. 63 fit the page table but are not stored.  Their slots (NaN here) count
    for nothing, their queries write zeros, in the same step and in later ones."""
    from nanosaur2_web_b200 import ops
    rng = np.random.default_rng(31)
    B, Hq, Hkv, D, P, rows = 2, 4, 2, 128, 16, 60
    cache = ops.kv4_cache(B * 4 + 1, Hkv, D, P, DEV)
    cache.codes.fill_(0xFF)
    cache.scales.fill_(float("nan"))
    table = t(rng.permutation(B * 4 + 1)[:B * 4].reshape(B, 4), torch.int32)
    w, cs = torch.ones(D, device=DEV), ops.ropeTable(rows, D, 1e4, DEV)

    def append(L, start, count=None):
        x = t(rng.standard_normal((B, L, (Hq + 2 * Hkv) * D)))
        out = torch.full((B, L, Hq * D), 9.0, dtype=BF, device=DEV)
        return ops.kv4_append(x, cache, table, t(start, torch.int32), count=None if count is None else t(count, torch.int32),
                              Hq=Hq, q_norm=w, k_norm=w, cs=cs, out=out)

    def attend(q, start):
        out = torch.full_like(q, 7.0)
        return ops.kv4_attention(q, cache, table, t(start, torch.int32), out=out)

    def check(got, q, start, counts):
        class Known:
            pass
        cd = Known()
        kv = n64(ops.kv4_read(cache, table, t([0, 0], torch.int32), 60)).reshape(B, 60, 2, Hkv, D)
        cd.k, cd.v, cd.D, cd.Hkv = kv[:, :, 0], kv[:, :, 1], D, Hkv
        want, tol = attend_oracle(cd, n64(q), start, counts, 0, 0, 1 / np.sqrt(D))
        got = n64(got)
        for b in range(B):
            assert (np.abs(got[b, :counts[b]] - want[b, :counts[b]]) <= tol[b, :counts[b]]).all(), b
            assert (got[b, counts[b]:] == 0).all(), b
    append(56, [0, 0], [56, 10])
    check_device()
    q = append(8, [56, 10])
    with pytest.raises(ops.NsaError, match="position"):
        check_device()
    assert (q[0, 4:] == 9).all()
    got = attend(q, [56, 10])
    with pytest.raises(ops.NsaError, match="position"):
        check_device()
    check(got, q, [56, 10], [4, 8])
    q = append(1, [62, 18])
    with pytest.raises(ops.NsaError, match="position"):
        check_device()
    got = attend(q, [62, 18])
    with pytest.raises(ops.NsaError, match="position"):
        check_device()
    check(got, q, [62, 18], [0, 1])
    out = torch.full((B, 4, 2 * Hkv * D), 5.0, dtype=BF, device=DEV)
    ops.kv4_read(cache, table, t([58, 0], torch.int32), 4, out=out)
    with pytest.raises(ops.NsaError, match="position"):
        check_device()
    assert (out[0, 2:] == 5).all() and not torch.isnan(out).any()
    # a longer table takes the same positions; another handle on the same memory is told the limit
    cs = ops.ropeTable(64, D, 1e4, DEV)
    q = append(2, [60, 19])
    attend(q, [60, 19])
    check_device()
    other = ops.Kv4Cache(cache.codes, cache.scales, positions=60)
    assert (ops.kv4_attention(q, other, table, t([60, 19], torch.int32))[0] == 0).all()
    with pytest.raises(ops.NsaError, match="position"):
        check_device()


@pytest.mark.parametrize("size", [1e-19, 1e-21, 3e-22, 1e-23, 1e-37, 1e18, 1e25, 1e37])
@pytest.mark.parametrize("D", [64, 256])
def test_kv4_append_keys_of_any_size_without_eps(D, size):
    """eps = 0 and heads whose squares are subnormal, zero or infinite in fp32: codes are those of fp64."""
    from nanosaur2_web_b200 import ops
    rng = np.random.default_rng(D)
    B, L, Hkv, P = 1, 700, 4, 16
    qkv = t(rng.standard_normal((B, L, 3 * Hkv * D)) * size)
    kw = t(1 + 0.2 * rng.standard_normal(D))
    mp = -(-L // P)
    cache, table = ops.kv4_cache(mp, Hkv, D, P, DEV), t(rng.permutation(mp).reshape(1, mp), torch.int32)
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    cs = ops.ropeTable(L, D, 1e4, DEV)
    ops.kv4_append(qkv, cache, table, start, Hq=Hkv, q_norm=kw, k_norm=kw, cs=cs, eps=0.0)
    kv = n64(ops.kv4_read(cache, table, start, L))[:, :, :Hkv * D]
    check_device()
    cos, sin = n64(cs.buf[:cs.sinOff]).reshape(L, 1, D // 2), n64(cs.buf[cs.sinOff:]).reshape(L, 1, D // 2)
    k = O4.norm_rope(n64(qkv[:, :, Hkv * D:2 * Hkv * D]).reshape(B, L, Hkv, D), n64(kw), cos, sin, 0.0)
    np.testing.assert_array_equal(kv, O4.values(*O4.quantise(k.reshape(B, L, -1), 32)))


@pytest.mark.parametrize("size", [1e-19, 1e-21, 1e-23, 1e-37, 1e18, 1e25, 1e37])
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("rope", [True, False])
def test_kv4_append_queries_of_any_size_without_eps(D, size, rope):
    """The same for q': unit rows whatever the input's size, to the tolerance of ordinary ones."""
    from nanosaur2_web_b200 import ops
    rng = np.random.default_rng(D + 1)
    B, L, Hq, P = 1, 20, 3, 32
    qkv = t(rng.standard_normal((B, L, (Hq + 2) * D)) * size)
    qkv[0, 3] = t(rng.standard_normal((Hq + 2) * D))                  # an ordinary token between them
    w = t(1 + 0.2 * rng.standard_normal(D))
    cache, table = ops.kv4_cache(1, 1, D, P, DEV), t([[0]], torch.int32)
    cs = ops.ropeTable(L, D, 1e4, DEV) if rope else None
    q = n64(ops.kv4_append(qkv, cache, table, t([0], torch.int32), Hq=Hq, q_norm=w, k_norm=w, cs=cs, eps=0.0)).reshape(L, Hq, D)
    check_device()
    cos = n64(cs.buf[:cs.sinOff]).reshape(L, 1, D // 2) if rope else None
    sin = n64(cs.buf[cs.sinOff:]).reshape(L, 1, D // 2) if rope else None
    x = n64(qkv)[0, :, :Hq * D].reshape(L, Hq, D)
    want, plain = O4.norm_rope(x, n64(w), cos, sin, 0.0), np.abs(O4.norm_rope(x, n64(w), None, None, 0.0))
    pair = plain + np.roll(plain, D // 2, -1)
    assert (np.abs(q - want) <= 2.0 ** -8 * np.abs(want) + 20 * 2.0 ** -24 * pair + 1e-30).all()


@pytest.mark.parametrize("D,group,L,T", [(128, 4, 1, 300), (256, 4, 1, 5000), (64, 2, 4, 9000), (128, 3, 4, 5000)])
def test_kv4_attention_of_the_largest_values(D, group, L, T):
    """Values of nearly 2^120, which the format holds, with scores that rise slowly (the running maximum lags behind), and
    with equal scores of thousands of tokens: the average is finite, so is the result."""
    from nanosaur2_web_b200.ops import kv4_attention
    rng = np.random.default_rng(T)
    cd = Cached(rng, 1, T, 1, D, 32)
    k = np.zeros((1, T, 1, D))
    k[..., :32] = 7.0 * np.linspace(-3, 3, T)[None, :, None, None]    # a group of equal values: stored as they are, nearly
    v = (0.9 + 0.1 * rng.random((1, T, 1, D))) * 2.0 ** 119.9
    cd.fill(k, v)
    for size in (0.0, 0.02, 0.3):
        q = t(size * np.ones((1, L, group * D)), BF)
        got = n64(kv4_attention(q, cd.cache, cd.table, t([T - L], torch.int32)))
        check_device()
        want, tol = attend_oracle(cd, n64(q), [T - L], [L], 0, 0, 1 / np.sqrt(D))
        assert (np.abs(got - want) <= tol).all(), (size, float(np.abs(got / want - 1).max()))


def test_append_refuses_an_empty_rope_table():
    """Without rows the table's pointer is null, which the C call takes as no rotation."""
    from nanosaur2_web_b200 import ops
    c = ops.kv4_cache(2, 1, 64, 16, DEV)
    table, start, w = t([[0, 1]], torch.int32), t([0], torch.int32), torch.ones(64, device=DEV)
    x = torch.zeros((1, 1, 3 * 64), device=DEV)
    none = ops.RopeTable(torch.empty(0, device=DEV), 0, 0, 64)
    with pytest.raises(ops.NsaError, match="head dim"):
        ops.kv4_append(x, c, table, start, Hq=1, q_norm=w, k_norm=w, cs=none)


def test_attention_refuses_a_scale_that_underflows():
    """A scale that is 0 in fp32 would be taken as the default, 1 / sqrt(D)."""
    from nanosaur2_web_b200 import ops
    c = ops.kv4_cache(2, 1, 64, 16, DEV)
    c.codes.fill_(0x9A)
    c.scales.fill_(1.0)
    table, start, q = t([[0, 1]], torch.int32), t([5], torch.int32), torch.ones((1, 1, 64), dtype=BF, device=DEV)
    with pytest.raises(ops.NsaError, match="scale"):
        ops.kv4_attention(q, c, table, start, scale=1e-46)
    ops.kv4_attention(q, c, table, start, scale=1e-44)
    check_device()


def test_kv4_attention_repeats_itself_whatever_the_workspace_held():
    """The same bits from every call, also over a workspace full of NaN, of ones, and of another call's sums."""
    from nanosaur2_web_b200 import ops
    rng = np.random.default_rng(40)
    for B, L, Hq, Hkv, D, P, T in ((40, 1, 32, 8, 128, 64, 1100), (1, 4, 32, 8, 128, 128, 20000)):
        mp = -(-T // P)
        cache = ops.kv4_cache(B * mp, Hkv, D, P, DEV)
        cache.codes.copy_(torch.randint(0, 256, cache.codes.shape, device=DEV, dtype=torch.uint8) | 0x11)
        cache.scales.copy_(torch.randint(16, 32, cache.scales.shape, device=DEV) / 64)
        table = t(rng.permutation(B * mp).reshape(B, mp), torch.int32)
        start = t([max(0, T - L - 17 * b) for b in range(B)], torch.int32)
        q, q2 = (torch.randn((B, L, Hq * D), device=DEV).to(BF) for _ in range(2))
        want = ops.kv4_attention(q, cache, table, start)
        ws = torch.empty(1 << 26, dtype=torch.uint8, device=DEV)
        for i in range(12):
            if i % 4 == 0:
                ws.fill_(0xFF)
            elif i % 4 == 1:
                ws.fill_(0)
                ws.view(torch.float32).fill_(1.0)
            elif i % 4 == 2:
                ops.kv4_attention(q2, cache, table, start, workspace=ws)
            assert torch.equal(ops.kv4_attention(q, cache, table, start, workspace=ws), want), i
    check_device()


def test_kv4_appends_with_rope_tables_of_several_lengths():
    """Sequences that enter with tables of their own lengths: a shorter table later does not hide the tokens of a longer one, nor
    one append without rotation any."""
    from nanosaur2_web_b200 import ops
    rng = np.random.default_rng(32)
    Hq, Hkv, D, P = 2, 1, 64, 16
    cache = ops.kv4_cache(8, Hkv, D, P, DEV)
    table, w = t([[0, 1, 2, 3], [4, 5, 6, 7]], torch.int32), torch.ones(D, device=DEV)
    for lengths in ((50, 20), (20, 50), (50, None), (20, None)):
        cache.positions = 0
        for b, rows in enumerate(lengths):
            n = rows or 50
            x = t(rng.standard_normal((1, n, (Hq + 2 * Hkv) * D)))
            ops.kv4_append(x, cache, table[b:b + 1], t([0], torch.int32), Hq=Hq, q_norm=w, k_norm=w,
                           cs=None if rows is None else ops.ropeTable(rows, D, 1e4, DEV))
        start = t([n - 1 for n in (lengths[0], lengths[1] or 50)], torch.int32)
        q = t(rng.standard_normal((2, 1, Hq * D)), BF)
        got = ops.kv4_attention(q, cache, table, start)
        check_device()
        assert torch.equal(got, ops.kv4_attention(q, ops.Kv4Cache(cache.codes, cache.scales), table, start)) and (got != 0).any(-1).all()
    check_device()
