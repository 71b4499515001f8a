"""GPU parity of the FP4 page pool (append, read) and the attention over it
(plain and differential) with the 64-bit oracle.

Append and read are exact.  Attention tolerances are sums of what the kernels
round, per output element (A = softmax . |V|):
  * P to a half: at most 2^-11 of each p, so 2^-11 A (fp32 queries: P as two halves, 2^-22 A);
  * a half's smallest step is 2^-24 and the largest p is scaled to at least 2^7, so a p (as a share of the largest,
    hence of the sum) is off by up to half a step over 2^7 = 2^-32 however small it is: 2^-32 sum |v|;
  * scores in fp32: D products summed, each rounding 2^-24 of at most the sum of magnitudes (reach); a score's
    error d moves the output by at most 2 d A; the query row rounds to a half for elements 2^-14 below its
    largest (2^-25 of it), which D * 2^-24 covers;
  * sums of p v and of p in fp32: 2^-24 per addition in blocks of 16, T / 16 + 64 of them at most;
  * exp2: 2^-22, and its argument (reach after the maximum) in fp32: another 2^-23 reach;
  * the output's own rounding, half a step.
"""

import math

import numpy as np
import pytest
import torch

from oracle import fp4 as of

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ia():
    import intent_attention
    return intent_attention


def _rows(g, shape, dtype):
    x = g.standard_normal(shape) * np.exp(0.7 * g.standard_normal(shape[:-2] + (1, shape[-1])))
    return torch.from_numpy(x.astype(np.float32)).cuda().to(DT[dtype])


def _np(t):
    return t.double().cpu().numpy()


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _cache(seed, B, Ht, D, PS, tokens, dtype="bf16", extra=3, dirty=False):
    """A pool filled to ``tokens`` (host list), its shuffled table, and the values it holds [B][Ht, T, D]."""
    ia = _ia()
    g = np.random.default_rng(seed)
    W = max(1, -(-max(tokens) // PS)) + 1
    P = B * Ht * W + extra
    table = _i32(g.permutation(P)[:B * Ht * W].reshape(B, Ht, W))
    pool = ia.Fp4Pool.allocate(P, PS, D)
    for t in pool.tensors():
        t.fill_(255 if dirty else 0)
    n = max(max(tokens), 1)
    k, v = _rows(g, (B, Ht, n, D), dtype), _rows(g, (B, Ht, n, D), dtype)
    ia.append_fp4(pool, k, v, table, counts=_i32(tokens))
    return pool, table, of.values(_np(k)), of.values(_np(v))


# --------------------------------------------------------------------------- #
#  Append and read
# --------------------------------------------------------------------------- #

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D,PS,n,start", [(64, 16, 1, 0), (64, 48, 37, 5), (128, 16, 64, 16), (128, 32, 33, 31),
                                          (256, 64, 129, 1), (256, 16, 2, 15), (128, 128, 500, 7)])
def test_append_read_exact(dtype, D, PS, n, start):
    ia = _ia()
    g = np.random.default_rng(D + PS + n)
    B, Ht = 3, 2
    W = (start + n + 4) // PS + 2
    table = _i32(g.permutation(B * Ht * W).reshape(B, Ht, W))
    pool = ia.Fp4Pool.allocate(B * Ht * W, PS, D, zero=True)
    pos, counts = [start, start + 1, start + 3], [n, max(0, n - 1), n // 2]
    k, v = _rows(g, (B, Ht, n, D), dtype), _rows(g, (B, Ht, n, D), dtype)
    ia.append_fp4(pool, k, v, table, _i32(pos), _i32(counts))
    for out_dtype in DT.values():
        gk, gv = ia.read_fp4(pool, table, _i32(pos), n + 1, _i32(counts), dtype=out_dtype)
        assert gk.shape == (B, Ht, n + 1, D) and gk.dtype == out_dtype
        for b in range(B):
            for got, x in ((gk, k), (gv, v)):
                want = np.zeros((Ht, n + 1, D))
                want[:, :counts[b]] = of.values(_np(x[b, :, :counts[b]]))
                np.testing.assert_array_equal(_np(got[b]), want)


def test_rounding_edges():
    """Ties, borders of the scale, saturation, zeros, tiny blocks, infinities and NaN."""
    ia = _ia()
    D = 128
    top = np.array([6.0, 6.0 * (1 + 2 ** -20), 5.9999995, 3.0, 2.0 ** -14 * 6, 2.0 ** -15, 2.0 ** -17, 2.0 ** -30, 0.0,
                    49152.0, 49153.0, 65504.0, 1e30, 3e38, 1e-40, np.inf], np.float32)
    edge = np.concatenate([of.GRID, of.BORDERS, of.BORDERS * (1 + 2 ** -12), of.BORDERS * (1 - 2 ** -12)])
    rows = np.zeros((len(top), D), np.float32)
    for i, a in enumerate(top):
        for blk in range(4):
            rows[i, 32 * blk] = a * (-1) ** blk
            if np.isfinite(a):
                e = np.clip(np.ceil(np.log2(a / 6)) if a > 0 else -14, -14, 13)
                rows[i, 32 * blk + 1: 32 * blk + 30] = np.where(
                    edge * 2.0 ** e <= a, edge * 2.0 ** e, 0) * (-1) ** np.arange(29)
    rows[3, 5] = np.nan
    rows[4, 40] = -np.inf
    x = torch.from_numpy(rows).cuda()[None, None]
    pool = ia.Fp4Pool.allocate(2, 16, D, zero=True)
    table = _i32([[[1]]])
    ia.append_fp4(pool, x, x.flip(2), table)
    k, v = ia.read_fp4(pool, table, None, len(top), dtype=torch.float32)
    want = of.values(rows)
    np.testing.assert_array_equal(_np(k[0, 0]), want)
    np.testing.assert_array_equal(_np(v[0, 0]), want[::-1])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_single_tokens_equal_one_prompt(D):
    """A token at a time, whatever the batch's parities, gives the planes that one call gives."""
    ia = _ia()
    g = np.random.default_rng(D)
    B, Ht, PS, T = 2, 2, 16, 35
    W = 4
    table = _i32(g.permutation(B * Ht * W).reshape(B, Ht, W))
    one, many = (ia.Fp4Pool.allocate(B * Ht * W, PS, D, zero=True) for _ in range(2))
    k, v = _rows(g, (B, Ht, T, D), "bf16"), _rows(g, (B, Ht, T, D), "bf16")
    ia.append_fp4(one, k, v, table, _i32([0, 1]))
    for t in range(T):
        ia.append_fp4(many, k[:, :, t:t + 1], v[:, :, t:t + 1], table, _i32([t, t + 1]))
    for a, b in zip(one.tensors(), many.tensors()):
        assert torch.equal(a, b)


def test_append_leaves_everything_else():
    """Bytes of no appended row keep their value; rows without a page are dropped and counted."""
    ia = _ia()
    g = np.random.default_rng(5)
    B, Ht, PS, D, W, P = 2, 2, 16, 128, 3, 9
    table = np.array([[[4, -1, 7], [2, 0, 9]], [[1, 3, 5], [8, -7, 6]]], np.int32)
    pool = ia.Fp4Pool.allocate(P, PS, D)
    for t in pool.tensors():
        t.copy_(torch.from_numpy(g.integers(113, 141, size=tuple(t.shape)).astype(np.uint8)))
    every = _i32(np.arange(P).reshape(P, 1, 1))
    k0, v0 = ia.read_fp4(pool, every, None, PS, dtype=torch.float32)
    n, pos, counts = 41, [3, -2], [41, 30]
    k, v = _rows(g, (B, Ht, n, D), "f32"), _rows(g, (B, Ht, n, D), "f32")
    dropped = torch.zeros(1, dtype=torch.int32, device="cuda")
    ia.append_fp4(pool, k, v, _i32(table), _i32(pos), _i32(counts), dropped=dropped)
    k1, v1 = ia.read_fp4(pool, every, None, PS, dtype=torch.float32)
    lost = 0
    for want, got, x in ((_np(k0), k1, k), (_np(v0), v1, v)):
        lost = 0
        xv = of.values(_np(x))
        for b in range(B):
            for h in range(Ht):
                for i in range(counts[b]):
                    t = pos[b] + i
                    pid = table[b, h, t // PS] if 0 <= t < W * PS else -1
                    if 0 <= pid < P:
                        want[pid, 0, t % PS] = xv[b, h, i]
                    else:
                        lost += 1
        np.testing.assert_array_equal(_np(got), want)
    assert int(dropped) == lost > 0


def test_strided_rows_and_out():
    ia = _ia()
    g = np.random.default_rng(11)
    B, Ht, n, D, PS = 2, 3, 21, 128, 16
    qkv = _rows(g, (B, n, 3 * Ht, D + 3), "f16")            # rows start on no 16-byte border
    k, v = (qkv[:, :, i * Ht:(i + 1) * Ht, 3:].transpose(1, 2) for i in (1, 2))
    big = _i32(g.permutation(B * Ht * 4).reshape(B, Ht, 4))
    table = big[:, :, 1:3]
    pool = ia.Fp4Pool.allocate(B * Ht * 4, PS, D, zero=True)
    ia.append_fp4(pool, k, v, table)
    out = torch.full((2, B, n, Ht, D + 1), 7.0, device="cuda", dtype=torch.bfloat16)
    views = tuple(out[i, :, :, :, 1:].transpose(1, 2) for i in range(2))
    gk, gv = ia.read_fp4(pool, table, None, n, out=views)
    np.testing.assert_array_equal(_np(gk), of.values(_np(k)))
    np.testing.assert_array_equal(_np(gv), of.values(_np(v)))
    assert (out[..., 0] == 7.0).all()
    # a last dimension that is not contiguous
    ia.append_fp4(pool, k.transpose(2, 3).contiguous().transpose(2, 3), v, table)
    np.testing.assert_array_equal(_np(ia.read_fp4(pool, table, None, n)[0]), of.values(_np(k)))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_beside_rows_never_written(D):
    """Two rows of V share their bytes: written ones are exact whatever their neighbours hold, and in a zeroed pool rows
    that were never written are 0 to reads and to attention."""
    ia = _ia()
    g = np.random.default_rng(D)
    PS, T, at = 16, 30, [1, 4, 5, 8, 17, 19, 22]             # odd and even rows alone, and a pair
    table = _i32([[[2, 0]]])
    k, v = _rows(g, (1, 1, T, D), "f32"), _rows(g, (1, 1, T, D), "f32")
    kd, vd = np.zeros((1, 1, T, D)), np.zeros((1, 1, T, D))
    for t in at:
        kd[:, :, t], vd[:, :, t] = of.values(_np(k[:, :, t])), of.values(_np(v[:, :, t]))
    for byte in (0, 111, 143, 255):
        pool = ia.Fp4Pool.allocate(3, PS, D, zero=True)
        pool.data.fill_(byte)
        for t in at:
            ia.append_fp4(pool, k[:, :, t:t + 1], v[:, :, t:t + 1], table, _i32([t]))
        for dtype in DT.values():
            gk, gv = ia.read_fp4(pool, table, None, T, dtype=dtype)
            np.testing.assert_array_equal(_np(gk)[:, :, at], kd[:, :, at])
            np.testing.assert_array_equal(_np(gv)[:, :, at], vd[:, :, at])
            if byte == 0:
                np.testing.assert_array_equal(_np(gk), kd)
                np.testing.assert_array_equal(_np(gv), vd)
        if byte == 0:
            # one row of V at a time decides the output, its score 12: its scale off by 2^-10 would be above the bounds
            for t in at:
                q = torch.from_numpy(12 * D ** -0.5 * kd[:, :, t] / np.square(kd[:, :, t]).mean()).float().cuda()
                _check(q, pool, table, [T], (kd, vd), ia.paged_decode_fp4(q, pool, table, _i32([T])))


# --------------------------------------------------------------------------- #
#  Attention
# --------------------------------------------------------------------------- #

def _tolerance(A, reach, v, D, split):
    p = 2.0 ** (-22 if split else -11)
    d = (D + 2) * 2.0 ** -24 * reach
    return A * (p + 2 * d[..., None] + (len(v) / 16 + 64) * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -32 * np.abs(v).sum(0)


def _check(q, pool, table, lengths, kv, got, scale=None, differential=None, absent=None):
    """Every output row against the oracle."""
    kd, vd = kv
    q4 = q if q.dim() == 4 else q[:, :, None]
    o4 = got if got.dim() == 4 else got[:, :, None]
    B, Hq, M, D = q4.shape
    Ht = table.shape[1]
    G = Hq // Ht
    cap = table.shape[2] * pool.page_size
    qd, od = _np(q4), _np(o4)
    split = q.dtype == torch.float32
    half_step = torch.finfo(got.dtype).eps / 2
    for b in range(B):
        n = min(max(int(lengths[b]), 0), cap)
        T = min(n, kd.shape[2])
        for h in range(Hq):
            k, v = kd[b, h // G, :T], vd[b, h // G, :T]
            seen = np.arange(T)[None, :] < (n - (M - 1 - np.arange(M)))[:, None]
            if absent is not None:
                seen = seen & ~absent[b, h // G, :T][None, :]
            if differential is None:
                s = 1 / math.sqrt(D) if scale is None else scale
                want, A, reach = of.attention(qd[b, h], k, v, seen, s)
                tol = _tolerance(A, reach, v, D, split)
            else:
                lam, w, eps, oscale = differential
                c = D // 2
                s = 1 / math.sqrt(c) if scale is None else scale
                x1, A1, r1 = of.attention(qd[b, h, :, :c], k[:, :c], v, seen, s)
                x2, A2, r2 = of.attention(qd[b, h, :, c:], k[:, c:], v, seen, s)
                x = x1 - lam[h] * x2
                tol = _tolerance(A1, r1, v, D, split) + abs(lam[h]) * _tolerance(A2, r2, v, D, split) \
                    + 2.0 ** -23 * np.abs(x)
                if w is None:
                    want, tol = oscale * x, abs(oscale) * tol
                else:
                    r = np.sqrt((x * x).mean(-1, keepdims=True) + eps)
                    want = oscale * w * x / r
                    # x off by tol moves the mean square's root by at most the root mean square of tol
                    moved = np.sqrt((tol * tol).mean(-1, keepdims=True))
                    tol = np.abs(oscale * w) / np.maximum(r - moved, 1e-30) * (tol + np.abs(x) * (moved / r + 2.0 ** -20))
            tol = tol + half_step * np.abs(want) + 2.0 ** -24 * (got.dtype == torch.float16)
            bad = np.abs(od[b, h] - want) > tol
            assert not bad.any(), (b, h, np.abs(od[b, h] - want).max(), tol[bad].min(), want[bad][:4], od[b, h][bad][:4])


SHAPES = [  # B, Ht, G, M, D, PS, lengths, dtype
    (1, 1, 1, 1, 64, 16, [1], "f16"),
    (4, 2, 4, 1, 128, 16, [0, 1, 16, 17], "bf16"),
    (3, 2, 8, 1, 128, 16, [255, 256, 257], "f16"),
    (2, 1, 8, 1, 64, 32, [33, 700], "f32"),
    (2, 2, 5, 1, 256, 64, [1000, 63], "bf16"),
    (3, 1, 1, 1, 128, 48, [2011, 96, 31], "f32"),
    (2, 2, 3, 4, 128, 16, [3, 400], "f16"),
    (2, 1, 4, 16, 64, 16, [15, 333], "bf16"),
    (1, 2, 7, 5, 256, 32, [777], "f32"),
    (2, 1, 32, 1, 128, 16, [900, 5], "bf16"),
    (1, 1, 48, 2, 128, 16, [600], "f16"),
    (40, 1, 2, 1, 64, 16, list(range(0, 400, 10)), "bf16"),
    (1, 3, 4, 1, 128, 128, [20011], "bf16"),
    (1100, 1, 2, 1, 64, 16, [(7 * i) % 301 for i in range(1100)], "f16"),
    (100, 2, 1, 2, 128, 16, [0] * 60 + [600] + [0] * 38 + [5], "bf16"),
]


@pytest.mark.parametrize("case", SHAPES, ids=[f"b{c[0]}h{c[1]}g{c[2]}m{c[3]}d{c[4]}p{c[5]}{c[7]}n{max(c[6])}" for c in SHAPES])
@pytest.mark.parametrize("kind", ["plain", "differential", "normed"])
def test_decode_matches_oracle(case, kind):
    ia = _ia()
    B, Ht, G, M, D, PS, lengths, dtype = case
    pool, table, kd, vd = _cache(B * 31 + D, B, Ht, D, PS, lengths, dirty=True)
    g = np.random.default_rng(9)
    q = _rows(g, (B, Ht * G, M, D), dtype)
    if M == 1:
        q = q[:, :, 0]
    if kind == "plain":
        got = ia.paged_decode_fp4(q, pool, table, _i32(lengths))
        _check(q, pool, table, lengths, (kd, vd), got)
        return
    lam = g.uniform(-0.3, 0.9, Ht * G).astype(np.float32)
    w = (1 + 0.2 * g.standard_normal(D)).astype(np.float32) if kind == "normed" else None
    tw = None if w is None else torch.from_numpy(w).cuda()
    got = ia.differential_decode_fp4(q, pool, table, _i32(lengths), torch.from_numpy(lam).cuda(), norm_weight=tw,
                                     eps=1e-5, out_scale=0.8)
    _check(q, pool, table, lengths, (kd, vd), got, differential=(lam.astype(float), w, 1e-5, 0.8))


@pytest.mark.parametrize("B,Ht,G,M,D,dtype", [(5000, 1, 1, 1, 64, "bf16"), (250, 8, 1, 1, 128, "f16"),
                                              (33, 40, 9, 1, 128, "bf16"), (310, 4, 2, 3, 256, "f32")])
def test_many_short_sequences(B, Ht, G, M, D, dtype):
    """More (sequence, head, column group) units than warps, empty and one-token sequences among them; one is long
    enough that units are cut."""
    ia = _ia()
    lengths = [(13 * i) % 140 if i % 5 else i % 2 for i in range(B)]
    lengths[B // 3] = 300
    pool, table, kd, vd = _cache(B, B, Ht, D, 16, lengths, dirty=True)
    q = _rows(np.random.default_rng(B), (B, Ht * G, M, D), dtype)
    ln = _i32(lengths)
    got = ia.paged_decode_fp4(q, pool, table, ln)
    some = sorted({B // 3, B - 1, *range(0, B, -(-B // 30))})
    _check(q[some], pool, table[some], [lengths[b] for b in some], (kd[some], vd[some]), got[some])
    # All of them against calls of 32 sequences, cut in other places: P rounds by 2^-11 at most (twice, as does l), the
    # output by half a step of its type, both relative to the largest |V|, on either side.
    again = torch.cat([ia.paged_decode_fp4(q[b:b + 32], pool, table[b:b + 32], ln[b:b + 32]) for b in range(0, B, 32)])
    tol = float(np.abs(vd).max()) * (torch.finfo(got.dtype).eps + 2.0 ** -8)
    assert float((got.float() - again.float()).abs().max()) <= tol


@pytest.mark.parametrize("D,Ht,G,M,lengths", [(128, 2, 4, 1, [40, 3000]), (64, 1, 40, 2, [5000]),
                                              (256, 2, 6, 3, [90, 12000, 0])])
def test_output_over_the_query(D, Ht, G, M, lengths):
    ia = _ia()
    B = len(lengths)
    pool, table, _, _ = _cache(D, B, Ht, D, 16, lengths)
    q = _rows(np.random.default_rng(D), (B, Ht * G, M, D), "bf16")
    ln, lam = _i32(lengths), torch.full((Ht * G,), 0.4, device="cuda")
    for f in (lambda x, **o: ia.paged_decode_fp4(x, pool, table, ln, **o),
              lambda x, **o: ia.differential_decode_fp4(x, pool, table, ln, lam, **o)):
        want, x = f(q), q.clone()
        assert f(x, out=x) is x and torch.equal(x, want)


def test_missing_pages_are_not_seen():
    ia = _ia()
    B, Ht, G, D, PS, n = 2, 2, 4, 128, 16, 200
    pool, table, kd, vd = _cache(3, B, Ht, D, PS, [n, n])
    absent = np.zeros((B, Ht, n), bool)
    t = table.clone()
    for b, h, w, x in ((0, 0, 0, -1), (0, 0, 5, pool.num_pages), (0, 1, 12, -9), (1, 0, 3, 2 ** 31 - 1)):
        t[b, h, w] = x
        absent[b, h, w * PS:(w + 1) * PS] = True
    t[1, 1, :] = -1
    absent[1, 1] = True
    q = _rows(np.random.default_rng(1), (B, Ht * G, 3, D), "f16")
    got = ia.paged_decode_fp4(q, pool, t, _i32([n, n]))
    _check(q, pool, t, [n, n], (kd, vd), got, absent=absent)
    assert (got[1, G:] == 0).all()


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 1e-30])
def test_scales(scale):
    ia = _ia()
    pool, table, kd, vd = _cache(4, 2, 1, 128, 16, [300, 40])
    q = _rows(np.random.default_rng(1), (2, 4, 128), "f32")
    got = ia.paged_decode_fp4(q, pool, table, _i32([300, 40]), sm_scale=scale)
    _check(q, pool, table, [300, 40], (kd, vd), got, scale=scale)


@pytest.mark.parametrize("size", [1e-30, 1e-5, 1e4, 3e37])
def test_query_sizes(size):
    """Queries far from 1 in either direction, the scale bringing the scores back."""
    ia = _ia()
    pool, table, kd, vd = _cache(8, 1, 2, 64, 16, [500])
    q = (_rows(np.random.default_rng(2), (1, 8, 64), "f32") * 0.1 * size).to(torch.bfloat16)
    got = ia.paged_decode_fp4(q, pool, table, _i32([500]), sm_scale=1.0 / size)
    _check(q, pool, table, [500], (kd, vd), got, scale=1.0 / size)


@pytest.mark.parametrize("T", [45, 9000])
@pytest.mark.parametrize("q_base,k_base,step,sm_scale,dtype", [
    (8192.0, 16384.0, 8192.0, 1.0, "f16"), (20480.0, 49152.0, 16384.0, 0.7, "f16"), (8192.0, 16384.0, 8192.0, 1.0, "f32"),
    (2.0 ** 60, 49152.0, 2.0 ** 60, -3.0, "bf16"), (2.0 ** 100, 24576.0, 2.0 ** 101, 1e30, "f32"),
    (2.0 ** 100, 24576.0, 2.0 ** 101, 1e30, "bf16"), (8.0, 1024.0, 0.25, 1.0, "f32"), (16.0, 512.0, 0.25, 0.9, "f16")])
def test_scores_far_from_zero(q_base, k_base, step, sm_scale, dtype, T):
    """A large score that all keys share and a difference of a few steps.  Every product is a small multiple of one power
    of two and the sums need 24 bits at most, so the scores are exact: the weights have to be right to the rounding of P
    and of exp2 (its argument, at most 150 before P leaves the floats, off by 2^-22 of itself with the scale's rounding),
    however large the scores are."""
    ia = _ia()
    g = np.random.default_rng(T)
    D, B, G = 128, 2, 4
    k = np.zeros((B, 1, T, D), np.float32)
    k[..., 0:32] = k[..., 64:96] = k_base
    more = np.array([0.0, 0.5, 1.0, 2.0, 4.0, 6.0], np.float32)[g.integers(0, 6, (2, B, 1, T))]
    k[..., 32], k[..., 96] = more
    v = g.standard_normal((B, 1, T, D)).astype(np.float32)
    table = _i32(g.permutation(B * (T // 16 + 1)).reshape(B, 1, -1))
    pool = ia.Fp4Pool.allocate(table.numel(), 16, D, zero=True)
    ia.append_fp4(pool, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), table)
    q = np.zeros((B, G, D))
    q[..., 0:32] = q[..., 64:96] = q_base
    q[..., 32] = step * np.array([1.0, -1.0, 2.0, 0.0])
    q[..., 96] = step * np.array([1.0, 1.0, 0.0, -2.0])
    tq = torch.from_numpy(q).to(DT[dtype]).cuda()
    lengths, lam = [T, T - 7], [0.5, -0.25, 1.0, 0.0]
    vd = of.values(v)
    np.testing.assert_array_equal(of.values(k), k)
    np.testing.assert_array_equal(_np(tq), q)
    plain = _np(ia.paged_decode_fp4(tq, pool, table, _i32(lengths), sm_scale=sm_scale, out_dtype=torch.float32))
    diff = _np(ia.differential_decode_fp4(tq, pool, table, _i32(lengths), torch.tensor(lam, device="cuda"),
                                          sm_scale=sm_scale, out_dtype=torch.float32))
    arg = 150 * 2.0 ** -22
    for b, n in enumerate(lengths):
        kb, vb, seen = k[b, 0, :n].astype(float), vd[b, 0, :n], np.ones((1, n), bool)
        for h in range(G):
            def part(lo, hi):
                out, A, _ = of.attention(q[b, h, None, lo:hi], kb[:, lo:hi], vb, seen, sm_scale)
                return out[0], (_tolerance(A, np.zeros(1), vb, D, dtype == "f32") + 2 * arg * A)[0]
            want, tol = part(0, D)
            assert (np.abs(plain[b, h] - want) <= tol + 2.0 ** -24 * np.abs(want)).all(), (b, h, plain[b, h][:4], want[:4])
            (w1, t1), (w2, t2) = part(0, D // 2), part(D // 2, D)
            want, tol = w1 - lam[h] * w2, t1 + abs(lam[h]) * t2 + 2.0 ** -22 * (np.abs(w1) + np.abs(w2))
            assert (np.abs(diff[b, h] - want) <= tol).all(), (b, h, diff[b, h][:4], want[:4])


def test_large_and_tiny_values():
    """The ends of what a row can hold: values up to 49152 and down to 2^-15, and one strong key."""
    ia = _ia()
    B, Ht, D, PS, n = 1, 1, 128, 16, 320
    g = np.random.default_rng(0)
    k = g.standard_normal((B, Ht, n, D)).astype(np.float32)
    v = g.standard_normal((B, Ht, n, D)).astype(np.float32)
    v[0, 0, :, :32] *= 30000.0
    v[0, 0, :, 32:64] *= 2.0 ** -13
    k[0, 0, 17] *= 40.0
    pool = ia.Fp4Pool.allocate(n // PS, PS, D)
    table = _i32(np.arange(n // PS).reshape(1, 1, -1))
    ia.append_fp4(pool, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), table)
    q = torch.from_numpy(g.standard_normal((1, 8, D)).astype(np.float32)).cuda()
    q[0, 0] = torch.from_numpy(k[0, 0, 17]).cuda()
    got = ia.paged_decode_fp4(q, pool, table, _i32([n]))
    _check(q, pool, table, [n], (of.values(k), of.values(v)), got)


def test_nan_query_gives_nan_in_its_rows_only():
    ia = _ia()
    pool, table, kd, vd = _cache(2, 2, 2, 128, 16, [300, 20])
    q = _rows(np.random.default_rng(1), (2, 8, 128), "f16")
    clean = ia.paged_decode_fp4(q, pool, table, _i32([300, 20]))
    q2 = q.clone()
    q2[0, 1, 7] = float("nan")
    q2[1, 6, 0] = float("inf")
    got = ia.paged_decode_fp4(q2, pool, table, _i32([300, 20]))
    assert torch.isnan(got[0, 1]).all() and torch.isnan(got[1, 6]).any()
    keep = torch.ones(2, 8, dtype=torch.bool, device="cuda")
    keep[0, 1] = keep[1, 6] = False
    assert torch.equal(got[keep], clean[keep])


def test_differential_row_of_zeros_stays_zero():
    """No token seen, or the maps cancel: 0 for every eps, eps 0 included."""
    ia = _ia()
    pool, table, kd, vd = _cache(2, 2, 1, 64, 16, [5, 5])
    q = torch.zeros(2, 4, 64, device="cuda")
    lam, w = torch.ones(4, device="cuda"), torch.ones(64, device="cuda")
    for eps in (0.0, 1e-5):
        got = ia.differential_decode_fp4(q, pool, table, _i32([0, 5]), lam, norm_weight=w, eps=eps)
        assert (got[0] == 0).all() and torch.isfinite(got).all()


@pytest.mark.parametrize("D,M,dtype", [(64, 1, "f32"), (128, 3, "bf16"), (256, 1, "f16")])
def test_equal_maps_cancel_exactly(D, M, dtype):
    """Equal halves of queries and keys with weight 1: 0 for every eps, for whole and cut units, not noise of rms 1."""
    ia = _ia()
    g = np.random.default_rng(D)
    lengths = [5, 9000, 300]
    B, T, W = len(lengths), max(lengths), -(-max(lengths) // 16)
    half, v = _rows(g, (B, 1, T, D // 2), "f32"), _rows(g, (B, 1, T, D), "f32")
    pool = ia.Fp4Pool.allocate(B * W, 16, D)
    table = _i32(g.permutation(B * W).reshape(B, 1, W))
    ia.append_fp4(pool, torch.cat([half, half], -1), v, table)
    q = _rows(g, (B, 4, M, D // 2), dtype)
    q = torch.cat([q, q], -1)
    lam, w = torch.ones(4, device="cuda"), torch.ones(D, device="cuda")
    for ln, norm, eps in ((lengths, w, 0.0), (lengths, w, 1e-5), (lengths, None, 0.0), ([5, 40, 90], w, 0.0)):
        t = table if ln is lengths else table[:, :, :6]                    # (few tiles: a warp a unit, nothing to join)
        got = ia.differential_decode_fp4(q, pool, t, _i32(ln), lam, norm_weight=norm, eps=eps)
        assert (got == 0).all()


def test_first_call_captured():
    """The very first call of a process, captured: nothing that a capture forbids happens in a call."""
    import subprocess
    import sys
    code = """
import sys, torch
sys.path.insert(0, "intent-attention-kernel_b200")
import intent_attention as ia
pool = ia.Fp4Pool.allocate(64, 16, 128, zero=True)
table = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 1, 64)
n = torch.tensor([900], dtype=torch.int32, device="cuda")
k = torch.randn(1, 1, 900, 128, device="cuda").half()
q = torch.randn(1, 4, 128, device="cuda").half()
lam = torch.full((4,), 0.5, device="cuda")
refs = torch.ones(64, dtype=torch.int32, device="cuda")
pages = ia.SequencePages(refs, table, n, 16)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ia.append_fp4(pool, k, k, table)
    a = ia.paged_decode_fp4(q, pool, table, n)
    d = ia.differential_decode_fp4(q, pool, table, n, lam)
    r = ia.read_fp4(pool, table, None, 900)
    c = ia.compact_pages(pool, pages)
g.replay()
torch.cuda.synchronize()
assert torch.equal(a, ia.paged_decode_fp4(q, pool, table, n)) and torch.equal(d, ia.differential_decode_fp4(q, pool, table, n, lam))
assert int(c) == 64 and bool(torch.isfinite(a).all()) and bool((a != 0).any())
"""
    root = __file__.rsplit("/tests/", 1)[0]
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_lengths_beyond_the_table_and_negative():
    ia = _ia()
    pool, table, kd, vd = _cache(2, 3, 1, 64, 16, [64, 64, 64])
    t = table[:, :, :4].contiguous()
    q = _rows(np.random.default_rng(1), (3, 2, 64), "bf16")
    got = ia.paged_decode_fp4(q, pool, t, _i32([1000, -5, 2 ** 31 - 1]))
    _check(q, pool, t, [64, 0, 64], (kd, vd), got)


def test_offsets_past_32_bits():
    """Pages whose code bytes lie beyond 2^32."""
    ia = _ia()
    PS, D, n = 128, 128, 300
    P = (1 << 32) // (PS * D // 2) + 64
    pool = ia.Fp4Pool.allocate(P, PS, D)
    table = _i32([[[P - 1, P - 40, P - 3]]])
    g = np.random.default_rng(0)
    k, v = _rows(g, (1, 1, n, D), "bf16"), _rows(g, (1, 1, n, D), "bf16")
    ia.append_fp4(pool, k, v, table)
    gk, gv = ia.read_fp4(pool, table, None, n, dtype=torch.float32)
    kd, vd = of.values(_np(k)), of.values(_np(v))
    np.testing.assert_array_equal(_np(gk), kd)
    np.testing.assert_array_equal(_np(gv), vd)
    q = _rows(g, (1, 4, D), "bf16")
    _check(q, pool, table, [n], (kd, vd), ia.paged_decode_fp4(q, pool, table, _i32([n])))


def test_strided_q_and_out_and_dtypes():
    ia = _ia()
    pool, table, kd, vd = _cache(2, 2, 2, 128, 16, [100, 77])
    big = _rows(np.random.default_rng(1), (2, 3, 8, 130), "bf16")
    q = big[:, :, :, 1:129].transpose(1, 2)                    # [B, Hq, M, D]
    out = torch.zeros(2, 3, 8, 256, dtype=torch.float32, device="cuda")
    got = ia.paged_decode_fp4(q, pool, table, _i32([100, 77]), out=out[..., ::1][..., 100:228].transpose(1, 2))
    _check(q, pool, table, [100, 77], (kd, vd), got)
    assert (out[..., :100] == 0).all() and (out[..., 228:] == 0).all()
    half = ia.paged_decode_fp4(q, pool, table, _i32([100, 77]), out_dtype=torch.float16)
    assert half.dtype == torch.float16 and torch.equal(half, got.half())


def test_repeatable_and_captured():
    """Two runs agree to the bit; two graphs captured over one pool replay on new inputs, in any order."""
    ia = _ia()
    lengths = [5000, 1, 777]
    pool, table, kd, vd = _cache(6, 3, 2, 128, 16, lengths)
    g = np.random.default_rng(3)
    ln = _i32(lengths)
    lam = torch.full((16,), 0.4, device="cuda")
    qs = [_rows(g, (3, 16, 128), "bf16") for _ in range(3)]
    eager = [(ia.paged_decode_fp4(q, pool, table, ln), ia.differential_decode_fp4(q, pool, table, ln, lam)) for q in qs]
    for q, (a, d) in zip(qs, eager):
        assert torch.equal(a, ia.paged_decode_fp4(q, pool, table, ln))
    q = qs[0].clone()
    graphs, outs = [], []
    for f in (lambda: ia.paged_decode_fp4(q, pool, table, ln),
              lambda: ia.differential_decode_fp4(q, pool, table, ln, lam)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(f())
        graphs.append(gr)
    for order in ((0, 1), (1, 0)):
        for x, want in zip(qs, eager):
            q.copy_(x)
            for i in order:
                graphs[i].replay()
            torch.cuda.synchronize()
            for i in range(2):
                assert torch.equal(outs[i], want[i])


def test_two_streams_at_once():
    ia = _ia()
    lengths = [3000, 2000]
    pool, table, _, _ = _cache(6, 2, 2, 128, 16, lengths)
    g = np.random.default_rng(3)
    ln = _i32(lengths)
    qs = [_rows(g, (2, 8, 128), "bf16") for _ in range(2)]
    want = [ia.paged_decode_fp4(q, pool, table, ln) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ia.paged_decode_fp4(qs[i], pool, table, ln))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_empty_calls():
    ia = _ia()
    pool = ia.Fp4Pool.allocate(0, 16, 128)
    table = torch.empty((2, 1, 0), dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 128, device="cuda")
    assert (ia.paged_decode_fp4(q, pool, table, _i32([5, 0])) == 0).all()
    k = torch.randn(2, 1, 3, 128, device="cuda")
    dropped = torch.zeros(1, dtype=torch.int32, device="cuda")
    ia.append_fp4(pool, k, k, table, dropped=dropped)
    assert int(dropped) == 6
    assert (ia.read_fp4(pool, table, None, 3)[0] == 0).all()
    none = torch.empty((0, 1, 4), dtype=torch.int32, device="cuda")
    assert ia.paged_decode_fp4(q[:0], pool, none, _i32([])).shape == (0, 4, 128)
    assert ia.paged_decode_fp4(q[:, :0], pool, table, _i32([1, 1])).shape == (2, 0, 128)
    assert ia.read_fp4(pool, table, None, 0)[0].shape == (2, 1, 0, 128)
    ia.append_fp4(pool, k[:, :, :0], k[:, :, :0], table)


def test_refusals():
    ia = _ia()
    pool = ia.Fp4Pool.allocate(4, 16, 128, zero=True)
    table, ln = _i32([[[0, 1]]]), _i32([20])
    q = torch.randn(1, 2, 128, device="cuda")
    k = torch.randn(1, 1, 4, 128, device="cuda")
    lam = torch.zeros(2, device="cuda")
    bad = [
        lambda: ia.paged_decode_fp4(q[..., :64], pool, table, ln),
        lambda: ia.paged_decode_fp4(q.double(), pool, table, ln),
        lambda: ia.paged_decode_fp4(q, pool, table[0], ln),
        lambda: ia.paged_decode_fp4(q, pool, table.long(), ln),
        lambda: ia.paged_decode_fp4(q, pool, table, ln.long()),
        lambda: ia.paged_decode_fp4(q, pool, table, _i32([1, 2])),
        lambda: ia.paged_decode_fp4(torch.randn(1, 2, 17, 128, device="cuda"), pool, table, ln),
        lambda: ia.paged_decode_fp4(torch.randn(1, 3, 128, device="cuda"), pool, _i32([[[0], [1]]]), ln),
        lambda: ia.paged_decode_fp4(q, pool, table, ln, out=torch.empty(1, 2, 64, device="cuda")),
        lambda: ia.paged_decode_fp4(q, pool, table, ln, sm_scale=float("nan")),
        lambda: ia.paged_decode_fp4(q, pool, table, ln, sm_scale=float("inf")),
        lambda: ia.differential_decode_fp4(q, pool, table, ln, lam[:1]),
        lambda: ia.differential_decode_fp4(q, pool, table, ln, lam.half()),
        lambda: ia.differential_decode_fp4(q, pool, table, ln, lam, norm_weight=torch.ones(64, device="cuda")),
        lambda: ia.differential_decode_fp4(q, pool, table, ln, lam, eps=-1.0),
        lambda: ia.append_fp4(pool, k, k[:, :, :2], table),
        lambda: ia.append_fp4(pool, k, k.half(), table),
        lambda: ia.append_fp4(pool, k, k, _i32([[[0, 1]], [[2, 3]]])),
        lambda: ia.append_fp4(pool, k, k, table, _i32([0, 1])),
        lambda: ia.append_fp4(pool, k, k, table, counts=torch.zeros(1, device="cuda")),
        lambda: ia.read_fp4(pool, table, None, -1),
        lambda: ia.read_fp4(pool, table, None, 4, dtype=torch.float64),
        lambda: ia.read_fp4(pool, table, None, 4, out=(k[:, :, :2], k)),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with pytest.raises(RuntimeError):
        ia.paged_decode_fp4(q.cpu(), pool, table, ln)
    with pytest.raises(RuntimeError):
        ia.append_fp4(pool, k.cpu(), k.cpu(), table)
