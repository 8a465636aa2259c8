"""GPU parity of the ops on drafted tokens and the int8 KV cache against plain
numpy in 64 bits: per-head norms with rotation, quantised rows, attention of
trees and chains, verification."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F = np.float32
U = 2.0 ** -24  # half a step of f32, relative


def tree(rng, rows, reach=5, pad=0):
    p = np.array([rng.integers(max(-1, i - reach), i) if i else -1 for i in range(rows)], np.int32)
    if pad:
        p[rows - pad:] = -2
    return p


def path_to(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


def chain(rows):
    return np.arange(-1, rows - 1, dtype=np.int32)


# ------------------------------------------------------- norms and rotation
@pytest.mark.parametrize("n_q,n_kv,hd", [(6, 6, 48), (32, 8, 128), (5, 1, 4), (9, 3, 100), (3, 3, 256), (40, 20, 64), (2, 1, 20)])
@pytest.mark.parametrize("kind", ["chain", "tree", "no_norm"])
def test_qk_norm_rope(hip, n_q, n_kv, hd, kind):
    B = hip.HipBackend
    rng = np.random.default_rng(hd + n_q)
    n_seq, rows = (3, 21) if kind == "tree" else (2, 67)
    start = np.array([0, 131071, 500][:n_seq])
    par = np.stack([tree(rng, rows, pad=3 * s) for s in range(n_seq)]) if kind == "tree" else np.stack([chain(rows)] * n_seq)
    heads = n_q + 2 * n_kv
    x = rng.normal(0, 1, (n_seq * rows, heads, hd)).astype(F)
    x[1, 0] = 0.0  # a head of zeros
    x[2, 0] *= F(1e15)
    fr = (10000.0 ** (-np.arange(0, hd, 2) / hd)).astype(F)
    qw, kw = rng.normal(1, 0.2, hd).astype(F), rng.normal(1, 0.2, hd).astype(F)
    eps, qs = 1e-6, 0.37
    norm = kind != "no_norm"
    got = B.qk_norm_rope(B.from_vec(x), start, rows, n_q, n_kv, hd, B.from_vec(fr), B.from_vec(qw) if norm else None,
                         B.from_vec(kw) if norm else None, eps, qs, parents=par if kind == "tree" else None)
    q, k, v = (g.to_vec().reshape(n_seq * rows, -1, hd) for g in got)
    pos = np.array([start[s] + max(0, len(path_to(par[s], i)) - 1 if par[s][i] != -2 else 0)
                    for s in range(n_seq) for i in range(rows)], np.float64)
    ang = pos[:, None, None] * fr.astype(np.float64)
    co, si = np.cos(ang), np.sin(ang)
    for name, out, lo, hi, w, scale in (("q", q, 0, n_q, qw, F(qs)), ("k", k, n_q, n_q + n_kv, kw, F(1))):
        h = x[:, lo:hi].astype(np.float64)
        if norm:
            h = h / np.sqrt((h * h).mean(-1, keepdims=True) + float(F(eps))) * w
        a, b = h[..., 0::2], h[..., 1::2]
        ref = np.stack((a * co - b * si, a * si + b * co), -1).reshape(h.shape) * float(scale)
        # the norm's factor: squares, a sum over at most 4 + 6 levels, mean, eps,
        # root, reciprocal: 14 roundings, halved by the root for the sum's part;
        # two products; cos and sin; the rotation's product and sum; the scale:
        # 20 half steps of (|a| + |b|) bound them
        size = (np.abs(ref[..., 0::2]) + np.abs(ref[..., 1::2])).repeat(2, -1)
        bad = np.abs(out - ref) > 20 * U * size + 1e-38
        assert not bad.any(), (name, np.argwhere(bad)[:4])
    assert np.array_equal(v, x[:, n_q + n_kv:])


def test_qk_norm_rope_agrees_with_rope(hip):
    """Without weights a chain is rope_with_freqs[_scaled]_preloaded of its parts."""
    B = hip.HipBackend
    rng = np.random.default_rng(5)
    rows, n_q, n_kv, hd = 33, 8, 2, 64
    x = rng.normal(0, 1, (rows, (n_q + 2 * n_kv) * hd)).astype(F)
    fr = B.from_vec((500000.0 ** (-np.arange(0, hd, 2) / hd)).astype(F))
    q, k, v = B.qk_norm_rope(B.from_vec(x), [77], rows, n_q, n_kv, hd, fr, q_scale=0.125)
    a = B.rope_with_freqs_scaled_preloaded(B.from_vec(x[:, :n_q * hd]), rows, n_q, hd, 77, fr, 0.125).to_vec()
    b = B.rope_with_freqs_preloaded(B.from_vec(x[:, n_q * hd:(n_q + n_kv) * hd]), rows, n_kv, hd, 77, fr).to_vec()
    # the same angles; products and sums may fuse otherwise: two roundings of |a| + |b|
    assert np.abs(q.to_vec() - a).max() <= 4 * U * 2 * np.abs(a).max()
    assert np.abs(k.to_vec() - b).max() <= 4 * U * 2 * np.abs(b).max()
    assert np.array_equal(v.to_vec().reshape(rows, -1), x[:, (n_q + n_kv) * hd:])


# ------------------------------------------------------------- the int8 cache
def quantised(x):
    """(q, s) of rows [.., hd] by the definition; the quotient of two f32 values
    is never nearer to a half than f64 resolves."""
    x64 = x.astype(np.float64)
    ok = np.isfinite(x).all(-1, keepdims=True)
    s = (np.abs(np.where(ok, x, 0)).max(-1, keepdims=True) / F(127)).astype(F)
    with np.errstate(divide="ignore", invalid="ignore"):
        r = np.where(s > 0, x64 / s.astype(np.float64), 0.0)
    q = np.where(ok, np.minimum(np.floor(np.abs(np.where(ok, r, 0)) + 0.5), 127) * np.sign(x64), 0)
    return np.nan_to_num(q).astype(np.int8), np.where(ok, s, F(np.nan)).astype(F)


def stored(x):
    q, s = quantised(x)
    return (q.astype(F) * s).astype(F)


def kv_rows(rng, *shape):
    x = rng.normal(0, 1, shape).astype(F)
    flat = x.reshape(-1, shape[-1])
    flat[0] = 0.0
    if len(flat) > 6:
        flat[1, 0], flat[2, -1] = np.nan, -np.inf
        flat[3] *= F(1e-42)   # subnormal scale
        flat[4] *= F(1e37)
        # quotients at and next to halves: max 127, so s = 1
        flat[5] = (np.arange(shape[-1]) % 127 - 63 + 0.5).astype(F)
        flat[5, 0] = 127.0
        flat[6] = np.nextafter(flat[5], F(0))
        flat[6, 0] = 127.0
    return x


@pytest.mark.parametrize("n_kv,hd,n_seq,rows,start", [
    (8, 128, 1, 1, [0]), (8, 128, 3, 5, [0, 63, 200]), (6, 48, 2, 64, [1, 127]), (1, 4, 2, 130, [5, 64]), (2, 100, 1, 300, [33]),
    (3, 20, 16, 3, list(range(60, 76))), (2, 256, 2, 67, [0, 3]), (32, 128, 1, 257, [0])])
def test_kv8_write_read(hip, n_kv, hd, n_seq, rows, start):
    B = hip.HipBackend
    rng = np.random.default_rng(hd * rows)
    size = [start[s] + rows + (s % 3) for s in range(n_seq)]
    caches = [B.kv8_new(size[s], n_kv, hd) for s in range(n_seq)]
    before = [rng.normal(0, 1, (size[s], n_kv, hd)).astype(F) for s in range(n_seq)]
    for s in range(n_seq):
        B.kv8_write([caches[s]], B.from_vec(before[s]), B.from_vec(before[s] * 2), [0], size[s])
    k, v = kv_rows(rng, n_seq, rows, n_kv, hd), kv_rows(rng, n_seq, rows, n_kv, hd)[::-1].copy()
    B.kv8_write(caches, B.from_vec(k), B.from_vec(v), start, rows)
    gk, gv = B.kv8_read(caches, start, rows)
    assert np.array_equal(gk.to_vec().reshape(k.shape), stored(k), equal_nan=True)
    assert np.array_equal(gv.to_vec().reshape(v.shape), stored(v), equal_nan=True)
    for s in range(n_seq):  # every other row of each cache is as it was
        a, b = (g.to_vec().reshape(before[s].shape) for g in B.kv8_read([caches[s]], [0], size[s]))
        for got, old, new in ((a, before[s], k[s]), (b, before[s] * 2, v[s])):
            want = stored(old)
            want[start[s]:start[s] + rows] = stored(new)
            assert np.array_equal(got, want, equal_nan=True), s


def test_kv8_unwritten_rows_are_zero(hip):
    B = hip.HipBackend
    for _ in range(2):
        c = B.kv8_new(130, 2, 36)
        k, v = B.kv8_read([c], [0], 130)
        assert not k.to_vec().any() and not v.to_vec().any()
        B.kv8_write([c], B.ones(130 * 72), B.ones(130 * 72), [0], 130)
        c.free()


@pytest.mark.parametrize("n_kv,hd", [(8, 128), (3, 20), (1, 100)])
def test_kv8_keep(hip, n_kv, hd):
    B = hip.HipBackend
    rng = np.random.default_rng(n_kv)
    starts, rows = [0, 37, 60], 64
    paths = np.full((3, 20), -1, np.int64)
    paths[0, :20] = np.sort(rng.choice(64, 20, replace=False))
    paths[1, :3] = [0, 1, 2]
    paths[2, :11] = [1, 2, 3, 9, 10, 12, 30, 31, 33, 62, 63]
    caches = [B.kv8_new(st + rows, n_kv, hd) for st in starts]
    data = [rng.normal(0, 1, (2, st + rows, n_kv, hd)).astype(F) for st in starts]
    for c, d, st in zip(caches, data, starts):
        B.kv8_write([c], B.from_vec(d[0]), B.from_vec(d[1]), [0], st + rows)
    B.kv8_keep(caches, starts, paths)
    for s, (c, d, st) in enumerate(zip(caches, data, starts)):
        n = int((paths[s] >= 0).sum())
        for got, x in zip(B.kv8_read([c], [0], st + rows), d):
            want = stored(x)
            want[st:st + n] = want[st + paths[s, :n]].copy()
            assert np.array_equal(got.to_vec().reshape(want.shape), want), s
    B.kv8_keep(caches, starts, np.full((3, 1), -1))  # empty paths: nothing moves


# ------------------------------------------------------------------ attention
def attend(q, k, v, lens, par, scale):
    """q [n, rows, n_q, hd]; k, v: per sequence [len + rows, n_kv, hd]. Returns
    the output and a bound of its error, per row and head."""
    n, rows, n_q, hd = q.shape
    out, tol = np.zeros(q.shape), np.zeros((n, rows, n_q, 1))
    for s in range(n):
        rep = n_q // k[s].shape[1]
        for i in range(rows):
            if par[s][i] == -2:
                continue
            keys = list(range(lens[s])) + [lens[s] + j for j in path_to(par[s], i)]
            for h in range(n_q):
                kk, vv = k[s][keys, h // rep].astype(np.float64), v[s][keys, h // rep].astype(np.float64)
                sc = kk @ q[s, i, h].astype(np.float64) * scale
                with np.errstate(invalid="ignore", over="ignore"):
                    p = np.exp(sc - sc.max())
                    out[s, i, h] = p @ vv / p.sum()
                    # a score: hd products and sums, q held to 24 bits of its largest
                    # value, two scales; a weight moves by twice that and exp's own
                    # steps; each sum takes at most a rounding a key, and a weight is
                    # held to 2^-23 of the largest
                    ds = (hd + 8) * U * scale * np.abs(q[s, i, h]).max() * np.abs(kk).sum(-1).max() + 4 * U * np.abs(sc).max()
                    tol[s, i, h] = (2 * ds + (4 * len(keys) + 32) * U) * np.abs(vv).max()
    return out, tol


def check_close(got, ref, tol):
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    ok = ~np.isnan(ref)
    err = np.abs(got - ref)
    assert (err[ok] <= np.broadcast_to(tol, ref.shape)[ok]).all(), (err[ok].max(), np.nanmax(tol))


CASES = [  # n_q, n_kv, hd, lens, rows, kind
    (6, 6, 48, [77], 1, "chain"), (6, 6, 48, [0], 1, "chain"), (8, 2, 64, [1, 0, 64, 63], 1, "chain"),
    (32, 8, 128, [300, 129], 26, "tree"), (32, 8, 128, [0, 5], 64, "tree"), (9, 3, 100, [65, 400], 17, "tree"),
    (5, 1, 4, [200], 33, "tree"), (10, 2, 80, [191, 192, 193], 7, "pad"), (4, 4, 128, [130], 70, "chain"),
    (8, 1, 256, [100, 31], 5, "tree"), (4, 2, 20, [1000], 130, "chain"), (40, 4, 64, [50], 3, "pad"),
    (2, 2, 64, [2500], 1, "chain"), (8, 8, 128, [3000, 10], 2, "chain"), (64, 2, 32, [90], 40, "tree"),
    (3, 1, 12, list(range(16)), 6, "pad")]


def attention_case(n_q, n_kv, hd, lens, rows, kind, seed=0):
    rng = np.random.default_rng(seed + hd + rows)
    n = len(lens)
    par = np.stack([chain(rows) if kind == "chain" else tree(rng, rows, pad=(rows // 2 if kind == "pad" and s % 2 == 0 else 0))
                    for s in range(n)])
    q = rng.normal(0, 1, (n, rows, n_q, hd)).astype(F)
    q[0, 0] *= F(6.0)  # a row whose softmax is sharp
    k = [rng.normal(0, 1, (ln + rows, n_kv, hd)).astype(F) for ln in lens]
    v = [rng.normal(0, 1, (ln + rows, n_kv, hd)).astype(F) for ln in lens]
    return q, k, v, par


@pytest.mark.parametrize("cache", ["f32", "int8"])
@pytest.mark.parametrize("n_q,n_kv,hd,lens,rows,kind", CASES)
def test_attention(hip, cache, n_q, n_kv, hd, lens, rows, kind):
    B = hip.HipBackend
    q, k, v, par = attention_case(n_q, n_kv, hd, lens, rows, kind)
    scale = 1.0 / math.sqrt(hd)
    pa = None if kind == "chain" else par
    extra = 37  # cache rows behind the last: whatever they hold stays out
    junk = np.full((extra, n_kv, hd), np.nan, F)
    full = [(np.concatenate((a, junk)), np.concatenate((b, junk))) for a, b in zip(k, v)]
    if cache == "f32":
        o = B.tree_attention(B.from_vec(q), [B.from_vec(a) for a, _ in full], [B.from_vec(b) for _, b in full], lens, rows, n_q,
                             n_kv, hd, scale, parents=pa)
    else:
        caches = []
        for a, b in full:
            caches.append(B.kv8_new(len(a), n_kv, hd))
            B.kv8_write(caches[-1:], B.from_vec(a), B.from_vec(b), [0], len(a))
        o = B.kv8_tree_attention(B.from_vec(q), caches, lens, rows, n_q, scale, parents=pa)
        k, v = [stored(a) for a in k], [stored(b) for b in v]
    ref, tol = attend(q, k, v, lens, par, float(F(scale)))
    check_close(o.to_vec().reshape(q.shape), ref, tol)


@pytest.mark.parametrize("cache", ["f32", "int8"])
@pytest.mark.parametrize("tiles", [1, 2, 3, 4, 5, 7])
@pytest.mark.parametrize("hd", [16, 60, 64, 68, 128, 132, 192, 196, 256])
def test_attention_every_shape_of_kernel(hip, cache, hd, tiles):
    """Head sizes about the 64-dimension blocks, columns about the 16-column
    tiles and groups of them, contexts that end in and at a step of keys."""
    B = hip.HipBackend
    n_q, n_kv = 2, 2
    rows = 16 * tiles - 3
    lens = [0, 63, 130, 64 * tiles - rows + 64]
    kind = "tree" if rows <= 64 else "chain"
    q, k, v, par = attention_case(n_q, n_kv, hd, lens, rows, kind, tiles)
    scale = 1.0 / math.sqrt(hd)
    pa = par if kind == "tree" else None
    if cache == "f32":
        o = B.tree_attention(B.from_vec(q), [B.from_vec(a) for a in k], [B.from_vec(b) for b in v], lens, rows, n_q, n_kv, hd,
                             scale, parents=pa)
    else:
        caches = []
        for a, b in zip(k, v):
            caches.append(B.kv8_new(len(a), n_kv, hd))
            B.kv8_write(caches[-1:], B.from_vec(a), B.from_vec(b), [0], len(a))
        o = B.kv8_tree_attention(B.from_vec(q), caches, lens, rows, n_q, scale, parents=pa)
        k, v = [stored(a) for a in k], [stored(b) for b in v]
    ref, tol = attend(q, k, v, lens, par, float(F(scale)))
    check_close(o.to_vec().reshape(q.shape), ref, tol)


@pytest.mark.parametrize("cache", ["f32", "int8"])
@pytest.mark.parametrize("n_q,n_kv,rows,ln", [(4, 1, 1, 20000), (2, 1, 20, 9000), (32, 1, 2, 6000), (64, 1, 16, 3000)])
def test_attention_long_contexts_in_splits(hip, cache, n_q, n_kv, rows, ln):
    """Key splits joined by the last workgroup, by groups of threads, by a thread
    per column: one sharp row (its key early, late) and broad ones."""
    B = hip.HipBackend
    hd = 64
    q, k, v, par = attention_case(n_q, n_kv, hd, [ln, ln // 3], rows, "chain", 5)
    q[1, 0, 0] = k[1][7, 0] * F(3)
    q[0, rows - 1, n_q - 1] = k[0][ln - 2, 0] * F(3)
    scale = 0.125
    if cache == "f32":
        o = B.tree_attention(B.from_vec(q), [B.from_vec(a) for a in k], [B.from_vec(b) for b in v], [ln, ln // 3], rows, n_q, n_kv,
                             hd, scale)
    else:
        caches = []
        for a, b in zip(k, v):
            caches.append(B.kv8_new(len(a), n_kv, hd))
            B.kv8_write(caches[-1:], B.from_vec(a), B.from_vec(b), [0], len(a))
        o = B.kv8_tree_attention(B.from_vec(q), caches, [ln, ln // 3], rows, n_q, scale)
        k, v = [stored(a) for a in k], [stored(b) for b in v]
    got = o.to_vec().reshape(q.shape)
    for s, n in enumerate((ln, ln // 3)):
        for i in range(rows):
            keys = n + i + 1
            sc = k[s][:keys, 0].astype(np.float64) @ q[s, i].astype(np.float64).T * scale  # [keys, n_q]
            p = np.exp(sc - sc.max(0))
            p /= p.sum(0)
            ref = p.T @ v[s][:keys, 0].astype(np.float64)
            # as attend(): a score's error, and the sums'; chunks of keys are summed
            # apart and joined, so no sum has more than 2^10 terms in a row, and the
            # weights' steps are at most 2^-23 of the largest
            ds = (hd + 8) * U * scale * np.abs(q[s, i]).max() * np.abs(k[s][:keys, 0]).sum(-1).max() + 4 * U * np.abs(sc).max()
            tol = (2 * ds + (4 * 1024 + 32) * U) * np.abs(v[s][:keys, 0]).max()
            assert np.abs(got[s, i] - ref).max() <= tol, (s, i, np.abs(got[s, i] - ref).max(), tol)


@pytest.mark.parametrize("n_seq", [1, 2])
@pytest.mark.parametrize("cache,ln", [("f32", 2000), ("int8", 4000)])
def test_attention_of_many_heads_in_few_splits(hip, cache, ln, n_seq):
    """One tile of columns of each of 40 KV heads, whose 16 (8) splits have more
    partial sums than the last workgroup of a head joins."""
    B = hip.HipBackend
    n_kv, hd, rows = 40, 128, 16
    lens = [ln, ln - 65][:n_seq]
    q, k, v, par = attention_case(n_kv, n_kv, hd, lens, rows, "chain", 6)
    scale = hd ** -0.5
    if cache == "f32":
        o = B.tree_attention(B.from_vec(q), [B.from_vec(a) for a in k], [B.from_vec(b) for b in v], lens, rows, n_kv, n_kv, hd, scale)
    else:
        caches = []
        for a, b in zip(k, v):
            caches.append(B.kv8_new(len(a), n_kv, hd))
            B.kv8_write(caches[-1:], B.from_vec(a), B.from_vec(b), [0], len(a))
        o = B.kv8_tree_attention(B.from_vec(q), caches, lens, rows, n_kv, scale)
        k, v = [stored(a) for a in k], [stored(b) for b in v]
    got = o.to_vec().reshape(q.shape)
    for s, n in enumerate(lens):
        seen = np.arange(n + rows)[:, None] <= n + np.arange(rows)  # [keys, rows]
        for h in range(n_kv):
            kk, vv = k[s][:, h].astype(np.float64), v[s][:, h].astype(np.float64)
            sc = np.where(seen, kk @ q[s, :, h].astype(np.float64).T * scale, -np.inf)
            p = np.exp(sc - sc.max(0))
            ref = (p / p.sum(0)).T @ vv
            # as in the long contexts above
            ds = (hd + 8) * U * scale * np.abs(q[s, :, h]).max(-1) * np.abs(kk).sum(-1).max() + 4 * U * np.abs(np.where(seen, sc, 0)).max(0)
            tol = (2 * ds + (4 * 1024 + 32) * U) * np.abs(vv).max()
            assert (np.abs(got[s, :, h] - ref).max(-1) <= tol).all(), (s, h)


@pytest.mark.parametrize("rows", [3, 30])
@pytest.mark.parametrize("cache", ["f32", "int8"])
def test_attention_scales_of_zero_and_below(hip, cache, rows):
    """Scale 0: equal weights; a negative scale: the queries turned round."""
    B = hip.HipBackend
    n_q, n_kv, hd, lens = 8, 2, 64, [70, 0]
    q, k, v, par = attention_case(n_q, n_kv, hd, lens, rows, "tree", 8)
    if cache == "f32":
        sk, sv = [B.from_vec(a) for a in k], [B.from_vec(b) for b in v]
    else:
        caches = []
        for a, b in zip(k, v):
            caches.append(B.kv8_new(len(a), n_kv, hd))
            B.kv8_write(caches[-1:], B.from_vec(a), B.from_vec(b), [0], len(a))
        k, v = [stored(a) for a in k], [stored(b) for b in v]
    for scale in (0.0, -0.2):
        x = B.from_vec(q)
        o = B.tree_attention(x, sk, sv, lens, rows, n_q, n_kv, hd, scale, parents=par) if cache == "f32" else \
            B.kv8_tree_attention(x, caches, lens, rows, n_q, scale, parents=par)
        check_close(o.to_vec().reshape(q.shape), *attend(-q, k, v, lens, par, -scale))


@pytest.mark.parametrize("cache", ["f32", "int8"])
def test_attention_hides_what_is_masked(hip, cache):
    """NaN and infinities in rows that a node does not see leave it alone; in
    rows that it sees, they reach it. Values of the type's lowest and highest."""
    B = hip.HipBackend
    n_q, n_kv, hd, ln, rows = 8, 2, 64, 70, 12
    q, k, v, _ = attention_case(n_q, n_kv, hd, [ln], rows, "chain", 3)
    par = np.array([[-1, 0, 1, 0, 3, -1, 5, 6, 2, -2, 5, 10]], np.int32)
    k[0][ln + 3], v[0][ln + 3] = np.nan, np.inf            # seen by 3 and 4
    v[0][ln + 7, 0, 5], k[0][ln + 10, 1] = -np.inf, np.inf  # 7; and 10, 11
    k[0][ln + 9], v[0][ln + 9] = np.nan, np.nan             # no node: seen by none
    v[0][ln + 8] = np.finfo(F).max / 4
    scale = 0.125
    if cache == "f32":
        o = B.tree_attention(B.from_vec(q), [B.from_vec(k[0])], [B.from_vec(v[0])], [ln], rows, n_q, n_kv, hd, scale, parents=par)
    else:
        c = B.kv8_new(ln + rows, n_kv, hd)
        B.kv8_write([c], B.from_vec(k[0]), B.from_vec(v[0]), [0], ln + rows)
        o = B.kv8_tree_attention(B.from_vec(q), [c], [ln], rows, n_q, scale, parents=par)
        k, v = [stored(k[0])], [stored(v[0])]
    got = o.to_vec().reshape(q.shape)[0]
    clean = [0, 1, 2, 5, 6, 9]
    assert np.isfinite(got[clean + [8]]).all() and not got[9].any()
    assert np.isnan(got[[3, 4]]).all()
    fin = [np.nan_to_num(x[0], nan=0, posinf=0, neginf=0)[None] for x in (k, v)]
    ref, tol = attend(q, fin[0], fin[1], [ln], par, scale)
    for i in clean + [8]:
        check_close(got[i], ref[0, i], tol[0, i])
    if cache == "f32":
        ref, tol = attend(q, k, v, [ln], par, scale)
        hit = np.zeros((n_q, hd), bool)
        hit[:4, 5] = True
        assert (got[7][hit] == -np.inf).all() and np.isfinite(got[7][~hit]).all()
        # an infinite key: a score of +inf has no softmax, one of -inf no weight
        assert np.isfinite(got[10, :4]).all() and np.array_equal(np.isnan(got[10, 4:]), np.isnan(ref[0, 10, 4:]))
    else:
        assert np.isnan(got[7, :4]).all() and np.isfinite(got[7, 4:]).all()
        assert np.isnan(got[10, 4:]).all() and np.isfinite(got[10, :4]).all()


@pytest.mark.parametrize("cache", ["f32", "int8"])
def test_attention_extreme_scores(hip, cache):
    """Scores far apart and of large size: the first key takes all, or none."""
    B = hip.HipBackend
    n_q, hd, ln = 2, 64, 333
    rng = np.random.default_rng(8)
    k = rng.normal(0, 1, (ln + 1, 1, hd)).astype(F)
    v = rng.normal(0, 1, (ln + 1, 1, hd)).astype(F)
    q = np.stack([k[100, 0], -k[100, 0]])[None, None].astype(F) * F(1e4)
    if cache == "f32":
        o = B.tree_attention(B.from_vec(q), [B.from_vec(k)], [B.from_vec(v)], [ln], 1, n_q, 1, hd, 1.0)
    else:
        c = B.kv8_new(ln + 1, 1, hd)
        B.kv8_write([c], B.from_vec(k), B.from_vec(v), [0], ln + 1)
        o = B.kv8_tree_attention(B.from_vec(q), [c], [ln], 1, n_q, 1.0)
        k, v = stored(k), stored(v)
    sc = k[:, 0].astype(np.float64) @ q[0, 0].astype(np.float64).T
    best = sc.argmax(0)
    assert best[0] == 100 and (np.sort(sc, 0)[-1] - np.sort(sc, 0)[-2] > 1e3).all()
    got = o.to_vec().reshape(2, hd)
    for h in range(2):  # one weight is 1, the others underflow
        assert np.abs(got[h] - v[best[h], 0]).max() <= 4 * U * np.abs(v[best[h], 0]).max()


@pytest.mark.parametrize("cache", ["f32", "int8"])
def test_attention_offsets_past_32_bits(hip, cache):
    """A cache above 4 GiB: keys of zero weigh the same, and a few rows at the
    end, past 2^32 bytes, take most of it."""
    B = hip.HipBackend
    n_kv, hd = 8, 128
    ln = 1_100_000 if cache == "f32" else 4_300_000
    rng = np.random.default_rng(2)
    new = rng.normal(0, 1, (64, n_kv, hd)).astype(F)
    val = rng.normal(0, 1, (64, n_kv, hd)).astype(F)
    q = (new[10] * 0.25).reshape(1, 1, n_kv, hd)  # head h's query is row 10's key
    if cache == "f32":
        kc, vc = B.zeros((ln + 1) * n_kv * hd), B.zeros((ln + 1) * n_kv * hd)
        for c, x in ((kc, new), (vc, val)):
            B.scatter_rows(c, B.from_vec(x), ln + 1, n_kv * hd, ln + 1 - 64, 64)
        o = B.tree_attention(B.from_vec(q), [kc], [vc], [ln], 1, n_kv, n_kv, hd, 1.0)
    else:
        c = B.kv8_new(ln + 1, n_kv, hd)
        B.kv8_write([c], B.from_vec(new), B.from_vec(val), [ln + 1 - 64], 64)
        a, b = B.kv8_read([c], [ln + 1 - 64], 64)
        assert np.array_equal(a.to_vec().reshape(new.shape), stored(new))
        assert np.array_equal(b.to_vec().reshape(new.shape), stored(val))
        o = B.kv8_tree_attention(B.from_vec(q), [c], [ln], 1, n_kv, 1.0)
        new, val = stored(new), stored(val)
    got = o.to_vec().reshape(n_kv, hd)
    for h in range(n_kv):
        sc = new[:, h].astype(np.float64) @ q[0, 0, h].astype(np.float64)
        p = np.exp(sc)
        ref = p @ val[:, h].astype(np.float64) / (p.sum() + ln - 63)
        # the keys of zero: ln terms of one weight, summed in f32: relative
        # rounding a term in the worst case would hide the rest, so the bound is
        # that of sums over blocks of 2^15 terms at most, joined: 2^-9 of 1
        assert np.abs(got[h] - ref).max() <= 2.0 ** -9 * np.abs(ref).max(), h


def test_attention_of_shared_caches_and_repeats(hip):
    """Two sequences over one cache, and the same call twice: the same bits."""
    B = hip.HipBackend
    n_q, n_kv, hd, ln, rows = 8, 2, 64, 2000, 5
    q, k, v, par = attention_case(n_q, n_kv, hd, [ln], rows, "tree", 11)
    q2 = B.from_vec(np.concatenate((q, q)))
    kc, vc = B.from_vec(k[0]), B.from_vec(v[0])
    c = B.kv8_new(ln + rows, n_kv, hd)
    B.kv8_write([c], kc, vc, [0], ln + rows)
    for call in (lambda: B.tree_attention(q2, [kc, kc], [vc, vc], [ln, ln], rows, n_q, n_kv, hd, 0.1, parents=par[0]),
                 lambda: B.kv8_tree_attention(q2, [c, c], [ln, ln], rows, n_q, 0.1, parents=par[0])):
        a, b = call(), call()
        x = a.to_vec().reshape(2, -1)
        assert np.array_equal(x[0], x[1]) and np.array_equal(x.ravel(), b.to_vec())


# --------------------------------------------------------------- verification
def pick(w, u):
    w = np.where((w > 0) & np.isfinite(w), w, 0.0).astype(np.float64)
    c = np.cumsum(w)
    return None if not c[-1] > 0 else int(np.searchsorted(c, u * c[-1], side="right"))


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(F)


def draft_ref(p, q, tok, u, count):
    V = p.shape[-1]
    n = next((i for i in range(count) if not u[i] * float(q[i, tok[i]]) < float(p[i, tok[i]])), count)
    w = p[n].astype(np.float64) - (q[n].astype(np.float64) if n < count else 0)
    t = pick(w, u[-1])
    if t is None:
        t = pick(p[n], u[-1])
    return n, int(u[-1] * V) if t is None else t


@pytest.mark.parametrize("V,n_seq,rows", [(1, 1, 1), (7, 2, 3), (2048, 1, 4), (2049, 3, 8), (32000, 1, 5), (50257, 16, 16),
                                          (128256, 2, 64), (300001, 1, 2)])
def test_verify_draft(hip, V, n_seq, rows):
    B = hip.HipBackend
    rng = np.random.default_rng(V + rows)
    seen = set()
    for trial in range(3):
        lg = rng.normal(0, 2, (n_seq, rows + 1, V))
        p = softmax(lg)
        q = softmax(lg[:, :rows] + rng.normal(0, [0.05, 0.5, 2][trial], (n_seq, rows, V)))
        tok = np.array([[min(V - 1, int(np.searchsorted(np.cumsum(q[s, i], dtype=np.float64), rng.random() * 0.999))) for i in range(rows)]
                        for s in range(n_seq)])
        u = rng.random((n_seq, rows + 1))
        counts = None if trial == 0 else rng.integers(0, rows + 1, n_seq)
        n, t = B.verify_draft(B.from_vec(p), B.from_vec(q), tok, u, V, counts)
        for s in range(n_seq):
            ref = draft_ref(p[s], q[s], tok[s], u[s], rows if counts is None else counts[s])
            assert (int(n[s]), int(t[s])) == ref, (s, ref)
            seen.add(ref[0])
    assert rows < 4 or len(seen) > 1


def test_verify_draft_edges(hip):
    """No residual, no mass, weights that are no numbers, numbers at both ends,
    a token that the draft could not have drawn."""
    B = hip.HipBackend
    V = 5000
    one = np.zeros(V, F)
    one[4321] = 1.0
    half = np.zeros(V, F)
    half[[10, 2047, 2048, 4999]] = 0.25
    bad = half.copy()
    bad[[0, 3000]], bad[4000] = np.nan, np.inf
    neg = half.copy()
    neg[20:40] = -1.0
    zero = np.zeros(V, F)
    top = np.nextafter(1.0, 0.0)
    cases = [  # p_0, q_0, p_1, token, u_0, u_1
        (one, one, half, 4321, 0.5, 0.0), (one, one, half, 4321, top, top), (one, half, half, 10, 0.0, 0.3),
        (half, half, one, 11, 0.0, 0.6), (zero, half, one, 10, 0.5, 0.7), (half, one, bad, 10, 0.2, 0.75), (bad, one, half, 0, 0.1, 0.5),
        (neg, zero, one, 25, 0.0, 0.49), (half, zero, half, 10, 0.9, top), (half, zero, bad, 10, 0.9, top), (zero, zero, zero, 0, 0.0, top),
        (half, zero, half, 10, 0.9, 0.25), (half, zero, half, 10, 0.9, np.nextafter(0.25, 0.0))]
    n_seq = len(cases)
    p = np.stack([np.stack((c[0], c[2])) for c in cases])
    q = np.stack([c[1][None] for c in cases])
    tok = np.array([[c[3]] for c in cases])
    u = np.array([[c[4], c[5]] for c in cases])
    n, t = B.verify_draft(B.from_vec(p), B.from_vec(q), tok, u, V)
    for s in range(n_seq):
        with np.errstate(invalid="ignore"):
            ref = draft_ref(p[s], q[s], tok[s], u[s], 1)
        assert (int(n[s]), int(t[s])) == ref, (s, ref)


@pytest.mark.parametrize("V,n_seq,rows", [(1, 1, 1), (33, 2, 5), (32000, 1, 26), (50257, 3, 64), (128256, 2, 9), (5000, 16, 64)])
def test_verify_tree(hip, V, n_seq, rows):
    B = hip.HipBackend
    rng = np.random.default_rng(V + rows)
    lg = rng.normal(0, 1, (n_seq, rows + 1, V))
    for s in range(n_seq):
        for r in range(rows + 1):
            lg[s, r, rng.integers(0, V, 3)] += 14.0
    p = softmax(lg)
    par = np.stack([tree(rng, rows, 4, pad=(rows // 3 if s % 2 else 0)) for s in range(n_seq)])
    tok = np.empty((n_seq, rows), np.int64)
    for s in range(n_seq):
        used = {}
        for i in range(rows):  # children hold the likeliest tokens; now and then one twice
            r = max(par[s, i], -1) + 1
            order = np.argsort(-p[s, r])
            tok[s, i] = order[min(V - 1, used.get(r, 0))]
            used[r] = used.get(r, 0) + (rng.random() < 0.8)
    tok[par == -2] = -5  # what is no node may hold anything
    u = rng.random((n_seq, rows + 1))
    paths, n, t = B.verify_tree(B.from_vec(p), tok, par, u, V)
    assert paths.shape == (n_seq, rows)
    for s in range(n_seq):
        cur, want = -1, []
        while True:
            x = pick(p[s, cur + 1], u[s, cur + 1])
            nxt = [i for i in range(rows) if par[s, i] == cur and tok[s, i] == x]
            if not nxt:
                break
            cur = nxt[0]
            want.append(cur)
        assert list(paths[s, :n[s]]) == want and (paths[s, n[s]:] == -1).all() and t[s] == x, s


def test_verify_behind_queued_work(hip):
    """Tens of milliseconds of other ops are queued before the call: it waits
    for them, and its results are its own."""
    B = hip.HipBackend
    rng = np.random.default_rng(4)
    V = 4000
    a = B.from_vec(rng.normal(0, 1, 4096 * 4096).astype(F))
    for turn in range(3):
        p = softmax(rng.normal(0, 2, (2, 4, V)))
        q = softmax(rng.normal(0, 2, (2, 3, V)))
        tok, u = q.argmax(-1), rng.random((2, 4))
        hp, hq = B.from_vec(p), B.from_vec(q)
        held = [B.matmul(a, a, 4096, 4096, 4096) for _ in range(40 if turn else 1)]
        n, t = B.verify_draft(hp, hq, tok, u, V)
        for s in range(2):
            assert (int(n[s]), int(t[s])) == draft_ref(p[s], q[s], tok[s], u[s], 3)
        del held


# ---------------------------------------------------------------- as they are used
@pytest.mark.parametrize("cache", ["f32", "int8"])
def test_a_speculative_run(hip, cache):
    """Three steps of a batch: qkv rows of a drafted tree are normed and turned,
    written, attended to, verified; the accepted path is kept, and what follows
    attends to the same rows as a run that had them in order all along."""
    B = hip.HipBackend
    rng = np.random.default_rng(21)
    n_seq, n_q, n_kv, hd, V, max_seq = 3, 8, 2, 64, 500, 300
    scale = 1.0 / math.sqrt(hd)
    fr = B.from_vec((10000.0 ** (-np.arange(0, hd, 2) / hd)).astype(F))
    qw, kw = (B.from_vec(rng.normal(1, 0.1, hd).astype(F)) for _ in range(2))
    lens = np.array([100, 3, 64])
    table = rng.normal(0, 1, (V, (n_q + 2 * n_kv) * hd)).astype(F)  # a token's qkv row

    def new_store():
        if cache == "int8":
            return [B.kv8_new(max_seq, n_kv, hd) for _ in range(n_seq)]
        return [(B.zeros(max_seq * n_kv * hd), B.zeros(max_seq * n_kv * hd)) for _ in range(n_seq)]

    def write(store, s, k, v, at, rows):
        if cache == "int8":
            B.kv8_write([store[s]], k, v, [at], rows)
        else:
            for c, x in zip(store[s], (k, v)):
                B.scatter_rows(c, x, max_seq, n_kv * hd, at, rows)

    def attention(store, q, lens, rows, parents):
        if cache == "int8":
            return B.kv8_tree_attention(q, store, lens, rows, n_q, scale, parents=parents)
        return B.tree_attention(q, [c[0] for c in store], [c[1] for c in store], lens, rows, n_q, n_kv, hd, scale, parents=parents)

    def feed(store, toks, lens, parents):
        """toks [n_seq, rows] through one layer: the attention's rows."""
        rows = toks.shape[1]
        q, k, v = B.qk_norm_rope(B.from_vec(table[toks]), lens, rows, n_q, n_kv, hd, fr, qw, kw, parents=parents)
        if cache == "int8":
            B.kv8_write(store, k, v, lens, rows)
        else:
            for s in range(n_seq):
                w = n_kv * hd
                write(store, s, B.gather_rows(k, n_seq * rows, w, s * rows, rows), B.gather_rows(v, n_seq * rows, w, s * rows, rows),
                      int(lens[s]), rows)
        return attention(store, q, lens, rows, parents).to_vec().reshape(n_seq, rows, n_q * hd)

    spec, plain = new_store(), new_store()
    text = [list(rng.integers(0, V, n)) for n in lens]
    for store in (spec, plain):
        for s in range(n_seq):
            rows = int(lens[s])
            q, k, v = B.qk_norm_rope(B.from_vec(table[text[s]]), [0], rows, n_q, n_kv, hd, fr, qw, kw)
            write(store, s, k, v, 0, rows)
    root = rng.integers(0, V, n_seq)  # the token to feed next
    head = rng.normal(0, 0.5, (n_q * hd, V)).astype(F)
    kept = 0
    for step in range(3):
        rows = 11
        par = np.stack([tree(rng, rows, 4) for _ in range(n_seq)])
        par[:, 0], par[:, 1:] = -1, np.maximum(par[:, 1:], 0)  # node 0 is the token to feed
        toks = rng.integers(0, V, (n_seq, rows))
        toks[:, 0] = root
        o = feed(spec, toks, lens, par)
        # the target's rows; the drafted tokens are made likely, some are not
        lg = B.matmul(B.from_vec(o), B.from_vec(head), n_seq * rows, n_q * hd, V).to_vec().reshape(n_seq, rows, V)
        for s in range(n_seq):
            for i in range(1, rows):
                if rng.random() < 0.6:
                    lg[s, par[s, i], toks[s, i]] += 30.0
        p = B.softmax(B.from_vec(lg), n_seq * rows, V)
        u = rng.random((n_seq, rows))
        paths, n, token = B.verify_tree(p, toks[:, 1:], par[:, 1:] - 1, u, V)
        whole = np.concatenate((np.zeros((n_seq, 1), np.int64), np.where(paths >= 0, paths + 1, -1)), 1)
        if cache == "int8":
            B.kv8_keep(spec, lens, whole)
        else:
            for s in range(n_seq):
                for i, j in enumerate(whole[s, :n[s] + 1]):
                    for c in spec[s]:
                        B.scatter_rows(c, B.gather_rows(c, max_seq, n_kv * hd, int(lens[s] + j), 1), max_seq, n_kv * hd, int(lens[s] + i), 1)
        # the plain run feeds the accepted tokens one by one
        longest = int(n.max()) + 1
        for i in range(longest):
            t = np.array([[toks[s, whole[s, min(i, n[s])]]] for s in range(n_seq)])
            at = lens + np.minimum(i, n)
            o1 = feed(plain, t, at, None)
            for s in range(n_seq):
                node = whole[s, min(i, n[s])]
                # the same keys, in another order of the sums; values of v up to ~4
                assert np.abs(o1[s, 0] - o[s, node]).max() <= (4 * (lens[s] + 12) + 32 + 4 * (hd + 8) * 8) * U * 5
        kept += int(n.sum())
        lens = lens + n + 1
        root = token
        for s in range(n_seq):
            a = (B.kv8_read([spec[s]], [0], int(lens[s])), B.kv8_read([plain[s]], [0], int(lens[s]))) if cache == "int8" else \
                ([B.gather_rows(c, max_seq, n_kv * hd, 0, int(lens[s])) for c in spec[s]],
                 [B.gather_rows(c, max_seq, n_kv * hd, 0, int(lens[s])) for c in plain[s]])
            for x, y in zip(*a):
                assert np.array_equal(x.to_vec(), y.to_vec()), (step, s)
    assert kept > 0


VIEWS = """
import gc, sys
sys.path.insert(0, sys.argv[1])
import numpy as np, torch
import esolearn_amd as E
E.init(0)
B = E.HipBackend
x = np.arange(1 << 20, dtype=np.float32)
a = B.from_vec(x)
t = torch.from_dlpack(a)
assert t.shape == (1 << 20,) and t.dtype == torch.float32 and t.is_cuda
t.mul_(2)
torch.cuda.synchronize()
assert np.array_equal(a.to_vec(), x * 2)
s = torch.cuda.Stream()
with torch.cuda.stream(s):  # an op's output, read on another stream right after the call
    for i in range(20):
        b = B.scale(a, float(i))
        assert np.array_equal(torch.from_dlpack(b).cpu().numpy(), x * 2 * i)
ptr = t.data_ptr()
a.free()  # the tensor still holds the values
others = [B.zeros(1 << 20) for _ in range(4)]
assert np.array_equal(t.cpu().numpy(), x * 2)
assert others[0].__dlpack_device__() == (10, 0)
for bad in (dict(copy=True), dict(dl_device=(1, 0))):
    try:
        others[0].__dlpack__(**bad)
    except BufferError:
        pass
    else:
        raise AssertionError(bad)
c = others[0].__dlpack__(stream=-1)
held = torch.from_dlpack(others[0]).data_ptr()
del c, others
gc.collect()
del t
gc.collect()
blocks = [B.zeros(1 << 20) for _ in range(5)]  # both come back to the pool
assert {ptr, held} <= {torch.from_dlpack(b).data_ptr() for b in blocks}
print("views ok")
"""


def test_device_views(hip):
    """Storages as torch tensors without a copy, in a process that imports torch
    first (both then use one HIP runtime)."""
    import os
    import subprocess
    import sys

    pytest.importorskip("torch")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", VIEWS, root], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "views ok" in r.stdout, r.stdout + r.stderr


def test_calls_from_several_threads(hip):
    """Overlapping calls of host threads are serialised: each has its results."""
    import threading

    B = hip.HipBackend
    rng = np.random.default_rng(9)
    n_q, n_kv, hd, V = 4, 2, 64, 3000
    bad = []

    def work(seed):
        try:
            q, k, v, par = attention_case(n_q, n_kv, hd, [700], 9, "tree", seed)
            h = [B.from_vec(x) for x in (q, k[0], v[0])]
            c = B.kv8_new(709, n_kv, hd)
            p = softmax(np.random.default_rng(seed).normal(0, 2, (1, 10, V)))
            tok, u = p[0, 1:].argmax(-1)[None], np.random.default_rng(seed).random((1, 10))
            hp = B.from_vec(p)
            first = None
            for _ in range(20):
                B.kv8_write([c], h[1], h[2], [0], 709)
                got = [B.tree_attention(h[0], [h[1]], [h[2]], [700], 9, n_q, n_kv, hd, 0.1, parents=par).to_vec(),
                       B.kv8_tree_attention(h[0], [c], [700], 9, n_q, 0.1, parents=par).to_vec(),
                       *B.verify_tree(hp, tok, par, u, V)]
                if first is None:
                    first = got
                if not all(np.array_equal(a, b) for a, b in zip(first, got)):
                    bad.append(seed)
        except Exception as e:  # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in rng.integers(0, 1000, 4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
