"""The 8-bit KV cache (gh_kv8_*) on the MI355X against plain numpy in 64 bits
(marked gpu).

Tolerances.  What the cache stores is compared exactly: the scale is a / 127
rounded once to f32, the code is x / scale rounded half to even, and the value
read back is code * scale rounded once, so every number has one right value.

Attention works on those exact values.  With e = 2^-24, per score it rounds q
to e times the row's largest magnitude (23 bits and sign), drops from the
exact integer product at most 2^-15 of q's largest times one code of K (4 e
max|q| max|k|, 127 codes being max|k|), and scales it by three f32 products:
  ds <= e ((sum |k| + 4 max|k|) max|q| / sqrt(hd) + 4 |s|).
A probability moves by a factor 1 + 2 ds (it and the sum) and is rounded to e
times the largest of the 64 or 256 tokens that are worked on together, which
is one of the sum's terms: 256 e of the sum at most.  Exponentials, the running
sum over up to 33 blocks and the scales are a further 44 e:
  max|V| (2 ds + 300 e), which `attend` computes from the case's own scores."""
from __future__ import annotations

import threading

import numpy as np
import pytest

import gemma_hip as gh

pytestmark = pytest.mark.gpu

B = gh.KV8_BLOCK
F32 = np.float32


def quantise(x):
    """(codes, scales [blocks, nkv], values f32) of x [n, nkv, hd], blocks from row 0."""
    n, nkv, hd = x.shape
    nb = -(-n // B)
    codes = np.zeros((n, nkv, hd), np.int64)
    scales = np.zeros((nb, nkv), F32)
    vals = np.zeros(x.shape, F32)
    with np.errstate(invalid="ignore"):
        for b in range(nb):
            for h in range(nkv):
                blk = x[b * B:(b + 1) * B, h]
                s = F32(np.nan) if not np.all(np.isfinite(blk)) else max(F32(np.abs(blk).max() / F32(127)), F32(2.0 ** -100))
                scales[b, h] = s
                c = np.zeros(blk.shape) if np.isnan(s) else np.rint(blk.astype(np.float64) / np.float64(s))
                codes[b * B:(b + 1) * B, h] = c
                vals[b * B:(b + 1) * B, h] = c.astype(F32) * s
    return codes, scales, vals


def attend(q, k, v, n_q, window, top=None):
    """(out, bound) in 64 bits; q [n_q, nq, hd], k, v [L, nkv, hd] as stored.
    top [L, nkv]: what stands for a token's largest |v| in the bound."""
    L, nkv, hd = k.shape
    nq = q.shape[1]
    out = np.zeros((n_q, nq, hd))
    bound = np.zeros((n_q, nq, 1))
    k, v, q64 = k.astype(np.float64), v.astype(np.float64), q.astype(np.float64)
    for t in range(n_q):
        pos = L - n_q + t
        lo = max(0, pos - window + 1) if window else 0
        if pos < 0:
            continue
        for h in range(nq):
            kk, vv = k[lo:pos + 1, h // (nq // nkv)], v[lo:pos + 1, h // (nq // nkv)]
            s = kk @ q64[t, h] / np.sqrt(hd)
            p = np.exp(s - s.max())
            out[t, h] = p @ vv / p.sum()
            eps = 2.0 ** -24
            ds = eps * ((np.abs(kk).sum(1).max() + 4 * np.abs(kk).max()) * np.abs(q64[t, h]).max() / np.sqrt(hd) + 4 * np.abs(s).max())
            largest = np.abs(vv).max() if top is None else top[lo:pos + 1, h // (nq // nkv)].max()
            bound[t, h] = largest * (2 * ds + 300 * eps)
    return out, bound


def rows(rng, n, nkv, hd, sigma=1.0):
    x = rng.normal(size=(n, nkv, hd)) * sigma
    x *= np.exp(rng.normal(size=(1, nkv, hd)) * 0.5)  # channels of different size
    return x.astype(F32)


def same_bits(a, b):
    a, b = np.asarray(a, F32), np.asarray(b, F32)
    nan = np.isnan(b)
    return a.shape == b.shape and np.array_equal(np.isnan(a), nan) and np.array_equal(a[~nan], b[~nan])


SHAPES = [(1, 256), (4, 256), (2, 128), (3, 64), (1, 32), (5, 32)]  # kv heads, head_dim


@pytest.mark.parametrize("nkv,hd", SHAPES)
@pytest.mark.parametrize("n", [1, 15, 63, 64, 65, 200])
def test_append_stores_the_quantised_rows(ctx, nkv, hd, n):
    rng = np.random.default_rng(n * 1000 + hd + nkv)
    k, v = rows(rng, n, nkv, hd), rows(rng, n, nkv, hd, 0.3)
    c = gh.KVCache8(ctx, 1, 256, nkv, hd)
    c.append([0], [n], k, v)
    assert c.cacheLength(0) == n
    gk, gv = c.read([0], [0], [n])
    assert same_bits(gk, quantise(k)[2]) and same_bits(gv, quantise(v)[2])


@pytest.mark.parametrize("nkv,hd", [(1, 256), (2, 128), (3, 64), (2, 32)])
@pytest.mark.parametrize("cuts", [[1] * 70, [63, 1, 1], [64, 64], [30, 100, 3], [1, 63, 65, 7], [100, 28, 200], [5, 59, 64, 1],
                                  [40, 152, 1]])
def test_a_cache_does_not_depend_on_how_its_tokens_were_cut(ctx, nkv, hd, cuts):
    """Rows of growing size raise the scale again and again; every prefix is
    what one append of it would have stored."""
    rng = np.random.default_rng(len(cuts) + hd)
    n = sum(cuts)
    grow = np.exp(np.linspace(0, 3, n))[:, None, None]
    k, v = (rows(rng, n, nkv, hd) * grow).astype(F32), (rows(rng, n, nkv, hd) * grow[::-1]).astype(F32)
    c = gh.KVCache8(ctx, 2, n, nkv, hd)  # the second sequence is left alone
    at = 0
    for m in cuts:
        c.append([0], [m], k[at:at + m], v[at:at + m])
        at += m
        if len(cuts) < 9 or at % 9 == 0:
            gk, gv = c.read([0], [0], [at])
            assert same_bits(gk, quantise(k[:at])[2]) and same_bits(gv, quantise(v[:at])[2]), at
    assert c.cacheLength(1) == 0


def test_rounding_is_half_to_even_and_exact_between_codes(ctx):
    """Values at and one ulp beside every middle between two codes, with scales
    whose quotients round the wrong way in f32."""
    hd, nkv = 256, 1
    rng = np.random.default_rng(5)
    for s in [F32(1.0), F32(0.37), F32(1.0000001), F32(3.1e-5), F32(2.0 ** -100), F32(7e30)] + list(
            np.exp(rng.uniform(-20, 20, 6)).astype(F32)):
        top = F32(127) * s
        s_eff = max(F32(top / F32(127)), F32(2.0 ** -100))
        mid = (np.arange(-127, 127) + 0.5) * np.float64(s_eff)
        x = np.concatenate([mid.astype(F32), np.nextafter(mid.astype(F32), F32(np.inf)),
                            np.nextafter(mid.astype(F32), F32(-np.inf)), [top]]).astype(F32)
        x = np.resize(x, 64 * hd).reshape(64, 1, hd).copy()
        x[0, 0, 0] = top
        x = np.clip(x, -top, top)
        c = gh.KVCache8(ctx, 1, 64, nkv, hd)
        c.append([0], [64], x, x)
        gk, gv = c.read([0], [0], [64])
        want = quantise(x)[2]
        assert same_bits(gk, want) and same_bits(gv, want), s


@pytest.mark.parametrize("fill", [0.0, 1e-45, 3e-39, 1e-30, 3.0e38])
def test_small_and_large_values(ctx, fill):
    x = np.full((70, 2, 64), fill, F32)
    x[3, 1] = -x[3, 1]
    c = gh.KVCache8(ctx, 1, 70, 2, 64)
    c.append([0], [70], x, 0.5 * x)
    gk, gv = c.read([0], [0], [70])
    assert same_bits(gk, quantise(x)[2]) and same_bits(gv, quantise((0.5 * x).astype(F32))[2])


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_value_that_is_not_finite_makes_its_block_nan_and_goes_with_its_token(ctx, bad):
    rng = np.random.default_rng(11)
    k, v = rows(rng, 150, 2, 128), rows(rng, 150, 2, 128)
    kb = k.copy()
    kb[70, 1, 5] = bad  # second block, head 1
    for cuts in ([150], [66, 4, 1, 79]):
        c = gh.KVCache8(ctx, 1, 150, 2, 128)
        at = 0
        for m in cuts:
            c.append([0], [m], kb[at:at + m], v[at:at + m])
            at += m
        gk, gv = c.read([0], [0], [150])
        assert np.isnan(gk[64:128, 1]).all() and same_bits(gk, quantise(kb)[2]) and same_bits(gv, quantise(v)[2])
    c = gh.KVCache8(ctx, 1, 150, 2, 128)
    c.append([0], [71], kb[:71], v[:71])
    c.truncate([0], [70])
    c.append([0], [80], k[70:], v[70:])
    gk, _ = c.read([0], [0], [150])
    assert same_bits(gk, quantise(k)[2])


@pytest.mark.parametrize("n,back,more", [(100, 80, 30), (100, 65, 1), (127, 66, 62), (64, 63, 1), (3, 1, 5), (128, 70, 10),
                                         (130, 127, 66)])
def test_truncate_within_the_last_block_leaves_no_trace(ctx, n, back, more):
    """128 and 130 tokens: the block's f32 rows are gone, the block's values
    take their place (next test); the others are as if never appended."""
    rng = np.random.default_rng(n + back)
    nkv, hd = 2, 64
    k, v = rows(rng, n, nkv, hd), rows(rng, n, nkv, hd)
    k[back:] *= 7  # the removed tokens hold the block's largest values
    k2, v2 = rows(rng, more, nkv, hd), rows(rng, more, nkv, hd)
    c = gh.KVCache8(ctx, 3, 256, nkv, hd)
    c.append([2], [n], k, v)
    c.truncate([2], [back])
    assert c.cacheLength(2) == back
    same = n // B == back // B
    first = back // B * B
    base = []
    for x in (k, v):
        y = x[:back].copy()
        if not same:
            y[first:] = quantise(x)[2][first:back]
        base.append(y)
    got = c.read([2], [0], [back])
    for y, x, g in zip(base, (k, v), got):
        want = quantise(y)[2] if same else np.concatenate([quantise(x)[2][:back]])
        assert same_bits(g, want)
    c.append([2], [more], k2, v2)
    got = c.read([2], [0], [back + more])
    for y, x, new, g in zip(base, (k, v), (k2, v2), got):
        whole = np.concatenate([y, new])
        want = quantise(whole)[2]
        if not same:  # that block's scale never shrinks below the one it was stored with
            codes, scales, _ = quantise(x)
            for h in range(nkv):
                blk = whole[first:first + B, h]
                s = max(scales[first // B, h], F32(np.abs(blk[back - first:]).max() / F32(127)))
                want[first:first + B, h] = np.rint(blk.astype(np.float64) / np.float64(s)).astype(F32) * s
        assert same_bits(g, want)


def test_truncate_to_a_block_boundary_and_to_nothing(ctx):
    rng = np.random.default_rng(3)
    k, v = rows(rng, 200, 1, 256), rows(rng, 200, 1, 256)
    c = gh.KVCache8(ctx, 1, 200, 1, 256)
    c.append([0], [200], k, v)
    c.truncate([0], [128])
    c.append([0], [5], k[:5], v[:5])
    gk, gv = c.read([0], [0], [133])
    assert same_bits(gk, np.concatenate([quantise(k)[2][:128], quantise(k[:5])[2]]))
    c.truncate([0], [0])
    assert c.cacheLength(0) == 0
    c.append([0], [1], k[9:10], v[9:10])
    gk, gv = c.read([0], [0], [1])
    assert same_bits(gk, quantise(k[9:10])[2]) and same_bits(gv, quantise(v[9:10])[2])


def test_batches_touch_their_sequences_alone_in_any_order(ctx):
    """300 sequences (two launches of a call), appended in a shuffled order
    with different counts, zero among them; read back in another order."""
    rng = np.random.default_rng(17)
    n, nkv, hd = 300, 1, 32
    c = gh.KVCache8(ctx, n, 130, nkv, hd)
    held = [[np.zeros((0, nkv, hd), F32)] * 2 for _ in range(n)]
    for _ in range(3):
        seqs = rng.permutation(n)[:280]
        counts = rng.integers(0, 44, size=280)
        k, v = rows(rng, int(counts.sum()), nkv, hd), rows(rng, int(counts.sum()), nkv, hd)
        c.append(seqs, counts, k, v)
        at = 0
        for s, m in zip(seqs, counts):
            held[s] = [np.concatenate([held[s][0], k[at:at + m]]), np.concatenate([held[s][1], v[at:at + m]])]
            at += m
    seqs = rng.permutation(n)
    lens = np.array([len(held[s][0]) for s in seqs])
    assert [c.cacheLength(int(s)) for s in seqs] == lens.tolist()
    begins = np.minimum(rng.integers(0, 70, size=n), lens)
    gk, gv = c.read(seqs, begins, lens)
    want = [np.concatenate([quantise(held[s][i])[2][b:] for s, b in zip(seqs, begins)]) for i in (0, 1)]
    assert same_bits(gk, want[0]) and same_bits(gv, want[1])


def _fill(c, rng, lens, sigma=1.0):
    ks = [rows(rng, n, c.n_kv_heads, c.head_dim, sigma) for n in lens]
    vs = [rows(rng, n, c.n_kv_heads, c.head_dim) for n in lens]
    c.append(np.arange(len(lens)), lens, np.concatenate(ks), np.concatenate(vs))
    return [quantise(x)[2] for x in ks], [quantise(x)[2] for x in vs]


def _check(got, ks, vs, q, counts, window, seqs=None):
    at = 0
    for i, t in enumerate(counts):
        s = i if seqs is None else seqs[i]
        want, bound = attend(q[at:at + t], ks[s], vs[s], t, window)
        g = got[at:at + t]
        assert np.all(np.isfinite(g))
        err = np.abs(g - want)
        assert np.all(err <= bound + 1e-30), (i, float((err / (bound + 1e-30)).max()))
        at += t


HEADS = [(4, 1, 256), (8, 4, 256), (8, 8, 128), (16, 2, 128), (6, 2, 64), (3, 3, 64), (20, 1, 64), (4, 1, 32), (12, 4, 32)]


@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("n", [1, 2, 17, 63, 64, 65, 130, 517])
def test_attention_of_single_tokens(ctx, nq, nkv, hd, n):
    rng = np.random.default_rng(n + 7 * nq + hd)
    c = gh.KVCache8(ctx, 1, n, nkv, hd)
    ks, vs = _fill(c, rng, [n])
    q = rows(rng, 1, nq, hd, 1.5)
    for window in (0, 1, 50, 512):
        _check(c.attention([0], [1], q, nq, window), ks, vs, q, [1], window)


@pytest.mark.parametrize("nq,nkv,hd", [(4, 1, 256), (8, 4, 256), (16, 2, 128), (6, 2, 64), (4, 1, 32)])
@pytest.mark.parametrize("n,t", [(5, 5), (64, 3), (70, 70), (129, 33), (200, 130), (300, 7)])
def test_attention_of_several_tokens_is_causal(ctx, nq, nkv, hd, n, t):
    rng = np.random.default_rng(n + t + nq + hd)
    c = gh.KVCache8(ctx, 1, n, nkv, hd)
    ks, vs = _fill(c, rng, [n])
    q = rows(rng, t, nq, hd, 1.5)
    for window in (0, 40, 65):
        _check(c.attention([0], [t], q, nq, window), ks, vs, q, [t], window)


@pytest.mark.parametrize("nq,nkv,hd", [(4, 1, 256), (16, 2, 128), (4, 1, 32)])
@pytest.mark.parametrize("up", [True, False])
def test_values_that_a_row_does_not_see_cost_it_no_precision(ctx, nq, nkv, hd, up):
    """V a thousand times as large, or as small, every 64 tokens (from the
    start, or from the end and so inside a block).  A probability is rounded to
    2^-24 of the largest, in units of the largest scale among the blocks that
    the row sees; times a code of at most 127 that is 2^-24 of the largest
    value of a block that it sees, be that one itself in sight or not: the
    bound goes by it, and by no block that the row does not see."""
    rng = np.random.default_rng(hd + up)
    n, t = 300, 300
    size = 1e3 ** (np.arange(n) // B - 2.0)
    k, v = rows(rng, n, nkv, hd), (rows(rng, n, nkv, hd) * (size if up else size[::-1])[:, None, None]).astype(F32)
    c = gh.KVCache8(ctx, 1, n, nkv, hd)
    c.append([0], [n], k, v)
    q = rows(rng, t, nq, hd)
    top = np.concatenate([np.broadcast_to(np.abs(v[b:b + B]).max((0, 2)), (len(v[b:b + B]), nkv)) for b in range(0, n, B)])
    for window in (0, 30):
        want, bound = attend(q, quantise(k)[2], quantise(v)[2], t, window, top)
        err = np.abs(c.attention([0], [t], q, nq, window) - want)
        assert np.all(err <= bound), float((err / bound).max())


def test_attention_of_a_ragged_batch_in_any_order_the_same_sequence_twice(ctx):
    rng = np.random.default_rng(23)
    lens = [1, 700, 64, 0, 129, 2100, 33]
    c = gh.KVCache8(ctx, len(lens), 2100, 2, 128)
    ks, vs = _fill(c, rng, lens)
    seqs, counts = [5, 1, 6, 3, 5, 0, 2, 4], [1, 4, 33, 0, 9, 1, 1, 0]
    q = rows(rng, sum(counts), 4, 128)
    for window in (0, 300):
        got = c.attention(seqs, counts, q, 4, window)
        _check(got, ks, vs, q, counts, window, seqs)


def test_queries_in_front_of_the_cache_see_nothing_and_give_zeros(ctx):
    """More queries than tokens: the first stand at negative positions."""
    rng = np.random.default_rng(29)
    c = gh.KVCache8(ctx, 2, 64, 1, 64)
    ks, vs = _fill(c, rng, [3])
    q = rows(rng, 21 + 2, 4, 64)
    for window in (0, 2, 2 ** 31 - 1):  # the last: further back than 32 bits count
        got = c.attention([0, 1], [21, 2], q, 4, window)
        assert np.array_equal(got[:18], np.zeros_like(got[:18])) and np.array_equal(got[21:], np.zeros_like(got[21:]))
        _check(got[18:21], ks, vs, q[18:21], [3], window)


def test_a_prompt_and_drafts_among_single_tokens(ctx):
    """One call of sizes far apart, which goes in several launches: 150
    sequences take one token each, one a prompt of 1200, a few take drafts."""
    rng = np.random.default_rng(30)
    n, nkv, nq, hd = 156, 4, 8, 32
    new = np.ones(n, int)
    new[[3, 50]], new[[7, 70, 101, 155]], new[20] = (1200, 90), (5, 2, 9, 17), 0
    old = rng.integers(1, 700, n)
    old[[3, 20, 60]] = 0, 5, 1500
    c = gh.KVCache8(ctx, n, 1600, nkv, hd)
    order = rng.permutation(n)
    held = [[rows(rng, a + b, nkv, hd) for a, b in zip(old, new)] for _ in (0, 1)]
    for lo, hi in ((np.zeros(n, int), old), (old, old + new)):
        c.append(order, (hi - lo)[order], *[np.concatenate([x[s][lo[s]:hi[s]] for s in order]) for x in held])
    stored = [[quantise(x)[2] for x in h] for h in held]
    begins = np.maximum(old + new - 40, 0)
    begins[3] = 0
    got = c.read(order, begins[order], (old + new)[order])
    for g, x in zip(got, stored):
        assert same_bits(g, np.concatenate([x[s][begins[s]:] for s in order]))
    q = rows(rng, int(new.sum()), nq, hd)
    for window in (0, 100):
        _check(c.attention(order, new[order], q, nq, window), *stored, q, new[order], window, order)


@pytest.mark.parametrize("t", [1, 3])
def test_a_long_sequence_among_short_ones(ctx, t):
    rng = np.random.default_rng(32 + t)
    lens = rng.integers(0, 100, 180)
    lens[77], lens[5] = 20000, 3000
    c = gh.KVCache8(ctx, 180, 20000, 2, 32)
    ks, vs = _fill(c, rng, lens)
    q = rows(rng, 180 * t, 4, 32)
    for window in (0, 4000):
        _check(c.attention(np.arange(180), [t] * 180, q, 4, window), ks, vs, q, [t] * 180, window)


def test_tokens_that_were_truncated_away_are_not_seen(ctx):
    """Stale codes behind a sequence's end, and a block whose scale is NaN
    behind it, take no part."""
    rng = np.random.default_rng(31)
    nkv, hd = 2, 256
    k, v = rows(rng, 200, nkv, hd), rows(rng, 200, nkv, hd)
    kb, vb = k.copy(), v.copy()
    kb[150], vb[190] = np.nan, np.inf
    c = gh.KVCache8(ctx, 1, 256, nkv, hd)
    c.append([0], [200], kb, vb)
    c.truncate([0], [100])
    q = rows(rng, 1, 4, hd)
    got = c.attention([0], [1], q, 4)
    _check(got, [quantise(k)[2][:100]], [quantise(v)[2][:100]], q, [1], 0)


def test_a_nan_block_reaches_the_queries_that_see_it_and_no_others(ctx):
    rng = np.random.default_rng(37)
    k, v = rows(rng, 300, 1, 64), rows(rng, 300, 1, 64)
    vb, kb = v.copy(), k.copy()
    vb[70, 0, 3] = np.nan  # tokens 64..127
    q = rows(rng, 300, 2, 64)
    c = gh.KVCache8(ctx, 2, 300, 1, 64)
    kb[70, 0, 3] = np.inf
    c.append([0, 1], [300, 300], np.concatenate([k, kb]), np.concatenate([vb, v]))
    for window in (0, 40):
        got = c.attention([0, 1], [300, 300], np.concatenate([q, q]), 2, window).reshape(2, 300, 2, 64)
        pos = np.arange(300)
        lo = np.maximum(0, pos - window + 1) if window else np.zeros(300, int)
        sees = (pos >= 64) & (lo < 128)
        for s in (0, 1):
            assert np.isnan(got[s][sees]).all()
            want, bound = attend(q, quantise(k)[2], quantise(v)[2], 300, window)
            err = np.abs(got[s] - want)[~sees]
            assert np.all(err <= (bound + np.zeros_like(want))[~sees])


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_query_that_is_not_finite_spoils_its_own_row_alone(ctx, bad):
    rng = np.random.default_rng(41)
    c = gh.KVCache8(ctx, 1, 100, 1, 128)
    ks, vs = _fill(c, rng, [100])
    q = rows(rng, 5, 4, 128)
    qb = q.copy()
    qb[2, 1, 77] = bad
    got, want = c.attention([0], [5], qb, 4), c.attention([0], [5], q, 4)
    assert np.isnan(got[2, 1]).all()
    got[2, 1] = want[2, 1]
    assert np.array_equal(got, want)


def test_sharp_and_flat_scores(ctx):
    """One score far above the rest, and all equal (the mean of V)."""
    rng = np.random.default_rng(43)
    c = gh.KVCache8(ctx, 1, 2000, 1, 256)
    ks, vs = _fill(c, rng, [2000], 3.0)
    q = np.concatenate([rows(rng, 1, 4, 256, 8.0), np.zeros((1, 4, 256), F32)])
    _check(c.attention([0], [2], q, 4), ks, vs, q, [2], 0)


@pytest.mark.parametrize("nq,hd", [(4, 256), (3, 128), (4, 64), (2, 32), (8, 256)])
def test_every_digit_of_millions_of_probabilities(ctx, nq, hd):
    """A probability's digits are taken by different lanes, which have to agree
    on it to the last bit: where they do not, one in some hundred thousand
    probabilities is off by 1/128 of its block's largest.  V is 1 at dim
    token % hd and 0 elsewhere, so that the output is sums of few
    probabilities and shows one.

    Bound for output d: a score's error changes every term by a factor of
    2 ds; rounding p to its digits costs half a 2^-23rd of the block's
    largest (of the four blocks' that more than 4 heads work on together: of
    the seven around it at most) for each of the 64 / hd + 1 tokens of a block,
    and of the sums' roundings each costs 2^-24 of them, 40 in a row at most."""
    rng = np.random.default_rng(67 + nq + hd)
    L, n = 20000, 64
    k, q = rows(rng, L, 1, hd, 1.2), rows(rng, n, nq, hd, 1.5)
    v = np.zeros((L, 1, hd), F32)
    v[np.arange(L), 0, np.arange(L) % hd] = 1
    c = gh.KVCache8(ctx, 1, L, 1, hd)
    c.append([0], [L], k, v)
    got = c.attention([0] * n, [1] * n, q, nq).reshape(n * nq, hd)
    kk, qq = quantise(k)[2][:, 0].astype(np.float64), q.reshape(n * nq, hd).astype(np.float64)
    s = qq @ kk.T / np.sqrt(hd)
    p = np.exp(s - s.max(1, keepdims=True))
    l = p.sum(1, keepdims=True)
    pad = -L % (64 * hd)
    pp = np.concatenate([p, np.zeros((n * nq, pad))], 1)
    want = pp.reshape(n * nq, -1, hd).sum(1) / l
    eps = 2.0 ** -24
    ds = eps * ((np.abs(kk).sum(1).max() + 4 * np.abs(kk).max()) * np.abs(qq).max(1, keepdims=True) / np.sqrt(hd) + 4 * np.abs(s).max(1, keepdims=True))
    largest = pp.reshape(n * nq, -1, 64).max(2)
    if nq > 4:
        padded = np.pad(largest, ((0, 0), (3, 3)))
        largest = np.max([padded[:, i:i + largest.shape[1]] for i in range(7)], axis=0)
    largest = largest.sum(1, keepdims=True)
    bound = want * (2 * ds + 40 * eps) + (64 // hd + 1) * eps * largest / l
    err = np.abs(got - want)
    assert np.all(err <= bound), (float((err / bound).max()), int((err > bound).sum()))


def test_results_do_not_change_from_call_to_call(ctx):
    rng = np.random.default_rng(47)
    lens = [900, 4000, 77]
    c = gh.KVCache8(ctx, 3, 4000, 4, 256)
    _fill(c, rng, lens)
    q = rows(rng, 3, 8, 256)
    first = c.attention([0, 1, 2], [1, 1, 1], q, 8)
    for _ in range(3):
        assert np.array_equal(first, c.attention([0, 1, 2], [1, 1, 1], q, 8))


def test_offsets_beyond_four_gigabytes(ctx):
    """The last of 40 sequences of 131072 tokens: its codes lie 5 GB in."""
    rng = np.random.default_rng(53)
    c = gh.KVCache8(ctx, 40, 131072, 1, 512 // 2)
    n = 300
    k, v = rows(rng, n, 1, 256), rows(rng, n, 1, 256)
    c.append([39], [n], k, v)
    gk, gv = c.read([39], [0], [n])
    ks, vs = quantise(k)[2], quantise(v)[2]
    assert same_bits(gk, ks) and same_bits(gv, vs)
    q = rows(rng, 1, 4, 256)
    _check(c.attention([39], [1], q, 4), [ks], [vs], q, [1], 0)
    c.close()


def test_captured_attention_and_reads_replay(ctx):
    """Launch-only calls under capture, replayed with eager work between."""
    rng = np.random.default_rng(59)
    c = gh.KVCache8(ctx, 2, 1500, 1, 256)
    ks, vs = _fill(c, rng, [1500, 40])
    q = rows(rng, 2, 4, 256)
    qb, ob = gh.DeviceBuffer.from_numpy(ctx, q), gh.DeviceBuffer(ctx, q.nbytes)
    kb = gh.DeviceBuffer(ctx, 4 * 40 * 256)
    eager = c.attention([0, 1], [1, 1], q, 4)
    try:
        for _ in range(3):
            ob.upload(np.full(q.shape, 7, F32))
            ctx.capture_begin()
            c.attention([0, 1], [1, 1], qb, 4, out=ob)
            c.read([1], [0], [40], k_out=kb)
            with pytest.raises(gh.GemmaHipError) as e:
                c.truncate([0], [10])
            assert e.value.name == "GH_ERR_STATE"
            with pytest.raises(gh.GemmaHipError) as e:
                c.append([1], [1], kb, kb)
            assert e.value.name == "GH_ERR_STATE"
            ctx.capture_replay(4)
            assert np.array_equal(ob.numpy().reshape(q.shape), eager)
            assert same_bits(kb.numpy().reshape(40, 1, 256), ks[1])
            assert np.array_equal(c.attention([0, 1], [1, 1], q, 4), eager)
        assert c.cacheLength(0) == 1500 and c.cacheLength(1) == 40
    finally:
        for b in (qb, ob, kb):
            b.free()


def test_a_captured_call_of_several_launches_replays(ctx):
    """Chunks that are joined, a prompt and single tokens in one captured call:
    its launches share the context's scratch one after the other."""
    rng = np.random.default_rng(61)
    lens = [3000, 600, 40, 2000] + [30] * 60
    counts = [1, 600, 7, 4] + [1] * 60
    c = gh.KVCache8(ctx, len(lens), 3000, 2, 64)
    ks, vs = _fill(c, rng, lens)
    q = rows(rng, sum(counts), 4, 64)
    seqs = np.arange(len(lens))
    eager = c.attention(seqs, counts, q, 4)
    _check(eager, ks, vs, q, counts, 0)
    qb, ob = gh.DeviceBuffer.from_numpy(ctx, q), gh.DeviceBuffer(ctx, q.nbytes)
    try:
        for _ in range(2):
            ob.upload(np.full(q.shape, 7, F32))
            ctx.capture_begin()
            c.attention(seqs, counts, qb, 4, out=ob)
            ctx.capture_replay(3)
            assert np.array_equal(ob.numpy().reshape(q.shape), eager)
            assert np.array_equal(c.attention(seqs, counts, q, 4), eager)
    finally:
        qb.free()
        ob.free()


def test_threads_share_a_context(ctx):
    """Calls of several threads, on one cache and on caches of their own, give
    what they give alone."""
    rng = np.random.default_rng(67)
    lens = [2500, 90, 700]
    c = gh.KVCache8(ctx, 3, 2500, 2, 128)
    _fill(c, rng, lens)
    jobs = [([0, 1], [1, 1]), ([2], [300]), ([1, 2, 0], [3, 1, 5]), ([0], [40])]
    qs = [rows(rng, sum(n), 8, 128) for _, n in jobs]
    logits = rng.normal(size=(4, 50000)).astype(F32)
    rules = gh.sampling(4, 0.9, [0, 40, 0, 3], 0.9, 0.0, rng.random(4).astype(F32))
    alone = [c.attention(s, n, q, 8) for (s, n), q in zip(jobs, qs)]
    tokens = gh.sample_rows(ctx, logits, 50000, rules)
    wrong = []

    def work(i):
        own = gh.KVCache8(ctx, 1, 200, 1, 32)
        x = rows(np.random.default_rng(i), 130, 1, 32)
        for turn in range(10):
            if not np.array_equal(c.attention(*jobs[i], qs[i], 8), alone[i]):
                wrong.append((i, turn, "attention"))
            if not np.array_equal(gh.sample_rows(ctx, logits, 50000, rules), tokens):
                wrong.append((i, turn, "tokens"))
            own.append([0], [13], x[13 * turn:13 * turn + 13], x[13 * turn:13 * turn + 13])
        if not same_bits(own.read([0], [0], [130])[0], quantise(x)[2]):
            wrong.append((i, "read"))
        own.close()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
