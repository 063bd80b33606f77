"""gh_sample_rows on the MI355X against plain numpy in 64 bits (marked gpu).

A token is a whole number and has to be equal.  The kernel's weights are
rounded to 2^-44 (262144 logits) of the largest one, numpy's to 2^-53: a draw
could differ only where u times the kept mass falls between the two sums of a
rank, a share of u below 2^18 * 2^-44 / 1 = 2^-26 of all; the fixed seeds here
have none (each case computes its distance from the nearest border and asks
for 2^-30 before it compares)."""
from __future__ import annotations

import numpy as np
import pytest

import gemma_hip as gh

pytestmark = pytest.mark.gpu

F32 = np.float32


def plain(l, r):
    """(token, distance of the draw from the nearest border between two tokens
    as a share of the mass) of one row."""
    if np.isnan(l).any() or not (l > -np.inf).any():
        return -1, 1.0
    order = np.lexsort((np.arange(l.size), -l.astype(np.float64)))
    v = l[order].astype(np.float64)
    if r["temperature"] == 0:
        return int(order[0]), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(v == v[0], 1.0, np.exp((v - v[0]) / np.float64(r["temperature"])))
    k = int(r["top_k"]) or l.size
    below = w < np.float64(r["min_p"])
    w = np.where(np.arange(l.size) < k, w, 0.0)
    mass = np.cumsum(w)
    before = np.concatenate([[0.0], mass[:-1]])
    keep = (before < np.float64(r["top_p"]) * mass[-1]) & ~below
    keep[0] = True
    total = mass[keep].max()
    t = np.float64(r["u"]) * total
    at = int((mass <= t).sum())
    return int(order[at]), float(np.abs(mass - t).min() / total) if r["u"] else 1.0


def check(ctx, logits, rules, exact_sums=False):
    """exact_sums: every weight is 1 (or 0), so that both sides' sums are whole
    numbers without rounding and a draw on a border is decided the same."""
    logits = np.atleast_2d(np.asarray(logits, F32))
    got = gh.sample_rows(ctx, logits, logits.shape[1], rules)
    assert got.dtype == np.int32 and got.shape == (len(rules),)
    for i, r in enumerate(rules):
        want, far = plain(logits[i], r)
        assert exact_sums or far > 2.0 ** -30, (i, r)
        assert got[i] == want, (i, r, got[i], want, logits[i][[got[i], want]])
    return got


def logits(rng, rows, vocab, sigma=2.0, ties=False):
    l = rng.normal(size=(rows, vocab)) * sigma
    l += np.where(rng.random((rows, vocab)) < min(0.5, 40 / vocab), rng.exponential(4, size=(rows, vocab)), 0)
    return (np.round(l * 8) / 8 if ties else l).astype(F32)


def mixed(rng, rows, vocab):
    r = gh.sampling(rows, u=rng.random(rows).astype(F32))
    r["temperature"] = rng.choice([0.3, 0.8, 1.0, 1.7, 5.0], rows)
    r["top_k"] = np.where(rng.random(rows) < 0.5, 0, np.exp(rng.uniform(0, np.log(vocab * 1.1), rows)).astype(int))
    r["top_p"] = rng.choice([1.0, 0.99, 0.9, 0.5, 0.1], rows)
    r["min_p"] = rng.choice([0.0, 0.0, 1e-4, 0.03, 0.5, 1.0], rows)
    return r


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 1000, 1024, 4097, 32003, 40007])
def test_mixed_rules(ctx, vocab, ties):
    rng = np.random.default_rng(vocab + ties)
    check(ctx, logits(rng, 40, vocab, ties=ties), mixed(rng, 40, vocab))


@pytest.mark.parametrize("ties", [False, True])
def test_the_models_vocabulary(ctx, ties):
    rng = np.random.default_rng(7 + ties)
    check(ctx, logits(rng, 24, 262144, ties=ties), mixed(rng, 24, 262144))


def test_more_rows_than_a_launch_takes(ctx):
    rng = np.random.default_rng(9)
    check(ctx, logits(rng, 300, 777), mixed(rng, 300, 777))


def test_a_million_logits(ctx):
    rng = np.random.default_rng(10)
    check(ctx, logits(rng, 2, 1_000_003), gh.sampling(2, [0.9, 1.2], [0, 5000], [0.9, 1.0], 0.0, [0.4, 0.93]))


@pytest.mark.parametrize("vocab", [5, 3000, 262144])
def test_all_logits_equal(ctx, vocab):
    """Ranks are indexes: rank floor(u n) of what is kept."""
    l = np.full((4, vocab), 1.25, F32)
    k = max(1, vocab // 3)
    r = gh.sampling(4, 0.7, [0, k, 0, 0], [1, 1, 0.25, 1], [0, 0, 0, 1.0], F32(0.70703125))
    got = check(ctx, l, r, exact_sums=True)
    assert got[0] == int(0.70703125 * vocab) and got[1] == int(0.70703125 * k)


@pytest.mark.parametrize("rows", [1, 7, 130])
def test_greedy_rows(ctx, rows):
    """All rows at temperature 0, and all but one; ties go to the lowest index."""
    rng = np.random.default_rng(11)
    l = logits(rng, rows, 40007, ties=True)
    l[0, 5] = np.nan
    if rows > 2:
        l[1], l[2, 30000:] = -np.inf, l[2].max() + 1
    r = gh.sampling(rows, 0.0, rng.integers(0, 50, rows), 0.5, 0.1, 0.25)
    got = check(ctx, l, r)
    assert got[0] == -1 and (rows < 3 or (got[1] == -1 and got[2] == 30000))
    r["temperature"][rows - 1] = 0.8
    check(ctx, l, r)


def test_borders_that_are_exact(ctx):
    """Powers of two as weights (T = 1 / ln 2 would round; equal logits do
    not): a mass that is exactly top_p of the whole is enough, a running mass
    that is exactly u times the kept is not passed yet."""
    l = np.zeros((1, 4), F32)
    for top_p, u, want in [(0.5, 0.5, 1), (0.5, 0.0, 0), (0.5, 0.99, 1), (0.25, 0.99, 0), (0.75, 0.5, 1), (1.0, 0.5, 2),
                           (1.0, 0.25, 1), (0.0, 0.9, 0), (1.0, 0.75, 3)]:
        assert gh.sample_rows(ctx, l, 4, gh.sampling(1, 1.0, 0, top_p, 0.0, u))[0] == want, (top_p, u)


def test_masked_logits_and_infinities(ctx):
    rng = np.random.default_rng(13)
    l = logits(rng, 6, 5000)
    l[0, rng.random(5000) < 0.99] = -np.inf           # a grammar's mask
    l[1, :] = -np.inf
    l[1, 4321] = -50.0                                # one token left
    l[2, [17, 900]] = np.inf                          # all the mass, shared
    l[3, :] = -np.inf                                 # nothing left
    l[4, 77] = np.nan
    l[5, :] = np.finfo(F32).min                       # a mask of the type's lowest value
    l[5, [5, 6]] = np.finfo(F32).max
    for u in (0.0, 0.3, 0.9999):
        got = check(ctx, l, gh.sampling(6, 0.9, 0, 1.0, 0.0, u))
        assert got[1] == 4321 and got[2] == (17 if u < 0.5 else 900) and got[3] == -1 and got[4] == -1
        got = check(ctx, l, gh.sampling(6, 0.9, 40, 0.9, 0.01, u))
        assert got[3] == -1 and got[4] == -1
    got = check(ctx, l, gh.sampling(6, 0.0))
    assert got[2] == 17 and got[3] == -1 and got[4] == -1 and got[5] == 5


@pytest.mark.parametrize("t", [1e-45, 1e-6, 1e4, 3e38])
def test_extreme_temperatures(ctx, t):
    rng = np.random.default_rng(15)
    l = logits(rng, 3, 4000, ties=True)
    check(ctx, l, gh.sampling(3, t, [0, 50, 0], [1, 1, 0.5], 0.0, [0.2, 0.6, 0.9]))


@pytest.mark.parametrize("vocab", [9, 700, 40000])
def test_logits_as_far_apart_as_f32_reaches(ctx, vocab):
    """Distances that f32 does not hold, at a temperature that leaves them a
    weight (exp(-2) at 3e38), beside masked ones."""
    rng = np.random.default_rng(16)
    l = rng.uniform(-3.4e38, 3.4e38, (5, vocab)).astype(F32)
    l[:, [1, 4]] = -np.inf, np.finfo(F32).max
    l[:, 7] = np.finfo(F32).min
    r = gh.sampling(5, [3.4e38, 1e38, 3.4e38, 2e38, 3e37], [0, 0, 5, 0, 0], [1, 0.9, 1, 1, 1], [0, 0, 0, 0.1, 0], 0.0)
    for u in (0.1, 0.6, 0.97):
        r["u"] = u
        check(ctx, l, r)
    l[0, 3] = np.inf
    assert check(ctx, l[:1], r[:1])[0] == 3


@pytest.mark.parametrize("mask", [-1e9, -65504.0, np.finfo(F32).min])
def test_flat_logits_under_a_finite_mask(ctx, mask):
    rng = np.random.default_rng(18)
    l = logits(rng, 12, 262144, 0.3)
    l[rng.random(l.shape) < 0.5] = mask
    l[:4, :200000] = mask
    check(ctx, l, mixed(rng, 12, 262144))


def test_zero_and_minus_zero_are_equal(ctx):
    l = np.array([[-0.0, 0.0, -1.0, 0.0]], F32)
    assert [int(gh.sample_rows(ctx, l, 4, gh.sampling(1, 1.0, 3, 1.0, 0.0, u))[0]) for u in (0.0, 0.4, 0.7)] == [0, 1, 3]
    assert gh.sample_rows(ctx, l, 4, gh.sampling(1, 0.0))[0] == 0


def test_top_k_one_and_u_zero_are_the_argmax(ctx):
    rng = np.random.default_rng(16)
    l = logits(rng, 5, 9999, ties=True)
    want = l.argmax(1)
    assert np.array_equal(gh.sample_rows(ctx, l, 9999, gh.sampling(5, 2.0, 1, 1.0, 0.0, 0.99)), want)
    assert np.array_equal(gh.sample_rows(ctx, l, 9999, gh.sampling(5, 2.0, 0, 1.0, 0.0, 0.0)), want)
    assert [gh.argmax(ctx, x) for x in l] == want.tolist()


def test_draws_follow_the_probabilities(ctx):
    """2048 evenly spread u: every token gets its share of them, to one draw."""
    rng = np.random.default_rng(18)
    l = logits(rng, 1, 50)
    n = 2048
    u = ((np.arange(n) + 0.5) / n).astype(F32)
    got = gh.sample_rows(ctx, np.repeat(l, n, 0), 50, gh.sampling(n, 1.5, 0, 1.0, 0.0, u))
    p = np.exp((l[0].astype(np.float64) - l.max()) / 1.5)
    assert np.all(np.abs(np.bincount(got, minlength=50) / n - p / p.sum()) <= 1.01 / n)


def test_captured_rows_replay(ctx):
    rng = np.random.default_rng(19)
    l = logits(rng, 8, 50000)
    r = mixed(rng, 8, 50000)
    eager = check(ctx, l, r)
    lb, tb = gh.DeviceBuffer.from_numpy(ctx, l), gh.DeviceBuffer(ctx, 32)
    try:
        for _ in range(3):
            tb.upload(np.full(8, -7, np.int32))
            ctx.capture_begin()
            gh.sample_rows(ctx, lb, 50000, r, out=tb)
            ctx.capture_replay(3)
            assert np.array_equal(tb.numpy(np.int32), eager)
            assert np.array_equal(gh.sample_rows(ctx, l, 50000, r), eager)
    finally:
        lb.free()
        tb.free()


def test_a_decode_step_of_a_batch(ctx):
    """Append, attend, project to logits and sample, as a serving loop runs
    them: three steps of four sequences, each against plain numpy."""
    from test_gpu_kv8 import attend, quantise
    rng = np.random.default_rng(61)
    nq, nkv, hd, vocab, n = 4, 1, 64, 2000, 4
    w = (rng.normal(size=(vocab, nq * hd)) * 0.3).astype(F32)
    emb = rng.normal(size=(vocab, (nq + 2 * nkv) * hd)).astype(F32)
    c = gh.KVCache8(ctx, n, 200, nkv, hd)
    lens = [1, 64, 100, 63]
    hist = [[rng.normal(size=(m, nkv, hd)).astype(F32) for m in lens] for _ in range(2)]
    c.append(range(n), lens, np.concatenate(hist[0]), np.concatenate(hist[1]))
    tok = np.arange(n)
    for step in range(3):
        qkv = emb[tok]
        q, k, v = (x.reshape(n, -1, hd) for x in np.split(qkv, [nq * hd, (nq + nkv) * hd], axis=1))
        c.append(range(n), [1] * n, k, v)
        hist = [[np.concatenate([h, x[i:i + 1]]) for i, h in enumerate(hh)] for hh, x in zip(hist, (k, v))]
        out = c.attention(range(n), [1] * n, q, nq)
        for i in range(n):
            want, bound = attend(q[i:i + 1], quantise(hist[0][i])[2], quantise(hist[1][i])[2], 1, 0)
            assert np.all(np.abs(out[i:i + 1] - want) <= bound)
        l = (out.reshape(n, -1).astype(np.float64) @ w.T.astype(np.float64)).astype(F32)
        tok = check(ctx, l, gh.sampling(n, [0.0, 0.8, 1.0, 1.2], [0, 50, 0, 20], [1, 0.9, 0.95, 1], [0, 0.01, 0, 0],
                                        rng.random(n).astype(F32)))
