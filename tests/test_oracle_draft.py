"""The oracle's steps of decoding with drafted tokens against its own one-token steps and against the laws that they have to keep."""
from fractions import Fraction

import numpy as np
import pytest

import exact_oracle as O


def branch_mask(parent):
    mask = []
    for i, p in enumerate(parent):
        mask.append((mask[p] if p >= 0 else 0) | 1 << i)
    return mask


@pytest.mark.parametrize("base", [0, 5])
def test_every_branch_of_a_tree_is_the_causal_attention_of_its_tokens(base):
    H, KV, hd, Smax = 4, 2, 16, 24
    parent = [-1, 0, 0, 1, 1, 2, 5]
    depth = [0, 1, 1, 2, 2, 2, 3]
    rng = np.random.default_rng(base)
    T, N = len(parent), (H + 2 * KV) * hd
    t, s = rng.integers(-(1 << 42), 1 << 42, (T, N)), rng.integers(0, 8, T)
    b = rng.integers(-(1 << 16), 1 << 16, N)
    cos, sin = O.rope_tables(Smax, hd, 1e4)
    inv = O.inv_sqrt_hd(hd)
    new = lambda: (rng0.integers(-32767, 32768, (1, KV, Smax, hd)), rng0.integers(0, 4, (1, KV, Smax)),
                   rng0.integers(-(1 << 20), 1 << 20, (1, KV, Smax, hd)))
    rng0 = np.random.default_rng(9)
    cache = new()
    got = O.tree_attention(t, s, b, cos, sin, [0], [base], [depth], [branch_mask(parent)], [T], cache, H, KV, hd, inv, Smax)
    for leaf in (3, 4, 6):
        way = [leaf]
        while parent[way[0]] >= 0:
            way.insert(0, parent[way[0]])
        rng0 = np.random.default_rng(9)
        kq, sk, v = new()
        y = O.round_shift(t[way], 28 - s[way][:, None]) + b
        y = y.reshape(len(way), H + 2 * KV, hd)
        pos = slice(base, base + len(way))
        for kh in range(KV):
            k, ks = O.qrow(O.rope(y[:, H + kh], cos[pos], sin[pos]))
            kq[0, kh, pos], sk[0, kh, pos], v[0, kh, pos] = k, ks[:, 0], y[:, H + KV + kh]
        for h in range(H):
            q, sq = O.qrow(O.rope(y[:, h], cos[pos], sin[pos]))
            kh, S = h // (H // KV), base + len(way)
            valid = np.arange(S)[None] <= base + np.arange(len(way))[:, None]
            want = O.attention_head_q(q, sq, kq[0, kh, :S], sk[0, kh, :S, None], v[0, kh, :S], valid, inv)
            assert np.array_equal(got.reshape(T, H, hd)[way, h], want), (leaf, h)


def test_nodes_outside_are_seen_by_nobody():
    H, KV, hd, Smax = 2, 1, 16, 8
    rng = np.random.default_rng(1)
    t = rng.integers(-(1 << 40), 1 << 40, (3, (H + 2 * KV) * hd))
    cos, sin = O.rope_tables(Smax, hd, 1e4)
    zero = lambda: (np.zeros((1, KV, Smax, hd), np.int64), np.zeros((1, KV, Smax), np.int64), np.zeros((1, KV, Smax, hd), np.int64))
    run = lambda base, depth, mask, nodes, keys=Smax: O.tree_attention(
        t, [0] * 3, None, cos, sin, [0], [base], [depth], [mask], [nodes], cache, H, KV, hd, O.inv_sqrt_hd(hd), keys)
    cache = zero()
    full = run(0, [0, 1, 2], [1, 3, 7], 3)
    assert full.any(1).all()
    cache = zero()
    assert np.array_equal(run(0, [0, 1, 99], [1, 3, 7], 3)[:2], full[:2]) and not cache[2][0, 0, 2].any()
    cache = zero()
    assert not run(0, [0, 1, 2], [0, 0, 0], 3).any()          # rows that see nothing
    cache = zero()
    assert np.array_equal(run(0, [0, 1, 2], [1, 7, 7], 2)[:2], full[:2])   # a bit of a padding node
    for base, keys in ((-1, Smax), (Smax, Smax), (3, 3)):
        cache = zero()
        assert not run(base, [0, 1, 2], [1, 3, 7], 3, keys).any() and not cache[0].any()


@pytest.mark.parametrize("case", ["near", "equal", "far", "no draft mass"])
def test_verified_tokens_follow_the_targets_distribution(case):
    """P(x) = q(x) / Q accepted(x) + (1 - sum of those) w(x) / W is p(x) / P, but for the 2^-20 of u's steps"""
    V = 12
    rng = np.random.default_rng(len(case))
    lg = rng.integers(-(3 << 16), 3 << 16, (2, V))
    p = O.isoftmax_row(lg[0])
    q = {"near": O.isoftmax_row(lg[0] + rng.integers(-(1 << 15), 1 << 15, V)), "equal": p, "far": O.isoftmax_row(-lg[0]),
         "no draft mass": np.where(np.arange(V) < 3, 1000, 0)}[case]
    P, Q = int(p.sum()), int(q.sum())
    w = [max(int(a) * Q - int(c) * P, 0) for a, c in zip(p, q)]
    step, left, prob = 1 << 20, Fraction(1), []
    for x in range(V):
        if q[x] == 0:
            prob.append(Fraction(0))
            continue
        lo, hi = 0, step   # the number of u that accept x, by the oracle itself
        while lo < hi:
            mid = (lo + hi) // 2
            got, n = O.verify_draft(lg, [q], [x], [mid, 0], 1 << 16, 1)
            lo, hi = (mid + 1, hi) if n == 1 else (lo, mid)
        prob.append(Fraction(int(q[x]), Q) * Fraction(lo, step))
        left -= prob[-1]
    for x in range(V):
        total = prob[x] + (left * Fraction(w[x], sum(w)) if sum(w) else 0)
        assert abs(total - Fraction(int(p[x]), P)) <= Fraction(V, step)


def test_verify_follows_the_sampler_after_the_last_token():
    rng = np.random.default_rng(5)
    lg = rng.integers(-(4 << 16), 4 << 16, (1, 50))
    for seed in range(20):
        ids, n = O.verify_draft(lg, [], [], [O.u20(seed, 3)], 70000, 0)
        assert n == 0 and ids == [O.sample_int(lg[0], seed, 3, 70000)[0]]
    ids, n = O.verify_draft(np.concatenate([lg, lg]), [O.isoftmax_row(lg[0])], [50], [0, 7], 70000, 1)
    assert n == 0 and len(ids) == 1   # a token outside the vocabulary


def test_tree_accept_takes_the_lowest_matching_child():
    assert O.tree_accept([7, 8, 8, 9], [1, 7, 7, 8], [-1, 0, 0, 1], 4) == ([0, 1, 3], [7, 8, 9])
    assert O.tree_accept([7, 8, 8, 9], [1, 7, 7, 8], [-1, 0, 0, 2], 4) == ([0, 1], [7, 8])
    assert O.tree_accept([7, 8], [1, 7], [-1, 0], 1) == ([0], [7])
    assert O.tree_accept([7], [1], [-1], 0) == ([], [])


def test_judged_rows_are_the_samplers_and_their_sums_are_bounded():
    """the usual table: isoftmax_row's p; tables with negative entries: sums below 2^23 as they are, none from there on"""
    rng = np.random.default_rng(6)
    sc = rng.integers(-(6 << 16), 6 << 16, 300)
    assert O.judged_row(sc) == O.isoftmax_row(sc).tolist()
    T = np.full(10242, -(1 << 14))
    T[0] = 1 << 24   # the row's largest gives 2^24, every other one within 40 takes 2^14 off
    for near, P in ((0, 1 << 20), (512, 1 << 21), (895, (1 << 30) // 129), (896, 0), (1023, 0), (1024, 0), (1500, 0)):
        row = np.full(2000, -(50 << 16))
        row[7], row[100:100 + near] = 0, -(1 << 16)
        assert sum(O.judged_row(row, T)) == P
