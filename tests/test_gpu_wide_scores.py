"""Scores and logits that leave int64, in every kernel that takes the exp LUT of a distance: two of them can lie 2^63 apart or more, where
the signed difference is negative. The distance is the unsigned one, checked here in Python integers; shifts and products wrap as numpy's."""
import numpy as np
import pytest
import torch

import exact_oracle as O
from exact_amd import ops
from exact_amd.tables import exp_t, host_tables
from test_gpu_draft import Tree, chain_reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
I8, I16, I32, I64 = torch.int8, torch.int16, torch.int32, torch.int64
EXP = [int(x) for x in exp_t()]


def dev(a, dt):
    return torch.tensor(np.ascontiguousarray(a), dtype=dt, device=DEV)


def probabilities(row):
    """Q20 probabilities of a row of Python integers"""
    mx, e = max(row), []
    for x in row:
        i, fr = (mx - x) >> 8, (mx - x) & 255
        e.append(EXP[i] - ((EXP[i] - EXP[i + 1]) * fr + 128 >> 8) if mx - x < 40 << 16 else 0)
    return [(a << 20) // sum(e) for a in e]


def far_apart(rows):
    return any(max(r) - min(r) >= 1 << 63 for r in rows)


def head(q, sq, k, sk, v, pos, inv):
    """attention of one head's rows, and whether some row's scores lie 2^63 apart"""
    out, rows = [], []
    for i, p in enumerate(pos):
        sc = O.round_shift((q[i] @ k[:p + 1].T) * inv, 32 - sq[i] - sk[:p + 1])
        rows.append([int(x) for x in sc])
        pr = np.array(probabilities(rows[-1]), np.int64)
        out.append(O.round_shift(pr @ v[:p + 1], 20))
    return np.stack(out), far_apart(rows)


def case(seed, H, KV, hd, S, R):
    """shifts of 60 and 61 together: scores are shifted left by 28 and 29"""
    rng = np.random.default_rng(seed)
    return (rng.integers(-32767, 32768, (R, H, hd)), rng.integers(30, 32, (R, H)), rng.integers(-32767, 32768, (KV, S, hd)),
            np.full((KV, S), 30), rng.integers(-(1 << 30), 1 << 30, (KV, S, hd)), np.arange(S - R, S))


@pytest.mark.parametrize("H,KV,hd", [(4, 2, 64), (3, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("path", ["blocks", "waves", "prefill"])
def test_attention_rows(H, KV, hd, path):
    if hd == 256 and path != "blocks":
        return
    R, S = 5, 31 if path == "waves" else 61
    q, sq, k, sk, v, pos = case(hd + H, H, KV, hd, S, R)
    inv = O.inv_sqrt_hd(hd)
    heads = [head(q[:, h], sq[:, h], k[h // (H // KV)], sk[h // (H // KV)], v[h // (H // KV)], pos, inv) for h in range(H)]
    want = np.stack([out for out, _ in heads], 1)
    assert all(far for _, far in heads)
    print(f"attention {path} H={H} KV={KV} hd={hd}", flush=True)
    cache = (dev(k, I16)[None], dev(sk, I32)[None], dev(v, I64)[None])
    qd, sd, pd, expt = dev(q, I16), dev(sq, I32), dev(pos, I32), dev(exp_t(), I32)
    out, ob = torch.empty((R, H * hd), dtype=I64, device=DEV), torch.empty((R, H), dtype=I32, device=DEV)
    if path == "prefill":
        ops.attention_prefill(qd, sd, cache, 0, pd, S, expt, out, H, KV, hd, inv, ops.prefill_workspace(R, H, KV, hd, S, DEV), ob)
    else:
        ops.attention(qd, sd, cache, torch.zeros(R, dtype=I32, device=DEV), pd, expt, out, H, KV, hd, inv, ob,
                      nkeys=S if path == "waves" else None)   # 32 keys: a wave a (row, head)
    assert np.array_equal(out.cpu().numpy().reshape(R, H, hd), want)
    assert np.array_equal(ob.cpu().numpy(), O.bitlen(np.abs(want).max(-1)))


@pytest.mark.parametrize("H,KV,hd,Smax,R", [(7, 1, 128, 300, 3), (14, 2, 64, 300, 2), (8, 1, 128, 1000, 2), (8, 1, 128, 1000, 4), (40, 8, 128, 200, 8),
                                            (4, 4, 256, 96, 2), (16, 16, 128, 500, 1)])
def test_decode_rows_match_two_launches(H, KV, hd, Smax, R):
    """totals of 61 bits against cached keys with shifts of 30: the fused launch, and the launches split over the keys"""
    rng = np.random.default_rng(H + Smax)
    N = (H + 2 * KV) * hd
    cache = (rng.integers(-32767, 32768, (R, KV, Smax, hd)), np.full((R, KV, Smax), 30), rng.integers(-(1 << 29), 1 << 29, (R, KV, Smax, hd)))
    t, s = dev(rng.integers(-(1 << 61), 1 << 61, (R, N)), I64), dev(rng.integers(0, 12, R), I32)
    slot, pos = dev(np.arange(R), I32), dev([Smax - 1 - 7 * r for r in range(R)], I32)
    tabs = host_tables(Smax, hd, 1e6)
    cos, sin, expt, inv = dev(tabs["cos"], I64), dev(tabs["sin"], I64), dev(exp_t(), I32), O.inv_sqrt_hd(hd)
    new = lambda: tuple(dev(x, dt) for x, dt in zip(cache, (I16, I32, I64)))
    qq, sq = torch.empty((R, H * hd), dtype=I16, device=DEV), torch.empty((R, H), dtype=I32, device=DEV)
    want, ob, a = torch.empty((R, H * hd), dtype=I64, device=DEV), torch.empty((R, H), dtype=I32, device=DEV), new()
    ops.qkv_rope_cache(t, s, None, cos, sin, slot, pos, a, qq, sq, H, KV, hd)
    print(f"decode H={H} KV={KV} hd={hd} Smax={Smax} R={R}", flush=True)
    ops.attention(qq, sq, a, slot, pos, expt, want, H, KV, hd, inv, ob)
    host = [x.cpu().numpy().astype(np.int64) for x in (qq.view(R, H, hd), sq, *a)]
    for r in range(R):
        got, _ = head(host[0][r:r + 1, 0], host[1][r:r + 1, 0], host[2][r, 0], host[3][r, 0], host[4][r, 0], [int(pos[r])], inv)
        assert np.array_equal(want.cpu().numpy()[r, :hd], got[0])
    keys = [1] + [Smax] * (ops.attention_keys_from(R, H, KV, hd, Smax) <= Smax)
    for k in keys:
        for obn in (1, 4):
            b, out = new(), torch.empty_like(want)
            ops.attention_qkv(t, s, None, cos, sin, slot, pos, b, expt, out, H, KV, hd, inv, None, obn=obn, keys=k)
            assert torch.equal(out, want), (k, obn)
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("Smax,H", [(250, 6), (500, 36), (700, 6), (1100, 6)])
def test_trees(hd, Smax, H):
    """totals of 61 bits, cached keys with shifts of 30: the trees' launches against the rows'"""
    x = Tree(H, 2, hd, Smax, 10, [Smax - 11, 3, Smax // 2], 8, masks="chain", smag=61)
    x.cache[1][:] = 30
    d = x.device()
    want = chain_reference(x, d)
    x.call(d)
    for a, b in zip((d["out"], d["obits"], *d["cache"]), (want[0], want[1], *want[2])):
        assert torch.equal(a, b)


def test_softmax_rows():
    rng = np.random.default_rng(1)
    x = rng.integers(-(1 << 63), (1 << 63) - 1, (6, 300), endpoint=True)
    x[0, :5] = [(1 << 63) - 1, (1 << 63) - 70000, -(1 << 63), -1, 0]
    x[1] = -(1 << 63) + np.arange(300) * 3000
    rows = [[int(a) for a in r] for r in x]
    assert far_apart(rows)
    p = ops.isoftmax(dev(x, I64), dev(exp_t(), I32)).cpu().numpy()
    assert [[int(a) for a in r] for r in p] == [probabilities(r) for r in rows]


@pytest.mark.parametrize("NE", [60, 130])
def test_routers(NE):
    """logits of whole int64 words; the experts of highest probability, ties to the lower one"""
    rng = np.random.default_rng(NE)
    R, k = 4, 4
    t = rng.integers(-(1 << 63), (1 << 63) - 1, (R, NE), endpoint=True)
    t[1, 7:9] = [(1 << 63) - 1, (1 << 63) - 40000]
    rows = [[int(a) for a in r] for r in t]
    assert far_apart(rows)
    p_sel, e_sel = torch.empty((R, k), dtype=I64, device=DEV), torch.empty((R, k), dtype=I32, device=DEV)
    ops.router_topk(dev(t, I64), dev(np.full(R, 28), I32), dev(exp_t(), I32), k, p_sel, e_sel)
    for r, row in enumerate(rows):
        p = probabilities(row)
        best = sorted(range(NE), key=lambda i: (-p[i], i))[:k]
        assert e_sel[r].tolist() == best and p_sel[r].tolist() == [p[i] for i in best]


@pytest.mark.parametrize("V", [1000, 20000])
def test_sampled_logits_of_wrapped_products(V):
    """logits whose product with the temperature leaves int64"""
    rng = np.random.default_rng(V)
    lg = rng.integers(-(1 << 63), (1 << 63) - 1, (3, V), endpoint=True)
    lg[1] >>= 40   # ... and a row that does not
    ids = torch.empty(3, dtype=I32, device=DEV)
    ops.sample(dev(lg, I64), 7, dev([0, 1, 2], I32), 81920, dev(exp_t(), I32), ids)
    for r in range(3):
        p = probabilities([int(x) for x in O.round_shift(lg[r] * 81920, 16)])
        target, c, j = O.u20(7, r) * sum(p) >> 20, 0, 0
        for a in p:
            c += a
            j += c <= target
        assert int(ids[r]) == j
