"""Operators of decoding with drafted tokens, each in plain torch and as the engine's call.

A case is a dict of plain values; its "kind" names the operator:
  tree    one attention layer over a tree of drafted tokens: q|k|v epilogue, RoPE at the nodes' depths, cache write, attention
  verify  drafted tokens of a draft model judged against the target's logits, and the token that follows them
  accept  the walk of a drafted tree along the target's own tokens
  keep    the accepted branch's keys and values moved up in every layer's cache
  fork    a sequence's cached prompt copied to other sequences, every layer
Everything is integers: probabilities in Q20, logits and values in Q16, `rs` the shift that rounds half up.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
I16, I32, I64, F64 = torch.int16, torch.int32, torch.int64, torch.float64
ONE = 1 << 16


def _ops():
    path = os.path.join(os.getcwd(), "exact-llm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from exact_amd import ops
    return ops


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # one user of the 0.5B heads, a small tree after a short prompt: launches and latency
        dict(name="tree_small", kind="tree", H=14, KV=2, hd=64, B=1, T=8, n0=37, Smax=512),
        # one user of the 7B heads deep in a document, a wide tree
        dict(name="tree_7b", kind="tree", H=28, KV=4, hd=128, B=1, T=26, n0=1793, Smax=2048),
        # a batch of the 14B heads with long contexts and full trees of different sizes
        dict(name="tree_batch_long", kind="tree", H=40, KV=8, hd=128, B=4, T=64, n0=6001, Smax=8192),
        # one drafted token of a small vocabulary
        dict(name="verify_small", kind="verify", B=1, K=1, V=1000, temp=0.8),
        # one user, four drafted tokens over a full vocabulary
        dict(name="verify_one", kind="verify", B=1, K=4, V=151936, temp=0.8),
        # a serving batch with up to seven drafted tokens each
        dict(name="verify_batch", kind="verify", B=8, K=7, V=152064, temp=1.0),
        # one sequence's tree, and a large batch of full trees
        dict(name="accept_one", kind="accept", B=1, T=16),
        dict(name="accept_batch", kind="accept", B=64, T=64),
        # the accepted branch of one sequence in the 0.5B layers, and of a batch of full trees in the 14B layers
        dict(name="keep_one", kind="keep", L=24, KV=2, hd=64, B=1, T=16, n0=37, Smax=512),
        dict(name="keep_batch", kind="keep", L=48, KV=8, hd=128, B=8, T=64, n0=801, Smax=1024),
        # a short prompt to a second sequence in the 0.5B layers, a document to three others in the 7B layers
        dict(name="fork_short", kind="fork", L=24, KV=2, hd=64, M=1, n0=137, Smax=512),
        dict(name="fork_long", kind="fork", L=28, KV=4, hd=128, M=3, n0=1793, Smax=2048),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(14, 2, 64), (28, 4, 128), (40, 8, 128), (16, 16, 128)]


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "verify", "verify", "accept", "keep", "fork"])
    if kind == "tree":
        H, KV, hd = rng.choice(HEADS)
        n0 = _log_int(rng, 1, 6000)
        T = _log_int(rng, 1, 64)
        return dict(kind=kind, H=H, KV=KV, hd=hd, B=_log_int(rng, 1, 4), T=T, n0=n0, Smax=n0 + T + rng.randint(0, 300))
    if kind == "verify":
        return dict(kind=kind, B=_log_int(rng, 1, 8), K=_log_int(rng, 1, 7), V=_log_int(rng, 1000, 152064),
                    temp=round(rng.uniform(0.3, 1.5), 3))
    if kind == "accept":
        return dict(kind=kind, B=_log_int(rng, 1, 64), T=_log_int(rng, 1, 64))
    H, KV, hd = rng.choice(HEADS[:3])
    L = rng.randint(2, 28)
    if kind == "keep":
        n0, T = _log_int(rng, 1, 900), _log_int(rng, 1, 64)
        return dict(kind=kind, L=L, KV=KV, hd=hd, B=_log_int(rng, 1, 8), T=T, n0=n0, Smax=n0 + T + rng.randint(0, 60))
    n0 = _log_int(rng, 1, 1000)
    return dict(kind=kind, L=L, KV=KV, hd=hd, M=rng.randint(1, 3), n0=n0, Smax=n0 + rng.randint(0, 300))


# ----------------------------------------------------------------------------- integer steps in plain torch
def _rs(a, n):
    """(a + 2^(n-1)) >> n for n > 0, a << -n otherwise; n an int or a tensor"""
    n = torch.as_tensor(n, device=a.device, dtype=I64)
    r = n.clamp(min=0)
    half = torch.where(r > 0, torch.ones_like(r) << (r - 1).clamp(min=0), torch.zeros_like(r))
    return ((a + half) >> r) << (-n).clamp(min=0)


def _bitlen(m):
    """bit length of 0 <= m < 2^53"""
    return torch.where(m > 0, torch.frexp(m.double())[1].to(I64), torch.zeros_like(m))


def _qrow(x):
    """15-bit rows with a power-of-two scale: (x >> s rounded, s)"""
    s = (_bitlen(x.abs().amax(-1, keepdim=True)) - 15).clamp(min=0)
    return _rs(x, s).clamp(-32767, 32767), s


def _exp_table():
    return torch.tensor([round(math.exp(-i / 256) * (1 << 24)) for i in range(256 * 40 + 2)], dtype=I32, device=DEV)


def _lut_exp(T, d):
    """Q24 exp(-d) of Q16 d >= 0, interpolated; 0 from 40 on"""
    i = (d >> 8).clamp(max=T.numel() - 2)
    a, b = T[i].to(I64), T[i + 1].to(I64)
    return torch.where(d < (40 << 16), a - _rs((a - b) * (d & 255), 8), torch.zeros_like(d))


def _softmax_q20(sc, valid, T):
    """integer softmax over the last axis; rows that see nothing give zeros"""
    mx = torch.where(valid, sc, torch.full_like(sc, -(1 << 62))).amax(-1, keepdim=True)
    e = torch.where(valid, _lut_exp(T, torch.where(valid, mx - sc, torch.zeros_like(sc))), torch.zeros_like(sc))
    return torch.div(e << 20, e.sum(-1, keepdim=True).clamp(min=1), rounding_mode="floor")


# ----------------------------------------------------------------------------- prepare
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + salt)
    return g


def _q16(g, shape, std):
    return (torch.randn(shape, generator=g, device=DEV) * (std * ONE)).round().to(I64)


def _rope_tables(n, hd):
    inv = 1.0 / (1e6 ** (torch.arange(0, hd, 2, dtype=F64) / hd))
    ang = torch.outer(torch.arange(n, dtype=F64), inv)
    ang = torch.cat([ang, ang], -1)
    return (ang.cos() * ONE).round().to(I64).to(DEV), (ang.sin() * ONE).round().to(I64).to(DEV)


def _fit(n, T):
    """real nodes of each tree of a batch: full ones and smaller ones"""
    return [max(1, T - (T // 5) * (b % 3)) for b in range(n)]


def _trees(g, B, T):
    """(parent, depth, mask of the ancestors and the node itself) of B random trees, parents before children"""
    i = torch.arange(T, device=DEV)
    r = torch.rand((B, T), generator=g, device=DEV)
    lo = (i // 3).clamp(max=i - 1).clamp(min=0)   # wide trees: a parent is one of the nodes not far behind
    parent = (lo + r * (i - lo)).long().clamp(max=(i - 1).clamp(min=0))
    parent[:, 0] = -1
    depth, mask = torch.zeros((B, T), dtype=I64, device=DEV), torch.ones((B, T), dtype=I64, device=DEV)
    for j in range(1, T):
        p = parent[:, j:j + 1]
        depth[:, j] = depth.gather(1, p)[:, 0] + 1
        mask[:, j] = mask.gather(1, p)[:, 0] | (1 << j if j < 63 else -(1 << 63))
    return parent.to(I32), depth.to(I32), mask


def _cache(g, L, B, KV, Smax, hd):
    """keys as the engine stores them (15-bit rows and their shifts) and Q16 values, the layers' caches in one tensor each"""
    kq, sk = torch.empty((L, B, KV, Smax, hd), dtype=I16, device=DEV), torch.empty((L, B, KV, Smax), dtype=I32, device=DEV)
    v = torch.empty((L, B, KV, Smax, hd), dtype=I64, device=DEV)
    for i in range(L):
        for b in range(B):
            q, s = _qrow(_q16(g, (KV, Smax, hd), 2.0))
            kq[i, b], sk[i, b] = q.to(I16), s[..., 0].to(I32)
            v[i, b] = _q16(g, (KV, Smax, hd), 1.0)
    return kq, sk, v


def _i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def prepare(case, seed):
    k = case["kind"]
    st = dict(case)
    if k == "tree":
        H, KV, hd, B, T, Smax = (case[n] for n in ("H", "KV", "hd", "B", "T", "Smax"))
        g = _gen(seed, 1)
        nq, R = (H + 2 * KV) * hd, B * T
        std = torch.cat([torch.full((H * hd,), 1.0), torch.full((KV * hd,), 2.0), torch.full((KV * hd,), 1.0)]).to(DEV)
        s = torch.randint(6, 11, (R,), generator=g, device=DEV, dtype=I32)
        y = torch.randn((R, nq), generator=g, device=DEV).double() * std * ONE
        st.update(t=(y * torch.exp2(28.0 - s.double())[:, None]).round().to(I64), s=s, b=_q16(g, (nq,), 0.15))
        _, depth, mask = _trees(g, B, T)
        base = _i32([max(0, case["n0"] - (case["n0"] // 23) * b) for b in range(B)])
        cos, sin = _rope_tables(Smax, hd)
        st.update(depth=depth, mask=mask, base=base, nodes=_i32(_fit(B, T)), cos=cos, sin=sin, expt=_exp_table(),
                  slot=_i32([(b + 1) % B for b in range(B)]), cache=tuple(x[0] for x in _cache(g, 1, B, KV, Smax, hd)),
                  inv=int(round((1 << 16) / math.sqrt(hd))), out=torch.zeros((R, H * hd), dtype=I64, device=DEV),
                  obits=torch.zeros((R, H), dtype=I32, device=DEV))
        return st
    if k == "verify":
        B, K, V = case["B"], case["K"], case["V"]
        g = _gen(seed, 2)
        lg, tnum, T = _q16(g, (B, K + 1, V), 3.0), int(round((1 << 16) / case["temp"])), _exp_table()
        near = lg[:, :K] + _q16(g, (B, K, V), 0.6)   # the draft model's logits: near the target's
        q = _softmax_q20(_rs(near * tnum, 16), torch.ones((), dtype=torch.bool, device=DEV), T)
        c = q.cumsum(-1)
        at = (torch.rand((B, K, 1), generator=g, device=DEV).double() * c[..., -1:]).long()
        tok = torch.searchsorted(c, at, right=True).clamp(max=V - 1)[..., 0].to(I32)
        u = torch.randint(0, 1 << 20, (B, K + 1), generator=g, device=DEV, dtype=I32)
        return dict(st, lg=lg, q=q, tok=tok, u=u, tnum=tnum, expt=T, drafted=_i32([max(1, K - b % 3) for b in range(B)]),
                    ids=torch.zeros((B, K + 1), dtype=I32, device=DEV), n=torch.zeros(B, dtype=I32, device=DEV))
    if k == "accept":
        B, T = case["B"], case["T"]
        g = _gen(seed, 3)
        parent, _, _ = _trees(g, B, T)
        tok = torch.randint(0, 2, (B, T), generator=g, device=DEV, dtype=I32) + 1000   # some siblings have the same token
        nxt = torch.randint(0, 2, (B, T), generator=g, device=DEV, dtype=I32) + 1000
        return dict(st, parent=parent, tok=tok, nxt=nxt, nodes=_i32(_fit(B, T)), path=torch.zeros_like(tok),
                    ids=torch.zeros_like(tok), n=torch.zeros(B, dtype=I32, device=DEV))
    L, KV, hd, Smax = (case[n] for n in ("L", "KV", "hd", "Smax"))
    g = _gen(seed, 4)
    if k == "keep":
        B, T = case["B"], case["T"]
        # the accepted nodes lie behind the rows that they move to, so that a pass can be repeated on what it left
        path, n = torch.full((B, T), -1, dtype=I32), []
        r = torch.Generator().manual_seed(seed)
        for b in range(B):
            a = min(1 + int(torch.randint(0, 6, (1,), generator=r)), (T + 1) // 2)
            path[b, 0] = 0
            path[b, 1:a] = (torch.randperm(T - a, generator=r)[:a - 1].sort()[0] + a).to(I32)
            n.append(a)
        base = [max(0, case["n0"] - (case["n0"] // 23) * b) for b in range(B)]
        return dict(st, cache=_cache(g, L, B, KV, Smax, hd), path=path.to(DEV), n=_i32(n), base=_i32(base),
                    slot=_i32([(b + 1) % B for b in range(B)]))
    M = case["M"]
    return dict(st, cache=_cache(g, L, M + 1, KV, Smax, hd), src=_i32([0] * M), dst=_i32(list(range(1, M + 1))),
                n=_i32([max(1, case["n0"] - m) for m in range(M)]))


# ----------------------------------------------------------------------------- one pass
def run(st):
    k = st["kind"]
    if own:
        ops = _ops()
        if k == "tree":
            ops.attention_tree(st["t"], st["s"], st["b"], st["cos"], st["sin"], st["slot"], st["base"], st["depth"], st["mask"],
                               st["nodes"], st["cache"], st["expt"], st["out"], st["H"], st["KV"], st["hd"], st["inv"], st["obits"],
                               keys=st["n0"] + st["T"])
            return dict(out=st["out"], obits=st["obits"], cache=st["cache"])
        if k == "verify":
            ops.verify_draft(st["lg"], st["q"], st["tok"], st["u"], st["tnum"], st["expt"], st["ids"], st["n"], st["drafted"])
            return dict(ids=st["ids"], n=st["n"])
        if k == "accept":
            ops.tree_accept(st["nxt"], st["tok"], st["parent"], st["path"], st["ids"], st["n"], st["nodes"])
            return dict(path=st["path"], ids=st["ids"], n=st["n"])
        if k == "keep":
            ops.cache_keep(st["cache"], st["slot"], st["base"], st["path"], st["n"])
        else:
            ops.cache_fork(st["cache"], st["src"], st["dst"], st["n"])
        return dict(cache=st["cache"])
    return dict(tree=_tree, verify=_verify, accept=_accept, keep=_keep, fork=_fork)[k](st)


def _tree(st):
    H, KV, hd, B, T = (st[n] for n in ("H", "KV", "hd", "B", "T"))
    kq, sk, v = st["cache"]
    dev, G = kq.device, H // KV
    y = (_rs(st["t"], 28 - st["s"].to(I64)[:, None]) + st["b"]).view(B, T, H + 2 * KV, hd)
    base, slot = st["base"].to(I64), st["slot"].to(I64)
    node = torch.arange(T, device=dev)
    real = node < st["nodes"].to(I64)[:, None]
    at = base[:, None] + st["depth"].to(I64)
    cos, sin = st["cos"][at][:, :, None], st["sin"][at][:, :, None]
    qk = y[:, :, :H + KV]
    rot = torch.cat([-qk[..., hd // 2:], qk[..., :hd // 2]], -1)
    z, sz = _qrow(_rs(qk * cos + rot * sin, 16))
    bi, ni = real.nonzero(as_tuple=True)   # the real nodes' rows of the cache
    row = (slot[bi], slice(None), base[bi] + ni)
    kq[row], sk[row], v[row] = z[bi, ni, H:].to(I16), sz[bi, ni, H:, 0].to(I32), y[bi, ni, H + KV:]
    S = st["n0"] + T
    kk, ks, vv = kq[slot, :, :S].double(), sk[slot, :, :S].to(I64), v[slot, :, :S].double()
    q = z[:, :, :H].reshape(B, T, KV, G, hd).transpose(1, 2).reshape(B, KV, T * G, hd)
    sq = sz[:, :, :H].reshape(B, T, KV, G, 1).transpose(1, 2).reshape(B, KV, T * G, 1)
    key = torch.arange(S, device=dev) - base[:, None]
    seen = ((st["mask"][:, :, None] >> key.clamp(0, 63)[:, None]) & 1).bool() & (key < st["nodes"][:, None])[:, None] & (key >= 0)[:, None]
    valid = ((key < 0)[:, None] | seen) & real[:, :, None]
    valid = valid[:, None, :, None].expand(B, 1, T, G, S).reshape(B, 1, T * G, S)
    dot = torch.matmul(q.double(), kk.transpose(-1, -2).contiguous()).to(I64)   # below 2^37: exact
    p = _softmax_q20(_rs(dot * st["inv"], 32 - sq - ks[:, :, None]), valid, st["expt"])
    o = _rs(torch.matmul(p.double(), vv).to(I64), 20)   # the p of a row sum to at most 2^20, v below 2^32: exact
    o = o.view(B, KV, T, G, hd).transpose(1, 2).reshape(B * T, H, hd)
    return dict(out=o.view(B * T, H * hd), obits=_bitlen(o.abs().amax(-1)).to(I32), cache=st["cache"])


def _verify(st):
    B, K, V = st["B"], st["K"], st["V"]
    dev, q = st["lg"].device, st["q"]
    p = _softmax_q20(_rs(st["lg"] * st["tnum"], 16), torch.ones((), dtype=torch.bool, device=dev), st["expt"])
    P, Q = p.sum(-1), q.sum(-1)
    tok, u, d = st["tok"].to(I64), st["u"].to(I64), st["drafted"].to(I64)
    px, qx = p[:, :K].gather(2, tok[..., None])[..., 0], q.gather(2, tok[..., None])[..., 0]
    ok = (u[:, :K] * qx * P[:, :K] < (px * Q << 20)) & (torch.arange(K, device=dev) < d[:, None])
    n = ok.to(I64).cumprod(1).sum(1)
    b = torch.arange(B, device=dev)
    pa, a = p[b, n], n.clamp(max=K - 1)
    w = (pa * Q[b, a][:, None] - q[b, a] * P[b, n][:, None]).clamp(min=0)
    w = torch.where(((n < d) & (w.sum(1) > 0))[:, None], w, pa)
    c = w.cumsum(1)
    last = (c <= ((u[:, K] * c[:, -1]) >> 20)[:, None]).sum(1)
    i = torch.arange(K + 1, device=dev)
    drafts = torch.cat([tok, tok[:, :1]], 1)
    ids = torch.where(i < n[:, None], drafts, torch.where(i == n[:, None], last[:, None], -torch.ones_like(drafts)))
    return dict(ids=ids.to(I32), n=n.to(I32))


def _accept(st):
    parent, tok, nxt = st["parent"].to(I64), st["tok"], st["nxt"]
    B, T = tok.shape
    i = torch.arange(T, device=tok.device)
    real = i < st["nodes"].to(I64)[:, None]
    ok = (nxt.gather(1, parent.clamp(min=0)) == tok) & (parent >= 0) & real
    # of siblings with the same token the first: no lower node with the same parent that matches
    same = (parent[:, :, None] == parent[:, None, :]) & ok[:, None, :] & (i[None, None, :] < i[None, :, None])
    ok = ok & ~same.any(-1)
    ok[:, 0] = real[:, 0]
    up, on = torch.where(parent < 0, torch.zeros_like(parent), parent), ok
    for _ in range(max(1, (T - 1).bit_length())):   # on the path: every ancestor matches too (pointer doubling)
        on = on & on.gather(1, up)
        up = up.gather(1, up)
    n = on.sum(1)
    order = torch.where(on, i, T).sort(1)[0]   # parents have lower numbers than their children
    inside = order < T
    path = torch.where(inside, order, -torch.ones_like(order))
    ids = torch.where(inside, nxt.gather(1, path.clamp(min=0)).to(I64), -torch.ones_like(order))
    return dict(path=path.to(I32), ids=ids.to(I32), n=n.to(I32))


def _keep(st):
    path, n, base, slot = (st[x].to(I64) for x in ("path", "n", "base", "slot"))
    bi, d = (torch.arange(st["T"], device=path.device) < n[:, None]).nonzero(as_tuple=True)
    to, fr, sl = base[bi] + d, base[bi] + path[bi, d], slot[bi]
    for x in st["cache"]:
        x[:, sl, :, to] = x[:, sl, :, fr]
    return dict(cache=st["cache"])


def _fork(st):
    src, dst, n = (st[x].to(I64) for x in ("src", "dst", "n"))
    m, i = (torch.arange(st["n0"], device=n.device) < n[:, None]).nonzero(as_tuple=True)
    for x in st["cache"]:
        x[:, dst[m], :, i] = x[:, src[m], :, i]
    return dict(cache=st["cache"])


# ----------------------------------------------------------------------------- work
def work(case):
    k = case["kind"]
    row = case.get("KV", 0) * (case.get("hd", 0) * 10 + 4)   # bytes of a position of a layer's cache
    if k == "tree":
        H, KV, hd, B, T = (case[n] for n in ("H", "KV", "hd", "B", "T"))
        nodes = _fit(B, T)
        base = [max(0, case["n0"] - (case["n0"] // 23) * b) for b in range(B)]
        keys = sum(base) + sum(nodes)
        return dict(bytes=sum(base) * row + sum(nodes) * (row + (H + 2 * KV) * hd * 8) + B * T * H * (hd * 8 + 4),
                    flops=sum(4 * n * (s + (n + 1) // 2) * H * hd for n, s in zip(nodes, base)) + keys)
    if k == "verify":
        B, K, V = case["B"], case["K"], case["V"]
        rows = sum(max(1, K - b % 3) for b in range(B))
        return dict(bytes=8 * V * (2 * rows + B), flops=20 * V * (2 * rows + B))
    if k == "accept":
        return dict(bytes=case["B"] * (case["T"] * 20 + 8), flops=case["B"] * case["T"])
    if k == "keep":
        return dict(bytes=2 * case["L"] * case["B"] * row * min(3, (case["T"] + 1) // 2), flops=1)
    return dict(bytes=2 * case["L"] * row * sum(max(1, case["n0"] - m) for m in range(case["M"])), flops=1)


# ----------------------------------------------------------------------------- the definitions, step by step
def _round_shift(a, n):
    """half up, on int64 tensors and one shift"""
    return a << -n if n <= 0 else (a + (1 << (n - 1))) >> n


def _row_bits(x):
    return int(x.abs().max()).bit_length()


def _exp_of(T, d):
    far = d >= 40 * ONE
    i = torch.where(far, torch.zeros_like(d), d // 256)
    e = T[i] - torch.div((T[i] - T[i + 1]) * (d - 256 * i) + 128, 256, rounding_mode="floor")
    return e.masked_fill(far, 0)


def _probs(sc, T):
    """softmax of one or more rows in which every entry counts"""
    e = _exp_of(T, sc.amax(-1, keepdim=True) - sc)
    return (e * (1 << 20)) // e.sum(-1, keepdim=True)


def exact(case, seed):
    """run()'s answer from the operators' definitions, one sequence (and KV head) after the other, in 64 bits"""
    st, k = prepare(case, seed), case["kind"]
    if k in ("keep", "fork"):
        new = tuple(x.clone() for x in st["cache"])
        if k == "keep":
            moves = [(s, s, b + p, b + d) for s, b, ps, n in zip(*(st[x].tolist() for x in ("slot", "base", "path", "n")))
                     for d, p in enumerate(ps[:n])]
            for a, b, fr, to in moves:
                for x, y in zip(st["cache"], new):
                    y[:, b, :, to] = x[:, a, :, fr]
        else:
            for a, b, n in zip(*(st[x].tolist() for x in ("src", "dst", "n"))):
                for x, y in zip(st["cache"], new):
                    y[:, b, :, :n] = x[:, a, :, :n]
        return dict(cache=new)
    if k == "accept":
        B, T = case["B"], case["T"]
        path, ids, ns = [], [], []
        for par, tok, nxt, nodes in zip(*(st[x].tolist() for x in ("parent", "tok", "nxt", "nodes"))):
            way = [0] if nodes else []
            while way:
                child = [j for j in range(1, nodes) if par[j] == way[-1] and tok[j] == nxt[way[-1]]]
                if not child:
                    break
                way.append(child[0])
            ns.append(len(way))
            path.append(way + [-1] * (T - len(way)))
            ids.append([nxt[j] for j in way] + [-1] * (T - len(way)))
        return dict(path=_i32(path), ids=_i32(ids), n=_i32(ns))
    if k == "verify":
        T, ids, ns = st["expt"].to(I64), [], []
        for b in range(case["B"]):
            K = case["K"]
            u, tok, d = st["u"][b].tolist(), st["tok"][b].tolist(), int(st["drafted"][b])
            got = []
            for i in range(d + 1):
                p = _probs(_round_shift(st["lg"][b, i] * st["tnum"], 16), T)
                P, w = int(p.sum()), p
                if i < d:
                    q = st["q"][b, i]
                    Q, x = int(q.sum()), tok[i]
                    if u[i] * int(q[x]) * P < int(p[x]) * Q << 20:
                        got.append(x)
                        continue
                    rest = (p * Q - q * P).clamp(min=0)
                    w = rest if int(rest.sum()) > 0 else p
                c = w.cumsum(0)
                got.append(int((c <= (u[K] * int(c[-1])) >> 20).sum()))
                break
            ns.append(len(got) - 1)
            ids.append(got + [-1] * (K + 1 - len(got)))
        return dict(ids=_i32(ids), n=_i32(ns))
    H, KV, hd, B, T = (case[n] for n in ("H", "KV", "hd", "B", "T"))
    tab, (kq, sk, v) = st["expt"].to(I64), (x.clone() for x in st["cache"])
    out, obits = torch.zeros((B * T, H, hd), dtype=I64, device=DEV), torch.zeros((B * T, H), dtype=I64, device=DEV)

    def turn(x, pos):   # RoPE of the heads x (rows, heads, hd) and their 15-bit rows
        h = hd // 2
        c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]
        lo, hi = x[..., :h], x[..., h:]
        z = _round_shift(torch.cat([lo * c[..., :h] - hi * s[..., :h], hi * c[..., h:] + lo * s[..., h:]], -1), 16)
        bits = torch.zeros(z.shape[:2], dtype=I64, device=DEV)
        top = z.abs().amax(-1)
        for j in range(15, 62):
            bits += top >= (1 << j)
        half = torch.where(bits > 0, (1 << bits) // 2, torch.zeros_like(bits))
        return torch.div(z + half[..., None], (1 << bits)[..., None], rounding_mode="floor").clamp(-32767, 32767), bits

    for b in range(B):
        n, p0, sl = int(st["nodes"][b]), int(st["base"][b]), int(st["slot"][b])
        t, s = st["t"][b * T:b * T + n], st["s"][b * T:b * T + n].tolist()
        y = torch.stack([_round_shift(row, 28 - e) for row, e in zip(t, s)]) + st["b"]
        y = y.view(n, H + 2 * KV, hd)
        z, bits = turn(y[:, :H + KV], p0 + st["depth"][b, :n].to(I64))
        kq[sl, :, p0:p0 + n] = z[:, H:].transpose(0, 1).to(I16)
        sk[sl, :, p0:p0 + n] = bits[:, H:].t().to(I32)
        v[sl, :, p0:p0 + n] = y[:, H + KV:].transpose(0, 1)
        S, words = p0 + n, st["mask"][b, :n].tolist()
        hidden = torch.zeros((n, S), dtype=torch.bool, device=DEV)
        hidden[:, p0:] = torch.tensor([[not (m >> j) & 1 for j in range(n)] for m in words], device=DEV)
        for h in range(H):
            kh = h // (H // KV)
            key, ks, val = kq[sl, kh, :S].to(I64), sk[sl, kh, :S].to(I64), v[sl, kh, :S]
            qd = z[:, h].double()
            dot = (qd @ (key >> 8).double().t().contiguous()).to(I64) * 256 + (qd @ (key & 255).double().t().contiguous()).to(I64)
            sh = 32 - bits[:, h:h + 1] - ks
            sc = torch.div(dot * st["inv"] + ((1 << sh) // 2), 1 << sh, rounding_mode="floor")
            sc = torch.where(hidden, torch.full_like(sc, -(1 << 50)), sc)
            p = _probs(sc, tab).masked_fill(hidden, 0).double()
            o = (p @ (val >> 16).double()).to(I64) * ONE + (p @ (val & 65535).double()).to(I64)
            o = _round_shift(o, 20)
            out[b * T:b * T + n, h] = o
            top = o.abs().amax(-1)
            for j in range(62):
                obits[b * T:b * T + n, h] += top >= (1 << j)
    return dict(out=out.view(B * T, H * hd), obits=obits.to(I32), cache=(kq, sk, v))
