"""The model's paths over drafted tokens: trees, a draft model, forked sequences. Drafts change how many tokens a pass gives, never
which, so receipts, tokens, logits and cache rows are compared with decoding one token at a time."""
import os
import random

import numpy as np
import pytest
import torch

import exact_oracle as O
import helpers
from exact_amd import ops, synth
from exact_amd.model import Cache, DeviceWeights, TModel, TreeDecoder, generate, lookup_draft, speculate, verify

pytestmark = pytest.mark.gpu
DEV = "cuda"


def model(name, Smax=96, batch=1, abits=15, seed=3):
    return TModel(DeviceWeights.synthetic(synth.CONFIGS[name], seed, DEV), Smax=Smax, batch=batch, abits=abits)


def guesses(true, seed, good):
    """a drafter that knows the tokens to come: trees in random order of one branch of true tokens (wrong after a while, with
    probability 1 - good a token) among branches of wrong ones"""
    rng = random.Random(seed)

    def draft(seen):
        ahead = true[len(seen):]
        toks, parents, last = [], [], -1
        for t in ahead[:6]:
            for _ in range(rng.randrange(3)):   # siblings before it, wrong ones and their children
                toks.append(rng.randrange(100))
                parents.append(rng.choice([last, len(toks) - 2]) if len(toks) > 1 else -1)
            toks.append(t if rng.random() < good else (t + 1) % 100)
            parents.append(last)
            last = len(toks) - 1
        return toks, parents

    return draft


@pytest.mark.parametrize("name,abits", [("tiny", 15), ("tiny-hd128", 15), ("tiny-moe", 15), ("tiny-tied", 15), ("tiny", 7)])
def test_drafted_generation_gives_the_same_receipt(name, abits):
    tm = model(name, abits=abits)
    prompt = helpers.prompt(7, 9, tm.cfg.V)
    want, greedy = generate(tm, prompt, 24, 5, 0.8)
    for nodes, good in ((1, 1.0), (16, 1.0), (24, 0.7), (5, 0.3), (64, 1.0)):
        got, g = generate(tm, prompt, 24, 5, 0.8, draft=guesses(prompt + want["tokens"], nodes, good), nodes=nodes)
        assert got == want and g == greedy, (nodes, good)
    got, _ = generate(tm, prompt, 24, 5, 0.8, draft=lookup_draft)
    assert got == want and verify(tm, got) == (True, None)
    one, _ = generate(tm, prompt, 1, 5, 0.8, draft=lookup_draft)
    assert one["tokens"] == want["tokens"][:1]


def test_drafted_generation_equals_the_oracle():
    cfg = synth.CONFIGS["tiny"]
    tm, om = model("tiny"), helpers.oracle_model(cfg, 3, T=96)
    prompt = helpers.prompt(8, 6, cfg.V)
    rec, greedy, _ = O.generate(om, prompt, 12, seed=9, temp=1.3)
    got, g = generate(tm, prompt, 12, 9, 1.3, draft=guesses(prompt + rec["tokens"], 1, 0.8))
    assert got == rec and g == greedy


def test_a_full_cache_is_filled_to_the_last_position():
    tm = model("tiny", Smax=32)
    prompt = helpers.prompt(3, 12, tm.cfg.V)
    want, _ = generate(tm, prompt, 21, 1, 1.0)   # the last token needs no position
    got, _ = generate(tm, prompt, 21, 1, 1.0, draft=guesses(prompt + want["tokens"], 2, 1.0), nodes=32)
    assert got == want
    with pytest.raises(ops.ExactError):
        generate(tm, prompt, 22, 1, 1.0, draft=lookup_draft)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("name,B", [("tiny", 3), ("tiny-hd128", 2), ("tiny-moe", 2)])
def test_batched_greedy_trees_equal_decoding_row_by_row(graph, name, B):
    tm = model(name, batch=B)
    ref, cache = tm.new_cache(), tm.new_cache()
    prompts = [helpers.prompt(b, 5 + 4 * b, tm.cfg.V) for b in range(B)]
    first = []
    for b, p in enumerate(prompts):
        first.append(int(tm.forward(p, ref, last_only=True, slot=b)[0].argmax()))
        tm.forward(p, cache, last_only=True, slot=b)
    true, logits, cur = [[t] for t in first], [], list(first)
    for _ in range(20):
        lg, ids = tm.decode_rows(cur, ref)
        logits.append(lg.clone())
        cur = ids.tolist()
        for b in range(B):
            true[b].append(cur[b])
    td = TreeDecoder(tm, cache, B, 12)
    if graph:
        td.capture()
    rng = random.Random(1)
    out = [[t] for t in first]
    for it in range(6):
        trees, parents = [], []
        for b in range(B):
            t, p = guesses(true[b], 10 * it + b, 0.85)(out[b])
            trees.append([out[b][-1]] + t[:11])
            parents.append([-1] + [x + 1 for x in p[:11]])
        new, paths = td.step(trees, parents)
        for b in range(B):
            for d, i in enumerate(paths[b]):
                assert torch.equal(td.logits_rows(b, [i])[0], logits[len(out[b]) - 1 + d][b]), (it, b, d)
            out[b] += new[b]
            assert out[b] == true[b][:len(out[b])]
        if min(len(o) for o in out) > 14:
            break
        if it == 2:   # eager work of the program in between
            torch.cuda.synchronize()
            rng.random()
    assert max(len(o) for o in out) > 8
    for b in range(B):
        n = cache.n[b]
        assert n == len(prompts[b]) + len(out[b]) - 1
        for x, y in zip(cache.stack, ref.stack):
            assert torch.equal(x[:, b, :, :n], y[:, b, :, :n])


@pytest.mark.parametrize("start", [235, 500])
def test_captured_trees_past_the_bounds_of_their_passes(start):
    """positions that pass 256 and 512, where another captured pass takes over, and the cache's end"""
    tm = model("tiny", Smax=start + 45, batch=2)
    ref, cache = tm.new_cache(), tm.new_cache()
    first, out = [], []
    for b in range(2):
        prompt = helpers.prompt(b, start - 30 * b, tm.cfg.V)
        first.append(int(tm.forward(prompt, ref, last_only=True, slot=b)[0].argmax()))
        tm.forward(prompt, cache, last_only=True, slot=b)
    true, cur = [[t] for t in first], list(first)
    for _ in range(44):
        _, ids = tm.decode_rows(cur, ref)
        cur = ids.tolist()
        for b in range(2):
            true[b].append(cur[b])
    td = TreeDecoder(tm, cache, 2, 8)
    td.capture()
    out, it = [[t] for t in first], 0
    while max(cache.n) < start + 36:
        trees, parents = [], []
        for b in range(2):
            t, p = guesses(true[b], 10 * it + b, 0.9)(out[b])
            trees.append([out[b][-1]] + t[:7])
            parents.append([-1] + [x + 1 for x in p[:7]])
        new, _ = td.step(trees, parents)
        for b in range(2):
            out[b] += new[b]
            assert out[b] == true[b][:len(out[b])], (it, b)
        it += 1
    assert len(td.graphs) == 2
    for b in range(2):
        for x, y in zip(cache.stack, ref.stack):
            assert torch.equal(x[:, b, :, :cache.n[b]], y[:, b, :, :cache.n[b]])


def test_two_tree_decoders_and_a_longer_cache():
    """captured passes of two caches, one longer than the model's tables, in turn"""
    tm = model("tiny-hd128", Smax=64)
    caches = [tm.new_cache(), Cache(tm.cfg, 1, 200, tm.dev, tm.cfg.NL)]
    prompt = helpers.prompt(5, 20, tm.cfg.V)
    want, _ = generate(tm, prompt, 12, 4, 1.0)
    tds, out = [], []
    for c in caches:
        tm.forward(prompt, c, last_only=True)
        tds.append(TreeDecoder(tm, c, 1, 8, seed=4, temp=1.0))
        tds[-1].capture()
        out.append(want["tokens"][:1])
    for i in range(8):
        for td, o in zip(tds, out):
            if len(o) < 12:
                t, p = guesses(prompt + want["tokens"], i, 0.9)(prompt + o)
                (new,), _ = td.step([[o[-1]] + t[:7]], [[-1] + [x + 1 for x in p[:7]]], [len(o)])
                o += new
    for o in out:
        assert o[:12] == want["tokens"][:len(o)] and len(o) >= 6


def test_tree_decoder_refusals():
    tm = model("tiny", Smax=32)
    cache = tm.new_cache()
    tm.forward([1, 2, 3], cache, last_only=True)
    for B, T in ((0, 4), (2, 4), (1, 0), (1, 65)):
        with pytest.raises(ops.ExactError):
            TreeDecoder(tm, cache, B, T)
    td = TreeDecoder(tm, cache, 1, 4)
    for tree in (([[]], [[]]), ([[1, 2]], [[-1]]), ([[1, 2]], [[-1, 1]]), ([[1, 2]], [[0, 0]]), ([[1, 2]], [[-1, -1]]), ([[1] * 5], [[-1, 0, 0, 0, 0]]),
                 ([[tm.cfg.V]], [[-1]]), ([[-1]], [[-1]]), ([[1], [1]], [[-1], [-1]])):
        with pytest.raises(ops.ExactError):
            td.step(*tree)
    cache.n[0] = 30
    with pytest.raises(ops.ExactError):
        td.step([[1, 2, 3]], [[-1, 0, 1]])
    assert cache.n[0] == 30
    with pytest.raises(ops.ExactError):
        td.finish()
    td.start([[1]], [[-1]])
    for again in (lambda: td.start([[1]], [[-1]]), td.capture):
        with pytest.raises(ops.ExactError):
            again()
    assert len(td.finish()[0][0]) == 1 and cache.n[0] == 31


def test_a_forked_prompt_continues_alike():
    tm = model("tiny-hd128", batch=4)
    cache, ref = tm.new_cache(), tm.new_cache()
    prompt = helpers.prompt(11, 33, tm.cfg.V)
    tm.forward(prompt, cache, last_only=True, slot=2)
    cache.fork(2, [0, 3, 1])
    for b in range(4):
        tm.forward(prompt, ref, last_only=True, slot=b)
    assert cache.n == ref.n == [33] * 4
    for x, y in zip(cache.stack, ref.stack):
        assert torch.equal(x, y)
    toks = [4, 5, 6, 7]
    for _ in range(3):
        (la, ia), (lb, ib) = tm.decode_rows(toks, cache), tm.decode_rows(toks, ref)
        assert torch.equal(la, lb) and torch.equal(ia, ib)
        toks = ia.tolist()
    for bad in ((2, [2]), (0, [1, 1]), (4, [1]), (0, [-1])):
        with pytest.raises(ops.ExactError):
            cache.fork(*bad)
    empty = tm.new_cache()
    empty.n[1] = 5
    empty.fork(0, [1])
    assert empty.n == [0] * 4


@pytest.mark.parametrize("dseed,k", [(3, 4), (4, 4), (4, 1)])
def test_speculation_follows_the_judging_rule(dseed, k):
    """every pass replayed on the host: the draft's samples from its own logits, the oracle's judging of them; the draft of the same
    weights has every token accepted"""
    tm, dm = model("tiny"), model("tiny", seed=dseed)
    prompt, n, seed, temp = helpers.prompt(2, 7, tm.cfg.V), 18, 31, 0.9
    toks, counts = speculate(tm, dm, prompt, n, seed, temp, k)
    assert len(toks) == n and (toks, counts) == speculate(tm, dm, prompt, n, seed, temp, k)
    tnum, dkey, jkey = ops.temp_num(temp), synth.key(seed, "draft"), synth.key(seed, "judge")
    lg = tm.forward(prompt, tm.new_cache(), last_only=True).cpu().numpy()
    got = [O.sample_int(lg[0], seed, 0, tnum)[0]]
    for a in counts:
        t0, d = len(got), min(k, n - len(got) - 1)
        seen, q, drafted = prompt + got, [], []
        for i in range(d):
            row = dm.forward(seen, dm.new_cache(), last_only=True).cpu().numpy()[0]
            x, p = O.sample_int(row, dkey, t0 + i, tnum)
            q.append(p)
            drafted.append(x)
            seen = seen + [x]
        lg = tm.forward(seen, tm.new_cache()).cpu().numpy()[-d - 1:]
        u = [O.splitmix64(jkey, (t0 + 1) * 65 + i) >> 44 for i in range(d + 1)]
        ids, acc = O.verify_draft(lg, q, drafted, u, tnum, d)
        assert acc == a
        got += ids
        if dseed == 3:
            assert acc == d
    assert got[:n] == toks
    if dseed != 3:
        assert any(a < k for a in counts)


def test_speculation_at_the_end_of_the_caches():
    tm, dm = model("tiny", Smax=24), model("tiny", Smax=20, seed=4)
    prompt = helpers.prompt(2, 12, tm.cfg.V)
    toks, _ = speculate(tm, dm, prompt, 13, 1, 1.0)
    assert len(toks) == 13
    with pytest.raises(ops.ExactError):
        speculate(tm, dm, prompt, 14, 1, 1.0)
    with pytest.raises(ops.ExactError):
        speculate(tm, model("tiny-tied"), prompt, 4, 1, 1.0)
    for k in (0, 65):
        with pytest.raises(ops.ExactError):
            speculate(tm, dm, prompt, 4, 1, 1.0, k)


def test_lookup_draft_shares_prefixes():
    assert lookup_draft([1, 2, 3, 4, 1, 2, 5, 6, 1, 2]) == ([5, 6, 1, 2, 3, 4, 1, 2, 5], [-1, 0, 1, 2, -1, 4, 5, 6, 7])
    assert lookup_draft([1, 2, 3, 9, 1, 2, 3, 8, 1, 2], length=2) == ([3, 8, 9], [-1, 0, 0])
    assert lookup_draft([1]) == lookup_draft([1, 2, 3]) == ([], [])


def sampled(tm, prompt, n, seed, temp, step0):
    """n sampled tokens one at a time, the sampler's steps from step0 on"""
    cache, ids, toks = tm.new_cache(B=1), torch.zeros(1, dtype=torch.int32, device=DEV), []
    lg = tm.forward(prompt, cache, last_only=True)
    for i in range(n):
        ops.sample(lg, seed, torch.full((1,), step0 + i, dtype=torch.int32, device=DEV), ops.temp_num(temp), tm.tab.exp, ids)
        toks.append(int(ids))
        lg, _ = tm.decode_rows(toks[-1:], cache)
    return toks


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("first", [(0, 0, 5), (0, 1 << 20, 0)])
def test_seeded_trees_of_a_batch(graph, first):
    """one seed for a forked prompt's two slots and another prompt's: the tokens of sampling one at a time at each sequence's own
    steps, so that equal steps continue the fork alike and steps apart differ"""
    tm, seed, temp = model("tiny-hd128", batch=3), 9, 1.2
    prompts = [helpers.prompt(1, 11, tm.cfg.V)] * 2 + [helpers.prompt(2, 6, tm.cfg.V)]
    true = [sampled(tm, p, 14, seed, temp, f) for p, f in zip(prompts, first)]
    assert (true[0] == true[1]) == (first[0] == first[1])
    cache = tm.new_cache()
    tm.forward(prompts[0], cache, last_only=True, slot=0)
    cache.fork(0, [1])
    tm.forward(prompts[2], cache, last_only=True, slot=2)
    td = TreeDecoder(tm, cache, 3, 7, seed=seed, temp=temp)
    if graph:
        td.capture()
    out = [t[:1] for t in true]
    for it in range(3):
        drafts = [guesses(true[b], it + b, 0.8)(out[b]) for b in range(3)]
        new, _ = td.step([[o[-1]] + t[:6] for o, (t, _) in zip(out, drafts)], [[-1] + [x + 1 for x in p[:6]] for _, p in drafts],
                         [f + len(o) for f, o in zip(first, out)])
        for b in range(3):
            out[b] += new[b]
            assert out[b][:14] == true[b][:len(out[b])]


def test_seeded_steps_have_to_be_given():
    """every pass would draw the random numbers of step 0 again"""
    tm = model("tiny", Smax=32)
    cache = tm.new_cache()
    tm.forward([1, 2, 3], cache, last_only=True)
    td = TreeDecoder(tm, cache, 1, 4, seed=5)
    for call in (td.step, td.start):
        with pytest.raises(ops.ExactError):
            call([[1]], [[-1]])
    assert cache.n[0] == 3 and len(td.step([[1]], [[-1]], [1])[0][0]) == 1 and cache.n[0] == 4
    assert len(TreeDecoder(tm, cache, 1, 4).step([[1]], [[-1]])[0][0]) == 1   # greedy ones take no steps


@pytest.mark.parametrize("graph", [False, True])
def test_a_pass_started_on_another_stream(graph):
    """finish() waits for the pass, whichever stream is current then"""
    tm = model("tiny")
    caches = [tm.new_cache(), tm.new_cache()]
    tds = []
    for c in caches:
        tm.forward([5, 6, 7, 8], c, last_only=True)
        tds.append(TreeDecoder(tm, c, 1, 4))
        if graph:
            tds[-1].capture()
    td, ref = tds
    tree = [[9, 3, 4, 5]], [[-1, 0, 0, 1]]
    want = ref.step(*tree)
    x = torch.randn((8192, 8192), dtype=torch.bfloat16, device=DEV)
    side, load = torch.cuda.Stream(), td._load

    def busy(*a):   # the pass lies behind some 50 ms of other work
        load(*a)
        for _ in range(50):
            x @ x

    td._load = busy
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        td.start(*tree)
    assert td.finish() == want
    lg = td.logits_rows(0, want[1][0])
    assert torch.equal(lg, ref.logits_rows(0, want[1][0]))


def test_trees_of_a_per_channel_model():
    """separate q, k, v linears with one scale a channel: receipts and logits of plain decoding"""
    z = np.load(os.path.join(os.path.dirname(__file__), "golden", "intmodel_tiny.npz"))
    cfg = synth.ModelConfig("channel", D=128, H=2, KV=1, hd=64, I=256, V=512, NL=2, theta=10000.0)
    arrays = {k: z[k] for k in z.files}
    arrays["emb"] = z["emb"].astype(np.int64)
    tm = TModel(DeviceWeights.from_arrays(cfg, arrays, DEV, mode="channel"), Smax=64)
    prompt = helpers.prompt(4, 8, cfg.V)
    want, greedy = generate(tm, prompt, 30, 2, 0.9)
    for nodes, good in ((1, 1.0), (4, 0.8), (20, 1.0), (40, 0.5)):
        got, g = generate(tm, prompt, 30, 2, 0.9, draft=guesses(prompt + want["tokens"], nodes, good), nodes=nodes)
        assert got == want and g == greedy, nodes


def test_captured_trees_with_eager_passes_between():
    """prompts, decode steps and other trees of the same model, run eagerly on another cache between the replays"""
    tm = model("tiny-moe")
    prompt = helpers.prompt(6, 10, tm.cfg.V)
    want, _ = generate(tm, prompt, 16, 8, 1.0)
    cache, other = tm.new_cache(), tm.new_cache()
    tm.forward(prompt, cache, last_only=True)
    td = TreeDecoder(tm, cache, 1, 8, seed=8, temp=1.0)
    td.capture()
    out, it = want["tokens"][:1], 0
    while len(out) < 12:
        t, p = guesses(prompt + want["tokens"], it, 0.8)(prompt + out)
        (new,), _ = td.step([[out[-1]] + t[:7]], [[-1] + [x + 1 for x in p[:7]]], [len(out)])
        out += new
        assert out[:16] == want["tokens"][:len(out)]
        other.n[0] = 0
        tm.forward(helpers.prompt(it, 20 + it, tm.cfg.V), other, last_only=True)
        tm.decode_rows([3], other)
        TreeDecoder(tm, other, 1, 5).step([[1, 2, 3]], [[-1, 0, 0]])
        it += 1
