"""Branching generation through the runner and the entry point: trees of drafted tokens against steps of single tokens, the cache that
they leave, beam searches against the same searches run from scratch, with pages, windows and recurrent states behind the beams."""
import math

import numpy as np
import pytest
import torch

import dryft_challenge_htn_2026_b200 as dk
import plain_qwen3 as plain
from dryft_challenge_htn_2026_b200.engine import Runner, load_model
from dryft_challenge_htn_2026_b200.engine import runner as runner_module
from helpers import TINY, make_folder, random_tokens, tolerance
from test_generate_gpu import teacher_forced_gap
from test_nilivik_gpu import make_model

pytestmark = pytest.mark.gpu


def guesses(seed, vocab, truth, kind):
    """A draft: the right tokens, the right ones among others in a tree, or anything."""
    rs = np.random.RandomState(seed)

    def draft(i, tokens):
        right = truth[i][len(tokens):len(tokens) + 6] if truth else []
        if kind == "right":
            return right
        if kind == "none":
            return []
        if kind == "wrong":
            return rs.randint(0, vocab, rs.randint(0, 7)).tolist()
        toks, parents, at = [], [], -1              # the right way, each node with some others beside it, in mixed order
        for t in right:
            for other in rs.randint(0, vocab, rs.randint(0, 3)).tolist():
                toks.append(int(other)), parents.append(at)
            toks.append(t), parents.append(at)
            at = len(toks) - 1
        return toks, parents
    return draft


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E", "F"])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_drafted_tokens_are_the_ones_that_single_steps_bring(tmp_path, name, temperature):
    vocab, n = TINY[name]["vocab_size"], 30
    eng = dk.Engine(make_folder(tmp_path, name, seed=17), dtype=torch.float32)
    prompts = [random_tokens(vocab, L, 40 + i) for i, L in enumerate([3, 61, 140])]
    steps = list(eng.generate(prompts, n, temperature=temperature, seed=5))
    want = [[s[i] for s in steps] for i in range(3)]
    truth = [p + w for p, w in zip(prompts, want)]
    counts = {}
    for kind in ("right", "tree", "wrong", "none"):
        got, counts[kind] = [[], [], []], 0
        for row in eng.generate_drafted(prompts, n, guesses(1, vocab, truth, kind), temperature=temperature, seed=5):
            counts[kind] += 1
            for g, r in zip(got, row):
                g += r
        assert got == want, kind
    assert counts["right"] == counts["tree"] == 1 + math.ceil((n - 1) / 7) and counts["none"] == n
    stop = want[1][4]                               # a sequence ends with the first of its tokens that stops it
    cut = [w[:w.index(stop) + 1] if stop in w else w for w in want]
    got = [[], [], []]
    for row in eng.generate_drafted(prompts, n, guesses(2, vocab, truth, "tree"), temperature=temperature, seed=5, stop_token_ids=(stop,)):
        for g, r in zip(got, row):
            g += r
    assert got == cut
    assert eng.runner.cache.slots.n_live == 0


@pytest.mark.parametrize("name", ["A", "C", "D", "E"])
def test_drafted_bfloat16_tokens_stay_within_rounding_of_plain(tmp_path, name):
    vocab = TINY[name]["vocab_size"]
    folder = make_folder(tmp_path, name, seed=18)
    cfg, t = plain.read_model(folder)
    eng = dk.Engine(folder, dtype=torch.bfloat16)
    prompts = [random_tokens(vocab, L, 50 + i) for i, L in enumerate([5, 90])]
    truth = [p + plain.greedy(cfg, t, p, 20) for p in prompts]
    scale = max(1.0, float(plain.forward(cfg, t, prompts[1]).abs().max()))
    for kind in ("tree", "wrong"):
        got = [[], []]
        for row in eng.generate_drafted(prompts, 20, guesses(3, vocab, truth, kind)):
            for g, r in zip(got, row):
                g += r
        for p, g in zip(prompts, got):
            assert len(g) == 20 and teacher_forced_gap(cfg, t, p, g) <= 0.12 * scale


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["B", "C", "E"])
def test_the_cache_behind_a_tree_is_that_of_its_accepted_tokens(tmp_path, name, dtype):
    vocab = TINY[name]["vocab_size"]
    model = load_model(make_folder(tmp_path, name, seed=19), getattr(torch, dtype))
    a, b = Runner(model, 64 * 24), Runner(model, 64 * 24)
    prompts = [random_tokens(vocab, L, 60 + i) for i, L in enumerate([59, 2, 130])]
    sa, sb = [a.begin() for _ in prompts], [b.begin() for _ in prompts]
    a.step([(s, p[:-1], []) for s, p in zip(sa, prompts) if len(p) > 1])
    tokens = [list(p) for p in prompts]
    rs = np.random.RandomState(4)
    for turn in range(4):
        trees = []
        for s, t in zip(sa, tokens):
            k = int(rs.randint(1, 40))
            trees.append((s, [t[-1]] + rs.randint(0, vocab, k - 1).tolist(), [-1] + [int(rs.randint(max(0, i - 3), i)) for i in range(1, k)]))
        new = a.step_tree(trees)
        for i, (s, t, n) in enumerate(zip(sa, tokens, new)):
            t += n
            assert a.length(s) == len(t) - 1
    la = a.step([(s, [t[-1]], [0]) for s, t in zip(sa, tokens)])
    lb = b.step([(s, t, [len(t) - 1]) for s, t in zip(sb, tokens)])
    assert float((la - lb).abs().max()) <= tolerance(dtype, lb)
    for r, slots in ((a, sa), (b, sb)):
        for s in slots:
            r.end(s)
        assert all(f == r.cache.num_pages for f in r.cache.pages_free())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "C"])
def test_steps_of_trees_replayed_as_graphs_are_those_that_are_launched(tmp_path, name, dtype):
    """Steps of one shape with other tokens, parents and lengths each time, over a page table that doubles and angle tables that grow."""
    vocab = TINY[name]["vocab_size"]
    model = load_model(make_folder(tmp_path, name, seed=23), getattr(torch, dtype))
    a, b = Runner(model, 64 * 40), Runner(model, 64 * 40)
    prompts = [random_tokens(vocab, L, 80 + i) for i, L in enumerate([488, 59, 2])]
    slots = [[r.begin() for _ in prompts] for r in (a, b)]
    for r, own in zip((a, b), slots):
        r.step([(s, p[:-1], []) for s, p in zip(own, prompts)])
    last, rs, replayed = [p[-1] for p in prompts], np.random.RandomState(6), 0
    for turn in range(14):
        sizes = [7, 3, 5] if turn % 5 else [5, 2, 3]            # steps of other sizes find the same shape
        trees = [([t] + rs.randint(0, vocab, k - 1).tolist(), [-1] + [int(rs.randint(0, i)) for i in range(1, k)]) for t, k in zip(last, sizes)]
        held = len(a._graphs)
        got = a.step_tree([(s, *t) for s, t in zip(slots[0], trees)], 0.7, [1, 2, 3], graph=True)
        replayed += len(a._graphs) == held > 0
        assert got == b.step_tree([(s, *t) for s, t in zip(slots[1], trees)], 0.7, [1, 2, 3])
        last = [g[-1] for g in got]
        assert [a.length(s) for s in slots[0]] == [b.length(s) for s in slots[1]]
        # more tokens, as if they had been accepted: the cache grows faster than these guesses make it
        more = [rs.randint(0, vocab, 3).tolist() for _ in prompts]
        for r, own in zip((a, b), slots):
            r.step([(s, [t] + m[:-1], []) for s, t, m in zip(own, last, more)])
        last = [m[-1] for m in more]
    assert replayed >= 9 and max(a.length(s) for s in slots[0]) > 512
    with pytest.raises(ValueError):
        a.step_tree([(s, [1] * k, [-1] + [k] * (k - 1)) for s, k in zip(slots[0], [7, 3, 5])], graph=True)
    la, lb = (r.step([(s, [t], [0]) for s, t in zip(own, last)]) for r, own in zip((a, b), slots))
    assert torch.equal(la, lb)


@pytest.mark.parametrize("name", ["A", "E"])
def test_drafts_of_all_lengths_find_captured_steps(tmp_path, monkeypatch, name):
    """Eight drafts of 0 to 39 tokens a step: few captures, the captured prompt step stays, the tokens are those of launched steps."""
    vocab = TINY[name]["vocab_size"]
    model = load_model(make_folder(tmp_path, name, seed=24), torch.float32)
    a, b = Runner(model, 64 * 60), Runner(model, 64 * 60)
    captures, real = [], torch.cuda.CUDAGraph
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda *args, **kw: captures.append(1) or real(*args, **kw))
    prompts = [random_tokens(vocab, 3 + 5 * i, 90 + i) for i in range(8)]
    for _ in range(2):                                        # a prompt step of this shape is captured the second time
        slots = [a.begin() for _ in prompts]
        a.step([(s, p[:-1], []) for s, p in zip(slots, prompts)], graph=True)
        for s in slots:
            a.end(s)
    prompt_step = next(iter(a._graphs))
    assert len(captures) == 1
    slots = [[r.begin() for _ in prompts] for r in (a, b)]
    for r, own in zip((a, b), slots):
        r.step([(s, p[:-1], []) for s, p in zip(own, prompts)])
    last, rs = [p[-1] for p in prompts], np.random.RandomState(7)
    for turn in range(60):
        trees = []
        for t in last:
            k = int(rs.randint(1, 41))
            trees.append(([t] + rs.randint(0, vocab, k - 1).tolist(), [-1] + [int(rs.randint(0, i)) for i in range(1, k)]))
        got = a.step_tree([(s, *t) for s, t in zip(slots[0], trees)], 0.8, list(range(8)), graph=True)
        assert got == b.step_tree([(s, *t) for s, t in zip(slots[1], trees)], 0.8, list(range(8)))
        last = [g[-1] for g in got]
    assert 1 <= len(captures) - 1 <= 8 and prompt_step in a._graphs
    la, lb = (r.step([(s, [t], [0]) for s, t in zip(own, last)]) for r, own in zip((a, b), slots))
    assert float((la - lb).abs().max()) <= tolerance("float32", lb)


def test_captured_steps_of_trees_stay_within_their_bytes(tmp_path, monkeypatch):
    """Shapes that take turns where the logits of one alone fit: never more than that, and a shape that was dropped is launched before it is
    captured again."""
    vocab = TINY["A"]["vocab_size"]
    model = load_model(make_folder(tmp_path, "A", seed=25), torch.float32)
    r, alone = Runner(model, 64 * 20), Runner(model, 64 * 20)
    monkeypatch.setattr(runner_module, "TREE_GRAPH_BYTES", 40 * vocab * 4)
    captures, real = [], torch.cuda.CUDAGraph
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda *args, **kw: captures.append(1) or real(*args, **kw))
    (s, u), last, rs = (x.begin() for x in (r, alone)), 5, np.random.RandomState(8)
    for turn in range(12):
        k = (32, 20)[turn // 2 % 2]                            # twice each in turn: launched, then captured
        tokens, parents = [last] + rs.randint(0, vocab, k - 1).tolist(), [-1] + [int(rs.randint(0, i)) for i in range(1, k)]
        got = r.step_tree([(s, tokens, parents)], graph=True)
        assert got == alone.step_tree([(u, tokens, parents)])
        last = got[0][-1]
        assert len(r._graphs) <= 1 and len(captures) == (turn + 1) // 2


def test_launched_steps_of_trees_keep_no_buffers(tmp_path):
    model = load_model(make_folder(tmp_path, "A", seed=26), torch.float32)
    r = Runner(model, 64 * 20)
    s = r.begin()
    r.step_tree([(s, [1, 2], [-1, 0])])
    held = len(r._scratch)
    for k in range(3, 20):
        r.step_tree([(s, [1] * k, list(range(-1, k - 1)))])
    assert len(r._scratch) == held


def test_trees_refusals(tmp_path):
    folder = make_folder(tmp_path, "A", seed=20)
    eng = dk.Engine(folder, dtype=torch.float32)
    r = Runner(eng.model, 64 * 8)
    s = r.begin()
    for tokens, parents in (([1, 2], [-1]), ([], []), ([1, 2], [-1, 1]), ([1, 2], [0, 0]), ([1, 2], [-1, -1]), ([1, 999], [-1, 0]),
                            ([1] * 1025, [-1] + [0] * 1024)):
        with pytest.raises(ValueError):
            r.step_tree([(s, tokens, parents)])
    for more in (dict(seeds=[1, 2]), dict(temperature=-1.0)):
        with pytest.raises(ValueError):
            r.step_tree([(s, [1], [-1])], **more)
    with pytest.raises(ValueError):
        r.step_tree([(s, [1], [-1]), (s, [2], [-1])])
    with pytest.raises(ValueError):
        list(eng.generate_drafted([[1]], 5, lambda i, t: [1] * 64))
    with pytest.raises(ValueError):
        list(eng.generate_drafted([[1]], 5, lambda i, t: ([1], [-1, 0])))
    assert eng.runner.cache.slots.n_live == 0
    with pytest.raises(ValueError):
        list(eng.generate_drafted([[1]], 5, lambda i, t: [], max_nodes=0))
    assert list(eng.generate_drafted([[1]], 0, lambda i, t: [])) == []
    other = load_model(make_model(tmp_path, "P")[0], torch.float32)
    assert not other.takes_trees
    with pytest.raises(ValueError, match="trees"):
        Runner(other, 64 * 8).step_tree([(0, [1], [-1])])


def search(score_of, prompt, beams, n, stops):
    """The same search from scratch: ``score_of(tokens)`` -> float64 log-probabilities of the token behind them."""
    live = [([], 0.0, False)]
    for _ in range(n):
        pool = []
        for b, (t, v, over) in enumerate(live):
            if over:
                pool.append((v, b, 0, t, True))
                continue
            lp = score_of(prompt + t) + v
            for k in np.argsort(-lp, kind="stable")[:beams]:
                pool.append((float(lp[k]), b, int(k), t + [int(k)], int(k) in stops))
        pool.sort(key=lambda x: (-x[0], x[1], x[2]))
        live = [(t, v, over) for v, _, _, t, over in pool[:beams]]
        if all(over for _, _, over in live):
            break
    return [(t, v) for t, v, _ in live]


def check_search(eng, score_of, prompts, beams, n, stops, tol):
    got = eng.beam_search(prompts, beams, n, stop_token_ids=stops)
    for p, rows in zip(prompts, got):
        want = search(score_of, p, beams, n, frozenset(stops))
        assert [len(r) for r in (rows, want)] == [beams, beams]
        assert all(rows[i][1] >= rows[i + 1][1] for i in range(beams - 1))
        for (t, v), (tw, vw) in zip(rows, want):
            assert abs(v - vw) <= tol, (v, vw)
            if t != tw:      # a near tie may fall the other way: then the tokens are as good as the score says
                again = 0.0
                for k in range(len(t)):
                    again += float(score_of(p + t[:k])[t[k]])
                assert abs(again - v) <= tol
    assert eng.runner.cache.slots.n_live == 0
    return got


@pytest.mark.parametrize("name,beams,n", [("A", 1, 6), ("A", 4, 12), ("B", 7, 9), ("C", 5, 70), ("E", 3, 20)])
def test_beam_search_float32(tmp_path, name, beams, n):
    folder = make_folder(tmp_path, name, seed=21)
    cfg, t = plain.read_model(folder)
    eng = dk.Engine(folder, dtype=torch.float32)
    prompts = [random_tokens(TINY[name]["vocab_size"], L, 70 + i) for i, L in enumerate([4, 63, 20])]
    score_of = lambda tokens: torch.log_softmax(plain.forward(cfg, t, tokens)[-1].double(), 0).numpy()
    tol = 2e-4 * n               # each of n log-probabilities within 2e-4, as single logits are held to
    got = check_search(eng, score_of, prompts, beams, n, (), tol)
    stop = got[0][0][0][min(2, n - 1)]
    check_search(eng, score_of, prompts, beams, n, (stop,), tol)
    if beams == 1:               # a search of width one is greedy
        assert [r[0][0] for r in got] == [[s[i] for s in list(eng.generate(prompts, n))] for i in range(3)]
    ranked = eng.beam_search(prompts[:1], beams, n, stop_token_ids=(stop,), length_penalty=1.0)[0]
    assert all(ranked[i][1] >= ranked[i + 1][1] for i in range(beams - 1))


@pytest.mark.parametrize("shape", ["P", "Q"])
def test_beam_search_moves_states_chunks_and_values_of_another_size(tmp_path, shape):
    """Attention over chunks with value heads of another size beside a recurrent state, looped layers."""
    eng = dk.Engine(make_model(tmp_path, shape)[0], dtype=torch.float32)
    runner = Runner(eng.model, 64 * 16)

    def score_of(tokens):
        s = runner.begin()
        logits = runner.step([(s, list(tokens), [len(tokens) - 1])])[0]
        runner.end(s)
        return torch.log_softmax(logits.double(), 0).cpu().numpy()

    prompts = [random_tokens(eng.model.spec.vocab_size, L, 80 + i) for i, L in enumerate([5, 37])]
    check_search(eng, score_of, prompts, 4, 30, (), 2e-4 * 30)


def test_beam_search_edges(tmp_path):
    eng = dk.Engine(make_folder(tmp_path, "B", seed=22), dtype=torch.bfloat16)
    assert eng.beam_search([], 3, 5) == [] and eng.beam_search([[1], [2]], 3, 0) == [[], []]
    for beams in (0, 33):
        with pytest.raises(ValueError):
            eng.beam_search([[1]], beams, 5)
    with pytest.raises(ValueError):
        eng.beam_search([[1], []], 2, 5)
    rows = eng.beam_search([[1, 2, 3]], 32, 3)[0]
    assert len(rows) == 32 and len({tuple(t) for t, _ in rows}) == 32 and all(len(t) == 3 and v < 0 for t, v in rows)
    once = eng.beam_search([[1, 2, 3], [7]], 6, 10)
    assert once == eng.beam_search([[1, 2, 3], [7]], 6, 10)
    # beside another request, the same search
    assert [t for t, _ in eng.beam_search([[7]], 6, 10)[0]][:1] == [t for t, _ in once[1]][:1]


def test_reorder_follows_parents_within_the_cache(tmp_path):
    model = load_model(make_folder(tmp_path, "C", seed=23), torch.float32)
    r = Runner(model, 64 * 40)
    vocab = TINY["C"]["vocab_size"]
    prompt, tails = random_tokens(vocab, 90, 1), [random_tokens(vocab, 45, 2 + i) for i in range(4)]
    slots = [r.begin() for _ in range(4)]
    r.step([(s, prompt, []) for s in slots])
    r.step([(s, t, []) for s, t in zip(slots, tails)])
    parents = [1, 0, 0, 3]
    r.cache.reorder([slots], [parents], [len(prompt)])
    got = r.step([(s, [5], [0]) for s in slots])
    for row, p in zip(got, parents):
        s = r.begin()
        ref = r.step([(s, prompt + tails[p] + [5], [len(prompt) + 45])])[0]
        r.end(s)
        assert float((row - ref).abs().max()) <= tolerance("float32", ref)
