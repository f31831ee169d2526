"""Trees of drafted tokens and beams: attention of a tree over the cache, the path that is accepted, the best continuations of beams,
and the moves of cache rows and states, each against a plain implementation in 64 bits (moves: against the same moves on the host)."""
import math
import threading

import numpy as np
import pytest
import torch

from dryft_challenge_htn_2026_b200.csrc import api

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = api.PAGE


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def normal(shape, dtype=torch.float32, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


def tree_of(rs, n):
    """Random parents of n nodes (-1 for the root)."""
    return [-1] + [int(rs.randint(max(0, i - 5), i)) for i in range(1, n)]


def ancestors(parents):
    """[n, n] bool: which nodes lie on the way from the root to each node, itself included."""
    n = len(parents)
    m = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if i and p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def bits_of(masks, words):
    """int32 words of the rows of several [n, n] masks one behind the other."""
    out = np.zeros((sum(len(m) for m in masks), words), np.uint32)
    row = 0
    for m in masks:
        for i in range(len(m)):
            for j in np.flatnonzero(m[i]):
                out[row, j // 32] |= np.uint32(1) << np.uint32(j % 32)
            row += 1
    return i32(out.view(np.int32))


def tree_case(before, nodes, nh, nkv, hd, dtype, seed=0, words=None, masks=None, extra_rows=0, width=None, strided=False):
    """Sequences of ``before`` cached tokens with trees of ``nodes`` nodes, pages in mixed order."""
    rs = np.random.RandomState(seed)
    parents = [tree_of(rs, n) if n else [] for n in nodes]
    masks = [ancestors(p) for p in parents] if masks is None else masks
    depth = []
    for p in parents:
        d = []
        for i, up in enumerate(p):
            d.append(0 if i == 0 else d[up] + 1)
        depth.append(d)
    need = [max(1, (b + n + PAGE - 1) // PAGE) for b, n in zip(before, nodes)]
    n_pages = sum(need) + 2
    order = rs.permutation(n_pages).tolist()
    table = -np.ones((len(nodes), width or max(need)), np.int64)
    for s, k in enumerate(need):
        table[s, :k] = [order.pop() for _ in range(k)]
    rows = sum(nodes) + extra_rows
    words = words or max(1, (max(nodes) + 31) // 32)
    tree = torch.cat([bits_of(masks, words), torch.zeros((extra_rows, words), dtype=torch.int32, device=DEV)])
    pos = [b + d for b, ds in zip(before, depth) for d in ds] + [0] * extra_rows
    q = normal((rows, nh * hd), dtype, seed + 1)
    if strided:
        q = torch.cat([normal((rows, 16), dtype, 5), q, normal((rows, 16), dtype, 6)], 1)[:, 16:16 + nh * hd]
    return dict(before=before, nodes=nodes, masks=masks, depth=depth, table=table, q=q, k=normal((n_pages, nkv, PAGE, hd), dtype, seed + 2),
                v=normal((n_pages, nkv, PAGE, hd), dtype, seed + 3), cu=i32(np.concatenate([[0], np.cumsum(nodes)])), pos0=i32(before),
                pos=i32(pos), tree=tree, page_table=i32(table), nh=nh, nkv=nkv, hd=hd, rows=rows, n_pages=n_pages)


def leave_numbers_behind():
    """Memory that the next call's scratch comes from holds large numbers: a part that nobody wrote shows."""
    for n in (1 << 18, 1 << 22, 1 << 24):
        torch.full((n,), 1e30, device=DEV)


def attend(c, window=0, scale=None, out=None, max_nodes=None):
    leave_numbers_behind()
    out = torch.full((c["rows"], c["nh"] * c["hd"]), 7.0, dtype=c["q"].dtype, device=DEV) if out is None else out
    api.attention_tree(c["q"], out, c["k"], c["v"], c["cu"], c["pos0"], c["pos"], c["tree"], c["page_table"], c["nh"], c["nkv"], c["hd"],
                       window, scale or c["hd"] ** -0.5, max_nodes or max(1, max(c["nodes"])))
    return out


def plain_attend(c, window=0, scale=None):
    """-> (float64 rows, a bound on the error of each number). A key on a page that is none is not seen."""
    scale = scale or c["hd"] ** -0.5
    G = c["nh"] // c["nkv"]
    q, k, v = (t.double().cpu() for t in (c["q"], c["k"], c["v"]))
    pos = c["pos"].cpu().numpy()
    out = torch.full((c["rows"], c["nh"] * c["hd"]), 7.0, dtype=torch.float64)
    tol = torch.zeros_like(out)
    half = torch.finfo(c["q"].dtype).eps / 2
    row = 0
    for s, (b, n) in enumerate(zip(c["before"], c["nodes"])):
        for i in range(n):
            keys, q_pos = [], int(pos[row])
            for place in range(b + n):
                p = place if place < b else int(pos[row - i + place - b])
                page = int(c["table"][s, place // PAGE]) if place // PAGE < c["table"].shape[1] else -1
                seen = place < b or bool(c["masks"][s][i, place - b])
                if seen and 0 <= page < c["n_pages"] and q_pos >= 0 and not (window and q_pos - p >= window):
                    keys.append((page, place % PAGE))
            if not keys:
                out[row], tol[row] = 0, 0
                row += 1
                continue
            pg, at = torch.tensor([x[0] for x in keys]), torch.tensor([x[1] for x in keys])
            for h in range(c["nh"]):
                cols = slice(h * c["hd"], (h + 1) * c["hd"])
                kk, vv, qq = k[pg, h // G, at], v[pg, h // G, at], q[row, cols]
                sc = kk @ qq * scale
                w = torch.softmax(sc, 0)
                out[row, cols] = w @ vv
                # float32 scores: hd products and sums, each half a step of the sum of their sizes; two of them set a weight. The sums
                # over the keys: one rounding a key, and a few a page. Storage: the weights may be rounded once, the result is.
                score = (kk.abs() @ qq.abs()).max() * scale * (c["hd"] + 4) * 2 ** -24
                sums = (len(keys) + 8 * (len(keys) // PAGE + 2)) * 2 ** -24
                big = vv.abs().max()
                tol[row, cols] = (2 * score + 2 * sums) * big + (half * (w @ vv.abs()) if c["q"].dtype == torch.bfloat16 else 0) \
                    + half * out[row, cols].abs() + 1e-30
            row += 1
    return out, tol


def check_attend(c, window=0, scale=None, **kw):
    got = attend(c, window, scale, **kw).double().cpu()
    ref, tol = plain_attend(c, window, scale)
    off = (got - ref).abs()
    assert bool((off <= tol).all()), f"off by {float(off.max())}, {float((off / tol.clamp(min=1e-30)).nan_to_num(0).max())} of what is allowed"


HEADS = [(4, 2, 64), (8, 1, 128), (3, 3, 48), (6, 2, 16), (2, 1, 256)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("before,nodes", [
    ([0], [1]), ([1], [1]), ([63], [1]), ([64], [2]), ([130], [7]),            # one sequence: from a single token on
    ([5, 200, 63], [9, 1, 33]), ([300, 1], [40, 64]),                          # unequal lengths, trees over two pages
    ([100, 0, 77], [5, 0, 3]),                                                 # a sequence without nodes
])
def test_tree_attention(dtype, heads, before, nodes):
    check_attend(tree_case(before, nodes, *heads, dtype, seed=len(before) + nodes[0]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 4, 64), (16, 1, 64), (3, 1, 32), (5, 1, 128), (14, 2, 64), (64, 1, 64)])
def test_tree_attention_long_contexts_and_large_trees(dtype, heads):
    check_attend(tree_case([900, 37, 2500], [12, 130, 3], *heads, dtype, seed=3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window", [1, 2, 5, 64, 150, 4000])
def test_tree_attention_window(dtype, window):
    c = tree_case([0, 130, 700], [20, 33, 6], 4, 2, 64, dtype, seed=window)
    for s, b in enumerate(c["before"]):                # pages that lie wholly before the window have been given back
        gone = max(0, b - window + 1) // PAGE
        c["table"][s, :gone] = -1
    c["page_table"] = i32(c["table"])
    check_attend(c, window)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 48, 128])
def test_tree_attention_any_bits_and_rows_that_see_nothing(dtype, hd):
    rs = np.random.RandomState(1)
    masks = [rs.rand(n, n) < 0.3 for n in (70, 5, 1)]
    masks[0][3] = False
    masks[2][0] = False
    c = tree_case([0, 40, 0], [70, 5, 1], 4, 2, hd, dtype, seed=9, masks=masks, extra_rows=3, width=5, words=4, strided=True)
    c["pos"][72] = -1                                   # a padding row
    c["tree"][:70, 3] = -1                              # bits of nodes that there are not
    c["tree"][70:76, 1:] = -1
    got = attend(c)
    assert bool((got[3] == 0).all()) and bool((got[75] == 0).all()) and bool((got[72] == 0).all())
    assert bool((got[76:] == 7).all())                  # rows behind the last sequence
    check_attend(c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 48, 128])
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, hd, odd):
    c = tree_case([60, 130], [9, 4], 4, 2, hd, dtype, seed=2)
    clean = attend(c)
    for s, (b, n) in enumerate(zip(c["before"], c["nodes"])):
        for place in range(b + n, c["table"].shape[1] * PAGE):          # behind the tree's last node
            page = c["table"][s, place // PAGE]
            if page >= 0:
                c["k"][page, :, place % PAGE], c["v"][page, :, place % PAGE] = odd, odd
    free = set(range(c["n_pages"])) - set(c["table"].reshape(-1).tolist())
    for page in free:
        c["k"][page], c["v"][page] = odd, odd
    assert torch.equal(attend(c), clean)
    # one node's key and value, and one of its values alone: only the rows that see the node are touched
    j = 3
    page, at = c["table"][0, (60 + j) // PAGE], (60 + j) % PAGE
    c["v"][page, 1, at, 5] = odd
    got = attend(c).view(-1, 4, hd)
    seen = torch.tensor(np.concatenate([c["masks"][0][:, j], np.zeros(4, bool)]), device=DEV)
    hurt = ~torch.isfinite(got)
    assert torch.equal(hurt[:, 2:, 5].all(1), seen) and int(hurt.sum()) == 2 * int(seen.sum())
    rest = clean.view(-1, 4, hd).clone()
    rest[hurt] = got[hurt]
    assert torch.equal(got.nan_to_num(1.5), rest.nan_to_num(1.5))
    c["k"][page, :, at] = odd
    got = attend(c)
    assert torch.equal(torch.isfinite(got).all(1), ~seen) and torch.equal(got[~seen], clean[~seen])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pages_that_are_none_hold_no_keys(dtype):
    c = tree_case([200, 70], [6, 3], 4, 2, 64, dtype, seed=4)
    c["table"][0, 1], c["table"][1, 0] = -1, c["n_pages"] + 5
    c["page_table"] = i32(c["table"])
    check_attend(c)
    short = dict(c, table=c["table"][:, :2], page_table=c["page_table"][:, :2].contiguous())     # a table that ends too soon
    check_attend(short)


def test_tree_attention_of_single_tokens_is_decode_attention():
    for dtype, hd in ((torch.bfloat16, 128), (torch.float32, 64)):
        c = tree_case([500, 3, 64], [1, 1, 1], 8, 2, hd, dtype, seed=6)
        out = torch.empty_like(c["q"])
        if dtype == torch.bfloat16:
            ws = api.attention_decode_ws(3, 8, hd, 2, DEV)
            api.attention_decode_bf16(c["q"], out, c["k"], c["v"], c["pos"], c["page_table"], 8, 2, hd, 0, hd ** -0.5, 2, *ws)
        else:
            api.attention_decode_f32(c["q"], out, c["k"], c["v"], c["pos"], c["page_table"], 8, 2, hd, 0, hd ** -0.5)
        _, tol = plain_attend(c)
        assert bool(((attend(c).double() - out.double()).abs().cpu() <= 2 * tol).all())


def test_tree_attention_captured_and_replayed_with_other_lengths():
    make = lambda before, seed: tree_case(before, [20, 9], 8, 2, 128, torch.bfloat16, seed=seed, width=12)
    c = make([640, 640], 7)
    out = torch.zeros_like(c["q"])
    attend(c, out=out, max_nodes=32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(c, out=out, max_nodes=32)
    for seed, before in enumerate(([100, 640], [0, 300], [641, 7])):
        d = make(before, seed)
        want = attend(d, max_nodes=32)
        for name in ("k", "v"):
            c[name][:d["n_pages"]] = d[name]
        for name in ("q", "pos0", "pos", "tree", "page_table"):
            c[name].copy_(d[name])
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv,n_seq,context,nodes", [
    (32, 8, 8, 8192, 2),      # bound by memory: pages come in late and out of turn, shares end one page into a tile
    (8, 1, 37, 577, 3), (16, 8, 41, 700, 40), (4, 4, 70, 64, 1),
])
def test_tree_attention_gives_the_same_bits_every_time(hd, nh, nkv, n_seq, context, nodes):
    rs = np.random.RandomState(n_seq)
    before = [int(b) for b in rs.randint(max(1, context // 2), context + 1, n_seq)]
    c = tree_case(before, [int(x) for x in rs.randint(1, nodes + 1, n_seq)], nh, nkv, hd, torch.bfloat16, seed=n_seq)
    first = attend(c)
    api.gemm_tc_check()
    out = torch.empty_like(first)
    for _ in range(50):
        attend_again = attend(c, out=out)
        assert torch.equal(attend_again, first)
    api.gemm_tc_check()
    ref, tol = plain_attend(dict(c, before=c["before"][:1], nodes=c["nodes"][:1], masks=c["masks"][:1]))
    rows = c["nodes"][0]
    assert bool(((first.double().cpu() - ref).abs() <= tol)[:rows].all())


def test_tree_attention_leaves_out_nodes_above_its_number():
    for dtype in (torch.bfloat16, torch.float32):
        c = tree_case([700, 3], [9, 40], 8, 2, 64, dtype, seed=12)
        got = attend(c, max_nodes=20)
        few = dict(c, nodes=[9, 20], masks=[c["masks"][0], c["masks"][1][:20, :20]], rows=29, q=c["q"][:29])
        ref, tol = plain_attend(few)
        assert bool(((got[:29].double().cpu() - ref).abs() <= tol).all()) and bool((got[29:] == 7).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_beyond_32_bits(dtype):
    """A store of more than 2^32 bytes and 2^31 numbers whose last pages are used, the rest whatever the memory held."""
    nkv, hd = 8, 128
    n_pages = (1 << 31) // (nkv * PAGE * hd) + 9
    store = torch.empty((1, 2, n_pages, nkv, PAGE, hd), dtype=dtype, device=DEV)
    c = tree_case([70, 130], [5, 33], 16, nkv, hd, dtype, seed=13)
    far = c["table"] + (n_pages - c["n_pages"])
    for page in range(c["n_pages"]):
        store[0, 0, n_pages - c["n_pages"] + page], store[0, 1, n_pages - c["n_pages"] + page] = c["k"][page], c["v"][page]
    d = dict(c, k=store[0, 0], v=store[0, 1], page_table=i32(np.where(c["table"] >= 0, far, -1)), n_pages=n_pages)
    assert torch.equal(attend(d), attend(c))
    small = torch.stack([c["k"], c["v"]])[None].clone()
    path, count = i32([[0, 2, 4, -1, -1]] * 2), i32([3, 3])
    for t, table in ((store, d["page_table"]), (small, c["page_table"])):
        api.kv_keep(t, table, c["pos0"], path, count)
        api.kv_reorder(t, table, i32([[1, 0]]), i32([2]), i32([90]))
    assert torch.equal(store[:, :, -c["n_pages"]:], small)
    del store, d
    torch.cuda.empty_cache()


def test_calls_on_two_streams_at_once():
    cases = [tree_case([900, 2000], [40, 7], 8, 2, 128, torch.bfloat16, seed=14 + i) for i in range(2)]
    logits = [normal((12, 50000), seed=20 + i, scale=3.0) for i in range(2)]
    scores = torch.zeros((3, 4), device=DEV)
    tree = ([3] * 12, [[-1] + list(range(11))], list(range(12)), [0.7], [[5, 6]])
    want = [(attend(c), select(x, scores, None, 8), accept(x, *tree)) for c, x in zip(cases, logits)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for st, c, x in zip(streams, cases, logits):
            with torch.cuda.stream(st):
                out = torch.empty_like(c["q"])
                api.attention_tree(c["q"], out, c["k"], c["v"], c["cu"], c["pos0"], c["pos"], c["tree"], c["page_table"], 8, 2, 128, 0, 128 ** -0.5, 40)
                best = torch.empty((3, 8), device=DEV), i32(np.zeros((3, 8))), i32(np.zeros((3, 8)))
                api.beam_select(x, scores, None, *best)
                got.append((out, best))
        torch.cuda.synchronize()
        for (out, best), (a, b, _) in zip(got, want):
            assert torch.equal(out, a) and all(torch.equal(p.cpu(), q) for p, q in zip(best, b))
    api.gemm_tc_check()


def test_scratch_memory_is_held_until_the_launches_are_made(monkeypatch):
    """Memory that is given back before the C entry is called is another thread's to take, on the same stream too: its first launch would lie
    between the two of this call."""
    real, held = api._entry, []

    def entry(lib, name, kinds):
        def call(*args):
            for size in [1 << k for k in range(9, 24)] * 8:              # what another thread may ask for meanwhile
                held.append(torch.empty(size, dtype=torch.uint8, device=DEV))
            took = [(t.data_ptr(), t.data_ptr() + t.numel()) for t in held]
            lost = [a for a in args if isinstance(a, int) and any(lo <= a < hi for lo, hi in took)]
            assert not lost, f"{name}: its scratch memory was taken"
            return real(lib, name, kinds)(*args)
        return call

    monkeypatch.setattr(api, "_entry", entry)
    cases = [lambda: attend(tree_case([900, 2000], [40, 7], 8, 2, 128, torch.bfloat16)),
             lambda: attend(tree_case([900, 2000], [40, 7], 8, 2, 64, torch.float32)),
             lambda: accept(normal((12, 50000), seed=2), [3] * 12, [[-1] + list(range(11))], list(range(12)), [0.7], [[5, 6]]),
             lambda: select(normal((12, 50000), seed=2), torch.zeros((3, 4), device=DEV), None, 8)]
    for case in cases:
        held.clear()
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        case()


def test_two_threads_on_one_stream():
    logits = [normal((64, 20000), seed=20 + i, scale=3.0) for i in range(2)]
    scores = torch.zeros((16, 4), device=DEV)
    tree = ([3] * 64, [[-1] + list(range(63))], list(range(64)), [0.7], [[5, 6]])
    want = [(select(x, scores, None, 16), accept(x, *tree)) for x in logits]
    wrong = []

    def work(k):
        for _ in range(200):
            got = select(logits[k], scores, None, 16), accept(logits[k], *tree)
            if not all(torch.equal(a, b) for a, b in zip(got[0], want[k][0])) or got[1] != want[k][1]:
                wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("before,width", [(60, 4), (700, 20)])       # tiles that are not split, and such that are
def test_values_that_are_none_in_some_of_many_tiles(hd, before, width):
    n_seq, nh, nkv = 70, 8, 4
    c = tree_case([before + s % 9 for s in range(n_seq)], [1 + s * 7 % 12 for s in range(n_seq)], nh, nkv, hd, torch.bfloat16, seed=9, width=width)
    clean = attend(c)
    for s, (b, n) in enumerate(zip(c["before"], c["nodes"])):
        page, at = c["table"][s, (b + n) // PAGE], (b + n) % PAGE        # the place behind the last node, where there is one
        if at and s % 3 == 0:
            c["v"][page, :, at:], c["k"][page, :, at:] = math.nan, math.inf
    assert torch.equal(attend(c), clean)
    hurt = torch.zeros((c["rows"], nh, hd), dtype=torch.bool, device=DEV)
    for s in range(0, n_seq, 4):                                         # the root's value for one kv head, in every fourth sequence
        b, row = c["before"][s], int(c["cu"][s])
        c["v"][c["table"][s, b // PAGE], s // 4 % nkv, b % PAGE, s % hd] = -math.inf
        hurt[row:row + c["nodes"][s], 2 * (s // 4 % nkv):2 * (s // 4 % nkv) + 2, s % hd] = True
    got = attend(c).view(-1, nh, hd)
    assert torch.equal(got == -math.inf, hurt) and torch.equal(got[~hurt], clean.view(-1, nh, hd)[~hurt])
    api.gemm_tc_check()


@pytest.mark.parametrize("hd,dtype", [(64, torch.float32), (128, torch.float32), (48, torch.bfloat16)])
def test_values_that_are_none_in_tiles_of_all_heights(hd, dtype):
    """Trees whose tiles have up to 16, up to 32 and up to 64 rows, side by side in a launch."""
    c = tree_case([61, 130, 5, 200], [40, 7, 13, 20], 4, 2, hd, dtype, seed=4)
    clean = attend(c)
    hurt = torch.zeros((c["rows"], 4, hd), dtype=torch.bool, device=DEV)
    for s, (b, n) in enumerate(zip(c["before"], c["nodes"])):
        row, j = int(c["cu"][s]), n // 2
        c["v"][c["table"][s, (b + j) // PAGE], 1, (b + j) % PAGE, 3 + s] = math.inf
        hurt[row:row + n, 2:, 3 + s] = torch.tensor(c["masks"][s][:, j], device=DEV)[:, None]
    got = attend(c).view(-1, 4, hd)
    assert torch.equal(got == math.inf, hurt) and torch.equal(got[~hurt], clean.view(-1, 4, hd)[~hurt])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("before", [30, 900])
def test_tree_attention_in_place(dtype, before):
    c = tree_case([before, 7, before + 99], [40, 9, 33], 8, 2, 128, dtype, seed=3, strided=True)
    want = attend(c)
    assert torch.equal(attend(c, out=c["q"]), want)


def test_operators_one_after_another_captured_and_replayed():
    """A step's choice and moves as one graph: accept, keep, then select, reorder of pages and states, with other contents each time."""
    V, n_pages, nkv, hd = 5000, 20, 2, 64
    rs = np.random.RandomState(1)
    parents = tree_of(rs, 30)
    logits, store = torch.zeros((30, V), device=DEV), torch.zeros((2, n_pages, nkv, PAGE, hd), dtype=torch.bfloat16, device=DEV)
    table, states = i32(rs.permutation(n_pages)[:16].reshape(4, 4)), torch.zeros((3, 6, 40), device=DEV)
    tok, parent, cu, pos, pos0 = i32(np.zeros(30)), i32(parents), i32([0, 30]), i32(range(100, 130)), i32([100])
    temp, seeds = torch.zeros(1, device=DEV), i32([[3, 4]])
    path, count, token = i32(np.zeros((1, 30))), i32([0]), i32([0])
    scores, slots, first, last = torch.zeros((1, 4), device=DEV), i32([4, 0, 3, 1]), i32([100]), i32([131])
    best, beam, which = torch.zeros((1, 4), device=DEV), i32(np.zeros((1, 4))), i32(np.zeros((1, 4)))

    def run():
        api.tree_accept(logits, tok, parent, cu, pos, temp, seeds, path, count, token)
        api.kv_keep(store, table[:1], pos0, path, count)
        api.beam_select(logits[:4], scores, None, best, beam, which)
        api.kv_reorder(store, table, beam, first, last)
        api.state_reorder(states, slots, beam)

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in range(4):
        logits.copy_(normal((30, V), seed=seed, scale=3.0))
        scores.copy_(normal((1, 4), seed=seed + 9))
        choice = logits.argmax(1).tolist()
        tok.copy_(i32([0] + [choice[p] if i % 4 else 1 for i, p in enumerate(parents) if i]))
        at = [(normal(tuple(store.shape), torch.bfloat16, seed)), normal(tuple(states.shape), seed=seed)]
        results = []
        for call in (run, graph.replay):
            store.copy_(at[0]), states.copy_(at[1])
            leave_numbers_behind()
            call()
            results.append([t.clone() for t in (store, states, path, count, token, best, beam, which)])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        assert results[1][2].tolist() == plain_accept(choice, tok.tolist(), [parents], 30)[0]
        want = plain_select(logits[:4], scores.cpu(), None, 4)
        assert np.array_equal(results[1][6].cpu().numpy(), want[1]) and np.array_equal(results[1][7].cpu().numpy(), want[2])
        b = want[1][0]
        assert torch.equal(states[:, [4, 0, 3, 1]], at[1][:, [[4, 0, 3, 1][x] for x in b]])


def test_tree_attention_refusals():
    c = tree_case([30], [4], 4, 2, 64, torch.bfloat16)
    good = dict(q=c["q"], out=torch.empty_like(c["q"]), k_store=c["k"], v_store=c["v"], cu_q=c["cu"], seq_pos0=c["pos0"], row_pos=c["pos"],
                tree=c["tree"], page_table=c["page_table"], n_heads=4, n_kv_heads=2, head_dim=64, window=0, scale=0.125, max_nodes=4)
    api.attention_tree(**good)
    for bad in (dict(max_nodes=0), dict(max_nodes=1025), dict(scale=0.0), dict(scale=-1.0), dict(window=-1), dict(head_dim=40), dict(n_heads=3),
                dict(n_kv_heads=4), dict(cu_q=c["cu"].long()), dict(cu_q=c["cu"][:1]), dict(row_pos=c["pos"][:3]), dict(tree=c["tree"][:2]),
                dict(out=torch.empty_like(c["q"]).float()), dict(k_store=c["k"].float()), dict(v_store=c["v"][:1]), dict(q=c["q"].cpu()),
                dict(q=c["q"][:, :128]), dict(page_table=c["page_table"].repeat(2, 1)), dict(q=c["q"].half(), out=c["q"].half()),
                dict(q=torch.zeros((4, 260), dtype=torch.bfloat16, device=DEV)[:, 1:257]), dict(k_store=c["k"].transpose(2, 3))):
        with pytest.raises(api.KernelError):
            api.attention_tree(**{**good, **bad})


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.bfloat16, 48), (torch.bfloat16, 128)])
@pytest.mark.parametrize("name", ["k", "v"])
def test_tree_attention_refuses_stores_that_are_not_aligned(dtype, hd, name):
    c = tree_case([30], [4], 4, 2, hd, dtype)
    attend(c)
    for off in (1, 16 // c["k"].element_size() - 1):
        odd = torch.zeros(c["k"].numel() + 16, dtype=dtype, device=DEV)[off:off + c["k"].numel()].view_as(c["k"])
        with pytest.raises(api.KernelError, match="16-byte"):
            attend(dict(c, **{name: odd}))


# ------------------------------------------------------------------------------------------------ accept
def sampler_choice(logits, pos, temperature, seeds):
    """The token ``sample`` chooses for each row."""
    n, V = logits.shape
    ws = n * api.sample_chunks(V)
    out = torch.empty(n, dtype=torch.int32, device=DEV)
    api.sample(logits, temperature, seeds, pos, None, torch.empty(ws, device=DEV), torch.empty(ws, dtype=torch.int32, device=DEV), out)
    return out.tolist()


def accept(logits, tok, parents, pos, temperature, seeds, max_nodes=None):
    nodes = [len(p) for p in parents]
    n, width = len(nodes), max_nodes or max(1, max(nodes))
    path, count, token = i32(np.full((n, width), 9)), i32(np.full(n, 9)), i32(np.full(n, 9))
    api.tree_accept(logits, i32(tok), i32([x for p in parents for x in p] or np.zeros(0)), i32(np.concatenate([[0], np.cumsum(nodes)])),
                    i32(pos), torch.tensor(temperature, dtype=torch.float32, device=DEV), i32(seeds), path, count, token)
    return path.tolist(), count.tolist(), token.tolist()


def plain_accept(choice, tok, parents, width):
    paths, counts, tokens, row = [], [], [], 0
    for p in parents:
        at, way = 0, [0] if p else []
        while p:
            nxt = [i for i in range(at + 1, len(p)) if p[i] == at and tok[row + i] == choice[row + at]]
            if not nxt:
                break
            at = nxt[0]
            way.append(at)
        paths.append(way + [-1] * (width - len(way)))
        counts.append(len(way))
        tokens.append(choice[row + at] if p else 0)
        row += len(p)
    return paths, counts, tokens


@pytest.mark.parametrize("vocab", [1, 7, 300, 4096, 4097, 50001, 151936])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_accept(vocab, temperature):
    rs = np.random.RandomState(vocab)
    nodes = [1, 40, 6, 0, 64, 33]
    parents = [tree_of(rs, n) if n else [] for n in nodes]
    rows = sum(nodes)
    logits = normal((rows, vocab), seed=vocab, scale=2.0)
    pos = rs.randint(0, 3000, rows).tolist()
    temps = [temperature] * 5 + [0.0]
    seeds = rs.randint(-2 ** 31, 2 ** 31 - 1, (6, 2))
    seq = np.repeat(np.arange(6), nodes)
    choice = sampler_choice(logits, i32(pos), i32([0] * rows).float() + torch.tensor(np.array(temps)[seq], dtype=torch.float32, device=DEV),
                            i32(seeds[seq]))
    tok, row = rs.randint(0, vocab, rows).tolist(), 0
    for p in parents:                                    # two of three drafted tokens are what their parent chose
        for i in range(1, len(p)):
            if i % 3:
                tok[row + i] = choice[row + p[i]]
        row += len(p)
    got = accept(logits, tok, parents, pos, temps, seeds)
    assert got == plain_accept(choice, tok, parents, 64)
    assert max(got[1]) > 3 or vocab > 10 ** 9


def noise_words(lo, hi, pos, V):
    """The top 24 bits of the sampler's hash of tokens 0 to V (the noise is -log(-log u), u = (word + 1/2) / 2^24)."""
    u32, m = np.uint32, 0xffffffff

    def mix(x):
        x = (x ^ x >> u32(16)) * u32(0x7FEB352D)
        x = (x ^ x >> u32(15)) * u32(0x846CA68B)
        return x ^ x >> u32(16)

    x = mix(np.arange(V, dtype=u32) ^ u32(0x9E3779B9))
    return mix(mix(x + u32((pos * 0x85EBCA6B + lo) & m)) ^ u32(hi)) >> u32(8)


def test_drawn_tokens_are_never_ones_that_have_no_chance():
    """All but 500 of 50,001 tokens are e^40 times less likely than the others. Among the hash values are some whose u would be 1 if it were
    rounded, and the noise infinite; the largest noise there may be is -log(-log(1 - 2^-24)) = 16.6."""
    V, rows, lo, hi = 50001, 1000, 12345, 0x9abcdef0
    logits = torch.full((rows, V), -40.0, device=DEV)
    logits[:, :500] = normal((rows, 500), seed=8)
    words = [noise_words(lo, hi, p + 1, V) for p in range(rows)]
    assert sum(int((w[500:] == 0xffffff).any()) for w in words) >= 2
    seeds = i32(np.array([[lo, hi]], np.uint32).view(np.int32))
    got = np.array(sampler_choice(logits, i32(range(rows)), torch.ones(rows, device=DEV), seeds.repeat(rows, 1)))
    assert got.max() < 500
    u = np.minimum((np.stack(words)[:, :500] + 0.5) / 2 ** 24, 1 - 2.0 ** -24)
    noise = -np.log(-np.log(u))
    value = logits[:, :500].double().cpu().numpy() + noise
    # u in float32 is off by half a step of 2^-24 at most, the noise by that over -u log u: 2.5e-4 where the noise is below 9; two tokens
    gap, row, best = value.max(1) - value[np.arange(rows), got], np.arange(rows), value.argmax(1)
    assert np.all((gap < 1e-3) | (np.maximum(noise[row, got], noise[row, best]) > 9)) and (gap == 0).mean() > 0.98
    for at in [p for p, w in enumerate(words) if (w == 0xffffff).any()] + list(range(0, rows, 97)):
        one = accept(logits[at:at + 1], [0], [[-1]], [at], [1.0], seeds.tolist())
        assert one == ([[0]], [1], [int(got[at])])


def test_the_largest_noise_wins_where_it_is_enough():
    """The token with the largest hash value has the noise -log(-log(1 - 2^-24)), in both operators: more than any other's."""
    V, lo, hi = 151936, 77, 0x1234567
    at = next(p for p in range(2000) if (noise_words(lo, hi, p + 1, V) == 0xffffff).any())
    token = int(np.flatnonzero(noise_words(lo, hi, at + 1, V) == 0xffffff)[0])
    u = np.minimum((noise_words(lo, hi, at + 1, V) + 0.5) / 2 ** 24, 1 - 2.0 ** -24)
    noise = -np.log(-np.log(u))
    second = np.sort(noise)[-2]
    seeds = i32([[lo, hi]])
    for temperature in (1.0, 0.5):
        for below in (-1.0, 1.0):                            # by so much the others' best falls short of the token, or is ahead of it
            logits = torch.zeros((1, V), device=DEV)
            logits[0, token] = (second - noise[token] - below) * temperature
            want = token if below < 0 else int(np.argsort(noise)[-2])
            assert sampler_choice(logits, i32([at]), torch.tensor([temperature], device=DEV), seeds) == [want]
            assert accept(logits, [0], [[-1]], [at], [temperature], [[lo, hi]]) == ([[0]], [1], [want])


def test_accept_takes_the_lowest_of_equal_children_ties_and_odd_logits():
    logits = torch.zeros((6, 500), device=DEV)
    logits[0, [7, 3]] = 5.0                              # a tie: the lower token
    logits[1] = -math.inf                                # nothing stands out: token 0
    logits[2, 4], logits[2, 9] = math.nan, 1.0           # an undefined logit is never chosen
    logits[3, 400] = math.inf
    parents = [[-1, 0, 0, 0, 1, 2]]
    tok = [1, 3, 3, 2, 0, 9]
    got = accept(logits, tok, parents, [5] * 6, [0.0], [[1, 2]])
    assert got == ([[0, 1, 4, -1, -1, -1]], [3], [0])
    assert accept(logits, [1, 2, 3, 3, 0, 9], parents, [5] * 6, [0.0], [[1, 2]]) == ([[0, 2, 5, -1, -1, -1]], [3], [0])
    assert accept(logits, [1, 2, 4, 3, 0, 9], parents, [5] * 6, [0.0], [[1, 2]]) == ([[0, 3, -1, -1, -1, -1]], [2], [400])
    assert accept(logits, [1, 3, 3, 3, 0, 0], [[-1, 3, 0, 0, 1, -7]], [5] * 6, [0.0], [[1, 2]])[0] == [[0, 2, -1, -1, -1, -1]]
    assert accept(logits, tok, parents, [-1] * 6, [0.9], [[1, 2]])[1:] == ([1], [0])     # padding rows


def test_accept_the_largest_tree():
    """A line of 1,024 nodes that is right to its end, one that goes wrong on the way, and 1,023 children of one node."""
    n = api.TREE_MAX_NODES
    logits = normal((3 * n, 40), seed=6)
    choice = logits.argmax(1).tolist()
    line = list(range(-1, n - 1))
    tok = [0] + choice[:n - 1] + [0] + choice[n:2 * n - 1] + [0] + [40] * (n - 2) + [choice[2 * n]]
    tok[n + 700] = (tok[n + 700] + 1) % 40
    parents = [line, line, [-1] + [0] * (n - 1)]
    args = logits, tok, parents, [5] * (3 * n), [0.0] * 3, [[1, 2]] * 3
    assert accept(*args) == plain_accept(choice, tok, parents, n)
    assert accept(*args)[1] == [n, 700, 2]


def test_accept_refusals():
    n, V, rows = 2, 50, 5
    good = dict(logits=torch.zeros((rows, V), device=DEV), tok=i32([0] * rows), parent=i32([0] * rows), cu_q=i32([0, 2, 5]), row_pos=i32([0] * rows),
                temperature=torch.zeros(n, device=DEV), seeds=i32(np.zeros((n, 2))), path=i32(np.zeros((n, 3))), n_path=i32([0, 0]), next_tok=i32([0, 0]))
    api.tree_accept(**good)
    for bad in (dict(logits=good["logits"].double()), dict(logits=good["logits"].T), dict(tok=i32([0])), dict(parent=good["parent"].long()),
                dict(seeds=i32([[0, 0]])), dict(temperature=good["temperature"][:1]), dict(path=i32(np.zeros((n, 1025)))), dict(path=i32(np.zeros((n, 0)))),
                dict(cu_q=i32([0, 5])), dict(n_path=i32([0])), dict(next_tok=good["next_tok"].cpu()), dict(logits=torch.zeros((rows, 0), device=DEV))):
        with pytest.raises(api.KernelError):
            api.tree_accept(**{**good, **bad})


# ------------------------------------------------------------------------------------------------ select
def select(logits, scores, ended, best):
    r = scores.shape[0]
    out = torch.full((r, best), 9.0, device=DEV), i32(np.full((r, best), 9)), i32(np.full((r, best), 9))
    api.beam_select(logits, scores, ended, *out)
    return tuple(t.cpu() for t in out)


def plain_select(logits, scores, ended, best):
    (r, b), z = scores.shape, logits.double().cpu().numpy()
    V = z.shape[1]
    score, beam, tok = np.full((r, best), -math.inf), np.zeros((r, best), np.int64), np.zeros((r, best), np.int64)
    for i in range(r):
        value = np.full((b, V), -math.inf)
        for j in range(b):
            x, own = z[i * b + j], float(scores[i, j])
            ok = np.isfinite(x)
            if not math.isfinite(own):
                continue
            if ended is not None and ended[i, j]:
                value[j, 0] = own
            elif ok.any():
                value[j, ok] = own + x[ok] - (x[ok].max() + np.log(np.exp(x[ok] - x[ok].max()).sum()))
        flat = value.reshape(-1)
        order = np.lexsort((np.arange(b * V), -flat))[:best]
        order = order[np.isfinite(flat[order])]
        score[i, :len(order)], beam[i, :len(order)], tok[i, :len(order)] = flat[order], order // V, order % V
    return score, beam, tok


def check_select(logits, scores, ended, best):
    got, want = select(logits, scores, ended, best), plain_select(logits, scores.cpu(), None if ended is None else ended.cpu(), best)
    assert np.array_equal(got[1].numpy(), want[1]) and np.array_equal(got[2].numpy(), want[2])
    # one rounding of the score to float32, and a sum of exponentials that is good to some 2^-22
    fine = np.isfinite(want[0])
    assert np.array_equal(np.isfinite(got[0].numpy()), fine)
    assert np.all(np.abs(got[0].numpy()[fine] - want[0][fine]) <= 2 ** -24 * np.abs(want[0][fine]) + 2 ** -22)


@pytest.mark.parametrize("vocab", [1, 2, 17, 300, 8192, 8195, 40000, 151936])
@pytest.mark.parametrize("requests,beams,best", [(1, 1, 1), (1, 4, 8), (3, 5, 10), (2, 16, 32), (1, 32, 64)])
def test_select(vocab, requests, beams, best):
    logits = normal((requests * beams, vocab), seed=vocab + best, scale=3.0)
    scores = -20 - 6 * torch.rand((requests, beams), generator=torch.Generator().manual_seed(best)).to(DEV)
    check_select(logits, scores, None, best)
    rs = np.random.RandomState(vocab)
    check_select(logits, scores, i32(rs.rand(requests, beams) < 0.4), best)


def test_select_ties_masks_and_beams_that_are_not_live():
    logits = torch.zeros((6, 9000), device=DEV)                      # equal everywhere: the lower beam, then the lower token
    scores = torch.tensor([[-1.0, -1.0, -1.0], [-2.0, -1.0, -1.0]], device=DEV)
    check_select(logits, scores, None, 10)
    logits[0, ::2] = -0.0
    check_select(logits, scores, None, 64)
    logits = normal((6, 9000), seed=1, scale=2.0)
    logits[:, 100:] = -math.inf                                      # masked tokens
    logits[1] = -math.inf                                            # a beam without a token
    logits[2, 5:50], logits[3, 7], logits[3, 60:80] = math.nan, math.inf, math.nan
    check_select(logits, scores, None, 64)
    scores[0, 0], scores[1, 1], scores[1, 2] = -math.inf, math.nan, math.inf
    check_select(logits, scores, None, 64)
    check_select(logits, scores, i32([[1, 1, 0], [0, 0, 1]]), 64)
    scores[:] = -math.inf
    check_select(logits, scores, None, 4)                            # nothing at all
    first = torch.tensor([[0.0] + [-math.inf] * 2] * 2, device=DEV)    # the first step of a search: one beam is live
    check_select(logits, first, None, 3)
    many = normal((6, 40), seed=2).repeat(1, 400) * 0.25             # every value 400 times
    check_select(many, torch.tensor([[-1.0, -1.0, -1.5], [-2.0, -1.0, -1.0]], device=DEV), None, 64)
    up = torch.arange(20000, device=DEV).float().repeat(6, 1) * 1e-3   # the best logits side by side, rising
    check_select(up, torch.tensor([[-1.0, -1.0, -1.5], [-2.0, -1.0, -1.0]], device=DEV), None, 64)


def exact_select(logits, scores, best):
    """``plain_select`` without ends, the maximum taken off before anything else is added, so that numbers of any size keep their differences."""
    (r, b), z = scores.shape, logits.double().cpu().numpy()
    V, out = z.shape[1], []
    for i in range(r):
        value = np.full((b, V), -math.inf)
        for j in range(b):
            x = z[i * b + j]
            ok = np.isfinite(x)
            if ok.any():
                d = x[ok] - x[ok].max()
                value[j, ok] = d + (float(scores[i, j]) - np.log(np.exp(d).sum()))
        flat = value.reshape(-1)
        order = np.lexsort((np.arange(b * V), -flat))[:best]
        out.append((flat[order], order // V, order % V))
    return [np.stack(x) for x in zip(*out)]


def check_exact_select(logits, scores, best):
    got, want = select(logits, scores, None, best), exact_select(logits, scores.cpu(), best)
    assert np.array_equal(got[1].numpy(), want[1]) and np.array_equal(got[2].numpy(), want[2])
    assert np.all(np.abs(got[0].numpy() - want[0]) <= 2 ** -24 * np.abs(want[0]) + 2 ** -22)      # as in check_select


LOWEST = torch.finfo(torch.float32).min


@pytest.mark.parametrize("masked", ["a piece", "the last piece", "all but a few", "a whole beam", "one beam's all but one"])
def test_select_with_the_lowest_number_as_a_mask(masked):
    """The lowest finite number is a logit like others: it weighs nothing beside ordinary ones, and a piece that holds nothing else costs a
    beam nothing."""
    logits = normal((6, 8192 * 2 + 500), seed=4, scale=3.0)
    scores = torch.tensor([[-3.0, -2.5, -4.0], [-20.0, -21.0, -20.5]], device=DEV)
    if masked == "a piece":
        logits[:, :8192 + 4] = LOWEST                       # (a row may begin up to three places into its first piece)
        logits[1, :], logits[1, 8300:8310] = LOWEST, torch.arange(10, device=DEV).float()
    elif masked == "the last piece":
        logits[:, 2 * 8192 - 4:] = LOWEST
    elif masked == "all but a few":
        keep = logits[:, [7, 9000, 16800]].clone()
        logits[:] = LOWEST
        logits[:, [7, 9000, 16800]] = keep
        return check_exact_select(logits, scores, 9)        # those of all three beams, and no more
    elif masked == "a whole beam":
        logits[1], logits[3] = LOWEST, LOWEST               # equal everywhere: its tokens are the best ones where its score is far above the others
        scores[0, 1] = 8.0
    else:
        logits[2] = LOWEST
        logits[2, 12000] = 1.5
    check_exact_select(logits, scores, 16)


def test_select_of_the_largest_numbers():
    logits = normal((4, 20000), seed=5, scale=3.0)
    logits[0, [5, 9000, 19000]] = torch.tensor([3.3e38, 3.4e38, -3.4e38], device=DEV)      # one token has all the weight
    logits[3] = logits[3] * 1e37
    check_exact_select(logits, torch.tensor([[-3.0, -2.0], [-1.0, -50.0]], device=DEV), 3)


@pytest.mark.parametrize("above", [0.0, 24.5, 315.25, 1000.125, -3000.5, 32768.0, 1048576.0])
def test_select_does_not_hang_on_a_number_added_to_all_logits(above):
    """Logits in steps of 1/8 (2^20 + 16 and that has its 24 bits), so the sum with ``above`` is exact and the log-probabilities are the same. Beams
    whose scores are one step of float32 apart take turns; their order is the one of the scores whichever of them is moved."""
    base = (normal((1, 30000), seed=6, scale=3.0) * 8).round() / 8
    base = base + torch.arange(30000, device=DEV).eq(777) * 4
    logits = base.repeat(8, 1)
    logits[1::4] += above
    logits[2::4] += above
    logits[3::4] -= above
    scores = torch.tensor([-20.0, -20.0 - 2 ** -19, -20.0, -20.0 + 2 ** -19, -9.5, -9.5 - 2 ** -20, -9.5 - 2 ** -19, -9.5], device=DEV).view(2, 4)
    got, same = select(logits, scores, None, 24), select(base.repeat(8, 1), scores, None, 24)
    assert torch.equal(got[1], same[1]) and torch.equal(got[2], same[2])
    assert torch.equal(got[0], same[0])
    check_exact_select(logits, scores, 24)


@pytest.mark.parametrize("vocab,beams,best", [(200003, 32, 64), (300000, 32, 57), (6500000, 1, 64), (2200000, 3, 64)])
def test_select_from_more_lists_than_a_block_has_room_for(vocab, beams, best):
    """The most beams and results over vocabularies from 196,606 on, or fewer beams over larger ones."""
    logits = normal((beams, vocab), seed=vocab, scale=3.0)
    scores = -20 - 2 * torch.rand((1, beams), generator=torch.Generator().manual_seed(best)).to(DEV)
    check_select(logits, scores, None, best)
    check_select(logits, scores, i32(np.arange(beams)[None] % 3 == 1), best)
    if beams == 32:
        two = torch.cat([logits, logits.flip(0)])               # two requests in a call
        both = select(two, torch.cat([scores, scores.flip(1)]), None, best)
        assert torch.equal(both[2][0], both[2][1]) and torch.equal(both[1][0], beams - 1 - both[1][1]) and torch.equal(both[0][0], both[0][1])
    logits = torch.zeros((beams, vocab), device=DEV)            # equal everywhere: the lower beam, then the lower token
    check_select(logits, torch.full((1, beams), -1.0, device=DEV), None, best)
    logits[:] = -math.inf
    logits[0, [5, vocab - 1, vocab // 2]], logits[beams - 1, 77] = 1.0, 2.0
    check_select(logits, torch.full((1, beams), -1.0, device=DEV), None, best)          # fewer candidates than asked for
    check_select(logits, torch.full((1, beams), -math.inf, device=DEV), None, best)


def test_select_from_memory_that_is_not_aligned_and_twice():
    base = normal((1 + 4 * 1000,), seed=3)
    logits = base[1:].view(4, 1000)
    scores = torch.zeros((2, 2), device=DEV)
    check_select(logits, scores, None, 5)
    a = select(logits, scores, None, 5)
    assert all(torch.equal(x, y) for x, y in zip(a, select(logits, scores, None, 5)))


def test_select_refusals():
    out = lambda r, k: dict(scores_out=torch.zeros((r, k), device=DEV), beam_out=i32(np.zeros((r, k))), tok_out=i32(np.zeros((r, k))))
    good = dict(logits=torch.zeros((4, 30), device=DEV), scores=torch.zeros((2, 2), device=DEV), ended=None, **out(2, 3))
    api.beam_select(**good)
    for bad in (dict(logits=good["logits"].double()), dict(logits=torch.zeros((5, 30), device=DEV)), dict(scores=torch.zeros((4, 1), device=DEV).half()),
                dict(ended=i32([[0, 0]])), out(2, 65), out(2, 0), dict(beam_out=i32(np.zeros((2, 2)))), dict(tok_out=good["tok_out"].long()),
                dict(logits=torch.zeros((66, 3), device=DEV), scores=torch.zeros((2, 33), device=DEV)), dict(logits=torch.zeros((4, 0), device=DEV)),
                dict(scores=torch.zeros((2, 2))), out(1, 3), dict(scores=good["scores_out"].view(-1)[1:5].view(2, 2)),
                dict(ended=good["tok_out"].view(-1)[:4].view(2, 2))):
        with pytest.raises(api.KernelError):
            api.beam_select(**{**good, **bad})


# ------------------------------------------------------------------------------------------------- moves
def paged(rs, lengths, width, extra=2):
    need = [(n + PAGE - 1) // PAGE for n in lengths]
    n_pages = sum(need) + extra
    order = rs.permutation(n_pages).tolist()
    table = -np.ones((len(need), width), np.int64)
    for s, k in enumerate(need):
        table[s, :k] = [order.pop() for _ in range(k)]
    return table, n_pages


def rows_of(store, table, s, place):
    return store[..., table[s, place // PAGE], :, place % PAGE, :]


def numbers(shape, dtype, seed):
    return torch.arange(int(np.prod(shape)), device=DEV).add(seed).remainder(251).view(shape).to(dtype)


SIZES = [(torch.bfloat16, 128), (torch.float32, 64), (torch.bfloat16, 20), (torch.float32, 3), (torch.bfloat16, 5)]


@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("lead", [(), (3,), (2, 2)])
def test_keep(dtype, size, lead):
    rs = np.random.RandomState(size)
    before, nodes = [0, 60, 129, 5, 300], [1, 64, 7, 0, 130]
    table, n_pages = paged(rs, [b + n for b, n in zip(before, nodes)], 8)
    table[4, 5] = -1                                       # a page that is not held: its rows neither come nor go
    store = numbers(lead + (n_pages, 3, PAGE, size), dtype, 1)
    path = np.full((5, 130), -1)
    count = [1, 9, 7, 0, 40]
    for s, c in enumerate(count):
        if c:
            path[s, :c] = np.concatenate([[0], np.sort(rs.choice(np.arange(1, max(2, nodes[s])), c - 1, replace=False))]) if c < nodes[s] else np.arange(c)
    want, old = store.clone(), store.clone()
    for s, b in enumerate(before):
        for k in range(count[s]):
            if table[s, (b + path[s, k]) // PAGE] >= 0 and table[s, (b + k) // PAGE] >= 0:
                rows_of(want, table, s, b + k).copy_(rows_of(old, table, s, b + path[s, k]))
    api.kv_keep(store, i32(table), i32(before), i32(path), i32(count))
    assert torch.equal(store, want)
    api.kv_keep(store, i32(table), i32(before), i32(path), i32([0] * 5))                # nothing moves
    assert torch.equal(store, want)


@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("requests,beams", [(1, 2), (3, 4), (2, 7), (2, 16), (1, 32)])
def test_reorder_pages(dtype, size, requests, beams):
    rs = np.random.RandomState(beams)
    first = rs.randint(0, 100, requests)
    last = first + np.maximum(0, rs.randint(-20, 150, requests))
    table, n_pages = paged(rs, np.repeat(np.maximum(last, 1), beams), 5)
    store = numbers((2, 2, n_pages, 2, PAGE, size), dtype, 3)
    parent = rs.randint(0, beams, (requests, beams))
    parent[0, :2] = [1, 0]                                 # two beams change places
    if requests > 1:
        parent[1, 1], parent[1, 0] = -1, beams             # no parents: left as they are
    want, old = store.clone(), store.clone()
    for r in range(requests):
        for b in range(beams):
            p = parent[r, b] if 0 <= parent[r, b] < beams else b
            for place in range(first[r], last[r]):
                rows_of(want, table, r * beams + b, place).copy_(rows_of(old, table, r * beams + p, place))
    api.kv_reorder(store, i32(table), i32(parent), i32(first), i32(last))
    assert torch.equal(store, want)


def test_reorder_leaves_out_pages_that_are_not_held():
    rs = np.random.RandomState(0)
    table, n_pages = paged(rs, [200, 200], 4)
    store = numbers((1, n_pages, 2, PAGE, 8), torch.float32, 0)
    want = store.clone()
    want[0, table[0, 1]] = store[0, table[1, 1]]
    table[0, 0], table[1, 2] = -1, n_pages
    api.kv_reorder(store, i32(table), i32([[1, 1]]), i32([-5]), i32([192]))
    assert torch.equal(store, want)
    want[0, table[0, 3], :, 250 - 3 * PAGE:] = store[0, table[1, 3], :, 250 - 3 * PAGE:]
    api.kv_reorder(store, i32(table), i32([[1, 1]]), i32([250]), i32([5000]))            # the table ends at place 256
    assert torch.equal(store, want)


@pytest.mark.parametrize("dtype,shape", [(torch.float32, (16, 128, 128)), (torch.bfloat16, (5,)), (torch.int32, (1,)), (torch.float32, (70, 3)),
                                         (torch.bfloat16, (3, 4, 8))])
@pytest.mark.parametrize("requests,beams", [(1, 1), (2, 3), (1, 8), (2, 12), (1, 32)])
def test_reorder_states(dtype, shape, requests, beams):
    rs = np.random.RandomState(beams)
    slots = requests * beams + 3
    store = numbers((2, slots) + shape, dtype, 5)
    slot = rs.permutation(slots)[:requests * beams]
    parent = rs.randint(0, beams, (requests, beams))
    want = store.clone()
    for r in range(requests):
        for b in range(beams):
            want[:, slot[r * beams + b]] = store[:, slot[r * beams + parent[r, b]]]
    api.state_reorder(store, i32(slot), i32(parent))
    assert torch.equal(store, want)
    odd = slot.copy()
    odd[0] = slots + 4                                      # a slot outside the store: neither read nor written
    parent[:] = 0
    api.state_reorder(store, i32(odd), i32(parent))
    for r in range(1, requests):
        for b in range(beams):
            want[:, slot[r * beams + b]] = want[:, slot[r * beams]]
    assert torch.equal(store, want)


def test_moves_refusals():
    store, table, par = torch.zeros((4, 1, PAGE, 8), device=DEV), i32([[0, 1], [2, 3]]), i32([[1, 0]])
    keep = dict(store=store, page_table=table, seq_pos0=i32([0, 0]), path=i32([[0, 1], [0, 1]]), n_path=i32([1, 1]))
    reorder = dict(store=store, page_table=table, parent=par, first=i32([0]), last=i32([9]))
    states = dict(store=torch.zeros((2, 3, 5), device=DEV), seq_slot=i32([0, 2]), parent=par)
    api.kv_keep(**keep), api.kv_reorder(**reorder), api.state_reorder(**states)
    odd = torch.zeros((4, 1, PAGE, 5), dtype=torch.uint8, device=DEV)
    for bad in (dict(store=store.cpu()), dict(store=store[:, :, :32]), dict(store=store.repeat(1, 2, 1, 1).transpose(0, 1)), dict(store=odd), dict(page_table=table.long()),
                dict(page_table=table[:1]), dict(seq_pos0=i32([0])), dict(n_path=i32([0])), dict(path=i32(np.zeros((2, 1025)))), dict(path=i32([0, 1]))):
        with pytest.raises(api.KernelError):
            api.kv_keep(**{**keep, **bad})
    for bad in (dict(store=store[0]), dict(page_table=table[:1]), dict(parent=i32([1, 0])), dict(parent=i32(np.zeros((1, 33)))), dict(first=i32([0, 0])),
                dict(last=i32([0]).float()), dict(store=odd)):
        with pytest.raises(api.KernelError):
            api.kv_reorder(**{**reorder, **bad})
    for bad in (dict(store=torch.zeros(4, device=DEV)), dict(store=torch.zeros((2, 3, 5), device=DEV).transpose(0, 2)), dict(seq_slot=i32([0])),
                dict(parent=par.long()), dict(store=torch.zeros((2, 3, 5), dtype=torch.uint8, device=DEV)), dict(parent=i32(np.zeros((1, 40))))):
        with pytest.raises(api.KernelError):
            api.state_reorder(**{**states, **bad})
