"""What branching generation decides on the host (no GPU): trees as arrays, drafts, and which beams may take whose place."""
import numpy as np
import pytest
import torch

from dryft_challenge_htn_2026_b200.cache import Cache, KVRequest, StateRequest
from dryft_challenge_htn_2026_b200.csrc import api, build
from dryft_challenge_htn_2026_b200.engine.batch import build_context, tree_arrays, tree_bucket, tree_shape
from dryft_challenge_htn_2026_b200.engine.branch import draft_tree

KV = KVRequest(2, 16, None, torch.float32)


def test_trees_as_arrays():
    depth, up, bits = tree_arrays([[-1, 0, 0, 1, 3], [-1], [-1] + list(range(39))])
    assert depth.tolist() == [0, 1, 1, 2, 3, 0] + list(range(40)) and up.tolist()[:6] == [-1, 0, 0, 1, 3, -1]
    assert bits.shape == (46, 2) and bits.view(np.uint32)[:6].tolist() == [[1, 0], [3, 0], [5, 0], [11, 0], [27, 0], [1, 0]]
    assert bits.view(np.uint32)[-1].tolist() == [0xffffffff, 0xff] and bits.view(np.uint32)[37].tolist() == [0xffffffff, 0]
    for bad in ([], [0], [-1, 1], [-1, -1], [-1, 0, 5]):
        with pytest.raises(ValueError):
            tree_arrays([[-1], bad])


def test_context_of_a_step_of_trees():
    cache = Cache([[KV]], max_tokens=64 * 4, max_slots=2, device="cpu")
    a, b = cache.begin(), cache.begin()
    cache.reserve(a, 70), cache.commit(a, 70)
    ctx = build_context(cache, [(a, [5, 6, 7], range(3)), (b, [8], range(1))], torch.device("cpu"), parents=[[-1, 0, 0], [-1]])
    assert ctx.row_pos.tolist() == [70, 71, 71, 0] and ctx.tree.place.tolist() == [70, 71, 72, 0] and not ctx.is_decode
    assert ctx.tree.parent.tolist() == [-1, 0, 0, -1] and ctx.tree.bits.tolist() == [[1], [3], [5], [1]] and ctx.tree.max_nodes == 3
    assert ctx.want_rows.tolist() == [0, 1, 2, 3] and ctx.seq_pos0.tolist() == [70, 0] and ctx.plans == {}
    one = build_context(cache, [(b, [8], [0])], torch.device("cpu"), parents=[[-1]])
    assert not one.is_decode and one.tree.max_nodes == 1
    assert build_context(cache, [(b, [8], [0])], torch.device("cpu")).tree is None


def test_context_of_a_padded_step_of_trees():
    assert [tree_bucket(n) for n in (1, 2, 3, 4, 5, 8, 9, 16, 17, 1024)] == [1, 2, 4, 4, 8, 8, 16, 16, 24, 1024]
    cache = Cache([[KV]], max_tokens=64 * 12, max_slots=2, device="cpu")
    a, b = cache.begin(), cache.begin()
    cache.reserve(a, 62), cache.commit(a, 62)
    ctx = build_context(cache, [(b, [8], range(1)), (a, [5, 6], range(2))], torch.device("cpu"), parents=[[-1], [-1, 0]], pad_to=8, max_nodes=40)
    assert ctx.row_pos.tolist() == [0, 62, 63] + [-1] * 5 and ctx.tree.place.tolist() == [0, 62, 63] + [-1] * 5
    assert ctx.tree.parent.tolist() == [-1, -1, 0] + [-2] * 5 and ctx.tree.bits.tolist() == [[1, 0], [1, 0], [3, 0]] + [[0, 0]] * 5
    assert ctx.cu_q.tolist() == [0, 1, 8] and ctx.row_seq.tolist() == [0] + [1] * 7 and ctx.tok.tolist() == [8, 5, 6] + [0] * 5
    assert ctx.want_rows.tolist() == list(range(8)) and ctx.n_tok == ctx.n_want == 8 and ctx.tree.max_nodes == 40
    assert ctx.tables[0].shape == (2, 8) and len(cache.groups[0].pages[a]) == 1          # padding asks for no pages
    few = build_context(cache, [(a, [5, 6], range(2))], torch.device("cpu"), parents=[[-1, 0]], pad_to=8)
    assert few.tree.max_nodes == 8


def test_drafts_as_trees():
    assert draft_tree(9, [1, 2, 3], 4) == ([9, 1, 2, 3], [-1, 0, 1, 2]) and draft_tree(9, [], 1) == ([9], [-1])
    assert draft_tree(9, ([1, 2, 3], [-1, -1, 0]), 8) == ([9, 1, 2, 3], [-1, 0, 0, 1])
    for draft in ([1, 2, 3, 4], ([1], []), ([1], [-1, 0])):
        with pytest.raises(ValueError):
            draft_tree(9, draft, 4)


def test_which_beams_may_take_whose_place(monkeypatch):
    cache = Cache([[KV, StateRequest((3,), torch.float32)]], max_tokens=64 * 8, max_slots=6, device="cpu")
    s = [cache.begin() for _ in range(6)]
    for x in s[:5]:
        cache.reserve(x, 10), cache.commit(x, 10)
    calls = []
    monkeypatch.setattr(api, "kv_reorder", lambda *a: calls.append(("kv", [t.tolist() for t in a[2:]])))
    monkeypatch.setattr(api, "state_reorder", lambda *a: calls.append(("state", [t.tolist() for t in a[1:]])))
    cache.reorder([s[:2], s[2:4]], [[0, 1], [0, 1]])                       # nobody moves
    assert not calls
    cache.reorder([s[:2], s[2:4]], [[1, 1], [0, 0]], [3, 10])
    assert calls == [("kv", [[[1, 1], [0, 0]], [3, 10], [10, 10]]), ("state", [s[:4], [[1, 1], [0, 0]]])]
    for slots, parents in (([s[:2]], [[0, 2]]), ([s[:2]], [[0, -1]]), ([[s[0], s[0]]], [[0, 0]]), ([[s[0], s[5]]], [[0, 0]]), ([s[:2]], [[0]]),
                           ([s[:2], s[2:5]], [[0, 0], [0, 0]]), ([s[:2]], [[0, 0], [0, 0]])):
        with pytest.raises(ValueError):
            cache.reorder(slots, parents)


def test_refusals_come_before_a_device_is_needed():
    """Tensors that are not on the GPU are refused by name, on a machine without one too."""
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(api.KernelError):
        api.attention_tree(torch.zeros(4, 64), torch.zeros(4, 64), torch.zeros(1, 1, 64, 64), torch.zeros(1, 1, 64, 64), i[:2], i[:1], i, i.view(4, 1),
                           i[:1].view(1, 1), 1, 1, 64, 0, 1.0, 4)
    with pytest.raises(api.KernelError):
        api.tree_accept(torch.zeros(4, 9), i, i, i[:2], i, torch.zeros(1), i[:2].view(1, 2), i.view(1, 4), i[:1], i[:1])
    with pytest.raises(api.KernelError):
        api.beam_select(torch.zeros(4, 9), torch.zeros(2, 2), None, torch.zeros(2, 2), i.view(2, 2), i.view(2, 2))
    with pytest.raises(api.KernelError):
        api.kv_keep(torch.zeros(1, 1, 64, 8), i[:1].view(1, 1), i[:1], i.view(1, 4), i[:1])
    with pytest.raises(api.KernelError):
        api.kv_reorder(torch.zeros(1, 1, 64, 8), i.view(4, 1), i.view(2, 2), i[:2], i[:2])
    with pytest.raises(api.KernelError):
        api.state_reorder(torch.zeros(1, 4, 8), i, i.view(2, 2))


@pytest.mark.parametrize("source,hd", [("attention_tree.cu", 64), ("attention_tree.cu", 16), ("attention_tree_tc.cu", 128)])
def test_addresses_that_are_not_aligned_are_refused_by_the_entry_points(source, hd):
    """Every address and row distance that the kernels take in 16 bytes; the answer comes before anything is asked of a device."""
    lib = build.load_lib(source, {"HD": hd})
    invalid, at = 1, 1 << 20                                               # cudaErrorInvalidValue; an address that nothing is read from

    def call(q=at, ldq=2 * hd, out=at, ldo=2 * hd, k=at, v=at, f32=0):
        body = (k, v, 4, at, at, at, at, 1, at, 64, 1, 2, 1, 0, 1.0, 4, at, at, 4)
        if source == "attention_tree_tc.cu":
            return api._entry(lib, "dk_attn_tree_tc", "pqpqq" + "ppippppipiiiiifippi" + "pp")(q, ldq, out, ldo, 4, *body, at, 0)
        return api._entry(lib, "dk_attn_tree", "ipqpq" + "ppippppipiiiiifippi" + "p")(f32, q, ldq, out, ldo, *body, 0)

    for f32 in (0, 1)[:1 if "tc" in source else 2]:
        for off in (2, 4, 8):
            for name in ("q", "out", "k", "v"):
                assert call(**{name: at + off}, f32=f32) == invalid, (name, off)
        for name in ("ldq", "ldo"):
            assert call(**{name: 2 * hd + 2}, f32=f32) == invalid, name


def test_shapes_of_captured_steps_of_trees_are_few():
    """Eight trees of 1 to 64 nodes, a thousand times: a handful of shapes, and the order of the trees makes no difference."""
    rs, shapes = np.random.RandomState(0), set()
    for _ in range(1000):
        nodes = rs.randint(1, 65, 8).tolist()
        rows, largest = tree_shape(nodes)
        assert sum(nodes) <= rows <= max(16, 1.5 * sum(nodes)) and max(nodes) <= largest <= min(rows, 2 * max(nodes))
        assert tree_shape(sorted(nodes)) == tree_shape(nodes[::-1]) == (rows, largest)
        shapes.add((rows, largest))
    assert len(shapes) <= 8
    assert [tree_shape([n]) for n in (1, 3, 17, 1024)] == [(1, 1), (4, 4), (24, 24), (1024, 1024)]
    assert tree_shape([1024] * 7) == (8192, 1024) and tree_shape([1, 1, 1]) == (4, 1)


def test_context_of_padding_beyond_the_largest_tree():
    """Padding that no tree has room for is not counted to the largest tree: its rows stand behind the last tree's real nodes."""
    cache = Cache([[KV]], max_tokens=64 * 12, max_slots=3, device="cpu")
    a, b = cache.begin(), cache.begin()
    ctx = build_context(cache, [(a, list(range(14)), range(14)), (b, [5, 6], range(2))], torch.device("cpu"),
                        parents=[list(range(-1, 13)), [-1, 0]], pad_to=24, max_nodes=16)
    assert ctx.tree.max_nodes == 16 and ctx.cu_q.tolist() == [0, 14, 24] and ctx.n_tok == 24
    assert ctx.row_pos.tolist()[14:] == [0, 1] + [-1] * 8 and ctx.tree.place.tolist()[14:] == [0, 1] + [-1] * 8 and ctx.tree.bits.shape == (24, 1)
    small = build_context(cache, [(a, list(range(14)), range(14)), (b, [5], range(1))], torch.device("cpu"),
                          parents=[list(range(-1, 13)), [-1]], pad_to=64, max_nodes=16)
    assert small.tree.max_nodes == 16 and small.cu_q.tolist() == [0, 14, 64]
