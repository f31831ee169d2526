"""The operators of branching generation, as calls and in their plain form.

A sequence branches where several continuations of it are looked at side by side: a tree of drafted tokens that the model
checks in one step, or the beams of a search. Four operators deal with that, beside the model's products and norms:

* "attention": every node of a tree of drafted tokens attends to its sequence's cached keys and to its own ancestors in the
  tree, whose keys lie in the cache behind them in the order of the nodes;
* "accept": from the nodes' logits, which path of the tree the model itself would have taken, and the token after it;
* "select": the best continuations of a request's beams, over all beams and the whole vocabulary;
* "move": the rows of the paged cache and the fixed-size states follow the choice. "keep" closes up the accepted nodes' rows
  behind a sequence; "beams" gives every beam its parent's rows or states.

A case names the operator and its sizes. Lengths lie between the two that a case gives, the first sequence at the upper one;
they follow from the case alone, everything else (values, pages, trees, parents) from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 64          # tokens a cache page
DEVICE = "cuda"
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEVICE)


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the smallest call: one sequence, the pending token and one drafted behind it, at the layer sizes of bench.py
        dict(name="tree of 2, short", op="attention", type="bfloat16", seqs=1, nodes_lo=2, nodes_hi=2, context_lo=130, context_hi=130,
             heads=32, kv_heads=8, dim=128, window=0),
        # a batch of eight with full trees at the lengths that decoding is benchmarked at
        dict(name="trees of 64, batch 8", op="attention", type="bfloat16", seqs=8, nodes_lo=40, nodes_hi=64, context_lo=1400,
             context_hi=4096, heads=32, kv_heads=8, dim=128, window=0),
        # a long context, few sequences
        dict(name="trees of 24, 32k tokens", op="attention", type="bfloat16", seqs=2, nodes_lo=13, nodes_hi=24, context_lo=30011,
             context_hi=32768, heads=32, kv_heads=8, dim=128, window=0),
        # the float32 path of a model, with a window and trees of unequal size
        dict(name="trees of 16, float32", op="attention", type="float32", seqs=4, nodes_lo=3, nodes_hi=16, context_lo=300,
             context_hi=1500, heads=32, kv_heads=8, dim=128, window=1024),
        # the tokens of a batch's trees, greedy
        dict(name="accept, batch 8 of 64", op="accept", seqs=8, nodes_lo=40, nodes_hi=64, vocab=151936, temperature=0.0),
        # one sequence with a short draft, sampled
        dict(name="accept, 5 sampled", op="accept", seqs=1, nodes_lo=5, nodes_hi=5, vocab=151936, temperature=0.7),
        # one request, four beams, twice as many candidates as beams
        dict(name="select, 1 of 4 beams", op="select", requests=1, beams=4, best=8, vocab=151936, ended=0),
        # a batch of searches, some of their beams at their end; a vocabulary that is no multiple of anything
        dict(name="select, 16 of 8 beams", op="select", requests=16, beams=8, best=16, vocab=100003, ended=1),
        # the cache of a whole model after a step of eight trees
        dict(name="keep, batch 8 of 64", op="keep", type="bfloat16", seqs=8, nodes_lo=40, nodes_hi=64, context_lo=70, context_hi=300,
             layers=36, kv_heads=8, dim=128),
        # a few layers in float32, one sequence
        dict(name="keep, 1 of 7", op="keep", type="float32", seqs=1, nodes_lo=7, nodes_hi=7, context_lo=121, context_hi=121, layers=4,
             kv_heads=2, dim=64),
        # what four searches have written since their prompts, in every layer
        dict(name="beams, pages", op="beams", type="bfloat16", requests=4, beams=4, shared_lo=33, shared_hi=200, written_lo=20,
             written_hi=120, layers=36, kv_heads=8, dim=128),
        # the recurrent states of two searches: 16 heads of 128 x 128 numbers a layer
        dict(name="beams, states", op="states", type="float32", requests=2, beams=8, layers=4, numbers=16 * 128 * 128),
    ]


def _span(rng, lo, hi):
    """A whole number, even over the logarithm where the range is wide."""
    if hi <= 10 * lo:
        return rng.randint(lo, hi)
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "accept", "accept", "select", "select", "keep", "beams", "states"])
    if op == "attention":
        kind = rng.choice(["bfloat16", "bfloat16", "float32"])
        dim = rng.choice([128, 128, 64, 64, 48])
        kv = rng.choice([1, 2, 3, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 8])
        hi = _span(rng, 1, 64 if kind == "bfloat16" else 16)
        far = _span(rng, 1, 32768 if kind == "bfloat16" else 1500)
        most = 8 * 4096 if kind == "bfloat16" else 4 * 1500
        seqs = min(_span(rng, 1, 16), max(1, most // far))
        return dict(op=op, type=kind, seqs=seqs, nodes_lo=rng.randint(1, hi), nodes_hi=hi, context_lo=rng.randint(max(1, far // 3), far),
                    context_hi=far, heads=heads, kv_heads=kv, dim=dim, window=rng.choice([0, 0, 0, rng.randint(17, 2000)]))
    if op == "accept":
        vocab, hi = _span(rng, 300, 151936), _span(rng, 1, 64)
        return dict(op=op, seqs=_span(rng, 1, 8), nodes_lo=rng.randint(1, hi), nodes_hi=hi, vocab=vocab,
                    temperature=rng.choice([0.0, 0.0, rng.choice([0.3, 0.7, 1.0, 1.3])]))
    if op == "select":
        beams = rng.randint(1, 16)
        return dict(op=op, requests=max(1, _span(rng, 1, 16) // (1 if beams <= 8 else 2)), beams=beams, best=rng.choice([beams, 2 * beams]),
                    vocab=_span(rng, 300, 151936), ended=rng.randint(0, 1))
    if op == "keep":
        hi, far = _span(rng, 2, 64), _span(rng, 1, 300)
        return dict(op=op, type=rng.choice(["bfloat16", "float32"]), seqs=rng.randint(1, 8), nodes_lo=rng.randint(1, hi), nodes_hi=hi,
                    context_lo=rng.randint(1, far), context_hi=far, layers=rng.randint(1, 16), kv_heads=rng.randint(1, 8),
                    dim=rng.choice([48, 64, 128]))
    if op == "beams":
        far, new = _span(rng, 1, 200), _span(rng, 1, 120)
        return dict(op=op, type=rng.choice(["bfloat16", "float32"]), requests=rng.randint(1, 4), beams=rng.randint(2, 8),
                    shared_lo=rng.randint(1, far), shared_hi=far, written_lo=rng.randint(1, new), written_hi=new,
                    layers=rng.randint(1, 16), kv_heads=rng.randint(1, 4), dim=rng.choice([48, 64, 128]))
    return dict(op=op, type=rng.choice(["bfloat16", "float32"]), requests=rng.randint(1, 4), beams=rng.randint(2, 8), layers=rng.randint(1, 4),
                numbers=_span(rng, 40, 16 * 128 * 128))


def _lengths(case, name, count):
    """``count`` whole numbers between the case's two, the first at the upper end; they follow from the case alone."""
    lo, hi = case[name + "_lo"], case[name + "_hi"]
    rng = random.Random("%s %d %d %d" % (name, lo, hi, count))
    return [hi] + [rng.randint(lo, hi) for _ in range(count - 1)]


# ---------------------------------------------------------------------------------------------- inputs
def _tree(rng, n):
    """Parents of n nodes, -1 for the root: a draft branches most near its root."""
    return [-1] + [rng.randint(max(0, i - 1 - i // 2), i - 1) if rng.random() < 0.7 else rng.randint(0, i - 1) for i in range(1, n)]


def _trees(rng, lens, width):
    """(parents, depths, bits of the nodes on the way from the root to each node itself) of the trees' nodes in one run."""
    parents, depths = np.full(sum(lens), -1, np.int64), np.zeros(sum(lens), np.int64)
    bits, row = np.zeros((sum(lens), width), np.uint32), 0
    for n in lens:
        for i, p in enumerate(_tree(rng, n)):
            if p >= 0:
                parents[row + i], depths[row + i] = p, depths[row + p] + 1
                bits[row + i] = bits[row + p]
            bits[row + i, i // 32] |= np.uint32(1 << (i % 32))
        row += n
    return parents, depths, bits.view(np.int32)


def _pages(rng, lengths):
    """A table of page ids for sequences of these lengths, in mixed order. Page 0 belongs to none."""
    need = [(n + PAGE - 1) // PAGE for n in lengths]
    order = list(range(1, 1 + sum(need)))
    rng.shuffle(order)
    table = np.full((len(need), max(need)), -1, np.int64)
    for s, n in enumerate(need):
        table[s, :n] = [order.pop() for _ in range(n)]
    return table, 1 + sum(need)


def _normal(gen, shape, kind):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(TYPES[kind])


def prepare(case, seed):
    rng, gen = random.Random(seed), torch.Generator(device=DEVICE).manual_seed(seed)
    s = dict(case)
    op = case["op"]
    if op in ("attention", "accept", "keep"):
        lens = _lengths(case, "nodes", case["seqs"])
        s["max_nodes"] = max(lens)
        parents, depths, bits = _trees(rng, lens, (max(lens) + 31) // 32)
        cu = np.concatenate([[0], np.cumsum(lens)])
        before = _lengths(case, "context", case["seqs"]) if op != "accept" else [rng.randint(1, 5000) for _ in lens]
        s.update(parent=_i32(parents), tree=_i32(bits), cu_q=_i32(cu), seq_pos0=_i32(before),
                 row_pos=_i32(np.repeat(before, lens) + depths))
    if op in ("attention", "keep"):
        table, pages = _pages(rng, [b + n for b, n in zip(before, lens)])
        s["page_table"] = _i32(table)
        shape = (pages, case["kv_heads"], PAGE, case["dim"])
    if op == "attention":
        s["q"] = _normal(gen, (sum(lens), case["heads"] * case["dim"]), case["type"])
        s["k_store"], s["v_store"] = _normal(gen, shape, case["type"]), _normal(gen, shape, case["type"])
        s["scale"] = case["dim"] ** -0.5
    elif op == "accept":
        # logits as a model's: a few tokens stand out. Most drafted tokens are the ones their parent's logits favour.
        s["logits"] = torch.randn((sum(lens), case["vocab"]), generator=gen, device=DEVICE) * 2
        tok, row = np.zeros(sum(lens), np.int64), 0
        liked = [rng.randrange(case["vocab"]) for _ in range(sum(lens))]
        for n in lens:
            for i in range(n):
                p = int(parents[row + i])
                tok[row + i] = liked[row + p] if p >= 0 and rng.random() < 0.6 else rng.randrange(case["vocab"])
            row += n
        s["logits"][torch.arange(sum(lens), device=DEVICE), _i32(liked).long()] += 14
        s["tok"] = _i32(tok)
        s["temperatures"] = torch.full((len(lens),), case["temperature"], device=DEVICE)
        s["seeds"] = _i32([[rng.randint(-2 ** 31, 2 ** 31 - 1), rng.randint(-2 ** 31, 2 ** 31 - 1)] for _ in lens])
    elif op == "select":
        r, b = case["requests"], case["beams"]
        s["logits"] = torch.randn((r * b, case["vocab"]), generator=gen, device=DEVICE) * 3
        s["scores"] = -20 - 6 * torch.rand((r, b), generator=gen, device=DEVICE)
        s["ended"] = _i32([[int(case["ended"] and rng.random() < 0.25) for _ in range(b)] for _ in range(r)])
    elif op == "keep":
        s["store"] = _normal(gen, (case["layers"], 2) + shape, case["type"])
        path, count, row = np.full((len(lens), max(lens)), -1, np.int64), [], 0
        for i, n in enumerate(lens):    # the way from the root to some node
            k, way = rng.randrange(n), []
            while k >= 0:
                way.append(k)
                k = int(parents[row + k])
            path[i, :len(way)] = way[::-1]
            count.append(len(way))
            row += n
        s["path"], s["n_path"] = _i32(path), _i32(count)
    elif op == "beams":
        r, b = case["requests"], case["beams"]
        first, new = _lengths(case, "shared", r), _lengths(case, "written", r)
        last = [f + n for f, n in zip(first, new)]
        table, pages = _pages(rng, np.repeat(last, b).tolist())
        s["store"] = _normal(gen, (case["layers"], 2, pages, case["kv_heads"], PAGE, case["dim"]), case["type"])
        s.update(page_table=_i32(table), first=_i32(first), last=_i32(last), most=max(new),
                 beam=_i32([[rng.randrange(b) for _ in range(b)] for _ in range(r)]))
    else:
        r, b = case["requests"], case["beams"]
        slots = rng.sample(range(r * b + 3), r * b)
        s["store"] = _normal(gen, (case["layers"], r * b + 3, case["numbers"]), case["type"])
        s.update(seq_slot=_i32(slots), beam=_i32([[rng.randrange(b) for _ in range(b)] for _ in range(r)]))
    return s


# --------------------------------------------------------------------------------------------- plain forms
def _visible(s):
    """[sequences, nodes, keys]: which places of its table's pages a node sees, and the sequences' node rows (clamped)."""
    cu, pos0, table = s["cu_q"].long(), s["seq_pos0"].long(), s["page_table"].long()
    node = torch.arange(s["max_nodes"], device=cu.device)
    lens = cu[1:] - cu[:-1]
    rows = (cu[:-1, None] + node).clamp(max=s["tree"].shape[0] - 1)
    key = torch.arange(table.shape[1] * PAGE, device=cu.device)
    j = key[None, :] - pos0[:, None]                                                       # the node that lies at a key's place
    inside = j.clamp(0, s["max_nodes"] - 1)
    words = torch.gather(s["tree"].long()[rows], 2, (inside // 32)[:, None, :].expand(-1, len(node), -1))
    seen = (j < 0)[:, None, :] | (((words >> (inside % 32)[:, None, :]) & 1 > 0) & ((j >= 0) & (j < lens[:, None]))[:, None, :])
    if s["window"] > 0:
        q_pos = s["row_pos"].long()[rows]
        k_pos = torch.where(j < 0, key[None, :], torch.gather(q_pos, 1, inside))
        seen &= q_pos[:, :, None] - k_pos[:, None, :] < s["window"]
    return seen, rows, lens


def _attention(s):
    nkv, dim = s["kv_heads"], s["dim"]
    group = s["heads"] // nkv
    seen, rows, lens = _visible(s)
    seqs, nodes, keys = seen.shape
    table = s["page_table"].long().clamp(min=0)
    k = s["k_store"][table].float().transpose(1, 2).reshape(seqs, nkv, keys, dim)
    v = s["v_store"][table].float().transpose(1, 2).reshape(seqs, nkv, keys, dim)
    q = s["q"][rows].float().view(seqs, nodes, nkv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, nkv, group * nodes, dim)
    score = (q @ k.transpose(2, 3)).view(seqs, nkv, group, nodes, keys) * s["scale"]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = weight.sum(-1, keepdim=True)
    o = (weight.view(seqs, nkv, group * nodes, keys) @ v).view(seqs, nkv, group, nodes, dim)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(seqs * nodes, -1)
    here = (torch.arange(nodes, device=lens.device)[None, :] < lens[:, None]).reshape(-1, 1)
    out = torch.zeros((s["q"].shape[0] + 1, o.shape[1]), device=o.device)                  # rows that are not there go to the last one
    out[torch.where(here[:, 0], rows.reshape(-1), torch.full_like(rows.reshape(-1), s["q"].shape[0]))] = o
    return out[:-1].to(s["q"].dtype)


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * (0x846CA68B & 0xFFFF) + ((x * (0x846CA68B >> 16) & 0xFFFF) << 16)) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _noise(seeds, pos, vocab):
    """The sampler's noise -log(-log(u)) of rows with these seeds [n, 2] at these positions, in 32 bits."""
    seeds = seeds.long() & 0xFFFFFFFF
    x = _mix(torch.arange(vocab, device=pos.device)[None, :] ^ 0x9E3779B9)
    x = _mix((x + ((pos * 0x85EBCA6B) & 0xFFFFFFFF)[:, None] + seeds[:, :1]) & 0xFFFFFFFF)
    x = _mix(x ^ seeds[:, 1:])
    u = ((x >> 8).float() + 0.5) * (1.0 / 16777216.0)
    return -torch.log(-torch.log(u))


def _sequence_of(s):
    rows = torch.arange(s["tok"].shape[0], device=DEVICE)
    return torch.searchsorted(s["cu_q"].long(), rows, right=True) - 1


def _accept(s):
    cu, tok, parent, seq = s["cu_q"].long(), s["tok"].long(), s["parent"].long(), _sequence_of(s)
    score = s["logits"]
    if s["temperature"] > 0:
        t = s["temperatures"][seq][:, None]
        score = score * (1.0 / t) + _noise(s["seeds"][seq], s["row_pos"].long() + 1, score.shape[1])
    choice = torch.nan_to_num(score, nan=-math.inf, posinf=math.inf, neginf=-math.inf).argmax(-1)
    # a node is accepted where every step from the root down to it takes the token that the parent's logits chose
    first = cu[:-1][seq]
    up = torch.where(parent >= 0, first + parent, first)
    twin = (seq[:, None] == seq[None, :]) & (parent[:, None] == parent[None, :]) & (tok[:, None] == tok[None, :])
    twin &= torch.ones_like(twin).tril(-1)
    step = (parent < 0) | ((choice[up] == tok) & ~twin.any(1))
    node = torch.arange(s["max_nodes"], device=cu.device)
    way = (s["tree"].long()[:, node // 32] >> (node % 32)) & 1 > 0                          # [rows, nodes]
    good = step[(first[:, None] + node).clamp(max=len(tok) - 1)]
    accepted = ~(way & ~good).any(1)
    lens = cu[1:] - cu[:-1]
    rows = (cu[:-1, None] + node).clamp(max=len(tok) - 1)
    there = accepted[rows] & (node[None, :] < lens[:, None])
    path = torch.where(there, node[None, :], torch.full_like(rows, s["max_nodes"])).sort(1).values
    count = there.sum(1)
    last = torch.gather(path, 1, count[:, None] - 1)[:, 0]
    path = torch.where(path < s["max_nodes"], path, torch.full_like(path, -1))
    return path.int(), count.int(), choice[cu[:-1] + last].int()


def _select(s):
    """Ranked in 64 bits, whose rounding decides no rank; equal values by the lower beam, then the lower token."""
    r, b = s["scores"].shape
    z = s["logits"].double()
    vocab = z.shape[1]
    top = z.amax(1, keepdim=True)
    total = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    value = s["scores"].double()[:, :, None] + (z - total).view(r, b, vocab)
    still = torch.full_like(value, -math.inf)
    still[:, :, 0] = s["scores"].double()
    value = torch.where(s["ended"][:, :, None] > 0, still, value).view(r, b * vocab)
    some = torch.topk(value, min(s["best"] + 32, b * vocab), dim=1)
    at = some.indices.sort(1).values
    order = torch.gather(value, 1, at).sort(dim=1, descending=True, stable=True)
    at = torch.gather(at, 1, order.indices[:, :s["best"]])
    return order.values[:, :s["best"]].float(), (at // vocab).int(), (at % vocab).int()


def _keep(s):
    store, path = s["store"], s["path"].long()
    k = torch.arange(path.shape[1], device=path.device)[None, :]
    on = k < s["n_path"].long()[:, None]
    place = lambda rows: s["seq_pos0"].long()[:, None] + torch.where(on, rows, torch.zeros_like(rows))    # off: the root onto itself
    src, dst = place(path), place(k.expand_as(path))
    page = lambda p: torch.gather(s["page_table"].long(), 1, p // PAGE)
    store[:, :, page(dst), :, dst % PAGE] = store[:, :, page(src), :, src % PAGE]
    return store


def _beams(s):
    store, beam = s["store"], s["beam"].long()
    r, b = beam.shape
    pos = s["first"].long()[:, None] + torch.arange(s["most"], device=beam.device)[None, :]
    on = (pos < s["last"].long()[:, None]).repeat_interleave(b, 0)
    pos = pos.repeat_interleave(b, 0)
    parent = (beam + b * torch.arange(r, device=beam.device)[:, None]).view(-1)
    table = s["page_table"].long()
    slot = torch.where(on, pos // PAGE, torch.zeros_like(pos))
    spare = torch.zeros_like(pos)                                                          # page 0, onto itself, where a row is off
    to = torch.where(on, torch.gather(table, 1, slot), spare)
    of = torch.where(on, torch.gather(table[parent], 1, slot), spare)
    store[:, :, to, :, pos % PAGE] = store[:, :, of, :, pos % PAGE]
    return store


def _states(s):
    r, b = s["beam"].shape
    slot = s["seq_slot"].long()
    parent = (s["beam"].long() + b * torch.arange(r, device=slot.device)[:, None]).view(-1)
    s["store"][:, slot] = s["store"][:, slot[parent]]
    return s["store"]


_PLAIN = dict(attention=_attention, accept=_accept, select=_select, keep=_keep, beams=_beams, states=_states)


# ------------------------------------------------------------------------------------------- the library's calls
def _call(s):
    from dryft_challenge_htn_2026_b200.csrc import api

    op = s["op"]
    if op == "attention":
        out = torch.empty_like(s["q"])
        api.attention_tree(s["q"], out, s["k_store"], s["v_store"], s["cu_q"], s["seq_pos0"], s["row_pos"], s["tree"], s["page_table"],
                           s["heads"], s["kv_heads"], s["dim"], s["window"], s["scale"], s["max_nodes"])
        return out
    if op == "accept":
        n = s["seq_pos0"].shape[0]
        path = torch.empty((n, s["max_nodes"]), dtype=torch.int32, device=DEVICE)
        count, token = torch.empty(n, dtype=torch.int32, device=DEVICE), torch.empty(n, dtype=torch.int32, device=DEVICE)
        api.tree_accept(s["logits"], s["tok"], s["parent"], s["cu_q"], s["row_pos"], s["temperatures"], s["seeds"], path, count, token)
        return path, count, token
    if op == "select":
        shape = (s["requests"], s["best"])
        score = torch.empty(shape, dtype=torch.float32, device=DEVICE)
        beam, token = torch.empty(shape, dtype=torch.int32, device=DEVICE), torch.empty(shape, dtype=torch.int32, device=DEVICE)
        api.beam_select(s["logits"], s["scores"], s["ended"], score, beam, token)
        return score, beam, token
    if op == "keep":
        api.kv_keep(s["store"], s["page_table"], s["seq_pos0"], s["path"], s["n_path"])
    elif op == "beams":
        api.kv_reorder(s["store"], s["page_table"], s["beam"], s["first"], s["last"])
    else:
        api.state_reorder(s["store"], s["seq_slot"], s["beam"])
    return s["store"]


def run(state):
    return _call(state) if own else _PLAIN[state["op"]](state)


# ------------------------------------------------------------------------------------------------- work
def _moved(b):
    """Beams of b whose parent, drawn evenly, is another one."""
    return b - 1


def work(case):
    op = case["op"]
    size = 2 if case.get("type") == "bfloat16" else 4
    if op == "attention":
        nodes, before = _lengths(case, "nodes", case["seqs"]), _lengths(case, "context", case["seqs"])
        if case["window"]:
            before = [min(b, case["window"] - 1) for b in before]
        row = size * case["dim"]
        keys = sum(b + n for b, n in zip(before, nodes))
        seen = sum(n * (b + max(1, n // 4)) for b, n in zip(before, nodes))
        return dict(bytes=2 * keys * case["kv_heads"] * row + 2 * sum(nodes) * case["heads"] * row, flops=4 * seen * case["heads"] * case["dim"])
    if op == "accept":
        n = sum(_lengths(case, "nodes", case["seqs"])) * case["vocab"]
        return dict(bytes=4 * n, flops=n)
    if op == "select":
        n = case["requests"] * case["beams"] * case["vocab"]
        return dict(bytes=4 * n, flops=2 * n)
    if op == "keep":        # a way down a tree of n nodes is some 0.3 n long on average here, all but its root moved
        rows = sum(max(1, int(0.3 * n)) for n in _lengths(case, "nodes", case["seqs"]))
        return dict(bytes=2 * rows * case["layers"] * 2 * case["kv_heads"] * case["dim"] * size, flops=0)
    if op == "beams":
        rows = sum(_lengths(case, "written", case["requests"])) * _moved(case["beams"])
        return dict(bytes=2 * rows * case["layers"] * 2 * case["kv_heads"] * case["dim"] * size, flops=0)
    return dict(bytes=2 * case["requests"] * _moved(case["beams"]) * case["layers"] * case["numbers"] * size, flops=0)


# ------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_attention(s):
    cu, before, table = s["cu_q"].tolist(), s["seq_pos0"].tolist(), s["page_table"].tolist()
    group, out = s["heads"] // s["kv_heads"], torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    words = s["tree"].cpu().numpy().view(np.uint32)
    pos = s["row_pos"].tolist()
    for i, p0 in enumerate(before):
        n = cu[i + 1] - cu[i]
        pages = torch.tensor(table[i][:(p0 + n + PAGE - 1) // PAGE], device=DEVICE)
        k = s["k_store"][pages].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :p0 + n]
        v = s["v_store"][pages].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :p0 + n]
        place = list(range(p0)) + pos[cu[i]:cu[i + 1]]
        mask = np.ones((n, p0 + n), bool)
        for a in range(n):
            mask[a, p0:] = [bool(words[cu[i] + a, c // 32] >> np.uint32(c % 32) & np.uint32(1)) for c in range(n)]
            if s["window"]:
                mask[a] &= pos[cu[i] + a] - np.array(place) < s["window"]
        mask = torch.from_numpy(mask).to(DEVICE)
        for h in range(s["heads"]):
            q = s["q"][cu[i]:cu[i + 1], h * s["dim"]:(h + 1) * s["dim"]].double()
            w = torch.softmax((q @ k[h // group].T * s["scale"]).masked_fill(~mask, -math.inf), 1)
            out[cu[i]:cu[i + 1], h * s["dim"]:(h + 1) * s["dim"]] = w @ v[h // group]
    return out


def exact(case, seed):
    if case["op"] == "accept":      # whole numbers only
        return None
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "select":
        r, b, scores, done = case["requests"], case["beams"], s["scores"].tolist(), s["ended"].tolist()
        out = np.zeros((r, case["best"]))
        for i in range(r):
            pool = []
            for j in range(b):
                if done[i][j]:
                    pool.append(np.array([scores[i][j]]))
                    continue
                z = s["logits"][i * b + j].cpu().numpy().astype(np.float64)
                z = scores[i][j] + z - np.logaddexp.reduce(z)
                pool.append(np.sort(z)[::-1][:case["best"]])
            out[i] = np.sort(np.concatenate(pool))[::-1][:case["best"]]
        return out, None, None
    store = s["store"].cpu()
    old = store.clone()
    if case["op"] == "keep":
        table, path = s["page_table"].tolist(), s["path"].tolist()
        for i, p0 in enumerate(s["seq_pos0"].tolist()):
            for k in range(int(s["n_path"][i])):
                a, c = p0 + path[i][k], p0 + k
                store[:, :, table[i][c // PAGE], :, c % PAGE] = old[:, :, table[i][a // PAGE], :, a % PAGE]
    elif case["op"] == "beams":
        table, beam = s["page_table"].tolist(), s["beam"].tolist()
        for i, (first, last) in enumerate(zip(s["first"].tolist(), s["last"].tolist())):
            for j, p in enumerate(beam[i]):
                to, of = table[i * case["beams"] + j], table[i * case["beams"] + p]
                for c in range(first, last):
                    store[:, :, to[c // PAGE], :, c % PAGE] = old[:, :, of[c // PAGE], :, c % PAGE]
    else:
        slot, beam = s["seq_slot"].tolist(), s["beam"].tolist()
        for i in range(case["requests"]):
            for j, p in enumerate(beam[i]):
                store[:, slot[i * case["beams"] + j]] = old[:, slot[i * case["beams"] + p]]
    return store.to(DEVICE, torch.float64)
