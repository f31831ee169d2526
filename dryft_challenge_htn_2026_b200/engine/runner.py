"""The step function: a model, its cache, and ``step`` over a batch of sequences.

``step`` runs exactly the tokens it is given as one batch, from what earlier steps left in the
cache, and returns the logits at the wanted places. Sequences of a step either all start (their
prompts, of any lengths, in one ragged pass) or each continue with the tokens given; nothing is
padded to a common length, and a sequence's result does not depend on the others in the batch.
"""
from collections import OrderedDict

import torch

from ..cache import Cache
from ..csrc import api
from ..sampling import seed_words
from .batch import build_context, tree_shape, tree_table_widths

GRAPH_MAX_TOKENS = 8192     # steps of more tokens are launched plainly (the reference's bound: engine/engine.py:30)
GRAPH_KEEP = 12             # captured step shapes kept, of steps and of steps of trees each, least recently used dropped first
TREE_GRAPH_BYTES = 1 << 30  # logits that the captured steps of trees may hold together (one of 512 nodes over 151,936 tokens: 311 MB)


class _StepGraph:
    def __init__(self):
        self.static = {}        # the step context's device buffer (engine.batch._pack)
        self.graph = None
        self.logits = None


class Runner:
    def __init__(self, model, max_tokens, max_slots=1024):
        """``max_tokens``: tokens all live sequences may hold together, each sequence rounded up
        to whole pages of 64."""
        self.model = model
        self.device = model.rt.device
        self.cache = Cache(model.entry_requests(), max_tokens, max_slots, self.device)
        self._scratch = {}
        self.vocab_size = model.spec.vocab_size
        self._seen = OrderedDict()      # step shapes run so far -> times
        self._graphs = OrderedDict()    # step shape -> _StepGraph
        self._generation = model.generation

    def begin(self):
        """A slot for a new sequence (its length starts at 0)."""
        return self.cache.begin()

    def end(self, slot):
        """Gives the sequence's pages and slot back."""
        self.cache.end(slot)

    def length(self, slot):
        return self.cache.length[slot]

    def _check(self, entries):
        for slot, tokens, _ in entries:
            if not self.cache.slots.is_live(slot):
                raise ValueError(f"slot {slot} is not live")
            if len(tokens) and (min(tokens) < 0 or max(tokens) >= self.vocab_size):
                raise ValueError(f"token id outside [0, {self.vocab_size})")
        if len({e[0] for e in entries}) != len(entries):
            raise ValueError("a slot appears twice in one step")

    def context(self, entries, pad_to=None, static=None, parents=None, max_nodes=0):
        self._check(entries)
        ctx = build_context(self.cache, entries, self.device, self._scratch, pad_to, self.model.step_plans, static, parents,
                            max_nodes)
        self.model.prepare(ctx.max_position + 1)     # tables grow here, never inside a step
        return ctx

    def _shape(self, entries):
        """What fixes every launch of a step: the new and the cached length of each sequence, how
        many places are wanted, and how wide the page tables are. Steps of equal shape differ in
        data only (token ids, slots, page ids, which places)."""
        cache = self.cache
        for slot, tokens, _ in entries:
            cache.reserve(slot, len(tokens))
        return (tuple(len(t) for _, t, _ in entries), tuple(cache.length[s] for s, _, _ in entries),
                sum(len(w) for _, _, w in entries),
                tuple(max(len(r) for r in cache.page_rows(g, [s for s, _, _ in entries])) for g in range(len(cache.groups))))

    @torch.inference_mode()
    def step(self, entries, tap=None, with_context=False, graph=False):
        """entries: list of (slot, tokens, want). Returns float32 logits [sum(len(want)), vocab]
        on the device, in the order of the entries and of each ``want``. ``tap``: see
        ``CausalLM.forward``. ``with_context``: also return the step's ``StepContext`` (the
        generation loop samples from the logits with its positions and wanted rows). Raises ``KernelError``
        where a kernel of the step gave up a wait, for which the step is waited for.
        ``graph``: a step shape that comes a second time is captured as a CUDA graph and replayed
        from then on (short steps are bound by the host's launches otherwise; the reference
        captures its prefill per length too: engine/engine.py:505-536). The logits of a replayed
        step live in the graph's memory and are overwritten by the next step of that shape."""
        n_tok = sum(len(t) for _, t, _ in entries)
        if graph and tap is None and n_tok <= GRAPH_MAX_TOKENS and self.device.type == "cuda":
            self._check(entries)
            return self._graph_step(entries, with_context)
        ctx = self.context(entries)
        logits = self.model.forward(ctx, self.cache, tap)
        for slot, tokens, _ in entries:
            self.cache.commit(slot, len(tokens))
        api.gemm_tc_check()      # single tokens too: their products wait within the kernel as well
        return (logits, ctx) if with_context else logits

    def _graph_step(self, entries, with_context):
        shape = self._shape(entries)
        logits, ctx = self._graph_forward(shape, max(p + n for n, p in zip(shape[0], shape[1])), entries)
        for slot, tokens, _ in entries:
            self.cache.commit(slot, len(tokens))
        api.gemm_tc_check()
        return (logits, ctx) if with_context else logits

    def _graph_forward(self, shape, positions, entries, **trees):
        """(logits, context) of a step of ``shape``, which reaches ``positions``; ``trees``: what ``context`` is told of them."""
        if self.model.prepare(positions) != self._generation:
            self._generation = self.model.generation
            self._graphs.clear()                      # they hold the addresses of the old tables
        sg = self._graphs.get(shape)
        if sg is None:
            times = self._seen.get(shape, 0)
            if times == 0:                            # the first time plainly: it sizes the kernels' scratch memory
                ctx = self.context(entries, **trees)
                logits = self.model.forward(ctx, self.cache)
            self._seen[shape] = times + 1
            self._seen.move_to_end(shape)
            while len(self._seen) > 64:
                self._seen.popitem(last=False)
            if times == 0:
                return logits, ctx
            sg = _StepGraph()
            ctx = self.context(entries, static=sg.static, **trees)
            torch.cuda.synchronize()
            sg.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(sg.graph):
                sg.logits = self.model.forward(ctx, self.cache)
            sg.ctx = ctx
            self._graphs[shape] = sg
            self._drop_graphs(bool(trees))
        else:
            self._graphs.move_to_end(shape)
            sg.ctx = self.context(entries, static=sg.static, **trees)   # same shape: the same views, new data
        sg.graph.replay()
        return sg.logits, sg.ctx

    def _drop_graphs(self, trees):
        """Keeps the graphs of steps (of trees, or the others) within their number, and those of trees within their bytes; the newest stays.
        A shape that was dropped is launched plainly when it comes next: capturing it each time would cost more than the launches."""
        own = [s for s in self._graphs if (s[0] == "trees") == trees]              # the least recently used first
        size = lambda s: self._graphs[s].logits.numel() * self._graphs[s].logits.element_size()
        while len(own) > 1 and (len(own) > GRAPH_KEEP or trees and sum(map(size, own)) > TREE_GRAPH_BYTES):
            shape = own.pop(0)
            del self._graphs[shape]
            self._seen.pop(shape, None)

    @torch.inference_mode()
    def step_tree(self, entries, temperature=0.0, seeds=None, graph=False):
        """Checks trees of drafted tokens. entries: list of (slot, tokens, parents): ``tokens[0]`` is the sequence's last token, which
        is not cached yet (``parents[0]`` = -1), ``tokens[i]`` was drafted to follow node ``parents[i]`` < i. One step runs all nodes;
        from the root on the way goes to the child that holds the token the model chooses (greedy, or drawn with ``temperature`` and the
        sequence's 64-bit seed in ``seeds``, as the sampler draws at that position), and ends at the first node without one. The nodes on
        the way stay cached as the sequence's next tokens, the others' rows are given up. Returns a list an entry: the drafted
        tokens on the way and the token chosen at its end, which is not cached: between 1 and the tree's depth + 1 tokens, the ones that
        steps of single tokens would have brought. Waits for the step. ``graph``: as in ``step``; what fixes the launches of a step of
        trees is how many sequences and nodes it has, the nodes of the largest tree, and how wide the page tables are, the latter three
        rounded up."""
        if not self.model.takes_trees:
            raise ValueError("a layer of this model cannot take trees of drafted tokens (it is no plain attention, or keeps a state)")
        for slot, tokens, parents in entries:
            if len(tokens) != len(parents) or not 1 <= len(tokens) <= api.TREE_MAX_NODES:
                raise ValueError(f"slot {slot}: {len(tokens)} tokens, {len(parents)} parents; a tree has 1 to {api.TREE_MAX_NODES} nodes")
        if seeds is None:
            seeds = [0] * len(entries)
        if len(seeds) != len(entries) or temperature < 0:
            raise ValueError("one seed an entry, and a temperature that is not negative")
        parents, entries = [list(p) for _, _, p in entries], [(s, t, range(len(t))) for s, t, _ in entries]
        nodes = [len(t) for _, t, _ in entries]
        if graph and self.device.type == "cuda" and 0 < sum(nodes) <= GRAPH_MAX_TOKENS:
            self._check(entries)
            for (slot, _, _), k in zip(entries, nodes):
                self.cache.reserve(slot, k)
            widths = tree_table_widths(self.cache, [s for s, _, _ in entries])
            reach = max(self.cache.length[s] + k for (s, _, _), k in zip(entries, nodes))
            rows, largest = tree_shape(nodes)
            logits, ctx = self._graph_forward(("trees", len(nodes), rows, largest, *widths), reach, entries, parents=parents, pad_to=rows,
                                              max_nodes=largest)
        else:
            ctx = self.context(entries, parents=parents)
            logits = self.model.forward(ctx, self.cache)
        n, width = len(entries), ctx.tree.max_nodes
        temps = torch.full((n,), float(temperature), device=self.device)
        words = torch.tensor([seed_words(s) for s in seeds], dtype=torch.int32, device=self.device)
        found = torch.empty(n * (width + 2), dtype=torch.int32, device=self.device)
        path, count, token = found[:n * width].view(n, width), found[n * width:n * (width + 1)], found[n * (width + 1):]
        api.tree_accept(logits, ctx.tok, ctx.tree.parent, ctx.cu_q, ctx.row_pos, temps, words, path, count, token)
        for g, table in zip(self.cache.groups, ctx.tables):
            for store in g.stores():
                api.kv_keep(store, table, ctx.seq_pos0, path, count)
        found = found.tolist()
        api.gemm_tc_check()
        out = []
        for i, (slot, tokens, _) in enumerate(entries):
            way = found[i * width:i * width + found[n * width + i]]
            self.cache.commit(slot, len(way))
            out.append([tokens[k] for k in way[1:]] + [found[n * (width + 1) + i]])
        return out
