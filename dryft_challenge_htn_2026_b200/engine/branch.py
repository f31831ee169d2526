"""Generation that branches: drafted tokens that the model checks several at a time, and searches over beams.

``run_drafted`` is the loop around ``Runner.step_tree``: somebody else's guess of how a sequence goes on (a small model, a table of
what followed the same words before) is run as a tree in one step, and what the model would have said itself is kept. The
tokens are the model's own, whatever the guess: a good one saves steps. ``run_beams`` keeps a request's best continuations side by
side: single tokens of all beams in the decode loop, their best continuations chosen on the device, the cache's rows and states
moved behind the choice."""
import torch

from ..csrc import api
from ..sampling import Sampler, seed_words
from .generate import BatchTracker, prefill_plan


def _prefill(runner, slots, prompts, limit, want):
    """Runs the prompts; ``want(ended, logits, ctx)`` gets the logits at the ends of those that ended with a step, in order."""
    for step in prefill_plan([len(p) for p in prompts], limit):
        ended = [i for i, _, p1 in step if p1 == len(prompts[i])]
        logits, ctx = runner.step([(slots[i], prompts[i][p0:p1], [p1 - p0 - 1] if p1 == len(prompts[i]) else []) for i, p0, p1 in step],
                                  with_context=True)
        if ended:
            want(ended, logits, ctx)


def draft_tree(last, draft, max_nodes):
    """(tokens, parents) of the tree that ``Runner.step_tree`` takes, from a sequence's last token and a draft: (tokens, parents) with
    -1 for the tokens drafted to follow the last one, or tokens alone, each drafted to follow the one before."""
    tokens, parents = draft if isinstance(draft, tuple) else (draft, range(-1, len(draft) - 1))
    tokens, parents = list(tokens), [p + 1 for p in parents]
    if len(tokens) != len(parents) or len(tokens) >= max_nodes:
        raise ValueError(f"a draft of {len(tokens)} tokens with {len(parents)} parents: as many of both, {max_nodes - 1} at most")
    return [last] + tokens, [-1] + parents


@torch.inference_mode()
def run_drafted(runner, prompts, params, seeds, draft, max_nodes, max_prefill_tokens=32768, graph=False):
    """Generator over the steps of one batch: yields, per step, a list with the list of new tokens of every sequence (empty once it has
    ended). ``draft(i, tokens)`` guesses how sequence i goes on behind its prompt and output ``tokens`` (see ``draft_tree``). ``graph``: see
    ``Runner.step_tree``."""
    n = len(prompts)
    tracker = BatchTracker(n, params.max_new_tokens, params.stop_token_ids)
    slots = []
    try:
        for _ in prompts:
            slots.append(runner.begin())
        dev = runner.device
        sampler, tok = Sampler(runner.vocab_size, n, dev), torch.empty(n, dtype=torch.int32, device=dev)
        temps = torch.full((n,), params.temperature, device=dev)
        words = torch.tensor([seed_words(s) for s in seeds], dtype=torch.int32, device=dev)

        def first(ended, logits, ctx):
            lo, hi = ended[0], ended[-1] + 1
            sampler(logits, temps[lo:hi], words[lo:hi], ctx.row_pos, ctx.want_rows, tok[lo:hi])

        _prefill(runner, slots, prompts, max_prefill_tokens, first)
        new = [[t] for t in tok.tolist()]
        who = list(range(n))
        while True:
            row = [[] for _ in range(n)]
            for i, tokens in zip(who, new):
                for t in tokens:
                    if tracker.finished[i]:
                        break
                    tracker.accept([i], [t])
                    row[i].append(t)
                if tracker.finished[i]:
                    runner.end(slots[i])
                    slots[i] = None
            yield row
            who = tracker.active(who)
            if not who:
                return
            trees = [draft_tree(tracker.outputs[i][-1], draft(i, list(prompts[i]) + tracker.outputs[i]), max_nodes) for i in who]
            new = runner.step_tree([(slots[i], *t) for i, t in zip(who, trees)], params.temperature, [seeds[i] for i in who], graph)
    finally:
        for s in slots:
            if s is not None:
                runner.end(s)


@torch.inference_mode()
def run_beams(loop, prompts, beams, max_new_tokens, stop_token_ids=(), max_prefill_tokens=32768):
    """The ``beams`` best continuations of each prompt that a search of that width finds: a list a prompt of (tokens, sum of their
    log-probabilities), best first. A continuation ends with a stop token, which it contains, or after ``max_new_tokens``. ``loop``: the
    ``DecodeLoop`` of the runner that holds the model and its cache."""
    runner = loop.runner
    n, dev, stops = len(prompts), runner.device, frozenset(stop_token_ids)
    slots = []
    try:
        for _ in range(n):
            slots.append([])
            for _ in range(beams):
                slots[-1].append(runner.begin())
        flat = [s for row in slots for s in row]
        for row, p in zip(slots, prompts):
            for s in row:
                runner.cache.reserve(s, len(p) + max_new_tokens)
        scores = torch.empty((n, beams), device=dev)
        beam, tok = torch.empty((n, beams), dtype=torch.int32, device=dev), torch.empty((n, beams), dtype=torch.int32, device=dev)

        def first(done, logits, ctx):
            lo, hi = done[0], done[-1] + 1
            api.beam_select(logits, torch.zeros((hi - lo, 1), device=dev), None, scores[lo:hi], beam[lo:hi], tok[lo:hi])

        _prefill(runner, [row[0] for row in slots], prompts, max_prefill_tokens, first)
        for row, p in zip(slots, prompts):
            for s in row[1:]:
                runner.cache.commit(s, len(p))
        runner.cache.reorder(slots, [[0] * beams] * n)          # every beam starts from the prompt that the first one ran
        found = [[[] for _ in range(beams)] for _ in prompts]
        ended = [[False] * beams for _ in prompts]
        other = torch.empty_like(scores)
        longest = max(len(p) for p in prompts) + max_new_tokens
        for made in range(1, max_new_tokens + 1):
            parents, tokens, values = beam.tolist(), tok.tolist(), scores.tolist()
            for r in range(n):
                was, over = found[r], ended[r]
                # a place that no candidate was found for stays out of the search
                ended[r] = [over[p] or v == -float("inf") or t in stops for p, t, v in zip(parents[r], tokens[r], values[r])]
                found[r] = [was[p] if over[p] or v == -float("inf") else was[p] + [t] for p, t, v in zip(parents[r], tokens[r], values[r])]
            if made == max_new_tokens or all(e for row in ended for e in row):
                break
            if made > 1:
                runner.cache.reorder(slots, parents, [len(p) for p in prompts])
            st = loop.state_for(n * beams, longest)
            st.fill([dict(slot=s, token=t, pos=runner.cache.length[s], temperature=0.0, seed=0) for s, t in zip(flat, (t for row in tokens for t in row))])
            loop.run()
            done = torch.tensor(ended, dtype=torch.int32, device=dev)
            scores, other = other, scores
            api.beam_select(st.logits[:n * beams], other, done, scores, beam, tok)
        api.gemm_tc_check()
        return [sorted(((t, v) for t, v in zip(f, row) if v > -float("inf")), key=lambda x: -x[1]) for f, row in zip(found, scores.tolist())]
    finally:
        torch.cuda.current_stream().synchronize()
        for row in slots:
            for s in row:
                runner.end(s)
