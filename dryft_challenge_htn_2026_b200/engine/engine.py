"""The Python entry point, in the manner of the reference's ``Engine`` (engine/engine.py:247-279,
683-732): ``Engine(model_path, dtype)`` and ``Engine.generate(input_ids, max_new_tokens)``, a
generator that yields one token per sequence per step. Beyond the reference: prompts of unequal
lengths run as one batch, sampling takes a temperature and a seed, sequences may end at stop
tokens, and ``generate_all`` runs as many batches one after another as there are requests.
"""
import torch

from ..csrc.api import MAX_BEAMS, PAGE, TREE_MAX_NODES
from ..registry import config_from_folder
from ..sampling import SamplingParams, request_seed
from ..weights import bind_random, load_weights
from ..weights.loader import list_tensors
from .branch import run_beams, run_drafted
from .generate import GpuBackend, plan_batches, run_batch
from .model import CausalLM
from .runner import Runner


def _dtype(dtype):
    if isinstance(dtype, str):
        try:
            return {"bfloat16": torch.bfloat16, "bf16": torch.bfloat16, "float32": torch.float32, "fp32": torch.float32}[dtype]
        except KeyError:
            raise ValueError(f"dtype must be bfloat16 or float32, not {dtype!r}") from None
    return dtype


def load_model(model_path, dtype=torch.bfloat16, device="cuda"):
    """The model class is chosen by config.json's ``architectures``; weights by tensor name."""
    config = config_from_folder(model_path)
    if hasattr(config, "with_shapes"):      # sizes that only the tensors' shapes give
        config = config.with_shapes({name: shape for name, (_, shape) in list_tensors(model_path).items()})
    model = CausalLM(config.to_spec(), _dtype(dtype), device)
    load_weights(model, model_path)
    return model


def random_model(config, seed=0, dtype=torch.bfloat16, device="cuda"):
    """A model of ``config`` with seeded random weights drawn on the device."""
    return bind_random(CausalLM(config.to_spec(), _dtype(dtype), device), seed)


class Engine:
    def __init__(self, model_path=None, dtype=torch.bfloat16, model=None, max_tokens=None, use_graph=True,
                 max_prefill_tokens=32768):
        """``model_path``: folder with config.json and safetensors (or pass a built ``model``).
        ``max_tokens``: cache size in tokens; by default the cache is sized by each call.
        ``max_prefill_tokens``: most prompt tokens one step runs; a batch of prompts beyond it is
        prefilled in several steps (whole sequences, a longer one in chunks), with equal results."""
        self.model = model if model is not None else load_model(model_path, dtype)
        self.use_graph = use_graph
        self.max_prefill_tokens = max_prefill_tokens
        self.runner = None
        self.backend = None
        self._fixed_tokens = max_tokens
        if max_tokens is not None:
            self._resize(max_tokens, 1024)

    def _resize(self, tokens, slots):
        self.backend = self.runner = None   # drop the old cache before the new one is allocated
        torch.cuda.empty_cache()
        self.runner = Runner(self.model, tokens, slots)
        self.backend = GpuBackend(self.runner, self.use_graph, self.max_prefill_tokens)

    def _ensure(self, prompts, max_new_tokens):
        if any(len(p) == 0 for p in prompts):
            raise ValueError("every prompt needs at least one token")
        need = sum((len(p) + max_new_tokens + PAGE - 1) // PAGE * PAGE for p in prompts)
        if self.runner is None or self.runner.cache.num_pages * PAGE < need or self.runner.cache.max_slots < len(prompts):
            if self._fixed_tokens is not None:
                raise ValueError(f"batch needs {need} cache tokens, engine was built with max_tokens={self._fixed_tokens}")
            self._resize(need, max(len(prompts), 64))

    def generate(self, input_ids, max_new_tokens, temperature=0.0, seed=0, stop_token_ids=(), first_index=0):
        """Yields, ``max_new_tokens`` times at most, a list with the next token of every sequence
        (None once a sequence has ended at a stop token). All sequences start together; their
        prompts may have different lengths. Greedy unless ``temperature`` > 0."""
        if max_new_tokens <= 0 or not input_ids:
            return
        params = SamplingParams(max_new_tokens, float(temperature), int(seed), tuple(stop_token_ids))
        self._ensure(input_ids, max_new_tokens)
        seeds = [request_seed(seed, first_index + i) for i in range(len(input_ids))]
        yield from run_batch(self.backend, [list(p) for p in input_ids], params, seeds)

    def generate_drafted(self, input_ids, max_new_tokens, draft, temperature=0.0, seed=0, stop_token_ids=(), max_nodes=64):
        """``generate`` with tokens that somebody else guesses and the model checks, several a step: the same tokens in fewer steps (up to the
        rounding of the logits: other numbers of rows take other product kernels, so in bfloat16 a near tie may fall the other way).
        ``draft(i, tokens)`` is asked before every step how sequence i goes on behind ``tokens`` (its prompt and what was generated) and
        answers with a list of tokens, or with (tokens, parents), a tree: ``parents[k]`` is the number of the drafted token that
        ``tokens[k]`` would follow, -1 for the last of ``tokens``. Up to ``max_nodes`` - 1 tokens. Yields a list of lists, the new
        tokens of every sequence (none once it has ended). For models whose layers are all attention that takes trees."""
        if max_new_tokens <= 0 or not input_ids:
            return
        if not 1 <= max_nodes <= TREE_MAX_NODES:
            raise ValueError(f"max_nodes must be between 1 and {TREE_MAX_NODES}")
        if not self.model.takes_trees:
            raise ValueError("a layer of this model cannot take trees of drafted tokens (it is no plain attention, or keeps a state)")
        params = SamplingParams(max_new_tokens, float(temperature), int(seed), tuple(stop_token_ids))
        self._ensure(input_ids, max_new_tokens + max_nodes)
        yield from run_drafted(self.runner, [list(p) for p in input_ids], params, [request_seed(seed, i) for i in range(len(input_ids))],
                               draft, max_nodes, self.max_prefill_tokens, self.use_graph)

    def beam_search(self, input_ids, beams, max_new_tokens, stop_token_ids=(), length_penalty=0.0):
        """The ``beams`` best continuations that a search of that width finds for each prompt: a list a prompt of (tokens, score), best
        first. The score is the sum of the tokens' log-probabilities over their number to the power ``length_penalty``; the search
        itself goes by the sum. A continuation ends with a stop token, which is returned, or after ``max_new_tokens``."""
        if not 1 <= beams <= MAX_BEAMS:
            raise ValueError(f"beams must be between 1 and {MAX_BEAMS}")
        if max_new_tokens <= 0 or not input_ids:
            return [[] for _ in input_ids]
        self._ensure([p for p in input_ids for _ in range(beams)], max_new_tokens)
        found = run_beams(self.backend.loop, [list(p) for p in input_ids], beams, max_new_tokens, stop_token_ids, self.max_prefill_tokens)
        scored = [[(t, v / len(t) ** length_penalty) for t, v in row] for row in found]
        return [sorted(row, key=lambda x: -x[1]) for row in scored]

    def generate_all(self, prompts, max_new_tokens, temperature=0.0, seed=0, stop_token_ids=(), batch_size=64):
        """Token lists for any number of requests, run ``batch_size`` at a time, one batch after
        another; a request's tokens do not depend on which batch it lands in."""
        out = [None] * len(prompts)
        for idx in plan_batches(len(prompts), batch_size):
            seqs = [[] for _ in idx]
            for row in self.generate([prompts[i] for i in idx], max_new_tokens, temperature, seed, stop_token_ids,
                                     first_index=idx.start):
                for k, t in enumerate(row):
                    if t is not None:
                        seqs[k].append(t)
            for k, i in enumerate(idx):
                out[i] = seqs[k]
        return out
