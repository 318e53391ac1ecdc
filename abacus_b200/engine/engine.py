"""The step function: a batch of sequences, their next tokens, the logits at the wanted places.

An Engine holds a model, its cache and the slots of the live sequences. A step
runs only the tokens it is given, as one batch, against what earlier steps left
in the cache: whole prompts of unequal lengths in one step, then one token per
sequence. This is abacus's forward(tokens, n, pos, logits, n_logits)
(src/model.c:315-327) for a batch of sequences instead of one.
"""
import os
from dataclasses import dataclass

import numpy as np

import torch

from ..cache import TOKENS_PER_PAGE, SequenceCache
from ..config.registry import load_config
from ..kernels.ops import KernelRefused
from ..models.model import Model
from ..parts.attention import KV8_ROWS_UP_TO
from ..weights.loader import load_folder
from ..weights.safetensors_io import folder_shapes
from .batch import Sequence, StepBatch
from .cstep import CStep
from .graphs import DecodeGraphs, PromptGraphs

DTYPES = {"bfloat16": torch.bfloat16, "bf16": torch.bfloat16, "float32": torch.float32, "fp32": torch.float32,
          "f32": torch.float32}


class StepError(ValueError):
    """A step that asks for what cannot be run (context full, unknown slot, no tokens)."""


def _device():
    if not torch.cuda.is_available():
        raise RuntimeError("abacus_b200 runs on a CUDA GPU (sm_100a); none is visible and there is no CPU path")
    return torch.device("cuda", torch.cuda.current_device())


def load_model(folder, dtype="bfloat16", device=None):
    """A Model from a folder with config.json and *.safetensors; the class is chosen by config.json."""
    dtype = DTYPES[dtype] if isinstance(dtype, str) else dtype
    arch, config = load_config(folder)
    if hasattr(arch, "complete_config"):  # sizes that config.json leaves to the tensors' shapes
        config = arch.complete_config(config, folder_shapes(folder))
    spec = config.to_spec()
    layout = arch.layout(spec)
    tensors = load_folder(folder, lambda available: arch.tensor_names(spec, available))
    model = Model(spec, layout, tensors, dtype, device or _device())
    model.config = config
    model.folder = os.path.abspath(folder)
    return model


@dataclass
class Scoring:
    """Where a step that scores leaves its numbers, for its wanted rows in order (ops.token_logprobs says what they are)."""
    tokens: torch.Tensor      # int32: the token whose log probability is wanted (-1: none)
    logprob: torch.Tensor     # float32
    entropy: torch.Tensor     # float32
    top_ids: torch.Tensor = None       # int32 [rows, k], or None
    top_logprobs: torch.Tensor = None  # float32 [rows, k]


# Tokens whose keys and values a pass over portions reads back from an 8-bit cache at a time (of one sequence, if it holds more): 0.5 GB with
# 8 kv heads of 128, which all layers use one after the other.
READ_BACK_TOKENS = 1 << 17

_ONE_TOKEN, _WANT_IT = np.zeros(1, dtype=np.int64), [0]


def capturable(model):
    """(single-token steps, steps of several tokens): whether the model's steps may be replayed from captured
    graphs. A captured graph replays device work only: a part whose forward decides anything on the host from the
    step's contents cannot be captured, and parts say so: `capturable = True` on every part for single-token
    steps; for steps of several tokens also no mixer with `capturable_prompts = False`. The second value is True,
    False, or "from_start": only steps whose sequences all start at their first token."""
    parts = list(model.parts())
    decode = all(getattr(part, "capturable", False) for part in parts)
    prompts = [getattr(part, "capturable_prompts", True) for part in parts]
    if not decode or not all(prompts):
        return decode, False
    # a part may allow captured prompt steps only where every sequence of the step starts at its first token
    # ("from_start"): what it decides on the host then holds for every step the graph is replayed for
    return decode, "from_start" if "from_start" in prompts else True


class Engine:
    def __init__(self, model, max_tokens, max_slots=None, max_context=None, use_graphs=True, cache=None):
        """cache: "int8" or "e4m3" keeps keys and values in 8 bits with scales (cache/kv8.py; models whose mixers are all plain attention
        in bfloat16, heads of 64 or 128): half the bytes a token, and an open block of 16 tokens in bfloat16 a slot beside them (a quarter
        of a 16-bit page; with a slot a page, the default, 0.75 of the 16-bit cache in all: give max_slots). None: in the model's type."""
        self.model = model
        if cache is not None:
            self._check_kv8(model, cache)
        spec = model.spec
        context = min(max_context or spec.max_positions, spec.max_positions)
        self.cache = SequenceCache(model.cache_needs(), model.cache_sources(), max_tokens, model.ctx.dtype,
                                   model.ctx.device, max_slots=max_slots, max_context=context,
                                   frame_need=model.frame_need(), form=cache)
        self.max_context = self.cache.max_context
        model.prepare(self.max_context)
        self.vocab = spec.vocab
        # the step function in C where the model is made of the library's own parts, else the parts' forward()
        self.cstep = CStep(model, self.cache) if cache is None and CStep.serves(model) else None
        decode_graphs, prompt_graphs = capturable(model)
        if cache is not None and prompt_graphs:
            # a step that reads an 8-bit cache back has its pages counted on the host: one with a sequence that goes on, and any
            # prompt step of a layer whose keys are another's
            prompt_graphs = "from_start" if all(e.source is None for e in model.schedule) else False
        self.graphs = DecodeGraphs(self) if use_graphs and decode_graphs else None
        prompts = use_graphs and prompt_graphs and os.environ.get("ABACUS_PROMPT_GRAPHS", "1") != "0"
        self.prompt_graphs = PromptGraphs(self, from_start_only=prompt_graphs == "from_start") if prompts else None
        self._step_batch = None
        self._graph_memory = None
        # the windowed layers of an 8-bit cache take several tokens of a sequence only at its start, or never (keys of another entry's ring)
        windowed = [e for e in model.schedule if cache is not None and model.blocks[e.layer].mixer.spec.window is not None]
        self._borrows = any(e.source is not None for e in model.schedule)
        self.takes_portions = not windowed
        self._single_only = any(e.source is not None for e in windowed)

    @staticmethod
    def _check_kv8(model, form):
        from ..cache.kv8 import FORMS
        from ..parts.attention import Attention
        if form not in FORMS:
            raise ValueError(f"cache {form!r}: keys and values are kept in the model's type (None) or as {' or '.join(FORMS)}")
        plain = all(type(b.mixer) is Attention and not b.mixer.general and b.mixer.spec.head_dim in (64, 128) for b in model.blocks)
        if not plain or model.ctx.dtype != torch.bfloat16:
            raise ValueError("an 8-bit cache serves bfloat16 models whose mixers are all plain attention with heads of 64 or 128")

    def graph_memory(self):
        """The memory pool of the engine's captured steps, by its id."""
        if self._graph_memory is None:
            self._graph_memory = torch.cuda.MemPool()
        return self._graph_memory.id

    @property
    def cache_tokens(self):
        """Tokens the cache has room for."""
        return self.cache.n_pages * TOKENS_PER_PAGE

    # ------------------------------------------------------------ sequences
    def open(self):
        """A slot for a new sequence."""
        return self.cache.open_slot()

    def close(self, slot):
        """The sequence is finished: what it holds is given back."""
        self.cache.close_slot(slot)

    def length(self, slot):
        return self.cache.length[slot]

    # ------------------------------------------------------------ the step
    def plan(self, entries):
        """entries: [(slot, tokens, want)] -> [Sequence]; checks them and makes room in the cache."""
        if not entries:
            raise StepError("a step needs at least one sequence")
        seqs, seen = [], set()
        for slot, tokens, want in entries:
            if slot not in self.cache.length:
                raise StepError(f"slot {slot} is not open")
            if slot in seen:
                raise StepError(f"slot {slot} appears twice in one step")
            seen.add(slot)
            tokens = np.asarray(tokens, dtype=np.int64).reshape(-1)
            if not tokens.size:
                raise StepError(f"slot {slot}: a step must bring at least one token")
            if tokens.min() < 0 or tokens.max() >= self.vocab:
                bad = tokens[(tokens < 0) | (tokens >= self.vocab)]
                raise StepError(f"slot {slot}: token {int(bad[0])} is outside the vocabulary of {self.vocab}")
            seqs.append(Sequence(slot, tokens, self.cache.length[slot], [int(w) for w in want]))
        if not self.takes_portions and any(len(s.tokens) > 1 and (s.start > 0 or self._single_only) for s in seqs):
            # (before anything is written: an 8-bit cache's open blocks would keep what the layers before put there)
            raise KernelRefused("windowed attention takes several tokens of a sequence only at its start, and only with keys of its own")
        self.cache.reserve_all([(s.slot, s.start + len(s.tokens)) for s in seqs])
        return seqs

    def step(self, entries):
        """Run one step; returns float32 logits [wanted rows, vocab] on the device, in the order of
        the entries and of each entry's `want`."""
        seqs = self.plan(entries)
        ways = self._ways(seqs)
        if len(ways) == 1:
            logits, self.last_batch = self._run(seqs)
            self._advance(seqs)
            return logits
        rows, out = self._rows(seqs), None
        for way in ways:
            part = [seqs[i] for i in way]
            logits, _ = self._run(part)
            self._advance(part)
            out = logits.new_empty((rows[-1], logits.shape[1])) if out is None else out
            self._put(out, logits, way, rows)
        self._fill_whole(seqs)
        return out

    def _run(self, seqs):
        """One forward pass over the sequences of a step: (logits, its StepBatch)."""
        if self.graphs is not None and self.graphs.takes(seqs):  # a plain decode step: replay its graph
            graph = self.graphs.get(seqs)
            return graph.run(seqs), graph.batch
        if self.prompt_graphs is not None and self.prompt_graphs.takes(seqs):  # a shape of prompts seen before
            return self.prompt_graphs.run(seqs)
        batch = self._room_for(sum(len(s.tokens) for s in seqs), len(seqs), sum(len(s.want) for s in seqs))
        batch.fill(seqs, exact=True)
        return self.forward(batch), batch

    def _advance(self, seqs):
        for s in seqs:
            self.cache.advance(s.slot, len(s.tokens))

    def _ways(self, seqs):
        """The places of a step's sequences by the forward passes they go through. One pass, but with an 8-bit cache: there whole prompts
        attend to their own keys as they came, sequences that bring a few tokens row by row to what the cache holds, and longer
        portions to pages read back into 16 bits (parts/attention.py: forward_kv8). Each way has a pass of its own, so that a
        sequence's numbers do not depend on what else is in the step; portions come READ_BACK_TOKENS of context at a time, so that their
        pages in 16 bits stay a small share of what the cache holds."""
        if self.cache.form is None or all(len(s.tokens) == 1 for s in seqs):
            return [list(range(len(seqs)))]
        from_start = all(s.start == 0 for s in seqs)
        ways, portions, held = {}, [[]], 0
        for i, s in enumerate(seqs):
            n = len(s.tokens)
            few = n <= KV8_ROWS_UP_TO
            if s.start == 0 and (n > 1 or from_start):
                # (only a layer whose keys are another's reads the cache for a whole prompt, by either way)
                ways.setdefault(("whole", few and self._borrows), []).append(i)
            elif few:
                ways.setdefault("few", []).append(i)
            else:
                if portions[-1] and held + s.start + n > READ_BACK_TOKENS:
                    portions.append([])
                    held = 0
                portions[-1].append(i)
                held += s.start + n
        ways = [way for way in [*ways.values(), *portions] if way]
        if len(ways) > 1:  # (a wanted place that is not there is refused before any pass runs)
            for s in seqs:
                for place in s.want:
                    if not 0 <= place < len(s.tokens):
                        raise StepError(f"wanted place {place} is outside the {len(s.tokens)} tokens given")
        return ways

    @staticmethod
    def _rows(seqs):
        """The wanted rows in front of each sequence's own, and of all."""
        return np.concatenate([[0], np.cumsum([len(s.want) for s in seqs])]).tolist()

    @staticmethod
    def _put(out, part, way, rows):
        """What a pass gave for the sequences at the places `way` of a step, to their rows of `out`."""
        index = [r for i in way for r in range(rows[i], rows[i + 1])]
        if index:
            out.index_copy_(0, torch.tensor(index, device=out.device), part)

    def _fill_whole(self, seqs):
        """last_batch for a step that ran in several passes: all of its sequences, in their order."""
        self.last_batch = self._room_for(sum(len(s.tokens) for s in seqs), len(seqs), sum(len(s.want) for s in seqs))
        self.last_batch.fill(seqs, exact=True)

    def score(self, entries, tokens, top=0):
        """A step (see step) that gives, for every wanted row, the log probability of the given token, the entropy and the `top` most
        likely tokens instead of logits, which are not kept. tokens: a token a wanted row, in the order of the entries and of each
        entry's `want` (-1: none). Returns (logprob, entropy, top_ids, top_logprobs) on the device, the last two None for top=0."""
        rows = sum(len(want) for _, _, want in entries)
        if len(tokens) != rows:
            raise StepError(f"{len(tokens)} tokens to score at {rows} wanted places")
        if not 0 <= top <= min(64, self.vocab):
            raise StepError(f"{top} most likely tokens: 0 to {min(64, self.vocab)} can be had")
        if not getattr(self.model.frame.logits, "scores", False):  # (before a recurrent state has moved on)
            raise StepError(f"the model's frame {self.model.spec.frame!r} makes logits of its own and cannot score")
        seqs = self.plan(entries)
        device = self.model.ctx.device
        given = torch.tensor(list(tokens), dtype=torch.int32).to(device)
        ways = self._ways(seqs)
        if len(ways) == 1:
            scoring = self._run_scoring(seqs, given, top)
        else:
            rows, scoring = self._rows(seqs), self._scoring(given, top)
            for way in ways:
                part = [seqs[i] for i in way]
                index = torch.tensor([r for i in way for r in range(rows[i], rows[i + 1])], dtype=torch.int64, device=device)
                got = self._run_scoring(part, given[index], top)
                for name in ("logprob", "entropy", "top_ids", "top_logprobs"):
                    if getattr(got, name) is not None:
                        self._put(getattr(scoring, name), getattr(got, name), way, rows)
            self._fill_whole(seqs)
        return scoring.logprob, scoring.entropy, scoring.top_ids, scoring.top_logprobs

    @staticmethod
    def _scoring(given, top):
        """Room for the numbers of a step that scores the tokens `given`."""
        rows, device = given.numel(), given.device
        number = lambda *shape: torch.empty(shape, dtype=torch.float32, device=device)
        return Scoring(given, number(rows), number(rows), torch.empty((rows, top), dtype=torch.int32, device=device) if top else None,
                       number(rows, top) if top else None)

    def _run_scoring(self, seqs, given, top):
        """One forward pass that scores."""
        batch = self._room_for(sum(len(s.tokens) for s in seqs), len(seqs), given.numel())
        batch.fill(seqs, exact=True)
        batch.scoring = self._scoring(given, top)
        try:
            self.model.forward(batch, self.cache)
            scoring = batch.scoring
        finally:
            batch.scoring = None
        self.last_batch = batch
        self._advance(seqs)
        return scoring

    def forward(self, batch):
        """The model's forward pass over a filled step: in one call to C where that serves the model."""
        if self.cstep is not None:
            return self.cstep.run(batch)
        return self.model.forward(batch, self.cache)

    def step_ahead(self, slots, tokens_dev):
        """A decode step (one token per sequence, its logits wanted) whose tokens are on the device, for instance
        where a sampler has just put them: the host need not have seen them. tokens_dev int32 [len(slots)], in the
        order of `slots`. Returns the logits like step(), or None if this engine runs such steps only from the
        host (no captured graphs), in which case nothing has happened."""
        if self.graphs is None:
            return None
        seqs = [Sequence(slot, _ONE_TOKEN, self.cache.length[slot], _WANT_IT) for slot in slots]
        if len(set(slots)) != len(slots) or not self.graphs.takes(seqs):
            return None
        self.cache.reserve_all([(s.slot, s.start + 1) for s in seqs])
        graph = self.graphs.get(seqs)
        logits = graph.run(seqs, tokens_dev=tokens_dev)
        self.last_batch = graph.batch
        for s in seqs:
            self.cache.advance(s.slot, 1)
        return logits

    def _room_for(self, n_rows, n_seqs, n_logits):
        """The engine's StepBatch for steps outside a graph; replaced by a larger one when a step outgrows it
        (pinned memory is slow to get, so it is not made anew for every step)."""
        b = self._step_batch
        if b is None or n_rows > b.cap_rows or n_seqs > b.cap_seqs or n_logits > b.cap_logits:
            grow = lambda n, least: max(least, 1 << max(0, int(n) - 1).bit_length())
            b = StepBatch(grow(max(n_rows, b.cap_rows if b else 0), 256), grow(max(n_seqs, b.cap_seqs if b else 0), 16),
                          grow(max(n_logits, b.cap_logits if b else 0), 64), self.model.ctx.device,
                          plans=self.model.step_plans())
            self._step_batch = b
        return b

    def check_status(self):
        """Raise if a kernel reported a fault (a bounded wait that ran out, a token out of range)."""
        from ..kernels import ops
        shared = ops.kernel_status(self.model.ctx.device)
        status = self.model.status.tolist() + shared.tolist()
        if any(status):
            self.model.status.zero_()
            shared.zero_()
            raise RuntimeError(f"a kernel reported a fault (a token outside the vocabulary, or a wait that "
                               f"ran out): status words {status}")
