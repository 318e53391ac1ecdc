"""The Python entry point: load a model folder and generate.

    from abacus_b200 import LM
    lm = LM("model_dir", dtype="bfloat16", max_tokens=65536)
    outs = lm.generate([[1, 2, 3], [4, 5]], max_new_tokens=32, temperature=0.0)
    scores = lm.score([[1, 2, 3, 4], [4, 5, 6]], top=5)   # how likely each token was, and the five likeliest in its place

Option names and meanings follow abacus's command line (src/main.c:9-23): max_new_tokens is -n,
temperature is --temp (0 = greedy, default 0.7), seed is --seed (default: the time, src/main.c:112);
top_k is the 20 that src/main.c:41 fixes. Prompts are token-id lists, or strings when the folder has a tokenizer.json
(then raw=False wraps each in the chat template of src/main.c:168, as -p does, and raw=True
does not, as --raw).
"""
import os
import time
from dataclasses import dataclass

import torch

from .engine import Engine, load_model
from .engine.generate import Generator, plan_batches, Request
from .sampling import Sampler

CHAT_TEMPLATE = "<|im_start|>user\n{}<|im_end|>\n<|im_start|>assistant\n<think>\n\n</think>\n\n"  # src/main.c:168
DEFAULT_CONTEXT = 4096   # abacus caps a sequence at 4,096 tokens (src/model.c:15)
DEFAULT_SEQUENCES = 8    # the cache's default room: this many sequences of that length


@dataclass
class Score:
    """What a model makes of a text: for every token but the first, its log probability after those before it (natural logarithm),
    the entropy of the distribution it was taken from, and that distribution's most likely tokens, [(token, log probability)]."""
    tokens: list
    logprobs: list
    entropies: list
    top: list = None

    @property
    def total(self):
        return sum(self.logprobs)


class LM:
    def __init__(self, folder, dtype="bfloat16", max_tokens=None, max_slots=None, max_context=None, cache=None):
        """cache: "int8" or "e4m3" keeps keys and values in 8 bits (see Engine); None: in the model's type."""
        self.model = load_model(folder, dtype)
        spec = self.model.spec
        if max_tokens is None:
            max_tokens = min(spec.max_positions, DEFAULT_CONTEXT) * DEFAULT_SEQUENCES
        self.engine = Engine(self.model, max_tokens=max_tokens, max_slots=max_slots, max_context=max_context, cache=cache)
        self.tokenizer = None
        if os.path.exists(os.path.join(folder, "tokenizer.json")):
            from .tokenizer import Tokenizer
            self.tokenizer = Tokenizer.from_file(os.path.join(folder, "tokenizer.json"))

    def stop_tokens(self):
        """<|im_end|> and <|endoftext|> when there is a tokenizer (src/main.c:176), and config.json's eos ids."""
        stops = set(self.model.spec.stop_tokens)
        if self.tokenizer is not None:
            stops.update(self.tokenizer.stop_ids())
        return sorted(stops)

    def encode(self, prompt, raw=False):
        if self.tokenizer is None:
            raise ValueError("this model folder has no tokenizer.json; give token ids")
        return self.tokenizer.encode(prompt if raw else CHAT_TEMPLATE.format(prompt))

    def generate(self, prompts, max_new_tokens=512, temperature=0.7, top_k=20, seed=None, stop_tokens=None,
                 batch_size=None, raw=False, return_requests=False, on_token=None, logprobs=None):
        """Returns one list of new token ids per prompt (strings instead, if the prompts were strings).
        seed None: the time, as abacus's command line does; give a seed to draw the same tokens again.
        on_token(request, token) is called for every kept token as soon as the host has it.
        logprobs: a number k from 0 on gives every kept token its log probability (at temperature 1, before any cut) and the k most
        likely tokens in its place, in the requests' `logprobs` and `top` (see return_requests)."""
        if seed is None:
            seed = int(time.time())
        as_text = bool(prompts) and isinstance(prompts[0], str)
        ids = [self.encode(p, raw) for p in prompts] if as_text else [list(p) for p in prompts]
        sampler = Sampler(self.model.ctx.device, temperature=temperature, top_k=top_k, seed=seed)
        stops = self.stop_tokens() if stop_tokens is None else list(stop_tokens)
        gen = Generator(self.engine, sampler, stops, on_token=on_token, logprobs=logprobs)
        requests = gen.generate(ids, max_new_tokens, batch_size=batch_size)
        self.last_stats = gen.stats
        if return_requests:
            return requests
        if as_text:
            return [self.tokenizer.decode(r.output) for r in requests]
        return [r.output for r in requests]

    def score(self, texts, top=0, raw=True, from_cache=False):
        """A Score for each text (token-id lists, or strings, which raw=False wraps as generate does): the log probability of every
        token after the first, and with top > 0 the `top` most likely tokens in its place. Texts go through in batches that
        fit the cache, and leave nothing there.
        from_cache: with an 8-bit cache a whole text attends to its own keys as they came, like a prompt, so that its score is the 16-bit
        model's. With from_cache=True every token attends to keys and values as the cache holds them, and the score shows what the
        8 bits cost: the first token goes in a step of its own and the others go on with it, one by one where a layer is windowed."""
        as_text = bool(texts) and isinstance(texts[0], str)
        ids = [self.encode(t, raw) for t in texts] if as_text else [[int(t) for t in text] for text in texts]
        engine, cache = self.engine, self.engine.cache
        scores = [None] * len(ids)
        requests = [Request(i, tokens, 0) for i, tokens in enumerate(ids)]
        for batch in plan_batches(requests, engine.cache_tokens, cache.max_slots, engine.max_context):
            longest = max(len(r.prompt) for r in batch)
            cuts = [0, longest] if not from_cache or cache.form is None else [0, 1, longest] if engine.takes_portions else list(range(longest + 1))
            of_row, numbers, slots = [], [], []  # the place in the batch of each row of numbers
            try:
                for r in batch:
                    slots.append(engine.open())
                for lo, hi in zip(cuts, cuts[1:]):
                    here = [(i, r, min(hi, len(r.prompt) - 1)) for i, r in enumerate(batch) if len(r.prompt) > lo]
                    if here:
                        entries = [(slots[i], r.prompt[lo:hi], list(range(end - lo))) for i, r, end in here]
                        numbers.append(engine.score(entries, [t for _, r, end in here for t in r.prompt[lo + 1:end + 1]], top))
                        of_row += [i for i, _, end in here for _ in range(lo, end)]
                logprob, entropy = (torch.cat([n[i] for n in numbers]).tolist() for i in (0, 1))
                best = [torch.cat([n[i] for n in numbers]).tolist() for i in (2, 3)] if top else None
            finally:
                for slot in slots:
                    engine.close(slot)
            made = [Score(r.prompt, [], [], [] if top else None) for r in batch]
            for row, i in enumerate(of_row):
                made[i].logprobs.append(logprob[row])
                made[i].entropies.append(entropy[row])
                if top:
                    made[i].top.append(list(zip(best[0][row], best[1][row])))
            for r, s in zip(batch, made):
                scores[r.index] = s
        self.engine.check_status()
        return scores


def generate(folder, prompts, dtype="bfloat16", max_tokens=None, cache=None, **options):
    """One call: load `folder` and generate for `prompts` (see LM.generate for the options)."""
    return LM(folder, dtype=dtype, max_tokens=max_tokens, cache=cache).generate(prompts, **options)
