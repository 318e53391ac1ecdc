"""Scoring at its edges: frames that cannot score, and generation that keeps log probabilities beside a step that runs ahead."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_frame_that_cannot_score_is_refused_before_anything_moves(tmp_path):
    """A registered frame with a logits() of its own: score() says so before the step has run (the sequence's recurrent states are as they
    were, and the next step gives what it would have given)."""
    import abacus_b200
    import temetar_models
    from abacus_b200.engine.engine import StepError
    lm = abacus_b200.LM(temetar_models.write_folder(tmp_path, "P")[0], max_tokens=512)
    engine, frame = lm.engine, lm.model.frame
    tokens, given = [5, 6, 7, 8, 9, 10, 11], type(frame)

    class Own(given):
        def logits(self, x, y, batch, ws):
            return torch.zeros((batch.n_logit_rows, self.vocab), device=batch.device)

    slot = engine.open()
    engine.step([(slot, tokens, [6])])
    before = engine.cache.save_states([slot])[1]
    frame.__class__ = Own
    try:
        with pytest.raises(StepError, match="cannot score"):
            engine.score([(slot, [1], [0])], [2])
    finally:
        frame.__class__ = given
    assert engine.length(slot) == 7 and before
    assert all(torch.equal(x, y) for x, y in zip(before, engine.cache.save_states([slot])[1]))
    assert engine.score([(slot, [1], [0])], [2])[0].isfinite().all()


@pytest.mark.parametrize("logprobs", [None, 0, 5])
def test_tokens_and_their_log_probabilities_do_not_wait_for_the_step_that_runs_ahead(logprobs):
    """An engine whose step ahead takes the GPU a tenth of a second: on_token has each token, with its log probability and the most likely
    ones, while that step is still running."""
    from abacus_b200.engine.generate import Generator
    from abacus_b200.sampling import Sampler

    class Engine:
        max_context, vocab = 64, 50

        class cache:
            n_pages, max_slots = 4, 2

        ended = None

        def open(self):
            return 0

        def close(self, slot):
            pass

        def logits(self, last):
            out = torch.zeros((1, 50), device="cuda")
            out[:, (last + 1) % 50].fill_(9.0)
            self.last, self.last_batch = last + 1, type("B", (), {"seq_slot": torch.zeros(1, dtype=torch.int32, device="cuda")})()
            return out

        def step(self, entries):
            return self.logits(entries[0][1][-1])

        def step_ahead(self, slots, tokens):
            torch.cuda._sleep(200_000_000)  # (cycles)
            out = self.logits(self.last)
            self.ended = torch.cuda.Event()
            self.ended.record()
            return out

    engine, seen = Engine(), []
    gen = Generator(engine, Sampler("cuda", temperature=0.0), logprobs=logprobs,
                    on_token=lambda r, token: seen.append((token, len(r.logprobs), engine.ended is not None and not engine.ended.query())))
    gen.generate([[1, 2]], max_new_tokens=2)  # (loads the kernels)
    seen.clear()
    engine.ended = None
    r = gen.generate([[1, 2]], max_new_tokens=5)[0]
    assert r.output == [3, 4, 5, 6, 7]
    has = 0 if logprobs is None else 1
    assert seen == [(3 + i, has * (i + 1), i < 4) for i in range(5)]
    if logprobs:
        assert all(top[0][0] == token and top[0][1] == p and len(top) == logprobs for token, p, top in zip(r.output, r.logprobs, r.top))


@pytest.mark.parametrize("dtype, rows, vocab, allowed", [("bfloat16", 32, 65536, None), ("bfloat16", 64, 49152, None), ("bfloat16", 64, 50257, None),
                                                         ("bfloat16", 600, 6000, None), ("float32", 500, 1500, None), ("float32", 64, 100001, 1000),
                                                         ("bfloat16", 8, 100001, 1000)])
def test_the_bound_on_candidates_holds_for_short_slices_and_ranges(dtype, rows, vocab, allowed):
    """Rows cut into slices of less than a turn of a CTA's threads, short rows, and rows of which a mask leaves one range of tokens: the 20
    most likely tokens are right and take at most 3 times as long as one (1.3 to 1.5 on a B200; 8 to 18 where every element is a
    candidate). The two take turns, the fastest of each counts."""
    from abacus_b200.kernels import ops
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn((rows, vocab), generator=g, device="cuda") * 2.0
    if allowed:
        x[:, :vocab // 3], x[:, vocab // 3 + allowed:] = -float("inf"), -float("inf")
    x = x.to(getattr(torch, dtype))
    tokens, out = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    top = {k: (torch.zeros((rows, k), dtype=torch.int32, device="cuda"), torch.zeros((rows, k), device="cuda")) for k in (1, 20)}
    fastest = {1: 1e9, 20: 1e9}
    for _ in range(5):
        for k, (ids, values) in top.items():
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            ops.token_logprobs(x, tokens, out, top_ids=ids, top_logprobs=values)
            torch.cuda._sleep(2_000_000)  # (the launches below are all there when the first runs)
            start.record()
            for _ in range(20):
                ops.token_logprobs(x, tokens, out, top_ids=ids, top_logprobs=values)
            end.record()
            torch.cuda.synchronize()
            fastest[k] = min(fastest[k], start.elapsed_time(end))
    want = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :20]
    assert torch.equal(top[20][0].long(), want) and torch.equal(top[1][0].long(), want[:, :1])
    assert fastest[20] <= 3 * fastest[1], fastest


def test_more_rows_than_a_launch_takes():
    """Rows in launches of 32,768: the last ones too, and nothing behind them."""
    from abacus_b200.kernels import ops
    n, vocab = 65600, 131
    x = (torch.randn((n + 1, vocab), generator=torch.Generator().manual_seed(2)) * 3.0).cuda()
    tokens = (torch.arange(n + 1, device="cuda") % vocab).to(torch.int32)
    logprob, entropy, values = (torch.full(s, 7.0, device="cuda") for s in ((n + 1,), (n + 1,), (n + 1, 3)))
    ids = torch.full((n + 1, 3), 9, dtype=torch.int32, device="cuda")
    ops.token_logprobs(x, tokens, logprob, entropy=entropy, top_ids=ids, top_logprobs=values, n_rows=n)
    logp = torch.log_softmax(x[:n].double(), dim=1)
    order = torch.sort(x[:n], dim=1, descending=True, stable=True).indices[:, :3]
    off = 2.0 ** -24 * 60  # (sums of 131 terms, each 2^-22 and 2^-23 of its distance off, as test_logprobs_gpu.compare counts them, and a logarithm)
    for got, want in ((logprob, logp.gather(1, tokens[:n].long()[:, None])[:, 0]), (values, logp.gather(1, order)),
                      (entropy, -(logp.exp() * logp).sum(dim=1))):
        assert ((got[:n].double() - want).abs() <= off * (2 + math.log(vocab)) + 2.0 ** -22 * want.abs()).all()
        assert (got[n] == 7.0).all()
    assert torch.equal(ids[:n].long(), order) and (ids[n] == 9).all()
