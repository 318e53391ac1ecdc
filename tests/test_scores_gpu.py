"""Scoring at its edges: frames that cannot score, and generation that keeps log probabilities beside a step that runs ahead."""
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
