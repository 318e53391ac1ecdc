"""What scoring refuses before anything runs: no GPU."""
import pytest

from abacus_b200.engine.generate import Generator
from test_cache_generation import FakeEngine, FakeSampler


def test_a_number_of_most_likely_tokens_that_cannot_be_had_is_refused_at_once():
    engine = FakeEngine()
    for k in (-1, 65, 2.5):
        with pytest.raises(ValueError, match="0 to 64"):
            Generator(engine, FakeSampler(), logprobs=k)
    engine.vocab = 7
    with pytest.raises(ValueError, match="0 to 7"):
        Generator(engine, FakeSampler(), logprobs=8)
    assert not engine.opened and Generator(engine, FakeSampler(), logprobs=7).logprobs == 7
    assert Generator(engine, FakeSampler()).logprobs is None
