"""Continuations of one prompt: what a forked cache's forwards refuse before any work."""
import pytest
import torch

from test_continuations_model_gpu import build, ids_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    return build()[0]


def test_a_prefix_that_was_written_again(model):
    """A prompt's cache set back and filled with other tokens, as many as before."""
    cache = model.new_cache(1, 60)
    model(ids_of(1, 40, 0).cuda(), past_key_values=cache)
    forked = cache.fork(2, 10)
    step = ids_of(2, 1, 1).cuda()
    model(step, past_key_values=forked)
    model(ids_of(1, 5, 2).cuda(), past_key_values=cache)
    model(step, past_key_values=forked)
    cache.length = 20
    model(ids_of(1, 30, 3).cuda(), past_key_values=cache)
    with pytest.raises(ValueError, match='no longer'):
        model(step, past_key_values=forked)
    assert forked.valid and forked.length == 42


def test_generating_past_the_model_s_positions(model):
    """Refused before the first token: the cache is as it was."""
    most = model.config.max_position_embeddings
    cache = model.new_cache(1, most)
    model(ids_of(1, most - 20, 0).cuda(), past_key_values=cache)
    forked = cache.fork(2, 100)
    tail = ids_of(2, 8, 1).cuda()
    with pytest.raises(ValueError, match='positions'):
        model.generate(tail, max_new_tokens=14, eos_token_id=[], pad_token_id=0, past_key_values=forked)
    assert forked.valid and forked.length == most - 20
    assert model.generate(tail, max_new_tokens=13, eos_token_id=[], pad_token_id=0, past_key_values=forked).shape == (2, 21)
    assert forked.length == most
