"""Sampling options beyond the reference's: what they accept, and what a request hands to the device."""

import numpy as np
import pytest

from matricxon_b200.sampling.config import SamplingConfig
from matricxon_b200.sampling.sampler import RequestSampler


def test_defaults_adjust_nothing_and_stay_where_they_were():
    config = SamplingConfig(0.5, 0.8, 10, 1.2, 100, 5, 3)
    assert (config.temperature, config.top_p, config.top_k, config.repeat_penalty, config.num_ctx, config.num_predict, config.seed) == (
        0.5, 0.8, 10, 1.2, 100, 5, 3)
    assert not config.adjusts_scores and config.largest_token_id == -1
    assert hash(config) == hash(SamplingConfig(0.5, 0.8, 10, 1.2, 100, 5, 3))


def test_biases_and_allowed_tokens_are_put_in_order():
    config = SamplingConfig(logit_bias={7: 1, 3: -2.5}, allowed_token_ids=[9, 2, 9])
    assert config.logit_bias == ((7, 1.0), (3, -2.5)) and config.allowed_token_ids == (2, 9)
    assert SamplingConfig(logit_bias=[(7, 1.0), (7, 4.0)]).logit_bias == ((7, 4.0),)
    assert config.adjusts_scores and config.largest_token_id == 9
    assert SamplingConfig(presence_penalty=0.1).adjusts_scores and SamplingConfig(frequency_penalty=-0.1).adjusts_scores
    assert not SamplingConfig(logit_bias={}).adjusts_scores and SamplingConfig(logit_bias=None).logit_bias == ()


@pytest.mark.parametrize("bad", [{"logit_bias": {1: float("inf")}}, {"logit_bias": {1: float("nan")}}, {"logit_bias": {-1: 1.0}},
                                 {"allowed_token_ids": ()}, {"allowed_token_ids": (3, -4)}, {"presence_penalty": float("nan")},
                                 {"frequency_penalty": float("inf")}])
def test_refusals(bad):
    with pytest.raises(ValueError):
        SamplingConfig(**bad)


@pytest.mark.parametrize("vocab", [10, 32, 33, 100])
def test_mask_words(vocab):
    sampler = RequestSampler(SamplingConfig(allowed_token_ids=(0, 5, 9, vocab - 1)))
    words = sampler.mask_words(vocab)
    assert words.dtype == np.int32 and words.shape == ((vocab + 31) // 32,)
    taken = {v for v in range(words.shape[0] * 32) if int(words[v // 32]) >> (v % 32) & 1}
    assert taken == {0, 5, 9, vocab - 1}
    assert RequestSampler(SamplingConfig()).mask_words(vocab) is None


def test_who_penalises_repeats():
    """The sampling kernel, unless the scores are adjusted before it."""
    plain, adjusted = RequestSampler(SamplingConfig(seed=1)), RequestSampler(SamplingConfig(seed=1, presence_penalty=0.5))
    for sampler in (plain, adjusted):
        for token in (4, 4, 7):
            sampler.accept(token)
    assert plain.penalty_ids() == [4, 7] and adjusted.penalty_ids() == []


@pytest.mark.parametrize("value", [1e39, -1e39, 3.5e38, -3.5e38, 1e308])
@pytest.mark.parametrize("name", ["logit_bias", "presence_penalty", "frequency_penalty"])
def test_numbers_beyond_the_scores_32_bits_are_refused(name, value):
    with pytest.raises(ValueError, match="32-bit"):
        SamplingConfig(**{name: {3: value} if name == "logit_bias" else value})


@pytest.mark.parametrize("value", [3.4e38, -3.4e38, float(np.finfo(np.float32).max), 1e-50])
def test_numbers_within_them_stay_finite(value):
    config = SamplingConfig(logit_bias={3: value}, presence_penalty=value, frequency_penalty=value)
    assert np.isfinite(np.asarray([config.logit_bias[0][1], config.presence_penalty, config.frequency_penalty], dtype=np.float32)).all()
