"""Generation where probabilities are no numbers, or all but one of them vanish."""
import math

import pytest
import torch

from test_decoding_cpu import _greedy, _llama


@pytest.mark.parametrize("drafted", [0, 1, 3])
@pytest.mark.parametrize("n", [1, 6])
def test_generate_refuses_probabilities_that_are_no_numbers(drafted, n):
    m = _llama()
    with torch.no_grad():
        m.lm_head[3] = math.nan
    with pytest.raises(RuntimeError, match="no numbers"):
        m.generate(torch.randint(0, 50, (2, 4)), n, 1.0, draft=_llama(1, 7) if drafted else None, drafted=max(drafted, 1))


def test_a_draft_whose_probabilities_are_no_numbers_is_refused_and_nothing_else():
    m, broken = _llama(), _llama(1, 7)
    with torch.no_grad():
        broken.lm_head.fill_(math.nan)
    ids = torch.randint(0, 50, (2, 4))
    out = m.generate(ids, 9, 1.0, draft=broken, drafted=2)
    assert out.shape == (2, 13) and torch.equal(out[:, :4], ids) and ((out >= 0) & (out < 50)).all()
    # next to no temperature: the likeliest token of the model each time
    assert torch.equal(m.generate(ids, 9, 1e-30, draft=broken, drafted=2), _greedy(m, ids, 9))


@pytest.mark.parametrize("temperature", [1e-6, 1e-30, 1e-45, 5e-324])
def test_generate_at_next_to_no_temperature(temperature):
    m = _llama()
    ids = torch.randint(0, 50, (2, 4))
    assert torch.equal(m.generate(ids, 9, temperature), _greedy(m, ids, 9))
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            m.generate(ids, 2, bad)


def test_other_temperatures_keep_their_probabilities_to_the_bit():
    m = _llama()
    h = torch.randn(7, 32)
    logits = h @ m.lm_head.T
    for t in (0.3, 0.8, 1.0, 2.5):
        assert torch.equal(m._probs(h, t), torch.softmax(torch.nn.functional.linear(h, m.lm_head)[:, :50] / t, -1))
    for t in (1e-38, 1e-45, 5e-324):
        assert torch.equal(m._probs(h, t).argmax(-1), logits[:, :50].argmax(-1)) and torch.equal(m._probs(h, t).amax(-1), torch.ones(7))
