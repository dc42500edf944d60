"""CPU: what the packed sampled paths refuse on the host."""

from types import SimpleNamespace

import pytest
import torch

from test_serving_host import _server
from utttcompanion_b200 import sampling
from utttcompanion_b200.dropin import uTTTModelB200
from utttcompanion_b200.model import UtttB200


def test_a_repetition_penalty_is_refused_where_nothing_applies_it(monkeypatch):
    eng, srv = _server(monkeypatch, capacity=2, max_batch=2)
    srv.max_sampled_tokens = 16
    srv.submit("a", [7, 8], 8, temperature=0.7)
    eng.repetition_penalty = 1.18
    srv.submit("a", [7, 8], 8)                                  # greedy turns are what they were
    with pytest.raises(ValueError, match="repetition"):
        srv.submit("a", [7, 8], 8, temperature=0.7)
    fake = SimpleNamespace(repetition_penalty=1.18)
    for call in (lambda: UtttB200.generate_replies(fake, torch.arange(6, 9), None, 4, 2),
                 lambda: UtttB200.generate_drafted(fake, torch.arange(6, 9), None, 4, None, temperature=0.5,
                                                   u=torch.zeros(4))):
        with pytest.raises(ValueError, match="repetition"):
            call()
    sampling.check_penalty(SimpleNamespace(), 1.0)               # an engine that names none


def test_the_model_and_its_engine_have_one_penalty():
    m = object.__new__(uTTTModelB200)
    m.engine = SimpleNamespace(repetition_penalty=1.0)
    m.repetition_penalty = 1.3
    assert m.engine.repetition_penalty == 1.3 and m.repetition_penalty == 1.3


@pytest.mark.parametrize("top_k", [float("inf"), float("nan"), -float("inf")])
def test_a_top_k_that_is_no_number_of_ids(top_k):
    with pytest.raises(ValueError):
        sampling.check_settings(top_k=top_k)


def test_a_sampled_row_is_not_left_with_another_turns_numbers():
    rows = sampling.SamplingRows(torch.device("cpu"), 2, 4)
    rows.set(0, 0.7, u=torch.tensor([0.25, 0.5]))
    for u in (None, torch.zeros(0)):
        with pytest.raises(ValueError):
            rows.set(0, 0.9, u=u)
    assert rows.temperature.tolist() == [pytest.approx(0.7), 0.0]
    rows.set(0)                                                  # greedy again: none needed
