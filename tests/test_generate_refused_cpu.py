"""A generate() that ends in an error leaves the model as it was: the host side, with stand-ins for the layers."""
from types import SimpleNamespace

import pytest
import torch

from eet_b200 import EET, modeling


class _Model:
    """Counts its calls; says no at the given one."""

    def __init__(self, refuse_at=None):
        self.layers, self.desc = [], SimpleNamespace(device=torch.device("cpu"), tp=None)
        self.pre_padding_len, self.calls, self.refuse_at = torch.empty(0).long(), 0, refuse_at
        self.reorder_state = torch.empty(0)

    def __call__(self, input_ids, first_pass=True, attention_mask=None, **_):
        self.calls += 1
        if self.calls == self.refuse_at:
            raise RuntimeError("Exceed the maximum step length")
        return torch.zeros(*input_ids.shape, 8)


class _Head:
    def greedy(self, hidden2d):
        return torch.zeros(hidden2d.shape[0], 1, dtype=torch.long)

    def sample(self, hidden2d, uniform, **settings):
        return EET.sample_rows(hidden2d, uniform, **settings)[0].view(-1, 1)   # (refused: not on a GPU)


def _lm(monkeypatch, refuse_at=None, graph=True):
    monkeypatch.setattr(EET, "check_device_status", lambda tp=None: None)
    lm = modeling._CausalLMBase(SimpleNamespace(), _Model(refuse_at), _Head())
    lm.use_cuda_graph = graph
    lm.decode_step = lambda ids: _Head().greedy(lm.model(ids, first_pass=False)[:, -1])
    return lm


IDS = torch.zeros(2, 4, dtype=torch.long)
MASK = torch.tensor([[0, 0, 1, 1], [1, 1, 1, 1]])


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("bad", [dict(temperature=-1.0), dict(top_p=2.0), dict(top_k=-3), dict(top_k=1.5), dict(min_p=torch.zeros(3)),
                                 dict(temperature=torch.zeros(2, dtype=torch.float64)), dict(min_p=float("nan"))])
def test_bad_settings_are_refused_in_front_of_the_prompt(monkeypatch, bad, graph):
    lm = _lm(monkeypatch, graph=graph)
    with pytest.raises(RuntimeError, match="sample_rows"):
        lm.generate(IDS, 3, attention_mask=MASK, do_sample=True, **bad)
    assert lm.model.calls == 0 and lm.model.pre_padding_len.numel() == 0 and lm._sampling is None and lm._graph is None


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("refuse_at,sample", [(1, False), (2, False), (3, False), (None, True), (1, True)])
def test_no_padding_stays_behind_an_error(monkeypatch, refuse_at, sample, graph):
    lm = _lm(monkeypatch, refuse_at, graph)
    with pytest.raises(RuntimeError, match="sample_rows" if refuse_at is None else "Exceed"):
        lm.generate(IDS, 5, attention_mask=MASK, do_sample=sample)
    assert lm.model.pre_padding_len.numel() == 0 and lm._sampling is None
    assert lm.generate(IDS, 2).shape == (2, 6)


def test_a_call_that_is_not_refused_takes_its_padding_and_leaves_none(monkeypatch):
    lm = _lm(monkeypatch)
    seen = []
    step = lm.decode_step
    lm.decode_step = lambda ids: seen.append(lm.model.pre_padding_len.flatten().tolist()) or step(ids)
    assert lm.generate(IDS, 3, attention_mask=MASK).shape == (2, 7)
    assert seen == [[2, 0], [2, 0]] and lm.model.pre_padding_len.numel() == 0
