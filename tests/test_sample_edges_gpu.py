"""EET.sample_rows where its settings or its rows are extreme, against the plain restatement in 64 bits (test_sample_gpu)."""
import math

import pytest
import torch

import test_sample_gpu
from test_sample_gpu import BF16, FP16, FP32, _check, _logits, _sample, kept64

pytestmark = pytest.mark.gpu

INF = math.inf


def _kept(x, temperature, top_k, top_p, min_p):
    """kept64, but for min_p = 1 at a finite temperature: exp(-d / T) is below 1 for every d > 0, so that only those equal to the largest stay.
    In 64 bits it is rounded to 1 where d / T is below 2^-54, and kept64, which compares that with min_p, would let such tokens stay."""
    if min_p < 1 or not 0 < torch.tensor(temperature, dtype=FP32) < INF:
        return kept64(x, temperature, top_k, top_p, min_p)
    order, w = kept64(x, temperature, top_k, top_p, 0.0)
    n = int((x[order] == x[order[:1]]).sum())
    return order[:n], w[:n]


@pytest.fixture(autouse=True)
def _oracle(monkeypatch):
    monkeypatch.setattr(test_sample_gpu, "kept64", _kept)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=1), dict(top_k=50), dict(top_k=900), dict(top_k=5000), dict(top_p=0.9), dict(top_p=0.0),
                                      dict(top_k=40, top_p=0.8), dict(top_k=6000, top_p=0.95), dict(min_p=0.02), dict(min_p=1.0),
                                      dict(top_k=100, top_p=0.9, min_p=0.5), dict(top_k=70, top_p=0.5, min_p=1.0)])
@pytest.mark.parametrize("temperature", [1e4, 1e30, 3e38, 1e39, INF])
@pytest.mark.parametrize("rows,vocab,dtype", [(3, 32001, FP16), (40, 1009, FP32), (5, 7, BF16)])
def test_sample_at_large_temperatures(settings, temperature, rows, vocab, dtype):
    """All tokens weigh nearly or exactly the same; what is -inf or NaN still cannot be drawn, the lowest number can."""
    logits, uniform = _logits(rows, vocab, dtype, 21)
    _check(logits, uniform, temperature=temperature, **settings)
    _check(logits, uniform, temperature=torch.tensor([temperature] * rows, dtype=torch.float64).float().cuda(), **settings)
    logits[:, vocab // 3:2 * vocab // 3] = -INF
    logits[:, -1] = math.nan
    _check(logits, uniform, temperature=temperature, **settings)
    logits[:, :vocab // 7] = torch.finfo(dtype).min
    _check(logits, uniform, temperature=temperature, **settings)


def test_sample_of_nothing_but_one_token_at_an_infinite_temperature():
    x = torch.full((4, 3000), -INF)
    for row, at in enumerate((0, 1499, 2999, 7)):
        x[row, at] = -5.0 * row
    tokens, logprobs = _sample(x.cuda(), torch.full((4,), 0.7, device="cuda"), temperature=INF, top_k=50, top_p=0.9, min_p=1.0)
    assert tokens.tolist() == [0, 1499, 2999, 7] and logprobs.tolist() == [0.0] * 4
