"""A generate() that is refused leaves no left padding behind, neither for the next call nor for one of another batch size."""
import pytest
import torch

from test_generate_sampling_gpu import _model

pytestmark = pytest.mark.gpu


def _logits(model, ids, **more):
    return model(ids, first_pass=True, **more).logits.clone()


@pytest.mark.parametrize("graph", [False, True])
def test_a_refused_call_with_padding_leaves_the_next_ones_as_they_were(graph):
    cfg, model = _model(3, 8, 24)
    gen = torch.Generator().manual_seed(8)
    ids = torch.randint(0, cfg.vocab_size, (3, 6), generator=gen).cuda()
    mask = torch.ones(2, 6, dtype=torch.long)
    mask[0, :3] = 0
    model.use_cuda_graph = graph
    plain = [_logits(model, ids[:b]) for b in (1, 2, 3)]
    assert not torch.equal(_logits(model, ids[:2], attention_mask=mask.cuda()), plain[1])      # (the tokens alone would not show it)
    tokens = [model.generate(ids[:b], 6) for b in (1, 2, 3)]
    padded = model.generate(ids[:2], 6, attention_mask=mask.cuda())
    for call in (dict(do_sample=True, top_p=2.0), dict(do_sample=True, temperature=torch.ones(3, device="cuda")), dict(max_new_tokens=100)):
        with pytest.raises(RuntimeError):
            model.generate(ids[:2], **dict(dict(max_new_tokens=6), **call), attention_mask=mask.cuda())
        for b in (1, 2, 3):
            assert torch.equal(_logits(model, ids[:b]), plain[b - 1])
            assert torch.equal(model.generate(ids[:b], 6), tokens[b - 1])
        assert torch.equal(model.generate(ids[:2], 6, attention_mask=mask.cuda()), padded)
