"""generate(do_sample=True): the tokens are those that EET.sample_rows draws from the logits of each step."""
import pytest
import torch

from model_util import random_hf_state_dict, tiny_config

pytestmark = pytest.mark.gpu


def _model(B, prompt, full, lm_head_int8=False):
    from eet_b200 import modeling
    cfg = tiny_config()
    sd = random_hf_state_dict(cfg, seed=5)
    sd["lm_head.weight"] = (sd["lm_head.weight"].float() * 20).half()     # logits of a few units: some tokens likelier than others
    return cfg, modeling.EETLlamaForCausalLM.from_eet(modeling.convert_llama_weights(sd, torch.int8), cfg, B, prompt, full, torch.int8,
                                                      lm_head_int8=lm_head_int8)


def _uniform(generator, steps, B):
    return torch.rand((steps, B), generator=generator, dtype=torch.float32, device="cuda")


@pytest.mark.parametrize("graph,lm_head_int8", [(False, False), (True, False), (False, True), (True, True)])
def test_tokens_are_drawn_from_the_logits_of_each_step(graph, lm_head_int8):
    from eet_b200 import EET
    B, S, new = 3, 5, 9
    cfg, model = _model(B, 8, 32, lm_head_int8)
    ids = torch.randint(0, cfg.vocab_size, (B, S), generator=torch.Generator().manual_seed(1)).cuda()
    settings = dict(temperature=torch.tensor([0.7, 1.5, 0.0], device="cuda"), top_k=40, top_p=torch.tensor([0.9, 1.0, 0.5], device="cuda"),
                    min_p=0.01)
    model.use_cuda_graph = graph
    got = model.generate(ids, new, do_sample=True, generator=torch.Generator("cuda").manual_seed(7), **settings)
    assert got.shape == (B, S + new) and torch.equal(got[:, :S], ids)
    # the same steps by hand: each step's logits, given the tokens before
    uniform = _uniform(torch.Generator("cuda").manual_seed(7), new, B)
    model.use_cuda_graph = False
    logits = model(ids, first_pass=True).logits[:, -1, :]
    for t in range(new):
        token, _ = EET.sample_rows(logits.contiguous(), uniform[t], **settings)
        assert torch.equal(token, got[:, S + t]), f"step {t}"
        logits = model.decode_logits(token.view(B, 1))[:, -1, :]


def test_the_same_generator_draws_the_same_and_another_other_tokens():
    cfg, model = _model(2, 8, 40)
    ids = torch.randint(0, cfg.vocab_size, (2, 6), generator=torch.Generator().manual_seed(2)).cuda()
    draw = lambda seed: model.generate(ids, 20, do_sample=True, generator=torch.Generator("cuda").manual_seed(seed))  # noqa: E731
    assert torch.equal(draw(1), draw(1))
    assert not torch.equal(draw(1), draw(2))


def test_without_drawing_or_at_temperature_zero_the_tokens_are_the_greedy_ones():
    cfg, model = _model(2, 8, 24)
    ids = torch.randint(0, cfg.vocab_size, (2, 6), generator=torch.Generator().manual_seed(3)).cuda()
    for graph in (False, True):
        model.use_cuda_graph = graph
        greedy = model.generate(ids, 8)
        assert torch.equal(model.generate(ids, 8, do_sample=True, temperature=0.0), greedy)
        # a captured step that draws is not what the next greedy call replays
        model.generate(ids, 8, do_sample=True, temperature=3.0)
        assert torch.equal(model.generate(ids, 8), greedy)


def test_bad_settings_are_refused_and_leave_the_model_as_it_was():
    cfg, model = _model(2, 8, 24)
    ids = torch.randint(0, cfg.vocab_size, (2, 6), generator=torch.Generator().manual_seed(4)).cuda()
    greedy = model.generate(ids, 6)
    for bad in (dict(temperature=-1.0), dict(top_p=2.0), dict(top_k=-3), dict(min_p=torch.zeros(3, device="cuda"))):
        with pytest.raises(RuntimeError, match="sample_rows"):
            model.generate(ids, 6, do_sample=True, **bad)
    assert torch.equal(model.generate(ids, 6), greedy)
