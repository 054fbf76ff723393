"""The driver's sampling (``model.py --temperature T --prompts S``) on the 0.6B shape: temperature 0 is the greedy
generation, and drawn texts score what their own tokens do when the decode kernel is fed them one by one."""
import pytest
import torch

from test_gpu_beam_driver import ARGS, NEW, _logits_along

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def driver():
    import model
    return model


def test_temperature_0_is_the_first_of_the_largest_logits(driver):
    import megakernel
    r = driver.run(ARGS + ["--temperature", "0", "--prompts", "2"])
    assert r["status"] == 0
    for prompt, (tokens, score) in zip(r["prompts"], r["texts"]):
        assert score == 0 and len(tokens) == NEW
        for lg, t in zip(_logits_along(megakernel.load(), r["inputs"], prompt + tokens[:-1], len(prompt)), tokens):
            assert lg[t] >= lg.max() - 2e-2  # two fp32-accurate paths, each logit within 1e-2


def test_texts_score_what_their_tokens_do(driver):
    import megakernel
    r = driver.run(ARGS + ["--temperature", "0.7", "--prompts", "3", "--seed", "5"])
    assert r["status"] == 0 and len(r["texts"]) == 3
    for prompt, (tokens, score) in zip(r["prompts"], r["texts"]):
        total = 0.0
        for lg, t in zip(_logits_along(megakernel.load(), r["inputs"], prompt + tokens[:-1], len(prompt)), tokens):
            total += torch.log_softmax(lg.double() / 0.7, 0)[t].item()
        assert abs(total - score) <= 2 * 1e-2 / 0.7 * NEW
    again = driver.run(ARGS + ["--temperature", "0.7", "--prompts", "3", "--seed", "5"])
    other = driver.run(ARGS + ["--temperature", "0.7", "--prompts", "3", "--seed", "6"])
    assert again["texts"] == r["texts"] and other["texts"] != r["texts"]
    few = driver.run(ARGS + ["--temperature", "0.7", "--top-k", "20", "--top-p", "0.9", "--min-p", "0.1", "--prompts", "2"])
    assert few["status"] == 0 and all(s <= 0 for _, s in few["texts"])


def test_command_line(driver):
    assert driver.main(ARGS + ["--temperature", "1.0", "--prompts", "4", "--eos", "7"]) == 0
