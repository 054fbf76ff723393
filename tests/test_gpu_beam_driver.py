"""The driver's beam search (``model.py --beams W --prompts S``) on the 0.6B shape: one beam is the greedy
generation, and every beam's score is what its own tokens score when the decode kernel is fed them one by one."""
import pytest
import torch

pytestmark = pytest.mark.gpu

NEW = 5
ARGS = ["--shape", "qwen3-0.6b", "--prompt", "24", "--max-seq", "64", "--new", str(NEW)]


@pytest.fixture(scope="module")
def driver():
    import model
    return model


def _logits_along(kernel, inp, ids, upto):
    """Logits after every prefix of ids from `upto` tokens on, by prefill and single-sequence decodes."""
    L, dev = len(inp["layer_weights"]) // 11, inp["embed"].device
    kd, vd = (torch.zeros(L, 8, inp["max_seq"], 128, dtype=torch.bfloat16, device=dev) for _ in range(2))
    w = (inp["embed"], inp["embed"], inp["final_norm"], inp["layer_weights"], inp["cos"], inp["sin"], kd, vd)
    out, _ = kernel.prefill(torch.tensor(ids[:upto], dtype=torch.int32, device=dev), *w, 0, inp["max_seq"])
    yield out
    for i in range(upto, len(ids)):
        yield kernel.decode(ids[i], *w, i, inp["max_seq"])


def test_beams_score_what_their_tokens_do(driver):
    import megakernel
    kernel = megakernel.load()
    r = driver.run(ARGS + ["--beams", "3", "--prompts", "2"])
    assert r["status"] == 0 and len(r["beams"]) == 2
    for prompt, group in zip(r["prompts"], r["beams"]):
        assert [s for _, s in group] == sorted((s for _, s in group), reverse=True)
        assert len({tuple(t) for t, _ in group}) == 3
        for tokens, score in group:
            assert len(tokens) == NEW
            total = 0.0
            for lg, t in zip(_logits_along(kernel, r["inputs"], prompt + tokens[:-1], len(prompt)), tokens):
                total += torch.log_softmax(lg.double(), 0)[t].item()
            # each step's logits from two fp32-accurate paths, within 1e-2 of each other
            assert abs(total - score) <= 2 * 1e-2 * NEW, (total, score)


def test_an_end_stops_a_beam(driver):
    """With the best first token as the end, the beam that takes it has no others and keeps its score."""
    r = driver.run(ARGS + ["--beams", "2"])
    first = r["beams"][0][0][0][0]
    e = driver.run(ARGS + ["--beams", "2", "--eos", str(first)])
    ended = [(t, s) for t, s in e["beams"][0] if t[-1] == first]
    assert ended and ended[0][0] == [first]
    assert e["beams"][0][0][0] == [first]  # nothing that goes on can pass it: log-probabilities only fall


def test_command_line(driver):
    assert driver.main(ARGS + ["--beams", "4", "--prompts", "3"]) == 0
    with pytest.raises(SystemExit):
        driver.main(ARGS + ["--beams", "17"])


def test_a_failed_prompt_leaves_the_others_their_search(driver):
    """One prompt's logits are NaN (as a failed call reports them): its group is reported as failed, and the other
    prompt's beams are those of a search in which nothing failed."""
    import megakernel
    r = driver.run(ARGS + ["--beams", "3", "--prompts", "2"])
    inp = r["inputs"]

    class Fails:
        def __getattr__(self, name):
            return getattr(megakernel.load(), name)

        def prefill_batch(self, *a):
            logits, tokens = megakernel.load().prefill_batch(*a)
            logits[0] = float("nan")
            return logits, tokens

    found = driver.beam_search(Fails(), r["prompts"], 3, NEW, -1, inp["embed"], inp["final_norm"], inp["layer_weights"],
                               inp["cos"], inp["sin"], inp["max_seq"])
    assert len(found[0]) == 3
    for tokens, score in found[0]:
        assert tokens == [] and score != score
    assert [t for t, _ in found[1]] == [t for t, _ in r["beams"][1]]
    assert [s for _, s in found[1]] == pytest.approx([s for _, s in r["beams"][1]], abs=1e-6)
