"""``model.sample_texts`` and its command line on the CPU, over a stand-in for the operators that keeps their contracts: a
row of NaN logits gets token -1, and a batched decode with a token out of range reports NaN for every sequence."""
import math

import pytest
import torch

VOCAB, NEW, MAX_SEQ = 50, 6, 32
PROMPTS = [[3, 1, 4], [1, 5, 9, 2, 6], [5, 3]]


class Operators:
    def __init__(self, failed=(), fails_at=0):
        self.failed, self.fails_at, self.samples, self.settings = failed, fails_at, 0, None

    def _logits(self, tokens, positions):
        return torch.stack([torch.randn(VOCAB, generator=torch.Generator().manual_seed(1000 * int(p) + int(t))) * 3
                            for t, p in zip(tokens, positions)])

    def prefill_batch(self, tokens, lengths, *rest):
        assert rest[-3].shape[0] == rest[-2].shape[0] == len(lengths) and rest[-1] == MAX_SEQ
        return self._logits(tokens[torch.tensor(lengths).cumsum(0) - 1], lengths), None

    def decode_batch(self, tokens, positions, *rest):
        if (tokens < 0).any() or (tokens >= VOCAB).any() or (positions >= MAX_SEQ).any():
            return torch.full((len(tokens), VOCAB), math.nan), None
        return self._logits(tokens, positions), None

    def sample(self, logits, uniforms, temperature, top_k, top_p, min_p):
        self.settings = [t.tolist() for t in (temperature, top_k, top_p, min_p)]
        p = torch.softmax(logits.double() / temperature.double()[:, None], 1)
        tokens = (p.cumsum(1) > uniforms.double()[:, None]).int().argmax(1).int()
        logprobs = p.gather(1, tokens.long()[:, None]).log()[:, 0].float()
        bad = logits.isnan().any(1)
        if self.samples == self.fails_at:
            bad[list(self.failed)] = True
        self.samples += 1
        tokens[bad], logprobs[bad] = -1, math.nan
        return tokens, logprobs


def texts(operators, eos=-1, seed=0):
    import model
    zero = torch.zeros(1, 1, dtype=torch.bfloat16)
    return model.sample_texts(operators, PROMPTS, NEW, eos, 0.75, 7, 0.5, 0.25, seed, zero, zero, [zero] * 11, zero, zero,
                              MAX_SEQ)


def test_the_random_numbers_decide():
    first, again, other = texts(Operators()), texts(Operators()), texts(Operators(), seed=1)
    assert first == again and first != other
    assert all(len(t) == NEW and all(0 <= x < VOCAB for x in t) and lp < 0 for t, lp in first)
    op = Operators()
    texts(op)
    assert op.settings == [[0.75] * 3, [7] * 3, [0.5] * 3, [0.25] * 3]


def test_an_end_stops_a_text():
    want = texts(Operators())
    eos = want[1][0][2]
    got = texts(Operators(), eos)
    for (tokens, lp), (full, total) in zip(got, want):
        cut = full.index(eos) + 1 if eos in full else NEW
        assert tokens == full[:cut] and (cut < NEW or lp == total)


@pytest.mark.parametrize("failed", [(0,), (1, 2)], ids=str)
@pytest.mark.parametrize("fails_at", [0, 3])
def test_a_failed_prompt_leaves_the_others_their_texts(failed, fails_at):
    want, got = texts(Operators()), texts(Operators(failed, fails_at))
    for i in range(3):
        if i in failed:
            assert got[i][0] == want[i][0][:fails_at] and math.isnan(got[i][1])
        else:
            assert got[i] == want[i]


@pytest.mark.parametrize("args", [["--beams", "2"], ["--device-loop"], ["--native-prefill"], ["--top-p", "1.5"], ["--min-p", "-1"],
                                  ["--top-k", "-2"], ["--prompts", "65"], ["--prompts", "0"], ["--prompt", "512"]], ids=" ".join)
def test_command_line_refusals(args, capsys):
    import model
    with pytest.raises(SystemExit):
        model.run(["--temperature", "0.8"] + args)
    assert "--temperature" in capsys.readouterr().err
    for bad in ("-1", "nan", "inf"):
        with pytest.raises(SystemExit):
            model.run(["--temperature", bad])
