"""``model.beam_search`` on the CPU, over a stand-in for the four operators that keeps their contracts: a group with
NaN logits or scores selects token -1, and a batched decode with a token out of range reports NaN for every
sequence. One failed prompt must not end the search of the others."""
import math

import pytest
import torch

VOCAB, BEAMS, NEW, MAX_SEQ = 50, 3, 5, 32


class Operators:
    def __init__(self, failed=(), fails_at=None):
        self.failed, self.fails_at, self.decodes = failed, fails_at, 0

    def _logits(self, tokens, positions):
        rows = [torch.randn(VOCAB, generator=torch.Generator().manual_seed(1000 * int(p) + int(t))) * 3
                for t, p in zip(tokens, positions)]
        return torch.stack(rows)

    def prefill_batch(self, tokens, lengths, *rest):
        assert rest[-3].shape[0] == rest[-2].shape[0] == len(lengths)
        ends = torch.tensor(lengths).cumsum(0) - 1
        logits = self._logits(tokens[ends], lengths)
        if self.fails_at is None:
            logits[list(self.failed)] = math.nan
        return logits, logits.argmax(1).int()

    def decode_batch(self, tokens, positions, *rest):
        self.decodes += 1
        if (tokens < 0).any() or (tokens >= VOCAB).any() or (positions >= MAX_SEQ).any():
            return torch.full((len(tokens), VOCAB), math.nan), torch.full_like(tokens, -1)
        logits = self._logits(tokens, positions)
        if self.decodes == self.fails_at:
            for g in self.failed:  # all of its rows: a finished one's logits are not looked at
                logits[BEAMS * g:BEAMS * (g + 1)] = math.nan
        return logits, logits.argmax(1).int()

    def beam_reorder(self, k, v, parents, begin, end, beams):
        assert ((parents // beams) == torch.arange(len(parents)) // beams).all()

    def beam_select(self, logits, scores, finished, beams, eos):
        out = ([], [], [], [])
        for g in range(0, len(scores), beams):
            rows = range(g, g + beams)
            if any(math.isnan(scores[r]) or (not finished[r] and logits[r].isnan().any()) for r in rows):
                picked = [(-1, r, math.nan, bool(finished[r])) for r in rows]
            else:
                cand = []
                for r in rows:
                    if finished[r]:
                        cand.append((-scores[r].item(), r, eos, True))
                    else:
                        logp = torch.log_softmax(logits[r].double(), 0) + scores[r].double()
                        cand += [(-s, r, t, t == eos) for t, s in enumerate(logp.tolist())]
                picked = [(t, r, -s, f) for s, r, t, f in sorted(cand)[:beams]]
            for column, values in zip(out, zip(*picked)):
                column.extend(values)
        return (torch.tensor(out[0], dtype=torch.int32), torch.tensor(out[1], dtype=torch.int32),
                torch.tensor(out[2]), torch.tensor(out[3]))


def search(operators, eos=-1):
    import model
    zero = torch.zeros(1, 1, dtype=torch.bfloat16)
    prompts = [[3, 1, 4], [1, 5, 9, 2, 6], [5, 3]]
    return model.beam_search(operators, prompts, BEAMS, NEW, eos, zero, zero, [zero] * 11, zero, zero, MAX_SEQ)


@pytest.mark.parametrize("eos", [-1, 7])
@pytest.mark.parametrize("failed", [(0,), (1,), (0, 2)], ids=str)
@pytest.mark.parametrize("fails_at", [None, 1, 3], ids=["in the prefill", "at the first step", "at a later one"])
def test_a_failed_prompt_leaves_the_others_their_search(failed, fails_at, eos):
    want = search(Operators(), eos)
    found = search(Operators(failed, fails_at), eos)
    for i in range(3):
        if i in failed:
            assert len(found[i]) == BEAMS
            assert all(tokens == [] and math.isnan(score) for tokens, score in found[i])
        else:
            assert found[i] == want[i] and all(0 <= t < VOCAB for tokens, _ in found[i] for t in tokens)
