"""``model.sample_texts`` at settings beyond what single precision and 32-bit integers hold, on the CPU over the stand-in of
``test_sample_texts``."""
import torch

from test_sample_texts import MAX_SEQ, NEW, PROMPTS, Operators


def settings(temperature, top_k, top_p=1.0, min_p=0.0):
    import model
    op, zero = Operators(), torch.zeros(1, 1, dtype=torch.bfloat16)
    texts = model.sample_texts(op, PROMPTS, NEW, -1, temperature, top_k, top_p, min_p, 0, zero, zero, [zero] * 11, zero, zero,
                               MAX_SEQ)
    assert all(len(t) == NEW for t, _ in texts)
    return [s[0] for s in op.settings]


def test_more_candidates_than_an_int32_counts_are_all():
    assert settings(1.0, 3_000_000_000)[1] == 2 ** 31 - 1
    assert settings(1.0, 2 ** 31 - 1)[1] == 2 ** 31 - 1


def test_temperatures_above_single_precision_are_its_largest():
    largest = torch.finfo(torch.float32).max
    assert settings(1e39, 0)[0] == largest
    assert settings(1e308, 0)[0] == largest
    assert settings(3e38, 0)[0] == torch.tensor(3e38).item()
