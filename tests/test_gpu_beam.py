"""Beam selection and cache reordering (``beam_select``, ``beam_reorder``) on the GPU against plain
implementations in 64 bits.

Tokens, parents and ends are whole numbers and must be equal: the oracle ranks by the same definition
(score in 64 bits, then row, then logit, then token). Its scores differ from the kernel's by the row sums'
fp32 rounding (about 2^-22 of the sum, at most), so two candidates of different rows may come out in another
order only where their scores are closer than that; the inputs here keep them apart. Scores are off by
half an fp32 step, 2^-24 of the score, and that sum's error, 2^-22."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def oracle(logits, scores, finished, beams, eos):
    x, sc = logits.cpu().double(), scores.cpu().double()
    fin = finished.cpu().tolist()
    out = {"tokens": [], "parents": [], "scores": [], "finished": []}
    for g in range(0, x.shape[0], beams):
        cand = []
        for r in range(g, g + beams):
            if eos >= 0 and fin[r]:
                cand.append((-sc[r].item(), r, 0.0, eos))
                continue
            lse = torch.logsumexp(x[r], 0)
            top = torch.sort(x[r], descending=True, stable=True)
            for value, token in zip(top.values[:beams].tolist(), top.indices[:beams].tolist()):
                s = -math.inf if value == -math.inf else (sc[r] + (value - lse)).item()
                cand.append((-s, r, -value, token))
        for s, r, _, t in sorted(cand)[:beams]:
            out["tokens"].append(t)
            out["parents"].append(r)
            out["scores"].append(-s)
            out["finished"].append(eos >= 0 and (fin[r] or t == eos))
    return out


def check(kernel, logits, scores, finished, beams, eos):
    print(f"[select] rows {tuple(logits.shape)} beams {beams} eos {eos}", flush=True)
    tokens, parents, out, fin = kernel.beam_select(logits, scores, finished, beams, eos)
    torch.cuda.synchronize()
    want = oracle(logits, scores, finished, beams, eos)
    assert tokens.dtype == torch.int32 and parents.dtype == torch.int32 and fin.dtype == torch.bool
    assert tokens.tolist() == want["tokens"]
    assert parents.tolist() == want["parents"]
    assert fin.tolist() == want["finished"]
    for a, b in zip(out.tolist(), want["scores"]):
        assert a == b or abs(a - b) <= 2.0 ** -24 * abs(b) + 2.0 ** -22, (a, b)


def inputs(rows, vocab, seed=0, done=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    logits = torch.randn(rows, vocab, generator=gen, device=DEV) * 3
    scores = -10 * torch.rand(rows, generator=gen, device=DEV)
    finished = torch.zeros(rows, dtype=torch.bool, device=DEV)
    finished[torch.randperm(rows, generator=gen, device=DEV)[:done]] = True
    return logits, scores, finished


@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 64, 257, 2047, 2048, 2049, 32003, 151936])
@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 4), (3, 3), (2, 16), (7, 2)])
def test_vocabularies_and_beams(kernel, vocab, groups, beams):
    logits, scores, finished = inputs(groups * beams, vocab, seed=vocab + beams, done=groups * beams // 3)
    check(kernel, logits, scores, finished, beams, eos=vocab // 2)


@pytest.mark.parametrize("groups,beams", [(2, 3), (1, 16)])
@pytest.mark.parametrize("vocab", [600001, 1 << 20])
def test_largest_vocabularies(kernel, vocab, groups, beams):
    """More chunks of a row than a wave has lanes, and more keys of them than its lanes read at once."""
    logits, scores, finished = inputs(groups * beams, vocab, seed=beams, done=1)
    check(kernel, logits, scores, finished, beams, eos=vocab - 1)
    logits[:] = 0.5  # all equal: the lowest tokens
    logits[:, vocab - 7:] = 2.0
    check(kernel, logits, scores, finished, beams, eos=3)


def test_first_step_from_one_live_beam(kernel):
    """Only the first beam of a group is live at the start: the others' scores are -infinity."""
    logits, scores, finished = inputs(8, 5000, seed=3)
    logits[:] = logits[:1]
    scores[:] = -math.inf
    scores[0] = scores[4] = 0.0
    check(kernel, logits, scores, finished, 4, -1)


def test_logits_shared_by_stride(kernel):
    logits, scores, finished = inputs(1, 3001, seed=4)
    scores = torch.tensor([0.0, -math.inf, -math.inf], device=DEV)
    check(kernel, logits.expand(3, -1), scores, finished.expand(3).contiguous(), 3, 7)
    wide = torch.randn(6, 4099, device=DEV)
    check(kernel, wide[:, 3:3003], torch.zeros(6, device=DEV) - torch.arange(6, device=DEV) * 0.37,
          torch.zeros(6, dtype=torch.bool, device=DEV), 3, 7)


@pytest.mark.parametrize("beams", [1, 5, 16])
def test_equal_logits_take_the_lowest_tokens(kernel, beams):
    """Whole rows of one value (more equals than a wave's short list holds), and of two."""
    for vocab in (40, 3000, 6001):
        logits = torch.zeros(beams, vocab, device=DEV)
        scores = -torch.arange(beams, device=DEV).float()
        fin = torch.zeros(beams, dtype=torch.bool, device=DEV)
        check(kernel, logits, scores, fin, beams, -1)
        logits[:, vocab // 2:] = 1.0
        logits[:, vocab // 3] = -0.0
        check(kernel, logits, scores, fin, beams, -1)


def test_masked_vocabulary(kernel):
    """-infinity logits (a constrained vocabulary) only fill up; a row of nothing else is no failure."""
    logits, scores, finished = inputs(6, 9000, seed=5)
    logits[:, 2:] = -math.inf
    logits[4] = -math.inf
    logits[0, 1] = -math.inf
    check(kernel, logits, scores, finished, 3, 1)
    logits[:] = -math.inf
    check(kernel, logits, scores, finished, 3, 1)


def test_all_finished(kernel):
    logits, scores, _ = inputs(8, 300, seed=6)
    check(kernel, logits, scores, torch.ones(8, dtype=torch.bool, device=DEV), 4, 299)
    check(kernel, logits, scores, torch.ones(8, dtype=torch.bool, device=DEV), 4, -1)  # nothing ends


@pytest.mark.parametrize("what", ["nan logit", "inf logit", "nan row", "nan score", "inf score"])
def test_a_failed_row_shows_in_its_group_alone(kernel, what):
    logits, scores, finished = inputs(12, 6000, seed=7, done=0)
    if what == "nan logit":
        logits[5, 4321] = math.nan
    elif what == "inf logit":
        logits[5, 17] = math.inf
    elif what == "nan row":
        logits[5] = math.nan
    else:
        scores[5] = math.nan if what == "nan score" else math.inf
    tokens, parents, out, fin = kernel.beam_select(logits, scores, finished, 4, 11)
    assert tokens[4:8].tolist() == [-1] * 4 and parents[4:8].tolist() == [4, 5, 6, 7]
    assert torch.isnan(out[4:8]).all() and not fin[4:8].any()
    keep = [0, 1, 2, 3, 8, 9, 10, 11]
    want = oracle(logits[keep], scores[keep], finished[keep], 4, 11)
    assert tokens[keep].tolist() == want["tokens"]
    assert parents[keep].tolist() == [keep[p] for p in want["parents"]]


# ---------------------------------------------------------------------------------------------------
def caches(rows, layers, max_seq, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(rows, layers, 8, max_seq, 128, generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2)]


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def reorder_check(kernel, k, v, parents, begin, end, beams):
    print(f"[reorder] {tuple(k.shape)} parents {parents} {begin} {end}", flush=True)
    want = []
    S = k.shape[3]
    for t in (k, v):
        new = t.clone()
        for b, p in enumerate(parents):
            if p // beams == b // beams and p >= 0:
                lo, hi = max(0, begin[b]), min(S, end[b])
                if lo < hi:
                    new[b, :, :, lo:hi] = t[p, :, :, lo:hi]
        want.append(new)
    kernel.beam_reorder(k, v, i32(parents), i32(begin), i32(end), beams)
    torch.cuda.synchronize()
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize("beams,parents", [
    (1, [0, 1]), (2, [1, 0, 2, 2]), (3, [1, 2, 0, 5, 5, 5]), (4, [0, 0, 0, 0, 7, 6, 5, 4]),
    (5, [4, 0, 1, 1, 0]), (16, [(7 * i + 3) % 16 for i in range(16)]),
    (8, [1, 0, 3, 2, 2, 2, 7, 6, 9, 10, 11, 12, 13, 14, 15, 8])], ids=str)
def test_reorder_maps(kernel, beams, parents):
    """Cycles, swaps and one parent for all, over ranges that fill no step."""
    rows = len(parents)
    k, v = caches(rows, 3, 77, seed=rows)
    begin = [5 + 3 * (b // beams) for b in range(rows)]
    reorder_check(kernel, k, v, parents, begin, [n + 41 for n in begin], beams)


def test_reorder_ranges(kernel):
    """Whole caches, nothing, ranges past both ends, and ranges of a group that differ."""
    for begin, end in (([0] * 4, [64] * 4), ([9] * 4, [9] * 4), ([-7] * 4, [1000] * 4), ([40] * 4, [3] * 4),
                       ([0, 10, 63, 64], [1, 20, 64, 64]), ([64] * 4, [70] * 4)):
        k, v = caches(4, 2, 64, seed=1)
        reorder_check(kernel, k, v, [3, 2, 1, 0], begin, end, 4)


def test_reorder_leaves_rows_whose_parent_is_elsewhere(kernel):
    k, v = caches(6, 2, 33, seed=2)
    reorder_check(kernel, k, v, [-1, 0, 3, 2, 9, 2 ** 31 - 1], [0] * 6, [33] * 6, 3)


# ---------------------------------------------------------------------------------------------------
def test_calls_on_two_streams_at_once(kernel):
    """Each call has a workspace of its own."""
    sets = [inputs(32, 100003, seed=20 + i, done=5) for i in range(2)]
    want = [kernel.beam_select(*s, 8, 77) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(8):
        for i, (stream, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(stream):
                got[i].append(kernel.beam_select(*s, 8, 77))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_a_step_in_a_graph(kernel):
    """Selection and reordering captured together and replayed on other logits and other caches."""
    rows, beams, L, S = 8, 4, 2, 96
    logits, scores, finished = inputs(rows, 20011, seed=30, done=1)
    k, v = caches(rows, L, S, seed=31)
    begin, end = i32([10] * 4 + [33] * 4), i32([60] * 4 + [90] * 4)

    def step():
        out = kernel.beam_select(logits, scores, finished, beams, 5)
        kernel.beam_reorder(k, v, out[1], begin, end, beams)
        return out

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (32, 33, 34):
        for old, new in zip((logits, scores, finished), inputs(rows, 20011, seed=seed, done=2)):
            old.copy_(new)
        for old, new in zip((k, v), caches(rows, L, S, seed=seed)):
            old.copy_(new)
        k0, v0 = k.clone(), v.clone()
        want = step()
        want_k, want_v = k.clone(), v.clone()
        k.copy_(k0)
        v.copy_(v0)
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_offsets_past_32_bits(kernel):
    """Caches whose elements, and logits whose bytes, pass 2^32."""
    rows, L, S = 16, 28, 4096
    k, v = (torch.zeros(rows, L, 8, S, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for t in (k, v):
        for b in range(rows):
            t[b, :, :, S - 40:] = torch.randn(L, 8, 40, 128, device=DEV, dtype=torch.bfloat16)
    tail = [t[:, :, :, S - 40:].clone() for t in (k, v)]
    parents = [15, 14, 13, 12, 0, 0, 0, 0, 8, 9, 1, 2, 3, 4, 5, 6]
    kernel.beam_reorder(k, v, i32(parents), i32([S - 33] * rows), i32([S] * rows), 16)
    for t, old in zip((k, v), tail):
        now = t[:, :, :, S - 40:]
        assert torch.equal(now[:, :, :, :7], old[:, :, :, :7])
        for b, p in enumerate(parents):
            assert torch.equal(now[b, :, :, 7:], old[p, :, :, 7:])
        assert (t[:, :, :, :S - 40] == 0).all()
    del k, v, tail
    wide = torch.zeros(1 << 31, device=DEV).view(4, 1 << 29)
    logits = wide[:, -50000:]
    logits.copy_(torch.randn(4, 50000, device=DEV))
    check(kernel, logits, torch.tensor([-1.0, -2.5, -1.25, -3.0], device=DEV),
          torch.zeros(4, dtype=torch.bool, device=DEV), 4, 9)


@pytest.mark.parametrize("gap", [3.0, 5.5, 7.3, 8.0, 9.77, 11.2, 15.9, 20.0])
@pytest.mark.parametrize("base", [0.0, -3.3, 40.7, -300.1], ids=str)
def test_sums_of_equal_logits_under_peaks(kernel, gap, base):
    """Rows of one value with a peak here and there: 151,936 equal terms, whose roundings all point one way."""
    rows, vocab = 6, 151936
    logits = torch.full((rows, vocab), base, device=DEV)
    logits[0:2, 5] = base + gap        # one peak
    logits[2:4, 5::2048] = base + gap  # one for each 2,048 logits
    logits[4:6, 5::8192] = base + gap
    scores = -torch.arange(rows, device=DEV) * 0.125
    check(kernel, logits, scores, torch.zeros(rows, dtype=torch.bool, device=DEV), 2, -1)


@pytest.mark.parametrize("apart", [6e-7, -6e-7])
@pytest.mark.parametrize("gap", [5.5, 7.3, 9.77])
def test_nearly_equal_candidates_of_two_rows(kernel, gap, apart):
    """The best of a row of peaks on a floor of equal logits, and of a scattered row, 6e-7 apart either way: more than
    the 2^-22 that the sums may be off."""
    vocab = 151936
    logits = torch.randn(2, vocab, generator=torch.Generator(device=DEV).manual_seed(9), device=DEV)
    logits[0] = 0.0
    logits[0, 5::2048] = gap
    logits[1, 77] = float(logits[1].max() + 1.0)
    for _ in range(40):  # the second row's best logit so that the rows are nearly equal, then its score
        x = logits.cpu().double()
        best = x[:, [5, 77]].diagonal() - torch.logsumexp(x, 1)
        logits[1, 77] += (best[0] - best[1]).item()
    scores = torch.tensor([0.0, (best[0] - best[1]).item() - apart], device=DEV)
    x = logits.cpu().double()
    best = x[:, [5, 77]].diagonal() - torch.logsumexp(x, 1) + scores.cpu().double()
    assert abs(best[0] - best[1] - apart).item() < 1e-7 and x[1].argmax() == 77
    check(kernel, logits, scores, torch.zeros(2, dtype=torch.bool, device=DEV), 2, -1)


@pytest.mark.parametrize("lowest", [-1e30, torch.finfo(torch.float32).min, -math.inf], ids=str)
def test_masks_of_the_lowest_value(kernel, lowest):
    """A constrained vocabulary masked with the type's lowest value. A row that holds nothing else is an even one, of
    probabilities 1 / vocabulary, and no row's best: the oracle takes the logits less their row's maximum, by which
    64 bits hold a logarithm of the sum beside such a number."""
    logits, scores, finished = inputs(6, 20000, seed=8)
    logits[:, 7000:] = lowest
    logits[3:] = lowest
    if lowest == -math.inf:
        logits[3:, 0] = -50.0
    logits[1] = lowest if lowest > -math.inf else 0.0
    want = oracle(logits.double() - logits.double().amax(1, keepdim=True), scores, finished, 3, 1)
    print(f"[select] masks of {lowest}", flush=True)
    tokens, parents, out, fin = kernel.beam_select(logits, scores, finished, 3, 1)
    assert tokens.tolist() == want["tokens"] and parents.tolist() == want["parents"]
    assert fin.tolist() == want["finished"]
    for a, b in zip(out.tolist(), want["scores"]):
        assert abs(a - b) <= 2.0 ** -24 * abs(b) + 2.0 ** -22, (a, b)
