"""Prefill of several prompts in one call (``prefill_batch``, C ABI ``mk_prefill_batch``) on the GPU, and
beam search with it: prefill_batch, beam_reorder, decode_batch and beam_select together.

Each prompt is held to what a prefill of its own is held to: the fp32 restatement's last logits within 5e-3
and its greedy token, every K/V row within one bf16 rounding step of the largest values."""
import math

import pytest
import torch

from oracle import hf, restate
from tests.gpu_common import DEV, Session, stats
from tests.test_gpu_beam import oracle as select_oracle
from tests.test_gpu_prefill import _check_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mini():
    return Session("mini", 512)


@pytest.fixture(scope="module")
def mini17():
    return Session("mini-1.7b", 512)


@pytest.fixture(scope="module")
def mini_2k():
    return Session("mini", 2048)


def _prompts(sess, lengths):
    return [hf.prompt_ids(n, sess.shape.vocab, seed=20 + i)[0].tolist() for i, n in enumerate(lengths)]


def _caches(sess, rows, fill=0.0):
    s = sess.shape
    return [torch.full((rows, s.layers, s.kv_heads, sess.max_seq, s.head_dim), fill, dtype=torch.bfloat16, device=DEV)
            for _ in range(2)]


def _prefill_batch(sess, prompts, kd, vd, **kw):
    tokens = torch.tensor([t for p in prompts for t in p], dtype=torch.int32, device=DEV)
    return sess.kernel.prefill_batch(tokens, [len(p) for p in prompts], sess.embed, sess.lm_head, sess.final_norm,
                                     sess.layers, sess.cos, sess.sin, kd, vd, sess.max_seq)


def _decode_batch(sess, toks, pos, kd, vd):
    return sess.kernel.decode_batch(toks, pos, sess.embed, sess.lm_head, sess.final_norm, sess.layers, sess.cos,
                                    sess.sin, kd, vd, sess.max_seq)


def _greedy(logits):
    """The argmax of the bf16-rounded logits, the lowest index on ties."""
    x = logits.to(torch.bfloat16)
    return int((x == x.max()).nonzero()[0])


@pytest.mark.parametrize("shape_fixture, lengths", [
    ("mini", (5,)), ("mini", (1, 1, 1)), ("mini", (3, 64, 1, 65, 17)),   # skinny products
    ("mini17", (7, 31, 50)),
    ("mini", (256, 1)), ("mini", (300, 5, 129, 64)),                     # tiles, QKV split over K
    ("mini17", (40, 90, 130)),
    ("mini", (512, 511, 257, 1, 33)),                                    # tiles with fused epilogues, whole caches
    ("mini_2k", (1500, 700, 900)), ("mini17", (400, 512, 300, 512, 37)),
    ("mini", tuple(1 + 7 * i for i in range(64))),                       # the most prompts
    ("mini", tuple(1 + i % 4 for i in range(64))),
], ids=str)
def test_matches_the_oracle_per_prompt(shape_fixture, lengths, request):
    sess = request.getfixturevalue(shape_fixture)
    prompts = _prompts(sess, lengths)
    kd, vd = _caches(sess, len(lengths))
    logits, toks = _prefill_batch(sess, prompts, kd, vd)
    assert logits.shape == (len(lengths), sess.shape.vocab) and toks.dtype == torch.int32
    assert sess.kernel.status() == 0
    for i in range(0, len(lengths), max(1, len(lengths) // 8)):  # of many prompts, some
        want, kw, vw = restate.prefill(sess.W, prompts[i], sess.cos_cpu, sess.sin_cpu, sess.max_seq)
        maxabs, cos = stats(logits[i].cpu(), want)
        print(f"[prefill_batch {shape_fixture}] prompt {i} of {lengths[i]}: max|d| {maxabs:.3e}", flush=True)
        assert maxabs < 5e-3 and cos > 0.999999
        assert int(toks[i]) == restate.argmax_bf16(want) == _greedy(logits[i])
        _check_cache(kd[i], kw, lengths[i], "k")
        _check_cache(vd[i], vw, lengths[i], "v")
    for i, n in enumerate(lengths):  # nothing behind a prompt
        assert kd[i, :, :, n:].abs().sum().item() == 0 and vd[i, :, :, n:].abs().sum().item() == 0


@pytest.mark.parametrize("lengths", [(9, 40, 3), (150, 222, 90)], ids=str)
def test_strided_caches_leave_the_others_alone(mini, lengths):
    prompts = _prompts(mini, lengths)
    kd, vd = _caches(mini, 3)
    want, _ = _prefill_batch(mini, prompts, kd, vd)
    ks, vs = _caches(mini, 9, fill=7.0)
    got, _ = _prefill_batch(mini, prompts, ks[1::3], vs[1::3])
    assert torch.equal(got, want)
    for i, n in enumerate(lengths):
        assert torch.equal(ks[3 * i + 1, :, :, :n], kd[i, :, :, :n]) and (ks[3 * i + 1, :, :, n:] == 7).all()
        assert torch.equal(vs[3 * i + 1, :, :, :n], vd[i, :, :, :n])
    for t in (ks, vs):
        assert (t[0::3] == 7).all() and (t[2::3] == 7).all()


@pytest.mark.parametrize("lengths", [(9, 40, 3), (150, 222, 90)], ids=str)
def test_out_of_range_token_is_reported_in_band(mini, lengths):
    prompts = _prompts(mini, lengths)
    prompts[1][2] = mini.shape.vocab
    logits, toks = _prefill_batch(mini, prompts, *_caches(mini, 3))
    assert torch.isnan(logits).all() and toks.tolist() == [-1] * 3
    prompts[1][2] = 0
    logits, toks = _prefill_batch(mini, prompts, *_caches(mini, 3))
    assert torch.isfinite(logits).all() and min(toks.tolist()) >= 0


@pytest.mark.parametrize("lengths", [(9, 40, 3), (150, 222, 90), (500, 512, 400)], ids=str)
def test_graph_replays_match_eager(mini, lengths):
    prompts = _prompts(mini, lengths)
    tokens = torch.tensor([t for p in prompts for t in p], dtype=torch.int32, device=DEV)
    kd, vd = _caches(mini, 3)

    def call():
        return mini.kernel.prefill_batch(tokens, list(lengths), mini.embed, mini.lm_head, mini.final_norm, mini.layers,
                                         mini.cos, mini.sin, kd, vd, mini.max_seq)

    want, want_tok = (t.clone() for t in call())
    want_k, want_v = kd.clone(), vd.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_tok = call()
    for _ in range(3):
        kd.zero_()
        vd.zero_()
        got.zero_()
        float(torch.randn(1 << 18, device=DEV).mul_(2).sum())  # unrelated eager work
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(got_tok, want_tok)
        assert torch.equal(kd, want_k) and torch.equal(vd, want_v)


def test_beam_search_of_several_prompts(mini):
    """The four calls as a search makes them, 2 prompts of 3 beams for 6 steps: every selection is the one
    the definition makes of the kernel's logits, and every beam that is left at the end has the score and the
    cache that its own tokens have in the oracle."""
    lengths, beams, steps, vocab = (21, 70), 3, 6, mini.shape.vocab
    prompts, rows = _prompts(mini, lengths), 6
    kd, vd = _caches(mini, rows)
    first, _ = _prefill_batch(mini, prompts, kd[::beams], vd[::beams])
    begin = torch.tensor([n for n in lengths for _ in range(beams)], dtype=torch.int32, device=DEV)
    heads = torch.tensor([b // beams * beams for b in range(rows)], dtype=torch.int32, device=DEV)
    mini.kernel.beam_reorder(kd, vd, heads, torch.zeros_like(begin), begin, beams)
    for b in range(rows):
        assert torch.equal(kd[b], kd[b // beams * beams]) and torch.equal(vd[b], vd[b // beams * beams])
    logits = first.repeat_interleave(beams, 0)
    scores = torch.full((rows,), -math.inf, device=DEV)
    scores[::beams] = 0
    finished = torch.zeros(rows, dtype=torch.bool, device=DEV)
    eos = int(torch.topk(first[0], 2).indices[1])  # a likely token, so that some beam ends
    paths, ended, pos = [[] for _ in range(rows)], [False] * rows, begin.clone()
    for step in range(steps):
        want = select_oracle(logits, scores, finished, beams, eos)
        tokens, parents, scores, finished = mini.kernel.beam_select(logits, scores, finished, beams, eos)
        assert tokens.tolist() == want["tokens"] and parents.tolist() == want["parents"]
        mini.kernel.beam_reorder(kd, vd, parents, begin, pos, beams)
        paths = [paths[p] + ([] if ended[p] else [t]) for p, t in zip(want["parents"], want["tokens"])]
        ended = finished.tolist()
        logits, _ = _decode_batch(mini, tokens, pos, kd, vd)
        pos = pos + 1
    assert mini.kernel.status() == 0
    for b in range(rows):
        ids = prompts[b // beams] + paths[b]
        assert len(set(map(tuple, paths[b // beams * beams:][:beams]))) == beams  # no two beams alike
        total = 0.0
        for i in range(lengths[b // beams], len(ids)):
            lg, _, _ = restate.prefill(mini.W, ids[:i], mini.cos_cpu, mini.sin_cpu, mini.max_seq)
            total += torch.log_softmax(lg.double(), 0)[ids[i]].item()
        # each step's log-probability from logits within 5e-3 of the oracle's
        assert abs(scores[b].item() - total) <= 2 * 5e-3 * len(paths[b]), (b, scores[b].item(), total)
        _, kw, vw = restate.prefill(mini.W, ids, mini.cos_cpu, mini.sin_cpu, mini.max_seq)
        n = len(ids)
        _check_cache(kd[b], kw, n, f"beam {b} k")
        _check_cache(vd[b], vw, n, f"beam {b} v")


def test_many_tokens(mini_2k):
    """64 prompts of 1,000 tokens, 64,000 rows: each as alone, to summation order."""
    s = mini_2k.shape
    prompts = [hf.prompt_ids(1000, s.vocab, seed=100 + i)[0].tolist() for i in range(64)]
    kd, vd = _caches(mini_2k, 64)
    logits, toks = _prefill_batch(mini_2k, prompts, kd, vd)
    for i in (0, 31, 63):
        k1, v1 = (t[0] for t in _caches(mini_2k, 1))
        tokens = torch.tensor(prompts[i], dtype=torch.int32, device=DEV)
        want, tok = mini_2k.kernel.prefill(tokens, mini_2k.embed, mini_2k.lm_head, mini_2k.final_norm, mini_2k.layers,
                                           mini_2k.cos, mini_2k.sin, k1, v1, 0, mini_2k.max_seq)
        maxabs, _ = stats(logits[i].cpu(), want.cpu())
        print(f"[prefill_batch] prompt {i} of 64,000 tokens: max|d| {maxabs:.3e}", flush=True)
        assert maxabs < 5e-3
        _check_cache(kd[i], k1.cpu(), 1000, "k")
        _check_cache(vd[i], v1.cpu(), 1000, "v")
    assert mini_2k.kernel.status() == 0
