"""The operators that serving several sequences at once needs beside the batched decode, and the calls
their speed is judged by: causal attention over packed prompts, beam search's selection over beams and
vocabulary, and the reordering of the beams' K/V caches.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` builds what a program
holds before the call, ``run`` makes one call: with ``own`` false in elementary torch operations, with ``own``
true through the framework's entry points. ``work`` counts the bytes and operations the call cannot do
without, ``exact`` computes the same outputs in 64 bits.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mega-kernel_amd")

# the models' geometry: 28 layers, 16 query and 8 K/V heads of 128, vocabulary 151936
LAYERS, HQ, HKV, D, VOCAB = 28, 16, 8, 128, 151936


def listed():
    return [
        # One short question: the smallest attention, where latency counts.
        {"name": "attention-32", "op": "attention", "dtype": "bf16", "hq": HQ, "hkv": HKV, "lengths": "32",
         "fused": False},
        # A few users' prompts of a chat, one of them a single token, straight from a fused projection.
        {"name": "attention-chat", "op": "attention", "dtype": "bf16", "hq": HQ, "hkv": HKV,
         "lengths": "131,7,64,300,1,48", "fused": True},
        # A server's batch of prompts at the precision of the framework's activations.
        {"name": "attention-16-fp32", "op": "attention", "dtype": "fp32", "hq": HQ, "hkv": HKV, "count": 16, "lo": 33,
         "hi": 288, "fused": False},
        # A busy server's batch: prompts of very different lengths.
        {"name": "attention-64", "op": "attention", "dtype": "bf16", "hq": HQ, "hkv": HKV, "count": 64, "lo": 64,
         "hi": 960, "fused": True},
        # A long document at the precision of the framework's activations.
        {"name": "attention-3584-fp32", "op": "attention", "dtype": "fp32", "hq": HQ, "hkv": HKV, "lengths": "3584",
         "fused": False},
        # Long documents together: the largest attention.
        {"name": "attention-long", "op": "attention", "dtype": "bf16", "hq": HQ, "hkv": HKV,
         "lengths": "8192,1801,4096", "fused": False},
        # One user's search with four beams: the smallest selection.
        {"name": "select-4", "op": "select", "groups": 1, "beams": 4, "vocab": VOCAB, "done": 0},
        # An odd number of users and beams over a vocabulary whose rows end anywhere.
        {"name": "select-5x3-odd", "op": "select", "groups": 5, "beams": 3, "vocab": 32003, "done": 2},
        # The largest batch of the batched decode, some of its beams at their end already.
        {"name": "select-8x8", "op": "select", "groups": 8, "beams": 8, "vocab": VOCAB, "done": 9},
        # One user's beams some way into an answer.
        {"name": "reorder-4", "op": "reorder", "groups": 1, "beams": 4, "max_seq": 512, "prompt_lo": 32,
         "prompt_hi": 32, "new": 128},
        # An odd number of users and beams, prompts of different lengths.
        {"name": "reorder-5x3", "op": "reorder", "groups": 5, "beams": 3, "max_seq": 1024, "prompt_lo": 7,
         "prompt_hi": 640, "new": 301},
        # The largest batch near the end of long answers.
        {"name": "reorder-8x8", "op": "reorder", "groups": 8, "beams": 8, "max_seq": 512, "prompt_lo": 33,
         "prompt_hi": 96, "new": 400},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "select", "select", "reorder"])
    if op == "attention":
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        hq, hkv = rng.choice([(HQ, HKV), (HQ, HKV), (HQ, HKV), (8, 8), (16, 2), (12, 4), (5, 1)])
        most = 4096 if dtype == "bf16" else 1792
        if rng.random() < 0.5:
            lens = [_spread(rng, 1, most) for _ in range(rng.randint(1, 4))]
            c = {"lengths": ",".join(str(n) for n in lens)}
        else:
            a, b = _spread(rng, 1, 1024), _spread(rng, 1, 1024)
            c = {"count": _spread(rng, 2, 64 if dtype == "bf16" else 24), "lo": min(a, b), "hi": max(a, b)}
        return {"op": op, "dtype": dtype, "hq": hq, "hkv": hkv, "fused": rng.random() < 0.5, **c}
    beams = rng.choice([1, 2, 3, 4, 5, 6, 8]) if op == "select" else rng.choice([2, 3, 4, 5, 6, 8])
    groups = _spread(rng, 1, 64 // beams)
    if op == "select":
        vocab = rng.choice([VOCAB, VOCAB, _spread(rng, 1000, VOCAB)])
        return {"op": op, "groups": groups, "beams": beams, "vocab": vocab, "done": rng.randint(0, groups * beams // 2)}
    max_seq = rng.choice([256, 512])
    lo = _spread(rng, 1, max_seq // 2)
    hi = rng.randint(lo, max_seq // 2)
    return {"op": op, "groups": groups, "beams": beams, "max_seq": max_seq, "prompt_lo": lo, "prompt_hi": hi,
            "new": _spread(rng, 1, max_seq - hi)}


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
def _even(lo, hi, count):
    return [lo + (hi - lo) * i // max(1, count - 1) for i in range(count)]


def _lengths(case):
    if "lengths" in case:
        return [int(n) for n in case["lengths"].split(",")]
    return _even(case["lo"], case["hi"], case["count"])


def _reorder_rows(case):
    """(changed rows, distinct parents of changed rows) of one group: half of the beams go on, the others
    are replaced by children of theirs."""
    stay = (case["beams"] + 1) // 2
    return case["beams"] - stay, min(stay, case["beams"] - stay)


def _inputs(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    order = random.Random(int(seed))
    s = {"case": case}
    if case["op"] == "attention":
        lens = _lengths(case)
        order.shuffle(lens)
        n, hq, hkv = sum(lens), case["hq"], case["hkv"]
        # queries and keys as their norms and rotations leave them (about 1; some heads attend sharply),
        # values as a projection of a normalised row
        q = torch.randn(n, hq, D, generator=gen, device=dev)
        q *= torch.exp(0.5 * torch.randn(1, hq, 1, generator=gen, device=dev))
        k = torch.randn(n, hkv, D, generator=gen, device=dev)
        v = torch.randn(n, hkv, D, generator=gen, device=dev) * 0.64
        if case["fused"] and case["dtype"] == "bf16":  # one projection's rows: q, k and v are slices of them
            rows = torch.cat([q, k, v], dim=1).to(torch.bfloat16)
            q, k, v = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:]
        else:
            q = q.to(torch.bfloat16) if case["dtype"] == "bf16" else q
            if case["fused"]:  # the keys and values of one projection
                rows = torch.cat([k, v], dim=1).to(torch.bfloat16)
                k, v = rows[:, :hkv], rows[:, hkv:]
            else:
                k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        s.update(q=q, k=k, v=v, lengths=lens)
    elif case["op"] == "select":
        n, vocab = case["groups"] * case["beams"], case["vocab"]
        # logits as a language model gives them: most far below a few favourites, of which beams share some
        x = torch.randn(n, vocab, generator=gen, device=dev) * 2
        likely = torch.randint(0, vocab, (n, 24), generator=gen, device=dev)
        x.scatter_add_(1, likely, 6 + 3 * torch.randn(n, 24, generator=gen, device=dev))
        done = torch.zeros(n, dtype=torch.bool)
        done[order.sample(range(n), case["done"])] = True
        s.update(logits=x, scores=-20 - 4 * torch.rand(n, generator=gen, device=dev), finished=done.to(dev),
                 eos=order.randrange(vocab))
    else:
        groups, beams, T = case["groups"], case["beams"], case["max_seq"]
        dims = (groups * beams, LAYERS, HKV, T, D)
        s["k"] = torch.randn(dims, generator=gen, device=dev, dtype=torch.bfloat16)
        s["v"] = torch.randn(dims, generator=gen, device=dev, dtype=torch.bfloat16).mul_(0.64)
        parents, first = [], _even(case["prompt_lo"], case["prompt_hi"], groups)
        order.shuffle(first)
        changed, _ = _reorder_rows(case)
        for g in range(groups):
            rows = list(range(g * beams, (g + 1) * beams))
            order.shuffle(rows)
            to = {r: r for r in rows[changed:]}
            to.update({r: rows[changed + i % (beams - changed)] for i, r in enumerate(rows[:changed])})
            parents += [to[r] for r in range(g * beams, (g + 1) * beams)]
        s["parents_list"] = parents
        s["begin_list"] = [n for n in first for _ in range(beams)]
        s["end_list"] = [n + case["new"] for n in s["begin_list"]]
        for name in ("parents", "begin", "end"):
            s[name] = torch.tensor(s[name + "_list"], dtype=torch.int32, device=dev)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        if _PACKAGE not in sys.path:
            sys.path.insert(0, _PACKAGE)
        import megakernel
        s["kernel"] = megakernel.load()
    return s


# ---------------------------------------------------------------------------------------------------
# one call
# ---------------------------------------------------------------------------------------------------
def _plain_attention(q, k, v, lengths):
    out, at = torch.empty(q.shape, dtype=q.dtype, device=q.device), 0
    heads = k.shape[1]
    g = q.shape[1] // heads
    for n in lengths:
        rows = slice(at, at + n)
        later = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        # the query heads of a K/V head in one product, the K/V heads as its batch
        qq = q[rows].float().view(n, heads, g, D).permute(1, 2, 0, 3).reshape(heads, g * n, D)
        sc = torch.bmm(qq, k[rows].float().permute(1, 2, 0).contiguous()).mul_(D ** -0.5).view(heads, g, n, n)
        sc.masked_fill_(later, -math.inf)
        p = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
        o = torch.bmm(p.view(heads, g * n, n), v[rows].float().transpose(0, 1).contiguous()).view(heads, g, n, D)
        out[rows] = (o / p.sum(-1, keepdim=True)).permute(2, 0, 1, 3).reshape(n, heads * g, D).to(q.dtype)
        at += n
    return out


def _plain_select(logits, scores, finished, beams, eos):
    """The candidates' scores in 64 bits, since two of them may lie closer than 32 bits tell apart."""
    n, vocab = logits.shape
    x = logits.double()
    m = x.amax(1, keepdim=True)
    lse = m + (x - m).exp().sum(1, keepdim=True).log()
    cand = x - lse + scores.double()[:, None]
    only = torch.full((1, vocab), -math.inf, dtype=cand.dtype, device=cand.device)
    only[0, eos] = 0
    cand = torch.where(finished[:, None], only + scores.double()[:, None], cand)
    cand = cand.view(n // beams, beams * vocab)
    index = torch.arange(beams * vocab, device=cand.device)
    best, where = [], []
    for _ in range(beams):  # the best of those left, the lowest index among equals
        top = cand.amax(1, keepdim=True)
        at = torch.where(cand == top, index, beams * vocab).amin(1, keepdim=True)
        best.append(top)
        where.append(at)
        cand.scatter_(1, at, -math.inf)
    where = torch.cat(where, 1)
    group = torch.arange(n // beams, device=cand.device)[:, None] * beams
    parents = (where // vocab + group).view(-1)
    tokens = (where % vocab).view(-1)
    return {"tokens": tokens.int(), "parents": parents.int(), "scores": torch.cat(best, 1).view(-1).float(),
            "finished": finished[parents] | (tokens == eos)}


def _plain_reorder(k, v, parents, begin, end, beams):
    for g in range(0, k.shape[0], beams):
        rows = [r for r in range(g, g + beams) if parents[r] != r]
        if rows:
            at = torch.tensor(rows, device=k.device)
            of = torch.tensor([parents[r] for r in rows], device=k.device)
            for t in (k, v):
                part = t[:, :, :, begin[g]:end[g]]
                part[at] = part[of]
    return {"k": k, "v": v}


def run(s):
    c = s["case"]
    if not own:
        if c["op"] == "attention":
            return _plain_attention(s["q"], s["k"], s["v"], s["lengths"])
        if c["op"] == "select":
            return _plain_select(s["logits"], s["scores"], s["finished"], c["beams"], s["eos"])
        return _plain_reorder(s["k"], s["v"], s["parents_list"], s["begin_list"], s["end_list"], c["beams"])
    kernel = s["kernel"]
    if c["op"] == "attention":
        return kernel.attention_packed(s["q"], s["k"], s["v"], s["lengths"])
    if c["op"] == "select":
        tokens, parents, scores, finished = kernel.beam_select(s["logits"], s["scores"], s["finished"], c["beams"],
                                                               s["eos"])
        return {"tokens": tokens, "parents": parents, "scores": scores, "finished": finished}
    kernel.beam_reorder(s["k"], s["v"], s["parents"], s["begin"], s["end"], c["beams"])
    return {"k": s["k"], "v": s["v"]}


def work(case):
    if case["op"] == "attention":
        lens, hq, hkv = _lengths(case), case["hq"], case["hkv"]
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": sum(lens) * D * (2 * hq * size + 2 * hkv * 2),
                "flops": 4.0 * hq * D * sum(n * (n + 1) // 2 for n in lens)}
    n = case["groups"] * case["beams"]
    if case["op"] == "select":  # a finished row's logits are not needed
        return {"bytes": (n - case["done"]) * case["vocab"] * 4 + n * (4 + 1 + 4 + 4 + 4 + 1),
                "flops": 4.0 * (n - case["done"]) * case["vocab"]}
    changed, parents = _reorder_rows(case)
    row = 2 * LAYERS * HKV * D * 2  # a position's keys and values
    return {"bytes": case["groups"] * (changed + parents) * case["new"] * row + 12 * n, "flops": 0.0}


# ---------------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "attention":
        q, k, v = (s[n].to(torch.float64) for n in ("q", "k", "v"))
        out = torch.zeros_like(q)
        first = 0
        for n in s["lengths"]:
            for head in range(case["hq"]):
                kh = head * case["hkv"] // case["hq"]
                kk, vv = (t[first:first + n, kh].contiguous() for t in (k, v))
                for a in range(0, n, 1024):  # a block of queries at a time
                    b = min(n, a + 1024)
                    w = (q[first + a:first + b, head].contiguous() @ kk[:b].T.contiguous()) / math.sqrt(D)
                    seen = torch.arange(b, device=w.device)[None] <= torch.arange(a, b, device=w.device)[:, None]
                    w = torch.softmax(torch.where(seen, w, torch.full_like(w, -math.inf)), dim=1)
                    out[first + a:first + b, head] = w @ vv[:b]
            first += n
        return out
    if case["op"] == "select":
        x, score = s["logits"].cpu().numpy().astype(np.float64), s["scores"].cpu().numpy().astype(np.float64)
        done, beams, vocab = s["finished"].cpu().numpy(), case["beams"], case["vocab"]
        got = {"tokens": [], "parents": [], "scores": [], "finished": []}
        for g in range(0, x.shape[0], beams):
            found = []  # (-score, row, token) of every row's own best
            for r in range(g, g + beams):
                if done[r]:
                    found.append((-score[r], r, s["eos"]))
                    continue
                peak = x[r].max()
                logp = x[r] - (peak + math.log(math.fsum(np.exp(x[r] - peak))))
                near = np.flatnonzero(x[r] >= np.partition(x[r], vocab - beams)[vocab - beams])
                found += [(-(score[r] + logp[t]), r, int(t)) for t in near]
            for value, r, t in sorted(found)[:beams]:
                got["tokens"].append(t)
                got["parents"].append(r)
                got["scores"].append(-value)
                got["finished"].append(bool(done[r]) or t == s["eos"])
        return {"tokens": torch.tensor(got["tokens"], dtype=torch.int32),
                "parents": torch.tensor(got["parents"], dtype=torch.int32),
                "scores": torch.tensor(got["scores"], dtype=torch.float64),
                "finished": torch.tensor(got["finished"])}
    k, v = s["k"].clone(), s["v"].clone()
    for b, p in enumerate(s["parents_list"]):
        for old, new in ((s["k"], k), (s["v"], v)):
            new[b, :, :, s["begin_list"][b]:s["end_list"][b]] = old[p, :, :, s["begin_list"][b]:s["end_list"][b]]
    return {"k": k, "v": v}
