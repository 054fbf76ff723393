"""The operators that a server needs beside the batched decode to keep its sequences in one pool of pages and to
answer with other than the likeliest token, and the calls their speed is judged by: a cache quantised as it is
written and read back, attention of each sequence's new token over its pages, and sampling from the logits with
temperature, top-k, top-p and min-p from given random numbers.

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

# the models' geometry: 16 query and 8 K/V heads of 128, vocabulary 151936
HQ, HKV, D, VOCAB = 16, 8, 128, 151936
KEY_ROWS = 160_000  # of 8 heads in bf16: no attention case reads more (0.66 GB)


def listed():
    return [
        # A decode step of a small batch: each sequence's new key and value go into 8-bit pages. Latency counts.
        {"name": "cache-8-new", "op": "cache", "dtype": "fp32", "pages": "e4m3", "hkv": HKV, "page_size": 16, "count": 8,
         "begin_lo": 33, "begin_hi": 480, "new_lo": 1, "new_hi": 1, "read": "written", "fused": True},
        # A server's batch of prompts, straight from a fused projection, stored and taken out again.
        {"name": "cache-prompts", "op": "cache", "dtype": "bf16", "pages": "e4m3", "hkv": HKV, "page_size": 64, "count": 16,
         "begin_lo": 0, "begin_hi": 0, "new_lo": 64, "new_hi": 664, "read": "written", "fused": True},
        # Conversations that go on: a chunk of each is added, and the whole of it read for the next chunk's attention.
        {"name": "cache-chunks", "op": "cache", "dtype": "fp32", "pages": "e4m3", "hkv": HKV, "page_size": 16, "count": 5,
         "begin_lo": 301, "begin_hi": 1801, "new_lo": 37, "new_hi": 400, "read": "all", "fused": False},
        # Long documents in bf16 pages: the largest cache.
        {"name": "cache-documents", "op": "cache", "dtype": "fp32", "pages": "bf16", "hkv": HKV, "page_size": 128, "count": 3,
         "begin_lo": 0, "begin_hi": 1000, "new_lo": 1801, "new_hi": 8192, "read": "all", "fused": False},
        # One user's next token after a short question: the smallest attention, where latency counts.
        {"name": "attention-1", "op": "attention", "dtype": "bf16", "pages": "bf16", "hq": HQ, "hkv": HKV, "page_size": 16,
         "count": 1, "lo": 300, "hi": 300, "max_seq": 512, "fused": False},
        # One user with a long document, at the precision of the framework's activations.
        {"name": "attention-1-long", "op": "attention", "dtype": "fp32", "pages": "bf16", "hq": HQ, "hkv": HKV,
         "page_size": 128, "count": 1, "lo": 30001, "hi": 30001, "max_seq": 32768, "fused": False},
        # A few users of very different lengths, an odd number of them, in 8-bit pages.
        {"name": "attention-13", "op": "attention", "dtype": "bf16", "pages": "e4m3", "hq": HQ, "hkv": HKV, "page_size": 64,
         "count": 13, "lo": 100, "hi": 1900, "max_seq": 2048, "fused": True},
        # The largest batch of the batched decode, at the precision of the framework's activations.
        {"name": "attention-64", "op": "attention", "dtype": "fp32", "pages": "e4m3", "hq": HQ, "hkv": HKV, "page_size": 16,
         "count": 64, "lo": 64, "hi": 960, "max_seq": 4096, "fused": False},
        # The same far into long answers: the largest attention.
        {"name": "attention-64-long", "op": "attention", "dtype": "bf16", "pages": "bf16", "hq": HQ, "hkv": HKV,
         "page_size": 64, "count": 64, "lo": 900, "hi": 4095, "max_seq": 4096, "fused": True},
        # One user's next token: the smallest choice over the whole vocabulary.
        {"name": "sample-1", "op": "sample", "rows": 1, "vocab": VOCAB, "filters": "top-p"},
        # An odd number of users with settings of their own over a vocabulary whose rows end anywhere.
        {"name": "sample-13-odd", "op": "sample", "rows": 13, "vocab": 32003, "filters": "mixed"},
        # The largest batch of the batched decode, every user with settings of their own.
        {"name": "sample-64", "op": "sample", "rows": 64, "vocab": VOCAB, "filters": "mixed"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "cache", "cache", "sample", "sample"])
    if op == "sample":
        return {"op": op, "rows": _spread(rng, 1, 64), "vocab": rng.choice([VOCAB, VOCAB, _spread(rng, 1000, VOCAB)]),
                "filters": rng.choice(["none", "top-k", "top-p", "min-p", "mixed", "mixed"]),
                "temperature": round(rng.uniform(0.3, 1.6), 2), "top_k": _spread(rng, 1, 2000),
                "top_p": round(rng.uniform(0.3, 0.99), 2), "min_p": round(rng.uniform(0.005, 0.3), 3)}
    pages, page_size = rng.choice(["bf16", "e4m3"]), rng.choice([1, 8, 16, 16, 32, 64, 128, 512])
    hq, hkv = rng.choice([(HQ, HKV), (HQ, HKV), (HQ, HKV), (8, 8), (16, 2), (12, 4), (5, 1), (40, 2)])
    common = {"op": op, "dtype": rng.choice(["bf16", "fp32"]), "pages": pages, "hkv": hkv, "page_size": page_size,
              "fused": rng.random() < 0.5}
    if op == "attention":
        count = _spread(rng, 1, 128)
        most = max(1, min(32000, KEY_ROWS * HKV // (count * hkv)))
        hi = _spread(rng, 1, most)
        return {**common, "hq": hq, "count": count, "lo": rng.choice([0, 1, hi, _spread(rng, 1, hi)]), "hi": hi,
                "max_seq": rng.randint(hi, 32768)}
    count = _spread(rng, 1, 64)
    new = _spread(rng, 1, max(1, 12000 // count))
    begin = rng.choice([0, _spread(rng, 1, max(1, 16000 // count))])
    return {**common, "count": count, "begin_lo": rng.randint(0, begin), "begin_hi": begin,
            "new_lo": rng.randint(1, new), "new_hi": new, "read": rng.choice(["written", "all"])}


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
def _even(lo, hi, count):
    return [lo + (hi - lo) * i // max(1, count - 1) for i in range(count)]


def _shuffled(values, order):
    values = list(values)
    order.shuffle(values)
    return values


def _tables(capacity, width, page_size, order):
    """(pages of the pool, block tables): each sequence's pages are any of the pool's, entries past them -1."""
    counts = [-(-n // page_size) for n in capacity]
    pool = list(range(sum(counts) + 5))
    order.shuffle(pool)
    table, at = np.full((len(capacity), width), -1, dtype=np.int32), 0
    for s, n in enumerate(counts):
        table[s, :n] = pool[at:at + n]
        at += n
    return len(pool), torch.from_numpy(table)


def _exponent(x):
    """The least e (at least -117) with |x| <= 448 * 2^e over the last dimension."""
    mantissa, exponent = torch.frexp(x.abs().amax(-1))
    return (exponent - 9 + (mantissa > 0.875)).clamp(min=-117)


def _quantised(x):
    """(e4m3 values, their power-of-two scales) of rows of 128 numbers."""
    e = _exponent(x)
    return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _pool(case, pages, gen):
    """The pages as earlier calls left them: keys as their norms and rotations leave them, values as a projection
    of a normalised row, (values, scales) of each."""
    dev = torch.device("cuda:0")
    shape = (pages, case["hkv"], case["page_size"], D)
    made = []
    for size in (1.0, 0.64):
        x = torch.randn(shape, generator=gen, device=dev)
        x.mul_(size)
        made.append(_quantised(x) if case["pages"] == "e4m3" else (x.to(torch.bfloat16), None))
    return made


def _inputs(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    order = random.Random(int(seed))
    s = {"case": case}
    if case["op"] == "sample":
        n, vocab = case["rows"], case["vocab"]
        # logits as a language model gives them: most far below a few favourites
        x = torch.randn(n, vocab, generator=gen, device=dev) * 2
        likely = torch.randint(0, vocab, (n, 24), generator=gen, device=dev)
        x.scatter_add_(1, likely, 6 + 3 * torch.randn(n, 24, generator=gen, device=dev))
        t = case.get("temperature", 0.8)
        kinds = {"none": (t, 0, 1.0, 0.0), "top-k": (t, case.get("top_k", 50), 1.0, 0.0),
                 "top-p": (t, 0, case.get("top_p", 0.9), 0.0), "min-p": (t, 0, 1.0, case.get("min_p", 0.05))}
        several = [kinds["top-p"], (0.6, 20, 0.95, 0.0), kinds["none"], (0.0, 0, 1.0, 0.0), kinds["min-p"],
                   (0.9, 1000, 0.8, 0.01), (1.5, 40, 1.0, 0.1), kinds["top-k"]]
        rows = [several[i % 8] if case["filters"] == "mixed" else kinds[case["filters"]] for i in range(n)]
        rows = _shuffled(rows, order)
        s.update(logits=x, uniforms=torch.rand(n, generator=gen, device=dev))
        for i, (name, kind) in enumerate((("temperature", torch.float32), ("top_k", torch.int32),
                                          ("top_p", torch.float32), ("min_p", torch.float32))):
            s[name] = torch.tensor([r[i] for r in rows], dtype=kind, device=dev)
        return s
    hkv, ps, kind = case["hkv"], case["page_size"], torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    if case["op"] == "attention":
        lens = _shuffled(_even(case["lo"], case["hi"], case["count"]), order)
        pages, table = _tables(lens, -(-case["max_seq"] // ps), ps, order)
        hq = case["hq"]
        q = torch.randn(case["count"], hq, D, generator=gen, device=dev)
        q *= torch.exp(0.5 * torch.randn(1, hq, 1, generator=gen, device=dev))  # some heads attend sharply
        if case["fused"]:  # one projection's rows, of which the queries are a slice
            q = torch.cat([q, torch.zeros(case["count"], 2 * hkv, D, device=dev)], dim=1).to(kind)[:, :hq]
        s.update(q=q.to(kind), lengths_list=lens, lengths=torch.tensor(lens, dtype=torch.int32, device=dev))
    else:
        begin = _shuffled(_even(case["begin_lo"], case["begin_hi"], case["count"]), order)
        new = _shuffled(_even(case["new_lo"], case["new_hi"], case["count"]), order)
        ends = [b + n for b, n in zip(begin, new)]
        pages, table = _tables(ends, max(-(-n // ps) for n in ends) + 1, ps, order)
        k = torch.randn(sum(new), hkv, D, generator=gen, device=dev)
        v = torch.randn(sum(new), hkv, D, generator=gen, device=dev) * 0.64
        if case["fused"]:  # the keys and values of one projection
            rows = torch.cat([k, v], dim=1).to(kind)
            k, v = rows[:, :hkv], rows[:, hkv:]
        first = [0] * len(begin) if case["read"] == "all" else begin
        s.update(k=k.to(kind), v=v.to(kind), begin_list=begin, new=new, first_list=first,
                 read=[e - f for e, f in zip(ends, first)])
        for name in ("begin", "first"):
            s[name] = torch.tensor(s[name + "_list"], dtype=torch.int32, device=dev)
    (s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"]) = _pool(case, pages, gen)
    s["tables"] = table.to(dev)
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ---------------------------------------------------------------------------------------------------
# one call
# ---------------------------------------------------------------------------------------------------
def _places(tables, first, counts, page_size):
    """(page, row in it) of the positions first[s] .. first[s] + counts[s] - 1 of every sequence, one after another."""
    dev = tables.device
    n = torch.tensor(counts, device=dev)
    total = sum(counts)
    seq = torch.repeat_interleave(torch.arange(len(counts), device=dev), n, output_size=total)
    at = torch.arange(total, device=dev) - (n.cumsum(0) - n)[seq] + first.long()[seq]
    return tables[seq, at // page_size].long(), at % page_size


def _plain_cache(s, page_size):
    page, row = _places(s["tables"], s["begin"], s["new"], page_size)
    back, at = _places(s["tables"], s["first"], s["read"], page_size)

    def one(x, pages, scales):
        if scales is None:
            pages[page, :, row] = x.to(torch.bfloat16)
            return pages[back, :, at]
        values, e = _quantised(x.float())
        # as bytes: indexing has no form for these types
        pages.view(torch.uint8)[page, :, row] = values.view(torch.uint8)
        scales.view(torch.uint8)[page, :, row] = e.view(torch.uint8)
        values = pages.view(torch.uint8)[back, :, at].view(torch.float8_e4m3fn).float()
        e = scales.view(torch.uint8)[back, :, at].int() - 127
        return torch.ldexp(values, e[..., None]).to(torch.bfloat16)

    return {"k": one(s["k"], s["k_pages"], s["k_scales"]), "v": one(s["v"], s["v_pages"], s["v_scales"])}


def _gathered(pages, scales, page, row):
    """[sequences, keys, heads, 128] in 32 bits of the places (page, row), [sequences, keys] each."""
    if scales is None:
        return pages[page, :, row].float()
    values = pages.view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn).float()
    return torch.ldexp(values, (scales.view(torch.uint8)[page, :, row].int() - 127)[..., None])


def _plain_attention(s, hkv, page_size):
    q, lengths = s["q"], s["lengths"].long()
    n, hq, longest = q.shape[0], q.shape[1], max(s["lengths_list"])
    if longest == 0:
        return torch.zeros_like(q)
    at = torch.arange(longest, device=q.device)
    seen = at[None] < lengths[:, None]  # [sequences, keys]
    # a key that is not seen is taken from wherever an entry of the table points, and left out below
    page, row = s["tables"][:, at // page_size].long().clamp(min=0), (at % page_size)[None].expand(n, -1)
    k = _gathered(s["k_pages"], s["k_scales"], page, row).permute(0, 2, 3, 1).reshape(n * hkv, D, longest)
    sc = torch.bmm(q.float().reshape(n * hkv, hq // hkv, D), k).mul_(D ** -0.5).view(n, hq, longest)
    sc.masked_fill_(~seen[:, None], -math.inf)
    p = torch.where(seen[:, None], sc.sub_(sc.amax(-1, keepdim=True)).exp_(), 0)
    v = _gathered(s["v_pages"], s["v_scales"], page, row).permute(0, 2, 1, 3).reshape(n * hkv, longest, D)
    o = torch.bmm(p.view(n * hkv, hq // hkv, longest), v).view(n, hq, D) / p.sum(-1, keepdim=True)
    return torch.where((lengths > 0)[:, None, None], o, 0).to(q.dtype)


def _plain_sample(logits, uniforms, temperature, top_k, top_p, min_p):
    """In 64 bits, since a border between two tokens may lie closer to a random number than 32 bits tell."""
    n, vocab = logits.shape
    x = logits.double()
    best = x.amax(1, keepdim=True)
    greedy = temperature == 0
    # a temperature of 0: all weight on the first of the largest
    z = (x - best) / torch.where(greedy, 1.0, temperature.double())[:, None]
    z, index = z.sort(dim=1, descending=True, stable=True)
    w = z.exp()
    rank = torch.arange(vocab, device=x.device)[None]
    limit = torch.where(top_k > 0, top_k, vocab).long()
    limit = torch.where(greedy, 1, limit)[:, None]
    w = torch.where(rank < limit, w, 0)
    before = w.cumsum(1) - w
    some = torch.where(top_p < 1, top_p.double() * w.sum(1), math.inf)[:, None]
    kept = (rank < limit) & ((rank == 0) | ((before < some) & (w >= min_p.double()[:, None])))
    w = torch.zeros_like(w).scatter_(1, index, torch.where(kept, w, 0))  # in the order of the vocabulary
    run_up = w.cumsum(1)
    total = run_up[:, -1:]
    tokens = ((run_up > uniforms.double()[:, None] * total) & (w > 0)).int().argmax(1)
    return {"tokens": tokens.int(), "logprobs": (w.gather(1, tokens[:, None]) / total).log()[:, 0].float()}


def run(s):
    c = s["case"]
    if not own:
        if c["op"] == "cache":
            return _plain_cache(s, c["page_size"])
        if c["op"] == "attention":
            return _plain_attention(s, c["hkv"], c["page_size"])
        return _plain_sample(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import megakernel
    kernel = megakernel.load()
    if c["op"] == "cache":
        kernel.cache_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["tables"], s["begin"], s["new"], s["k_scales"],
                           s["v_scales"])
        k, v = kernel.cache_read(s["k_pages"], s["v_pages"], s["tables"], s["first"], s["read"], s["k_scales"],
                                 s["v_scales"])
        return {"k": k, "v": v}
    if c["op"] == "attention":
        return kernel.attention_paged(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lengths"], s["k_scales"],
                                      s["v_scales"])
    tokens, logprobs = kernel.sample(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return {"tokens": tokens, "logprobs": logprobs}


def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * 4 + 4 + 16 + 8), "flops": 4.0 * case["rows"] * case["vocab"]}
    size, row = 2 if case["dtype"] == "bf16" else 4, D * 2 if case["pages"] == "bf16" else D + 1
    hkv, ps = case["hkv"], case["page_size"]
    if case["op"] == "attention":
        lens = _even(case["lo"], case["hi"], case["count"])
        return {"bytes": sum(lens) * hkv * 2 * row + case["count"] * case["hq"] * D * 2 * size +
                4 * sum(1 - (-n // ps) for n in lens), "flops": 4.0 * case["hq"] * D * sum(lens)}
    new = sum(_even(case["new_lo"], case["new_hi"], case["count"]))
    read = new + (sum(_even(case["begin_lo"], case["begin_hi"], case["count"])) if case["read"] == "all" else 0)
    return {"bytes": 2 * hkv * (new * (D * size + row) + read * (row + D * 2)) + 4 * (2 * (new + read) // ps), "flops": 0.0}


# ---------------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------------
def _rounded(x, bits, least):
    """x to `bits` significant bits, to even on ties, in steps of at least 2^least."""
    step = torch.exp2((torch.frexp(x)[1] - bits).clamp(min=least).double())
    return torch.round(x / step) * step


def _value(pages, scales):
    if scales is None:
        return pages.double()
    return pages.double() * torch.exp2(scales.view(torch.uint8).double() - 127)[..., None]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "sample":
        x, u = s["logits"].cpu().numpy().astype(np.longdouble), s["uniforms"].cpu().numpy().astype(np.longdouble)
        t, k, p, m = (s[name].cpu().numpy() for name in ("temperature", "top_k", "top_p", "min_p"))
        tokens, logprobs = [], []
        for r in range(case["rows"]):
            order = np.argsort(-x[r], kind="stable")
            if t[r] == 0:
                tokens.append(int(order[0]))
                logprobs.append(0.0)
                continue
            kept = order[:k[r]] if k[r] > 0 else order
            w = np.exp((x[r][kept] - x[r][kept[0]]) / np.longdouble(t[r]))
            upto = np.cumsum(w)
            if p[r] < 1:  # the fewest whose weights reach the share
                kept = kept[:int(np.argmax(upto >= np.longdouble(p[r]) * upto[-1])) + 1]
                w = w[:len(kept)]
            kept, w = kept[w >= np.longdouble(m[r])], w[w >= np.longdouble(m[r])]
            by = np.argsort(kept)
            upto = np.cumsum(w[by])
            at = int(np.argmax(upto > u[r] * upto[-1]))
            tokens.append(int(kept[by][at]))
            logprobs.append(float(np.log(w[by][at] / upto[-1])))
        return {"tokens": torch.tensor(tokens, dtype=torch.int32), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}
    tables, ps = s["tables"].cpu().tolist(), case["page_size"]
    kp, vp = _value(s["k_pages"], s["k_scales"]), _value(s["v_pages"], s["v_scales"])

    def rows(pages, q, first, count):
        """[count, heads, 128]: the positions of sequence q from `first` on."""
        if count == 0:
            return pages[:0, :, 0]
        used = tables[q][first // ps:(first + count - 1) // ps + 1]
        whole = pages[used].transpose(1, 2).reshape(-1, pages.shape[1], D)
        return whole[first % ps:first % ps + count]

    if case["op"] == "attention":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        g = case["hq"] // case["hkv"]
        for b, n in enumerate(s["lengths_list"]):
            if n == 0:
                continue
            k, v = rows(kp, b, 0, n), rows(vp, b, 0, n)
            for h in range(case["hkv"]):
                w = s["q"][b, h * g:(h + 1) * g].double() @ k[:, h].T.contiguous() / math.sqrt(D)
                out[b, h * g:(h + 1) * g] = torch.softmax(w, dim=1) @ v[:, h].contiguous()
        return out
    got = {}
    for name, pages in (("k", kp), ("v", vp)):
        x = s[name].double()
        if case["pages"] == "bf16":
            x = _rounded(x, 8, -133)
        else:
            least = x.abs().amax(-1, keepdim=True) / 448  # the smallest power of two that is not below this
            scale = torch.exp2(torch.ceil(torch.log2(least)).clamp(min=-117))
            x = _rounded(x / scale, 4, -9) * scale
        parts, at = [], 0
        for q, (begin, new, first) in enumerate(zip(s["begin_list"], s["new"], s["first_list"])):
            parts += [rows(pages, q, first, begin - first), x[at:at + new]]
            at += new
        got[name] = torch.cat(parts)
    return got
