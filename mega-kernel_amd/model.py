"""Greedy decoding driver: the reference's Python surface on the MI355X decode kernel.

Mirrors ``/root/reference/model.py`` step for step:
  * build the model (``:23-27``). The Hub checkpoint is unreachable offline, so this builds a seeded
    random-init Qwen3 of the requested shape (normal std 0.02, norms 1, tied embeddings,
    rope_theta 1e6) on the CPU and casts it to bf16. The Transformers prefill runs on the CPU
    (torch's bf16 batched products on this GPU are avoided); its weights, RoPE tables and K/V are
    then copied to the GPU;
  * flatten the 11 weights per layer (``:30-44``) and build the RoPE tables (``:47-53``, taken from
    the model's own rotary module, see ``megakernel.rope_tables``);
  * prefill with Transformers (``:72-73``) and copy its K/V into the ``[L, 8, max_seq, 128]`` cache
    (``:79-87``);
  * greedy loop calling the same ``decode`` entry point (``:95-127``), timed with device events.
    The fused device argmax (``decode_greedy``) replaces the separate ``argmax().item()`` per token;
    the host reads each token back only to feed the next call, as the reference does.
  * ``--device-loop``: the same greedy generation as one ``decode_steps`` call, which feeds each
    step's argmax to the next launch on the device; the host reads the tokens once at the end.
  * ``--native-prefill``: the prompt goes through the batched prefill kernel (``prefill``: all
    prompt tokens at once on the matrix cores, writing the ``[L, 8, max_seq, 128]`` cache
    directly) instead of the Transformers prefill and cache copy.
  * ``--beams W`` (and ``--prompts S``): beam search instead of the greedy loop, S prompts of different
    lengths with W beams each (S * W <= 64). ``prefill_batch`` fills the first beam's cache of every
    prompt in one call and ``beam_reorder`` spreads it over the others; each step is ``beam_select``,
    ``beam_reorder`` of the rows generated so far, and ``decode_batch`` of all beams. Nothing is read
    back until the last step.
  * ``--temperature T`` (with ``--top-k``, ``--top-p``, ``--min-p``, ``--seed`` and ``--prompts S``): S prompts of
    different lengths are continued together with tokens drawn from their logits (S <= 64). ``prefill_batch`` fills
    their caches, and each step is ``sample`` and ``decode_batch``. Nothing is read back until the last step.

    python mega-kernel_amd/model.py [--shape qwen3-0.6b] [--prompt 32] [--max-seq 512] [--new 64]
                                    [--device-loop] [--native-prefill] [--beams 4 [--prompts 2] [--eos ID]]
                                    [--temperature 0.8 [--top-k 50] [--top-p 0.9] [--min-p 0.05] [--seed 0]]
"""
import argparse
import os
import sys
import time

HERE = os.path.dirname(os.path.abspath(__file__))
if HERE not in sys.path:
    sys.path.insert(0, HERE)

SHAPES = {  # hidden, intermediate (28 layers, 16 q / 8 kv heads of 128, vocab 151936)
    "qwen3-0.6b": (1024, 3072),
    "qwen3-1.7b": (2048, 6144),
}


def build_model(shape, max_positions, seed=0):
    import torch
    from transformers import Qwen3Config, Qwen3ForCausalLM
    hidden, inter = SHAPES[shape]
    cfg = Qwen3Config(hidden_size=hidden, intermediate_size=inter, num_hidden_layers=28, num_attention_heads=16,
                      num_key_value_heads=8, head_dim=128, vocab_size=151936, tie_word_embeddings=True,
                      rms_norm_eps=1e-6, rope_parameters={"rope_type": "default", "rope_theta": 1e6},
                      max_position_embeddings=max_positions, initializer_range=0.02)
    torch.manual_seed(seed)
    return Qwen3ForCausalLM(cfg).to(torch.bfloat16).eval()


def beam_search(kernel, prompts, beams, new, eos, embed, final_norm, layer_weights, cos, sin, max_seq):
    """The best ``beams`` continuations of up to ``new`` tokens of each prompt (lists of token ids), best first, as
    (tokens, score) with the score the sum of their log-probabilities; a continuation ends with ``eos`` (-1: none
    does). All calls are queued without reading anything back, so ``new`` steps are always made. A prompt whose
    logits fail (NaN) has beams of no tokens and the score NaN; the others' searches go on."""
    import torch
    dev, rows = embed.device, len(prompts) * beams
    lengths = [len(p) for p in prompts]
    shape = (rows, len(layer_weights) // 11, 8, max_seq, 128)
    k, v = (torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(2))
    packed = torch.tensor([t for p in prompts for t in p], dtype=torch.int32, device=dev)
    weights = (embed, embed, final_norm, layer_weights, cos, sin)
    first, _ = kernel.prefill_batch(packed, lengths, *weights, k[::beams], v[::beams], max_seq)
    begin = torch.tensor(lengths, dtype=torch.int32, device=dev).repeat_interleave(beams)
    heads = torch.arange(rows, dtype=torch.int32, device=dev) // beams * beams
    kernel.beam_reorder(k, v, heads, torch.zeros_like(begin), begin, beams)
    logits = first.repeat_interleave(beams, 0)
    scores = torch.full((rows,), -float("inf"), device=dev)
    scores[::beams] = 0  # a prompt's beams are one until the first selection
    finished = torch.zeros(rows, dtype=torch.bool, device=dev)
    position, steps = begin.clone(), []
    for i in range(new):
        tokens, parents, scores, finished = kernel.beam_select(logits, scores, finished, beams, eos)
        steps.append((tokens, parents, finished))
        if i + 1 < new:
            kernel.beam_reorder(k, v, parents, begin, position, beams)
            # a failed group's tokens are -1, which would fail the decode of every sequence
            logits, _ = kernel.decode_batch(tokens.clamp(min=0), position, *weights, k, v, max_seq)
            position = position + 1
    steps, scores = [tuple(t.tolist() for t in s) for s in steps], scores.tolist()
    found = []
    for s in range(len(prompts)):
        group = []
        for row in range(s * beams, (s + 1) * beams):
            path, at = [], row
            for i in reversed(range(new)) if scores[row] == scores[row] else ():  # NaN: failed
                tokens, parents, _ = steps[i]
                if i == 0 or not steps[i - 1][2][parents[at]]:  # not the repeated end of a finished one
                    path.append(tokens[at])
                at = parents[at]
            group.append((path[::-1], scores[row]))
        found.append(group)
    return found


def sample_texts(kernel, prompts, new, eos, temperature, top_k, top_p, min_p, seed, embed, final_norm, layer_weights, cos,
                 sin, max_seq):
    """Up to ``new`` tokens after each prompt (lists of token ids), drawn with ``sample``, as (tokens, the sum of their
    log-probabilities); a continuation ends with ``eos`` (-1: none does). All calls are queued without reading
    anything back, so ``new`` steps are always made. A prompt whose logits fail (NaN) ends there, with the sum NaN; the
    others go on."""
    import torch
    dev, rows = embed.device, len(prompts)
    lengths = [len(p) for p in prompts]
    shape = (rows, len(layer_weights) // 11, 8, max_seq, 128)
    k, v = (torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(2))
    packed = torch.tensor([t for p in prompts for t in p], dtype=torch.int32, device=dev)
    weights = (embed, embed, final_norm, layer_weights, cos, sin)
    # the largest of their types where they are larger: as good as no limit, as even weights as can be
    temperature, top_k = min(temperature, torch.finfo(torch.float32).max), min(top_k, 2 ** 31 - 1)
    settings = [torch.full((rows,), x, dtype=t, device=dev) for x, t in (
        (temperature, torch.float32), (top_k, torch.int32), (top_p, torch.float32), (min_p, torch.float32))]
    numbers = torch.rand(new, rows, generator=torch.Generator().manual_seed(seed)).to(dev)
    logits, _ = kernel.prefill_batch(packed, lengths, *weights, k, v, max_seq)
    position, steps = torch.tensor(lengths, dtype=torch.int32, device=dev), []
    for i in range(new):
        tokens, logprobs = kernel.sample(logits, numbers[i], *settings)
        steps.append((tokens, logprobs))
        if i + 1 < new:
            # a failed row's token is -1, which would fail the decode of every sequence
            logits, _ = kernel.decode_batch(tokens.clamp(min=0), position, *weights, k, v, max_seq)
            position = position + 1
    steps = [(t.tolist(), p.tolist()) for t, p in steps]
    found = []
    for row in range(rows):
        text, total = [], 0.0
        for tokens, logprobs in steps:
            if tokens[row] < 0:
                total = float("nan")
                break
            text.append(tokens[row])
            total += logprobs[row]
            if tokens[row] == eos:
                break
        found.append((text, total))
    return found


def run(argv=None, keep_prefill_cache=False):
    """Runs the driver and returns what it did: the generated tokens (the prefill's greedy token
    first), the prompt length, the device status after the loop, ms per token, and, with
    ``keep_prefill_cache``, a copy of the K/V cache as the prefill left it together with the decode
    operator's other inputs (so a caller can replay the decode from the same state)."""
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--shape", default="qwen3-0.6b", choices=sorted(SHAPES))
    ap.add_argument("--prompt", type=int, default=32, help="random prompt length (token ids, seed 1)")
    ap.add_argument("--max-seq", type=int, default=512)
    ap.add_argument("--new", type=int, default=64, help="tokens to generate")
    ap.add_argument("--device-loop", action="store_true", help="generate with one decode_steps call")
    ap.add_argument("--native-prefill", action="store_true",
                    help="fill the cache with the batched prefill kernel (prefill) instead of the Transformers "
                         "prefill and cache copy")
    ap.add_argument("--beams", type=int, default=0, help="beam search with this many beams per prompt (1 to 16)")
    ap.add_argument("--prompts", type=int, default=1, help="with --beams or --temperature: prompts taken together")
    ap.add_argument("--eos", type=int, default=-1, help="with --beams or --temperature: the token that ends a continuation")
    ap.add_argument("--temperature", type=float, default=None, help="draw the tokens at this temperature (0: the likeliest)")
    ap.add_argument("--top-k", type=int, default=0, help="with --temperature: from the k largest logits (0: all)")
    ap.add_argument("--top-p", type=float, default=1.0, help="with --temperature: from the fewest that reach this share")
    ap.add_argument("--min-p", type=float, default=0.0, help="with --temperature: from those this likely against the likeliest")
    ap.add_argument("--seed", type=int, default=0, help="with --temperature: of the random numbers")
    a = ap.parse_args(argv)
    if a.temperature is not None:
        if a.beams or a.device_loop or a.native_prefill:
            ap.error("--temperature goes without --beams, --device-loop and --native-prefill")
        if not (0 <= a.temperature < float("inf") and 0 <= a.top_p <= 1 and 0 <= a.min_p <= 1 and a.top_k >= 0):
            ap.error("--temperature and --top-k must be at least 0, --top-p and --min-p between 0 and 1")
        if not 1 <= a.prompts <= 64:
            ap.error("--temperature takes 1 to 64 prompts")
        if not 1 <= a.prompt < a.max_seq:
            ap.error("--temperature needs a prompt that leaves room in --max-seq")
    if a.beams and (a.beams > 16 or a.beams < 0 or a.prompts < 1 or a.beams * a.prompts > 64):
        ap.error("--beams takes 1 to 16 beams per prompt, and at most 64 in all")
    if a.beams and not 1 <= a.prompt < a.max_seq:
        ap.error("--beams needs a prompt that leaves room in --max-seq")
    import torch
    import megakernel

    kernel = megakernel.load()  # the HIP operator; raises if it is not built
    dev = torch.device("cuda:0")
    model = build_model(a.shape, max(4096, a.max_seq))
    ids = torch.randint(0, 151936, (1, a.prompt), generator=torch.Generator().manual_seed(1))
    layer_weights = [t.to(dev) for t in megakernel.layer_weight_list(model)]
    embed = model.model.embed_tokens.weight.detach().to(dev)
    final_norm = model.model.norm.weight.detach().to(dev)
    cos, sin = megakernel.rope_tables(model, a.max_seq, dev)

    # prompts of different lengths, the longest of --prompt tokens: pieces of the same random ids
    prompts = [ids[0, :max(1, a.prompt - 5 * i)].tolist() for i in range(a.prompts)]
    if a.temperature is not None:
        new = min(a.new, a.max_seq - a.prompt)
        t0 = time.perf_counter()
        found = sample_texts(kernel, prompts, new, a.eos, a.temperature, a.top_k, a.top_p, a.min_p, a.seed, embed,
                             final_norm, layer_weights, cos, sin, a.max_seq)
        wall = time.perf_counter() - t0
        for i, (tokens, score) in enumerate(found):
            print(f"prompt {i} ({len(prompts[i])} tokens): " + (
                f"{score:.3f} {tokens[:8]}{' ...' if len(tokens) > 8 else ''}" if score == score else "failed"))
        print(f"sampling: {a.prompts} prompts, {new} steps in {wall * 1e3:.1f} ms, device status {kernel.status()}")
        return {"prompt": a.prompt, "prompts": prompts, "texts": found, "status": kernel.status(),
                "generated": [t for tokens, score in found for t in (tokens if score == score else [-1])],
                "inputs": {"embed": embed, "final_norm": final_norm, "layer_weights": layer_weights, "cos": cos,
                           "sin": sin, "max_seq": a.max_seq}}

    if a.beams:
        new = min(a.new, a.max_seq - a.prompt)
        t0 = time.perf_counter()
        found = beam_search(kernel, prompts, a.beams, new, a.eos, embed, final_norm, layer_weights, cos, sin, a.max_seq)
        wall = time.perf_counter() - t0
        for i, group in enumerate(found):
            print(f"prompt {i} ({len(prompts[i])} tokens): " + "; ".join(
                f"{score:.3f} {tokens[:8]}{' ...' if len(tokens) > 8 else ''}" if score == score else "failed"
                for tokens, score in group))
        print(f"beam search: {a.prompts} x {a.beams} beams, {new} steps in {wall * 1e3:.1f} ms, device status "
              f"{kernel.status()}")
        return {"prompt": a.prompt, "prompts": prompts, "beams": found, "status": kernel.status(),
                "generated": [t for group in found for tokens, score in group
                              for t in (tokens if score == score else [-1])],  # -1: a failed beam
                "inputs": {"embed": embed, "final_norm": final_norm, "layer_weights": layer_weights, "cos": cos,
                           "sin": sin, "max_seq": a.max_seq}}

    k_cache, v_cache = megakernel.empty_cache(len(model.model.layers), a.max_seq, dev)
    if a.native_prefill:
        prompt = ids[0].to(device=dev, dtype=torch.int32)
        p0, p1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        p0.record()
        _, first = kernel.prefill(prompt, embed, embed, final_norm, layer_weights, cos, sin, k_cache, v_cache, 0,
                                  a.max_seq)
        p1.record()
        position, token = a.prompt, int(first.item())
        print(f"prefill: {a.prompt} tokens in {p0.elapsed_time(p1):.2f} ms (batched prefill kernel)")
    else:
        with torch.inference_mode():
            out = model(ids, use_cache=True)
        position = megakernel.copy_prefill_cache(out.past_key_values, k_cache, v_cache)
        token = int(out.logits[0, -1].float().argmax())
    result = {"prompt": position, "first_token": token}
    if keep_prefill_cache:
        result["prefill_cache"] = (k_cache.clone(), v_cache.clone())
        result["inputs"] = {"embed": embed, "final_norm": final_norm, "layer_weights": layer_weights, "cos": cos,
                            "sin": sin, "max_seq": a.max_seq}

    generated = [token]
    steps = min(a.new, a.max_seq - position)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0 = time.perf_counter()
    start.record()
    if a.device_loop and steps > 1:
        tokens = torch.zeros(steps, dtype=torch.int32, device=dev)
        tokens[0] = token
        kernel.decode_steps(tokens, steps - 1, True, embed, embed, final_norm, layer_weights, cos, sin, k_cache,
                            v_cache, position, a.max_seq)
    else:
        for _ in range(steps - 1):
            _, tok = kernel.decode_greedy(token, embed, embed, final_norm, layer_weights, cos, sin, k_cache,
                                          v_cache, position, a.max_seq)
            token = int(tok.item())
            generated.append(token)
            position += 1
    end.record()
    end.synchronize()
    wall = time.perf_counter() - t0
    if a.device_loop and steps > 1:
        generated = tokens.tolist()
    n = max(steps - 1, 1)
    result.update(generated=generated, status=kernel.status(), ms_per_token=start.elapsed_time(end) / n)
    print(f"generated {len(generated)} tokens: {generated[:16]}{' ...' if len(generated) > 16 else ''}")
    print(f"decode: {result['ms_per_token']:.3f} ms/token (device events), {n / wall:.1f} tokens/s wall, "
          f"device status {result['status']}")
    return result


def main(argv=None):
    """The command line: 0 when the device status is clean and every generated token is valid."""
    r = run(argv)
    return 0 if r["status"] == 0 and all(t >= 0 for t in r["generated"]) else 1


if __name__ == "__main__":
    sys.exit(main())
