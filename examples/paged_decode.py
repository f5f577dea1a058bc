"""Beam decoding with a decoder layer over a paged 8-bit KV cache.

Random-init Llama-3-8B-shaped layers (``ntops_b200.chain``) and a random output head take ragged
prompts, then continue each with a few beams: pages are reserved (``extend``), keys and values
quantised into them (``store``), attended over (``attention``), beams forked and dropped
(``reorder``), and the pool packed at the end (``compact``).  The scores are meaningless; the calls,
their order and their shapes are those of a serving loop.

    python examples/paged_decode.py [--layers 2] [--requests 4] [--beams 4] [--prompt 300] [--steps 32]
"""

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ntops_b200 import chain, kv_cache  # noqa: E402
import ntops_b200.torch as nt  # noqa: E402

VOCAB = 1024  # of the random output head


def decode(layers=2, requests=4, beams=4, prompt=300, steps=32, page_size=16, dtype=torch.float8_e4m3fn, seed=0,
           device="cuda"):
    """Runs the loop; returns a dict of its final state and timings."""
    g = torch.Generator(device=device).manual_seed(seed)
    wts = [chain.LayerWeights(device, seed=seed + i) for i in range(layers)]
    head = (torch.randn((chain.HIDDEN, VOCAB), generator=g, device=device) * 0.02).to(torch.bfloat16)
    embed = torch.randn((VOCAB, chain.HIDDEN), generator=g, device=device).to(torch.bfloat16)
    sin, cos = chain.rope_tables(prompt + steps, device)
    i32 = dict(dtype=torch.int32, device=device)

    m = -(-(prompt + steps) // page_size)
    cache = kv_cache.PagedKVCache.allocate(layers, requests * beams * m + 8, chain.KV_HEADS, page_size, chain.HEAD_DIM,
                                           dtype=dtype, device=device)
    refs = torch.zeros(cache.num_pages, **i32)
    table = torch.full((requests, m), -1, **i32)

    def forward(tokens, start, lengths):
        x = embed[tokens]
        for i in range(layers):
            x = nt.add(x, chain.layer_step(x, wts[i], sin, cos, cache.layer(i), table, start, lengths))
        return x

    def log_probs(x):  # [rows, VOCAB]
        return torch.log_softmax(nt.mm(x, head).float(), -1)

    # ragged prompts, right after one another in each row
    lengths = torch.tensor([prompt - 7 * i % prompt for i in range(requests)], **i32)
    tokens = torch.randint(0, VOCAB, (requests, prompt), generator=g, device=device)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    table, refs, missing = kv_cache.extend(cache, table, refs, lengths)
    x = forward(tokens, torch.zeros_like(lengths), lengths)
    last = x[torch.arange(requests, device=device), lengths.long() - 1]
    torch.cuda.synchronize()
    t1 = time.perf_counter()

    # each request's best tokens start its beams
    score, tok = log_probs(last).topk(beams)  # [requests, beams]
    parents = torch.arange(requests, device=device).view(-1, 1).expand(-1, beams).reshape(-1).int()
    table, lengths, refs, short = kv_cache.reorder(cache, table, lengths, refs, parents)
    missing = missing + short
    history = tok.reshape(-1, 1)
    for _ in range(steps - 1):
        start, lengths = lengths, lengths + 1
        table, refs, short = kv_cache.extend(cache, table, refs, lengths)
        missing = missing + short
        x = forward(history[:, -1:], start, lengths)
        s = (score.reshape(-1, 1) + log_probs(x[:, 0])).view(requests, beams * VOCAB)
        score, best = s.topk(beams)
        group = torch.arange(requests, device=device).view(-1, 1) * beams
        parents = (group + best // VOCAB).reshape(-1).int()
        table, lengths, refs, short = kv_cache.reorder(cache, table, lengths, refs, parents)
        missing = missing + short
        history = torch.cat((history[parents.long()], (best % VOCAB).reshape(-1, 1)), 1)
    table, refs, used = kv_cache.compact(cache, table, refs)
    torch.cuda.synchronize()
    t2 = time.perf_counter()
    return dict(cache=cache, table=table, lengths=lengths, refs=refs, used=int(used), missing=int(missing),
                history=history.view(requests, beams, -1), score=score, prompt_s=t1 - t0, decode_s=t2 - t1)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    kw = dict(layers=a.layers, requests=a.requests, beams=a.beams, prompt=a.prompt, steps=a.steps)
    decode(**kw)  # warm-up
    r = decode(**kw)
    rows = a.requests * a.beams
    print(f"prompts: {a.requests * a.prompt / r['prompt_s']:.0f} tokens/s; decode: {rows * a.steps / r['decode_s']:.0f} "
          f"tokens/s ({r['decode_s'] / a.steps * 1e3:.2f} ms a step of {rows} beams)")
    print(f"pages in use: {r['used']} of {r['cache'].num_pages}; entries without a page: {r['missing']}")


if __name__ == "__main__":
    main()
