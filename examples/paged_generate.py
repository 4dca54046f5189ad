"""Serving with the paged cache: prompts in chunks, tokens one by one, a budget.

    python examples/paged_generate.py [--layers 2] [--prompts 300,17,64] [--new 24]
                                      [--chunk 128] [--budget 0] [--recent 32]

A small decoder (the package's transformer blocks, random weights) serves several
sequences from one :class:`ssa_b200.PagedCache`: every step mixes chunks of prompts
that are still coming in with single tokens of the sequences that are generating,
each layer appends the step's keys and values to the pages and attends over
everything its sequences have cached, and with ``--budget`` a cache that outgrows it
is cut back to the slots that received the most attention.  Without a budget the
last step's logits are checked against the same model run densely over the whole
sequence.
"""

import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import ssa_b200 as ssa  # noqa: E402


class Decoder(nn.Module):
    """Token embedding, ``layers`` blocks, tied output head."""

    def __init__(self, layers=2, hidden=256, num_q_heads=8, num_kv_heads=2, head_dim=64, vocab=512):
        super().__init__()
        self.embed = nn.Embedding(vocab, hidden)
        self.blocks = nn.ModuleList(
            ssa.ToyTransformerBlock(hidden_size=hidden, num_q_heads=num_q_heads, num_kv_heads=num_kv_heads,
                                    head_dim=head_dim) for _ in range(layers))
        self.norm = nn.LayerNorm(hidden)

    def logits(self, x):
        return self.norm(x) @ self.embed.weight.T

    def dense(self, tokens):
        """Logits of every position of one sequence, each layer attending densely."""
        x = self.embed(tokens).unsqueeze(0)
        for block in self.blocks:
            x = block(x, use_dense=True)
        return self.logits(x[0])

    def step(self, cache, batch, tokens):
        """Logits of the step's rows; the cache holds what came before them."""
        x = self.embed(tokens)
        for i, block in enumerate(self.blocks):
            a, h = block.attn, block.norm1(x)
            q = a.q_proj(h).view(-1, a.num_q_heads, a.head_dim)
            k = a.k_proj(h).view(-1, a.num_kv_heads, a.head_dim)
            v = a.v_proj(h).view(-1, a.num_kv_heads, a.head_dim)
            cache.append(batch, k, v, layer=i)
            x = x + a.o_proj(cache.attend(batch, q, layer=i).flatten(1))
            x = x + block.ffn(block.norm2(x))
        return self.logits(x)


@torch.no_grad()
def serve(model, prompts, new_tokens, chunk, budget=0, recent=32, page_size=16):
    """Greedy continuations of ``prompts`` (1-D int64 tensors) by ``new_tokens``
    tokens -> (sequences, logits of the last step, the cache)."""
    attn = model.blocks[0].attn
    device, dtype = model.embed.weight.device, model.embed.weight.dtype
    longest = max(len(p) for p in prompts) + new_tokens
    pages = (len(prompts) + 1) * (-(-longest // page_size) + 1)
    cache = ssa.PagedCache(pages, page_size, attn.num_kv_heads, attn.head_dim, num_layers=len(model.blocks),
                           dtype=dtype, device=device, track_weights=budget > 0)
    ids = [cache.add() for _ in prompts]
    seqs = [p.tolist() for p in prompts]
    total = [len(p) + new_tokens for p in prompts]
    fed = [0] * len(prompts)                       # rows of the sequence the cache has seen
    last = [None] * len(prompts)
    while True:
        # a sequence is done when its last token needs no successor
        live = [i for i in range(len(seqs)) if fed[i] < total[i] - 1]
        if not live:
            return seqs, last, cache
        rows = [min(chunk, len(seqs[i]) - fed[i]) for i in live]
        batch = cache.extend([ids[i] for i in live], rows)
        tokens = torch.tensor([t for i, n in zip(live, rows) for t in seqs[i][fed[i]:fed[i] + n]], device=device)
        logits = model.step(cache, batch, tokens)
        at = 0
        for i, n in zip(live, rows):
            at += n
            fed[i] += n
            if fed[i] == len(seqs[i]):             # its newest token is in: the next one
                last[i] = logits[at - 1]
                seqs[i].append(int(last[i].argmax()))
        if budget:
            cache.evict([ids[i] for i in live], budget, recent)


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--prompts", default="300,17,64", help="prompt lengths")
    p.add_argument("--new", type=int, default=24)
    p.add_argument("--chunk", type=int, default=128)
    p.add_argument("--budget", type=int, default=0, help="cached slots per KV head a sequence may keep (0: all)")
    p.add_argument("--recent", type=int, default=32)
    args = p.parse_args()
    lengths = [int(n) for n in args.prompts.split(",")]
    if min(lengths) < 1 or args.new < 1 or args.chunk < 1:
        p.error("prompts, --new and --chunk: at least one token each")
    if args.budget and not 0 <= args.recent <= args.budget:
        p.error("--recent must be within --budget")
    torch.manual_seed(0)
    model = Decoder(args.layers).cuda()
    prompts = [torch.randint(0, 512, (n,)) for n in lengths]
    seqs, last, cache = serve(model, prompts, args.new, args.chunk, args.budget, args.recent)
    ssa.check_errors()
    for i, (prompt, seq) in enumerate(zip(prompts, seqs)):
        line = f"sequence {i}: {len(prompt)} + {len(seq) - len(prompt)} tokens, {cache.length(i)} slots cached"
        if not args.budget:
            with torch.no_grad():
                ref = model.dense(torch.tensor(seq[:-1], device="cuda"))[-1]
            line += f", logits off the dense model's by {float((last[i] - ref).abs().max()):.1e}"
        print(line)


if __name__ == "__main__":
    main()
