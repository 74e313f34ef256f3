"""A small paged-cache server: prompts in chunks, beams that share pages, single-token steps, compaction.

A toy decoder (random weights, synthetic tokens) whose cache is only ever touched by the serving-step operators:
``fork_pages`` gives the rows their pages, ``rotary_append`` turns the new tokens' queries and keys and appends to the
cache, ``paged_chunk_attention`` attends over it, ``compact_pages`` closes the gaps. Lengths, offsets and tables stay on
the device throughout.

    python -m fgw_b200.examples.serving_step [--beams 4 --steps 16 ...]
"""
import argparse

import torch

from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
from fgw_b200.operators.mha.page_ops import compact_pages, fork_pages
from fgw_b200.operators.mha.rotary_append import rotary_append, rotary_table


class Decoder:
    """Weights of the toy decoder: per layer one fused query/key/value projection and one output projection, and a head."""

    def __init__(self, layers, heads, kv_heads, dim, vocab, positions, dtype=torch.bfloat16, seed=0):
        gen = torch.Generator().manual_seed(seed)
        width = heads * dim
        self.layers, self.heads, self.kv_heads, self.dim, self.dtype = layers, heads, kv_heads, dim, dtype

        def weight(*shape):
            return (torch.randn(*shape, generator=gen) * shape[0] ** -0.5).to(dtype).cuda()

        self.embedding = torch.randn(vocab, width, generator=gen).to(dtype).cuda()
        self.qkv = [weight(width, (heads + 2 * kv_heads) * dim) for _ in range(layers)]
        self.out = [weight(width, width) for _ in range(layers)]
        self.head = weight(width, vocab)
        # twice as many positions as "trained": linear scaling by two
        self.cos_sin = rotary_table(positions, dim, scaling="linear", factor=2.0)


class Server:
    """The rows of a batch over one page pool per layer and K/V."""

    def __init__(self, model, rows, pages, page, width):
        self.model, self.page = model, page
        shape = (pages * page, model.kv_heads, model.dim)
        self.pools = [torch.zeros(shape, dtype=model.dtype, device="cuda") for _ in range(2 * model.layers)]
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(rows, dtype=torch.int32, device="cuda")

    def fork(self, parents, more):
        """Row i goes on from row ``parents[i]`` (-1: it is free) with room for ``more[i]`` tokens; returns the status."""
        reserve = torch.where(parents >= 0, self.lens[parents.clamp(min=0)], 0) + more
        self.table, self.lens, status = fork_pages(self.pools, self.table, self.lens, parents, self.page,
                                                   reserve_seqlens=reserve.int())
        return status

    def step(self, tokens, counts):
        """Run ``tokens`` (``counts[b]`` new ones of each row, end to end) through the layers; returns their states."""
        m = self.model
        offsets = torch.zeros(counts.numel() + 1, dtype=torch.int32, device="cuda")
        offsets[1:] = torch.cumsum(counts, 0)
        self.lens = self.lens + counts
        x = m.embedding[tokens]
        for layer in range(m.layers):
            k_cache, v_cache = self.pools[2 * layer], self.pools[2 * layer + 1]
            normal = torch.nn.functional.rms_norm(x, x.shape[-1:])
            qkv = (normal @ m.qkv[layer]).view(-1, m.heads + 2 * m.kv_heads, m.dim)
            q, k, v = qkv.split([m.heads, m.kv_heads, m.kv_heads], 1)
            q = rotary_append(q, k, v, k_cache, v_cache, self.table, self.lens, offsets, m.cos_sin, self.page)
            attended = paged_chunk_attention(q, k_cache, v_cache, self.table, self.lens, offsets, self.page)
            x = x + attended.flatten(1) @ m.out[layer]
        return x

    def compact(self):
        """Move the live pages to the pools' start; returns (live pages, pages moved) on the device."""
        self.table, status = compact_pages(self.pools, self.table, self.lens, self.page)
        return status


def beam_decode(model, prompts, beams, steps, page=16, chunk=64):
    """Beam search from ``prompts`` (lists of tokens); returns (tokens [prompts * beams][...], scores, last states).

    Every prompt runs in chunks on its first row, forks into its beams, and each step keeps the best ``beams`` of their
    continuations, forking and freeing rows as the choice says.
    """
    rows = len(prompts) * beams
    longest = max(map(len, prompts)) + steps
    width = -(-longest // page) + 1
    server = Server(model, rows, pages=rows * width, page=page, width=width)
    first = torch.arange(len(prompts), device="cuda") * beams  # each prompt's first row
    own = torch.arange(rows, dtype=torch.int32, device="cuda")
    state = None
    for start in range(0, max(map(len, prompts)), chunk):
        parts = [p[start:start + chunk] for p in prompts]
        counts = torch.zeros(rows, dtype=torch.int32, device="cuda")
        counts[first] = torch.tensor([len(p) for p in parts], dtype=torch.int32, device="cuda")
        server.fork(own, counts)
        x = server.step(torch.tensor([t for p in parts for t in p], device="cuda"), counts)
        ends = torch.cumsum(counts[first], 0).long() - 1
        state = x[ends.clamp(min=0)] if state is None else torch.where((counts[first] > 0)[:, None],
                                                                       x[ends.clamp(min=0)], state)
    one = torch.ones(rows, dtype=torch.int32, device="cuda")
    tokens = torch.empty(rows, 0, dtype=torch.long, device="cuda")
    scores = torch.zeros(rows, device="cuda")
    for step in range(steps):
        logp = torch.log_softmax((state @ model.head).float(), -1)  # [prompts or rows, vocab]
        vocab = logp.shape[-1]
        if step == 0:
            best, at = torch.topk(logp, beams, -1)
            parents = first.repeat_interleave(beams)
            chosen, scores = at.flatten(), best.flatten()
        else:
            total = (scores[:, None] + logp).view(len(prompts), beams * vocab)
            best, at = torch.topk(total, beams, -1)
            parents = (first[:, None] + at // vocab).flatten()
            chosen, scores = (at % vocab).flatten(), best.flatten()
        server.fork(parents.int(), one)
        tokens = torch.cat([tokens[parents], chosen[:, None]], 1)
        state = server.step(chosen, one)
        if step == steps // 2:
            server.compact()
    return tokens, scores, state


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("layers", 4), ("heads", 8), ("kv-heads", 2), ("dim", 128), ("vocab", 1000), ("prompts", 4),
                        ("beams", 4), ("steps", 16), ("length", 300)):
        parser.add_argument("--" + name, type=int, default=value)
    args = parser.parse_args(argv)
    model = Decoder(args.layers, args.heads, args.kv_heads, args.dim, args.vocab, args.length + args.steps)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(args.vocab, (args.length - 37 * i % args.length,), generator=gen).tolist()
               for i in range(args.prompts)]
    tokens, scores, _ = beam_decode(model, prompts, args.beams, args.steps)
    for i in range(args.prompts):
        row = i * args.beams
        print(f"prompt {i} ({len(prompts[i])} tokens): {tokens[row].tolist()} ({scores[row].item():.3f})")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
