"""Serving a small decoder: whole prompts first, then a token of every sequence
a step, out of a paged 8-bit cache.

    python -m examples.serve [--steps 16] [--code float8_e4m3fn|int8]

One attention layer with random weights between an embedding and its transpose
as the output head: enough to run every serving operator as a server does.

  prompts   q/k/v projection -> paged_append (rotates q and k, stores k and v)
            -> prompt_attention over the rotated prompt -> output projection
  a step    q/k/v projection -> paged_append -> paged_attention -> output
            projection, for one new token of each sequence
"""

import argparse

import torch

from ninetoothed_b200 import programs


class PagedCache:
    """Pages of 8-bit keys and values with their scales, handed out to sequences as they grow."""

    def __init__(self, pages, kv_heads, page, head_dim, code, max_tokens, batch, device="cuda"):
        shape = (pages, kv_heads, page, head_dim)
        self.page = page
        self.key, self.value = (torch.empty(shape, dtype=code, device=device) for _ in range(2))
        self.key_scale, self.value_scale = (torch.zeros(shape[:2], device=device) for _ in range(2))
        self.free = list(range(pages))
        self.table = torch.zeros((batch, -(-max_tokens // page)), dtype=torch.int32, device=device)
        self.owned = [0] * batch

    @property
    def tensors(self):
        return self.key, self.value, self.key_scale, self.value_scale

    def reserve(self, lengths):
        """Pages for sequences of these lengths."""
        for s, length in enumerate(lengths):
            while self.owned[s] * self.page < length:
                self.table[s, self.owned[s]] = self.free.pop()
                self.owned[s] += 1


class Decoder:
    """attention(norm(x)) W_o, then the embedding's transpose."""

    def __init__(self, vocabulary=512, heads=8, kv_heads=2, head_dim=64, max_tokens=1024, seed=0, device="cuda"):
        gen = torch.Generator(device).manual_seed(seed)
        width = heads * head_dim

        def weight(rows, cols):
            return (torch.randn((rows, cols), generator=gen, device=device) * rows**-0.5).half()

        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.embedding = weight(vocabulary, width) * vocabulary**0.5
        self.qkv, self.out = weight(width, (heads + 2 * kv_heads) * head_dim), weight(width, width)
        self.cos, self.sin = programs.rotary_tables(max_tokens, head_dim, device=device)

    def project(self, tokens):
        normed = torch.nn.functional.layer_norm(self.embedding[tokens], self.embedding.shape[-1:])
        qkv = programs.matmul(normed, self.qkv).view(len(tokens), -1, self.head_dim)
        return qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)

    def logits(self, attended):
        return programs.matmul(programs.matmul(attended.flatten(1), self.out), self.embedding.T)

    def prompts(self, tokens, offsets, cache):
        """Logits of every token of packed prompts, which are stored in the cache."""
        query, key, value = self.project(tokens)
        past = torch.zeros_like(offsets[1:])
        query, key = programs.paged_append(key, value, offsets, past, cache.table, *cache.tensors, query=query,
                                           cos=self.cos, sin=self.sin, return_key=True)
        return self.logits(programs.prompt_attention(query, key, value, offsets))

    def step(self, tokens, lengths, cache):
        """Logits of one new token of each sequence that had `lengths` tokens."""
        query, key, value = self.project(tokens)
        offsets = torch.arange(len(tokens) + 1, dtype=torch.int32, device=tokens.device)
        query, _ = programs.paged_append(key, value, offsets, lengths, cache.table, *cache.tensors, query=query,
                                         cos=self.cos, sin=self.sin)
        attended = programs.paged_attention(query[:, None], *cache.tensors, cache.table, lengths + 1)
        return self.logits(attended[:, 0])


def serve(prompt_lengths=(37, 5, 200, 64), steps=16, code=torch.float8_e4m3fn, seed=0):
    """Continues random prompts greedily; returns each sequence's tokens and the
    logits that chose its continuation [steps, batch, vocabulary]."""
    model = Decoder(seed=seed)
    batch, lengths = len(prompt_lengths), list(prompt_lengths)
    longest = max(lengths) + steps
    cache = PagedCache(batch * -(-longest // 16), model.kv_heads, 16, model.head_dim, code, longest, batch)
    gen = torch.Generator("cuda").manual_seed(seed + 1)
    tokens = torch.randint(0, len(model.embedding), (sum(lengths),), generator=gen, device="cuda")
    offsets = torch.tensor([sum(lengths[:i]) for i in range(batch + 1)], dtype=torch.int32, device="cuda")
    cache.reserve(lengths)
    logits = model.prompts(tokens, offsets, cache)[offsets[1:].long() - 1]
    sequences, chosen = [list(s) for s in torch.split(tokens, lengths)], []
    held = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for _ in range(steps):
        chosen.append(logits)
        tokens = logits.argmax(dim=-1)
        for sequence, token in zip(sequences, tokens):
            sequence.append(token)
        lengths = [n + 1 for n in lengths]
        cache.reserve(lengths)
        logits = model.step(tokens, held, cache)
        held += 1
    return [torch.stack(s) for s in sequences], torch.stack(chosen)


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=16)
    parser.add_argument("--code", choices=("float8_e4m3fn", "int8"), default="float8_e4m3fn")
    args = parser.parse_args()
    sequences, _ = serve(steps=args.steps, code=getattr(torch, args.code))
    for s, sequence in enumerate(sequences):
        print(f"sequence {s}: {len(sequence) - args.steps} prompt tokens, then {sequence[-args.steps:].tolist()}")


if __name__ == "__main__":
    main()
