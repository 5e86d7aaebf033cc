"""Serving a small decoder: whole prompts first, then a token of every sequence
a step, out of a paged 8-bit cache.

    python -m examples.serve [--steps 16] [--code float8_e4m3fn|int8] [--piece 64] [--int4]

One attention layer with random weights between an embedding and its transpose
as the output head: enough to run every serving operator as a server does.

  prompts   q/k/v projection -> paged_append (rotates q and k, stores k and v)
            -> prompt_attention over the rotated prompt -> output projection
  a step    q/k/v projection -> paged_append -> paged_attention -> output
            projection, for one new token of each sequence

With --piece the prompts come in pieces of so many tokens, which attend over the
cache (chunk_attention); with --int4 the projections have 4-bit weights
(int4_matmul) and the rows before the first are normed to 8 bits (rms_norm).
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

    def __init__(self, vocabulary=512, heads=8, kv_heads=2, head_dim=64, max_tokens=1024, seed=0, device="cuda",
                 int4=False):
        gen = torch.Generator(device).manual_seed(seed)
        width = heads * head_dim

        def weight(rows, cols):
            return (torch.randn((rows, cols), generator=gen, device=device) * rows**-0.5).half()

        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.embedding = weight(vocabulary, width) * vocabulary**0.5
        self.qkv, self.out = weight(width, (heads + 2 * kv_heads) * head_dim), weight(width, width)
        self.cos, self.sin = programs.rotary_tables(max_tokens, head_dim, device=device)
        self.int4 = int4
        if int4:
            self.norm = torch.ones(width, dtype=torch.float16, device=device)
            self.qkv, self.out = (programs.int4_quantize(w.T.contiguous(), 64, symmetric=False) for w in (self.qkv, self.out))

    def project(self, tokens):
        if self.int4:
            codes, scale = programs.rms_norm(self.embedding[tokens], self.norm, code_dtype=torch.float8_e4m3fn)
            qkv = programs.int4_matmul(codes, *self.qkv, input_scale=scale)
        else:
            normed = torch.nn.functional.layer_norm(self.embedding[tokens], self.embedding.shape[-1:])
            qkv = programs.matmul(normed, self.qkv)
        qkv = qkv.view(len(tokens), -1, self.head_dim)
        return qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)

    def logits(self, attended):
        attended = attended.flatten(1)
        hidden = programs.int4_matmul(attended, *self.out) if self.int4 else programs.matmul(attended, self.out)
        return programs.matmul(hidden, self.embedding.T)

    def prompts(self, tokens, offsets, cache):
        """Logits of every token of packed prompts, which are stored in the cache."""
        query, key, value = self.project(tokens)
        past = torch.zeros_like(offsets[1:])
        query, key = programs.paged_append(key, value, offsets, past, cache.table, *cache.tensors, query=query,
                                           cos=self.cos, sin=self.sin, return_key=True)
        return self.logits(programs.prompt_attention(query, key, value, offsets))

    def pieces(self, tokens, offsets, past, cache):
        """Logits of every token of packed pieces of prompts that had `past` tokens."""
        query, key, value = self.project(tokens)
        query, _ = programs.paged_append(key, value, offsets, past, cache.table, *cache.tensors, query=query,
                                         cos=self.cos, sin=self.sin)
        lengths = past + offsets[1:] - offsets[:-1]
        return self.logits(programs.chunk_attention(query, *cache.tensors, cache.table, offsets, lengths))

    def step(self, tokens, lengths, cache):
        """Logits of one new token of each sequence that had `lengths` tokens."""
        query, key, value = self.project(tokens)
        offsets = torch.arange(len(tokens) + 1, dtype=torch.int32, device=tokens.device)
        query, _ = programs.paged_append(key, value, offsets, lengths, cache.table, *cache.tensors, query=query,
                                         cos=self.cos, sin=self.sin)
        attended = programs.paged_attention(query[:, None], *cache.tensors, cache.table, lengths + 1)
        return self.logits(attended[:, 0])


def offsets_of(lengths):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")


def by_pieces(model, prompts, cache, piece):
    """The last logits of each prompt, which come `piece` tokens at a time."""
    last = [None] * len(prompts)
    for start in range(0, max(map(len, prompts)), piece):
        parts = [prompt[start : start + piece] for prompt in prompts]
        past = torch.tensor([min(start, len(prompt)) for prompt in prompts], dtype=torch.int32, device="cuda")
        offsets = offsets_of([len(part) for part in parts])
        logits = model.pieces(torch.cat(parts), offsets, past, cache)
        for s, end in enumerate(offsets[1:].tolist()):
            if len(parts[s]):
                last[s] = logits[end - 1]
    return torch.stack(last)


def serve(prompt_lengths=(37, 5, 200, 64), steps=16, code=torch.float8_e4m3fn, seed=0, piece=None, int4=False):
    """Continues random prompts greedily; returns each sequence's tokens and the
    logits that chose its continuation [steps, batch, vocabulary]."""
    model = Decoder(seed=seed, int4=int4)
    batch, lengths = len(prompt_lengths), list(prompt_lengths)
    longest = max(lengths) + steps
    cache = PagedCache(batch * -(-longest // 16), model.kv_heads, 16, model.head_dim, code, longest, batch)
    gen = torch.Generator("cuda").manual_seed(seed + 1)
    tokens = torch.randint(0, len(model.embedding), (sum(lengths),), generator=gen, device="cuda")
    offsets = offsets_of(lengths)
    cache.reserve(lengths)
    if piece:
        logits = by_pieces(model, torch.split(tokens, lengths), cache, piece)
    else:
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
    parser.add_argument("--piece", type=int)
    parser.add_argument("--int4", action="store_true")
    args = parser.parse_args()
    sequences, _ = serve(steps=args.steps, code=getattr(torch, args.code), piece=args.piece, int4=args.int4)
    for s, sequence in enumerate(sequences):
        print(f"sequence {s}: {len(sequence) - args.steps} prompt tokens, then {sequence[-args.steps:].tolist()}")


if __name__ == "__main__":
    main()
