"""Serves several continuations of one prompt from the 8-bit paged KV cache.

A small decoder with random Q6_K weights reads a prompt once (in chunks), forks
the sequence, which shares the prompt's pages, decodes the forks together, ends
some of them, packs the pages that are left and decodes on:

    python examples/serve_paged.py --prompt 700 --forks 6 --steps 24 --format e4m3
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from vibrant_b200 import kv8, synth, tensor, vkq  # noqa: E402


class Decoder:
    """RMSNorm, attention and a SiLU feed-forward in each layer; weights stay packed."""

    def __init__(self, layers=3, width=512, heads=8, kv_heads=2, head_dim=64, hidden=1024, vocab=1024, seed=0,
                 device="cuda:0"):
        self.heads, self.kv_heads, self.head_dim, self.width = heads, kv_heads, head_dim, width
        gen = torch.Generator(device=device).manual_seed(seed)

        def weight(k, n, i):
            data = synth.weights_device(vkq.Q6_K, k, n, seed * 1000 + i, device)
            return tensor.QuantWeight(vkq.Q6_K, k, n, data, device=device)

        self.embedding = torch.randn(vocab, width, generator=gen, device=device)
        self.norm = torch.ones(width, device=device)
        shapes = [(width, heads * head_dim), (width, kv_heads * head_dim), (width, kv_heads * head_dim),
                  (heads * head_dim, width), (width, hidden), (width, hidden), (hidden, width)]
        self.layers = [[weight(k, n, 10 * i + j) for j, (k, n) in enumerate(shapes)] for i in range(layers)]
        self.head = weight(width, vocab, 10 * layers)
        self.device = torch.device(device)

    def normed(self, x):
        out = torch.empty_like(x)
        vkq.rms_norm(x.data_ptr(), self.norm.data_ptr(), out.data_ptr(), x.shape[0], x.shape[1], 1e-6,
                     device=self.device.index, stream=torch.cuda.current_stream(self.device))
        return out

    def step(self, tokens, cache, batch, cos, sin, last):
        """Logits of the rows `last` of the new tokens, which join the cache."""
        x = self.embedding[tokens]
        for i, (wq, wk, wv, wo, gate, up, down) in enumerate(self.layers):
            h = self.normed(x)
            q, k, v = (tensor.matmul(h, w).unflatten(1, (-1, self.head_dim)) for w in (wq, wk, wv))
            q = cache.append(i, batch, k, v, q=q, cos=cos, sin=sin, layout="half")
            x = x + tensor.matmul(cache.attend(i, batch, q).flatten(1), wo)
            h = self.normed(x)
            g, u = tensor.matmul(h, gate), tensor.matmul(h, up)
            vkq.silu_mul(g.data_ptr(), u.data_ptr(), g.data_ptr(), g.numel(), device=self.device.index,
                         stream=torch.cuda.current_stream(self.device))
            x = x + tensor.matmul(g, down)
        return tensor.matmul(self.normed(x[last]), self.head)


def serve(prompt=700, chunk=256, forks=6, steps=24, fmt="e4m3", page=32, compact=True, model=None):
    """Tokens [forks, steps] that the forks chose (-1 after their end), the logits
    of the last step, and the bookkeeping at the end."""
    model = model or Decoder()
    dev = model.device
    most = prompt + steps + 1
    max_pages = -(-most // page)
    # the prompt's pages once, and each fork's own
    pages = -(-prompt // page) + forks * (2 + -(-steps // page))
    cache = kv8.Cache(len(model.layers), pages, page, model.kv_heads, model.head_dim, fmt, device=dev)
    seqs = kv8.Sequences(cache, forks + 1, max_pages)
    cos, sin = tensor.rotary_tables(model.head_dim, 1e4, most, "yarn", factor=2.0, orig_len=max(most // 2, 1), device=dev)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731

    # the prompt, in row 0, a chunk at a time
    text = torch.randint(0, model.embedding.shape[0], (prompt,), generator=torch.Generator().manual_seed(1)).to(dev)
    parent = ints([0])
    for at in range(0, prompt, chunk):
        n = min(chunk, prompt - at)
        seqs.extend(parent, ints([n]))
        batch = seqs.batch(parent, tokens=n, cu_tokens=ints([0, n]), max_tokens=n, max_len=at + n)
        logits = model.step(text[at:at + n], cache, batch, cos, sin, slice(n - 1, n))

    # rows 1 .. forks go on from it with its likeliest tokens, one each
    rows = list(range(1, forks + 1))
    seqs.fork(ints([0] * forks), ints(rows))
    seqs.free(parent)
    tokens = logits[0].topk(forks).indices
    chosen = torch.full((forks, steps), -1, dtype=torch.int64, device=dev)
    for i in range(steps):
        if i == steps // 2 and forks > 1:  # half of them end here
            seqs.free(ints(rows[1::2]))
            tokens, rows = tokens[0::2], rows[0::2]
            if compact:
                seqs.compact()
        slots = ints(rows)
        chosen[slots.long() - 1, i] = tokens
        seqs.extend(slots, torch.ones_like(slots))
        batch = seqs.batch(slots, tokens=len(rows), max_len=prompt + i + 1)
        logits = model.step(tokens, cache, batch, cos, sin, slice(None))
        tokens = logits.argmax(dim=1)
    torch.cuda.synchronize(dev)
    status = vkq.device_status(dev.index)
    if status != vkq.OK:
        raise RuntimeError(f"device status {status}")
    return chosen, logits, cache, seqs


def main():
    a = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    a.add_argument("--prompt", type=int, default=700)
    a.add_argument("--chunk", type=int, default=256)
    a.add_argument("--forks", type=int, default=6)
    a.add_argument("--steps", type=int, default=24)
    a.add_argument("--format", choices=sorted(kv8.FORMATS), default="e4m3")
    args = a.parse_args()
    chosen, _, cache, seqs = serve(args.prompt, args.chunk, args.forks, args.steps, args.format)
    for i, row in enumerate(chosen.tolist()):
        print(f"fork {i}: {' '.join(str(t) for t in row if t >= 0)}")
    used = int((seqs.refs > 0).sum())
    print(f"{used} of {cache.num_pages} pages in use, {int(seqs.lens.sum())} tokens of {int((seqs.lens > 0).sum())} sequences")


if __name__ == "__main__":
    main()
