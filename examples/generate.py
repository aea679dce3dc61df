"""Greedy generation by an encoder-decoder next to MonarchAttention.

The shape of the reference's BART summarisation (bart/model.py, bart/pipeline.py)
with random weights: the encoder's layers attend with MonarchAttention under the
source's key-padding mask; their keys and values for the decoder's cross
attention are stored once in a paged cache, the decoder's own token by token,
both in the type asked for; every new token attends to both with
decode_attention.  At the end the decoder's cached context of the first layer is
read back as the dense tensors and mask that MonarchAttention takes.

    python examples/generate.py [--cache e4m3] [--tokens 64]
"""
import argparse
import os
import sys
import time

import torch
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
import monarch_attention_b200 as mab  # noqa: E402

CACHES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class Model:
    """Pre-norm encoder and decoder layers of width heads * dim, random weights."""

    def __init__(self, layers, heads, dim, vocab, block, dtype, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        width = heads * dim
        w = lambda *s: (torch.randn(s, generator=g, device=device) / s[-1] ** 0.5).to(dtype)
        self.heads, self.dim, self.width = heads, dim, width
        self.embed = torch.randn(vocab, width, generator=g, device=device).to(dtype)
        block_of = lambda: {"qkv": w(3 * width, width), "out": w(width, width),
                            "up": w(2 * width, width), "down": w(width, 2 * width)}
        self.encoder = [block_of() for _ in range(layers)]
        self.decoder = [{**block_of(), "cross_q": w(width, width), "cross_kv": w(2 * width, width),
                         "cross_out": w(width, width)} for _ in range(layers)]
        self.attention = mab.MonarchAttention(block, 2, mab.PadType.post)

    def norm(self, x):
        return F.layer_norm(x, (self.width,))

    def split(self, x, n):
        """(E, T, n * width) -> n views (E, heads, T, dim), no copy."""
        E, T, _ = x.shape
        return [t.view(E, T, self.heads, self.dim).permute(0, 2, 1, 3) for t in x.chunk(n, -1)]

    def merge(self, x):
        return x.transpose(1, 2).reshape(x.shape[0], x.shape[2], self.width)

    def feed(self, p, x):
        return x + F.gelu(self.norm(x) @ p["up"].t()) @ p["down"].t()

    def encode(self, source, mask):
        x = self.embed[source]
        for p in self.encoder:
            q, k, v = self.split(self.norm(x) @ p["qkv"].t(), 3)
            x = x + self.merge(self.attention(q, k, v, mask)) @ p["out"].t()
            x = self.feed(p, x)
        return x

    def step(self, token, own, cross, mask):
        """Logits of the next token of every sequence; `own` grows by one token."""
        x = self.embed[token][:, None]
        for p, mine, theirs in zip(self.decoder, own, cross):
            q, k, v = self.split(self.norm(x) @ p["qkv"].t(), 3)
            mine.append(k, v)
            x = x + self.merge(mine.attend(q)) @ p["out"].t()
            (q,) = self.split(self.norm(x) @ p["cross_q"].t(), 1)
            x = x + self.merge(theirs.attend(q, mask)) @ p["cross_out"].t()
            x = self.feed(p, x)
        return (self.norm(x) @ self.embed.t())[:, 0]


@torch.no_grad()
def generate(batch=4, source_len=1024, tokens=64, layers=2, heads=12, dim=64, vocab=1000, block=32,
             cache="bf16", dtype=torch.bfloat16, device="cuda", seed=0):
    """Greedy tokens (batch, tokens), all steps' logits, the model, its caches and inputs."""
    g = torch.Generator(device=device).manual_seed(seed + 1)
    model = Model(layers, heads, dim, vocab, block, dtype, device, seed)
    source = torch.randint(0, vocab, (batch, source_len), generator=g, device=device)
    lengths = torch.randint(source_len // 2, source_len + 1, (batch,), generator=g, device=device)
    mask = torch.arange(source_len, device=device)[None] < lengths[:, None]

    def new_cache(max_len):
        pages = batch * -(-max_len // 64)
        return mab.PagedKVCache(pages, heads, dim, max_seqs=batch, max_len=max_len, page_size=64,
                                dtype=CACHES[cache], device=device)

    memory = model.norm(model.encode(source, mask))
    cross = [new_cache(source_len) for _ in range(layers)]
    for p, c in zip(model.decoder, cross):
        c.append(*model.split(memory @ p["cross_kv"].t(), 2))
    own = [new_cache(tokens) for _ in range(layers)]
    token = torch.zeros(batch, dtype=torch.long, device=device)
    out, logits = [], []
    for _ in range(tokens):
        logits.append(model.step(token, own, cross, mask))
        token = logits[-1].argmax(-1)
        out.append(token)
    mab.check_status(torch.device(device, torch.cuda.current_device())
                     if device == "cuda" else torch.device(device))
    return dict(tokens=torch.stack(out, 1), logits=torch.stack(logits, 1), model=model, own=own,
                cross=cross, source=source, mask=mask, memory=memory)


@torch.no_grad()
def dense_logits(r):
    """The same decoder over all generated tokens at once in fp32, with dense
    causal and cross attention instead of the caches."""
    m, tokens, mask = r["model"], r["tokens"], r["mask"]
    f = lambda p: {k: v.float() for k, v in p.items()}
    T = tokens.shape[1]
    inputs = torch.cat([torch.zeros_like(tokens[:, :1]), tokens[:, :-1]], 1)
    x = m.embed.float()[inputs]
    causal = torch.ones(T, T, dtype=torch.bool, device=x.device).tril()

    def attend(q, k, v, ok):
        s = (q @ k.transpose(-1, -2)) * m.dim ** -0.5
        return torch.softmax(s.masked_fill(~ok, -torch.inf), -1) @ v

    for p in map(f, m.decoder):
        q, k, v = m.split(m.norm(x) @ p["qkv"].t(), 3)
        x = x + m.merge(attend(q, k, v, causal)) @ p["out"].t()
        (q,) = m.split(m.norm(x) @ p["cross_q"].t(), 1)
        k, v = m.split(r["memory"].float() @ p["cross_kv"].t(), 2)
        x = x + m.merge(attend(q, k, v, mask[:, None, None])) @ p["cross_out"].t()
        x = m.feed(p, x)
    return m.norm(x) @ m.embed.float().t()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--cache", choices=sorted(CACHES), default="bf16")
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--source-len", type=int, default=1024)
    a = ap.parse_args()
    dtype = torch.float16 if a.cache == "f16" else torch.bfloat16  # 16-bit pages have the queries' type
    args = dict(batch=a.batch, source_len=a.source_len, tokens=a.tokens, cache=a.cache, dtype=dtype)
    generate(**args)  # first use of every kernel
    torch.cuda.synchronize()
    t = time.perf_counter()
    r = generate(**args)
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    err = (r["logits"].float() - dense_logits(r)).abs().max() / r["logits"].float().abs().max()
    k, v, mask = r["own"][0].read()
    print(f"{a.batch} x {a.tokens} tokens from {a.source_len} with a {a.cache} cache: {t * 1e3:.1f} ms; "
          f"logits within {err:.2g} of the dense fp32 decoder; read back {tuple(k.shape)}, "
          f"{int(mask.sum())} valid tokens")


if __name__ == "__main__":
    main()
