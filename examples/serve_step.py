"""One attention layer of a quantized decoder served to a batch of conversations
over a common document:

- the projections are ``fp4_linear`` (microscaled 4-bit weights and activations);
- keys and values go into a ``paged_kv_cache`` (int8 or int4 codes);
- the document's pages are written once and read once a step for the whole
  batch (``prefix_table``), each conversation's own tokens follow.

    python examples/serve_step.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import qtpytorch_b200 as mxb  # noqa: E402


class AttentionLayer:
    """Grouped-query attention with quantized projections and cache."""

    def __init__(self, dim=1024, heads=8, kv_heads=2, pages=256, page_size=32, fmt="nvfp4",
                 cache_dtype="int8d", seed=0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, dim // heads

        def proj(n, k):
            lin = torch.nn.Linear(k, n, bias=False, device="cuda")
            with torch.no_grad():
                lin.weight.copy_(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
            return mxb.fp4_linear.from_linear(lin, fmt)

        self.qkv = proj(dim + 2 * kv_heads * self.head_dim, dim)
        self.out = proj(dim, dim)
        self.cache = mxb.paged_kv_cache(pages, kv_heads, self.head_dim, cache_dtype, page_size)
        self._free = list(range(pages))

    def take_pages(self, n: int) -> list:
        taken, self._free = self._free[:n], self._free[n:]
        if len(taken) < n:
            raise RuntimeError("the cache has no free pages")
        return taken

    def write(self, x: torch.Tensor, slots: torch.Tensor):
        """Project tokens x [T, dim], store their keys and values; their queries."""
        q, k, v = self.qkv(x).split([self.heads * self.head_dim] + 2 * [self.kv_heads * self.head_dim], -1)
        self.cache.write(k.unflatten(-1, (self.kv_heads, self.head_dim)),
                         v.unflatten(-1, (self.kv_heads, self.head_dim)), slots)
        return q.unflatten(-1, (self.heads, self.head_dim))

    def step(self, x, slots, table, lengths, prefix_table, prefix_len):
        """x [B, T, dim]: the T newest tokens of each conversation, already
        counted in ``lengths``."""
        B, T, dim = x.shape
        q = self.write(x.reshape(B * T, dim), slots.reshape(-1))
        o = mxb.paged_attention(q.reshape(B, T, self.heads, self.head_dim), self.cache, table, lengths,
                                prefix_table=prefix_table, prefix_len=prefix_len)
        return self.out(o.reshape(B, T, dim))


def slots_of(pages: torch.Tensor, positions: torch.Tensor, page_size: int) -> torch.Tensor:
    """Slots of token positions of a sequence whose pages are ``pages``."""
    return pages[positions // page_size].long() * page_size + positions % page_size


def main(batch=6, document=300, steps=5, cache_dtype="int8d", fmt="nvfp4"):
    layer = AttentionLayer(cache_dtype=cache_dtype, fmt=fmt)
    page = layer.cache.page_size
    g = torch.Generator("cuda").manual_seed(1)

    def tokens(*shape):
        return torch.randn(*shape, 1024, generator=g, device="cuda").bfloat16()

    doc_pages = torch.tensor(layer.take_pages(-(-document // page)), device="cuda")
    layer.write(tokens(document), slots_of(doc_pages, torch.arange(document, device="cuda"), page))
    table = torch.tensor([layer.take_pages(-(-steps // page)) for _ in range(batch)], device="cuda")
    outs = []
    for i in range(steps):
        at = torch.full((batch,), i, device="cuda")
        slots = torch.stack([slots_of(table[b], at[b:b + 1], page) for b in range(batch)])
        lengths = torch.full((batch,), i + 1, dtype=torch.int32, device="cuda")
        outs.append(layer.step(tokens(batch, 1), slots, table, lengths, doc_pages, document))
    return layer, torch.cat(outs, 1)


if __name__ == "__main__":
    for cache_dtype, fmt in (("int8d", "nvfp4"), ("int4d", "mxfp4")):
        layer, y = main(cache_dtype=cache_dtype, fmt=fmt)
        torch.cuda.synchronize()
        print(f"{fmt} projections, {layer.cache}: out {tuple(y.shape)}, rms {y.float().square().mean().sqrt():.4f}")
