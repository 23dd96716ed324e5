"""A decoder layer's serving step over NF4 weights and a paged key/value cache: the fused layer's
projections (layer.py:871-929) with its training attention replaced by the cache's.

One `step` takes the new tokens of every sequence (whole prompts, chunks of prompts, or a token
each while decoding; any mixture with `cu_q`):

    q|k|v projection -> paged_append (rotation, k and v into the cache) -> attention over the
    cache -> o projection -> residual + RMSNorm -> gate|up + SwiGLU -> down projection

`shared` > 0 says that all sequences start with the same `shared` positions (a system prompt,
whose pages every table row names): attention then reads those keys once for the whole batch.
The page table and the lengths are the caller's tensors, shared by all layers of a model and
updated in place between steps, so a decoding step can be captured in a graph and replayed.
"""

from __future__ import annotations

import torch

from . import kernels
from .quant_state import quantize_4bit
from .stack import Qwen2Shape


class DecoderLayer:
    """`weights`: {"q", "k", "v", "o", "gate", "up", "down"} -> (packed, quant_state); `norm_in`,
    `norm_post`: fp32 RMSNorm weights and `eps` theirs; `bias`: of q|k|v, or None; `window`,
    `sinks`: sliding-window attention (0: full)."""

    def __init__(self, weights: dict, norm_in: torch.Tensor, norm_post: torch.Tensor,
                 bias: torch.Tensor | None = None, window: int = 0, sinks: int = 0,
                 eps: float = 1e-6):
        self.qkv = [weights[n] for n in ("q", "k", "v")]
        self.o, self.gate, self.up, self.down = (weights[n] for n in ("o", "gate", "up", "down"))
        rows = sum(int(qs.shape[0]) for _, qs in self.qkv)
        if bias is not None and tuple(bias.shape) != (rows,):
            raise ValueError(f"the bias of q|k|v is a tensor of {rows} numbers")
        self.norm_in, self.norm_post, self.bias = norm_in, norm_post, bias
        self.window, self.sinks, self.eps = window, sinks, eps

    @classmethod
    def synthetic(cls, shape: Qwen2Shape, device="cuda", seed: int = 0, std: float = 0.02, **kw):
        """Seeded N(0, std) weights of `shape`, norms of ones."""
        g = torch.Generator(device=device).manual_seed(seed)
        w = {n: quantize_4bit(torch.randn(s, generator=g, device=device) * std)
             for n, s in shape.weights().items()}
        one = torch.ones(shape.hidden, device=device)
        return cls(w, one, one.clone(), **kw)

    def step(self, x: torch.Tensor, cache: kernels.PagedKV, cos: torch.Tensor, sin: torch.Tensor,
             cu_q: torch.Tensor | None = None, shared: int = 0, max_q: int = 0,
             max_len: int = 0) -> torch.Tensor:
        """The residual stream after the layer, of the new tokens' x [tokens, hidden] (the cache's
        dtype).  `cos`, `sin`: kernels.rope_table; the rest as in kernels.paged_attention."""
        h, _ = kernels.add_rmsnorm(x, self.norm_in, self.eps)
        bias = None if self.bias is None else self.bias.to(h.dtype).contiguous()
        qkv = kernels.linear_fwd(h, self.qkv, bias=bias)
        q = kernels.paged_append(qkv, cos, sin, cache, cu_q=cu_q)
        kw = dict(cu_q=cu_q, window=self.window, sinks=self.sinks, max_q=max_q, max_len=max_len)
        if shared:
            a = kernels.shared_prefix_attention(q, cache, shared, **kw)
        else:
            a = kernels.paged_attention(q, cache, **kw)
        x = x + kernels.linear_fwd(a.flatten(1), [self.o])
        h, _ = kernels.add_rmsnorm(x, self.norm_post, self.eps)
        return x + kernels.linear_fwd(kernels.linear_swiglu_fwd(h, self.gate, self.up), [self.down])
