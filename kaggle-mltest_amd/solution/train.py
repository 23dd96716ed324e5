"""A decoder layer's training step over NF4 weights, on a packed batch (FusedDecoderLayer,
layer.py:850-1091): frozen weights, norms and bias, LoRA adapters on q and v with their dropout.

    RMSNorm -> q|k|v projection (+ LoRA of the dropped input) -> rotation and attention ->
    o projection -> residual + RMSNorm -> SwiGLU MLP -> residual

The attention's probabilities, the MLP's activations and the dropout's masks and outputs are not kept:
the backward pass forms them again (`layer.RopeAttention`, `mlp.RecomputedMLP`, `kernels.dropout`).
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import kernels
from .layer import LoraAdapter, ProjectionSpec, project, rope_attention
from .mlp import RecomputedMLP


def _rows2(t):
    """A [tokens, hidden] tensor as the norm's kernels take it: contiguous, 16-byte aligned."""
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


class AddNorm(torch.autograd.Function):
    """apply(x, d or None, weight, eps, dtype) -> (x + d, RMSNorm(x + d) in the GEMM dtype); the norm's
    weight is frozen."""

    @staticmethod
    def forward(ctx, x, d, weight, eps, dtype):
        x, d = _rows2(x), None if d is None else _rows2(d)
        y, rstd = kernels.add_rmsnorm(x, weight, eps, d=d, dtype=dtype)
        ctx.save_for_backward(x, d, weight, rstd)
        ctx.dtype = dtype
        return x.view_as(x) if d is None else x + d.to(x.dtype), y

    @staticmethod
    @once_differentiable
    def backward(ctx, dres, dy):
        x, d, weight, rstd = ctx.saved_tensors
        dx = kernels.rmsnorm_bwd(x, weight, rstd, dy=_rows2(dy), d=d, dres=_rows2(dres), dtype=ctx.dtype)
        return dx, None if d is None else dx.to(d.dtype), None, None, None


class TrainLayer:
    """`weights`: {"q", "k", "v", "o", "gate", "up", "down"} -> (packed, quant_state); `norm_in`,
    `norm_post`: fp32 RMSNorm weights and `eps` theirs; `bias`: of q|k|v, or None; `lora`: (A_q, B_q,
    A_v, B_v), A [rank, hidden] and B [rows, rank]; `alpha` their scale times the rank; `dropout`: of the
    adapters' inputs; `index`: the layer's number in its model (its dropout sites are 2 index and
    2 index + 1)."""

    def __init__(self, weights: dict, norm_in: torch.Tensor, norm_post: torch.Tensor, n_heads: int,
                 n_kv: int, lora, alpha: float = 32.0, dropout: float = 0.0, index: int = 0,
                 bias: torch.Tensor | None = None, window: int = 0, eps: float = 1e-6):
        self.qkv = [weights[n] for n in ("q", "k", "v")]
        self.o, self.gate, self.up, self.down = (weights[n] for n in ("o", "gate", "up", "down"))
        if len(lora) != 4 or lora[0].shape[0] != lora[1].shape[1] or lora[2].shape[0] != lora[3].shape[1]:
            raise ValueError("lora is (A_q [rank, hidden], B_q [rows, rank], A_v, B_v)")
        self.norm_in, self.norm_post, self.bias, self.eps = norm_in, norm_post, bias, eps
        self.n_heads, self.n_kv, self.window, self.lora = n_heads, n_kv, window, tuple(lora)
        self.loras = [LoraAdapter(seg, alpha / lora[2 * i].shape[0], dropout=dropout, site=2 * index + i)
                      for i, seg in enumerate((0, 2))]

    @kernels._on_its_device
    def forward(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                cu_seqlens: torch.Tensor | None = None, max_len: int = 0,
                seed: torch.Tensor | None = None, dtype=None) -> torch.Tensor:
        """The residual stream after the layer, of x [tokens, hidden] (fp32, or the GEMM dtype `dtype`).
        `cos`, `sin`: fp32 [tokens, head_dim], of every token's position; `seed`: as kernels.dropout
        takes it (None: no dropout, as in evaluation)."""
        dtype = dtype or (x.dtype if x.dtype in kernels.GEMM_DTYPES else torch.float16)
        x, h = AddNorm.apply(x, None, self.norm_in, self.eps, dtype)
        loras = self.loras if seed is not None else \
            [LoraAdapter(ad.seg, ad.scale) for ad in self.loras]
        bias = None if self.bias is None else self.bias.to(dtype)
        qkv = project(h, ProjectionSpec(self.qkv, loras, seed), bias, self.lora)
        a = rope_attention(qkv, cos, sin, self.n_heads, self.n_kv, cu_seqlens, window=self.window,
                           max_len=max_len)
        a = project(a.flatten(1), ProjectionSpec([self.o]))
        x, h = AddNorm.apply(x, a, self.norm_post, self.eps, dtype)
        m = RecomputedMLP.apply(h, *self.gate, *self.up, *self.down)
        return x + m.to(x.dtype)
