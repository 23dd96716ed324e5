"""The served decoder layer in its other forms (bfloat16, heads of 128, a q|k|v bias, a norm's
epsilon) against the same layer in 64 bits on whole sequences."""

import math

import pytest
import torch

from tests.gpu_util import banner, oracle_w16

pytestmark = pytest.mark.gpu

PAGE, INTER, BASE = 16, 512, 1e4


def _whole(layer, x, heads, kv, dim, bias, eps):
    """The layer on one whole sequence x [n, hidden] in float64, weights as dequantized to x's
    dtype."""
    name = "bf16" if x.dtype == torch.bfloat16 else "f16"
    w = {n: oracle_w16(*p, name).double() for n, p in
         zip(("q", "k", "v", "o", "gate", "up", "down"),
             (*layer.qkv, layer.o, layer.gate, layer.up, layer.down))}
    x, n = x.double(), x.shape[0]
    b = torch.zeros((heads + 2 * kv) * dim) if bias is None else bias.cpu()
    bq, bk, bv = b.double().split((heads * dim, kv * dim, kv * dim))

    def norm(t):
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps)

    def rotate(t):
        ang = torch.arange(n).double()[:, None] * BASE ** (-torch.arange(0, dim, 2).double() / dim)
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        lo, hi = t[..., :dim // 2], t[..., dim // 2:]
        return torch.cat((lo * c - hi * s, hi * c + lo * s), -1)

    h = norm(x)
    q = rotate((h @ w["q"].t() + bq).view(n, heads, dim))
    k = rotate((h @ w["k"].t() + bk).view(n, kv, dim)).repeat_interleave(heads // kv, 1)
    v = (h @ w["v"].t() + bv).view(n, kv, dim).repeat_interleave(heads // kv, 1)
    s = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) / math.sqrt(dim)
    s = s.masked_fill(torch.arange(n) > torch.arange(n)[:, None], -math.inf)
    a = torch.matmul(torch.softmax(s, -1), v.transpose(0, 1).contiguous())
    x = x + a.transpose(0, 1).reshape(n, -1) @ w["o"].t()
    h = norm(x)
    return x + (torch.nn.functional.silu(h @ w["gate"].t()) * (h @ w["up"].t())) @ w["down"].t()


def _close(got, want, dtype):
    """Some ten roundings of half a step one after the other (norm, q|k|v, rotation, weights of
    the attention, its output, o, sum, norm, gate|up, product, down, sum), each on values of a few
    units: 32 half steps of the largest value hold every element, 8 half steps the root mean
    square (a rounding's own is 0.6 of half a step, and the products of random weights neither add
    up nor amplify them)."""
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    off = got.double().cpu() - want
    assert off.abs().max() <= 32 * half * want.abs().max(), float(off.abs().max())
    assert off.pow(2).mean().sqrt() <= 8 * half * want.pow(2).mean().sqrt()


FORMS = [  # dtype, heads, kv, dim, bias, eps
    (torch.float16, 4, 2, 64, True, None),
    (torch.bfloat16, 4, 2, 64, False, None),
    (torch.bfloat16, 2, 1, 128, True, None),
    (torch.float16, 4, 1, 128, False, None),
]


def _run_form(cuda, dtype, heads, kv, dim, bias, eps, size=1.0):
    from solution import kernels
    from solution.decode import DecoderLayer
    from solution.stack import Qwen2Shape

    g = torch.Generator().manual_seed(6)
    kw = {}
    if bias is True:
        bias = torch.randn((heads + 2 * kv) * dim, generator=g).to(dtype).to(cuda)
    if bias is not False:
        kw["bias"] = bias
    if eps is not None:
        kw["eps"] = eps
    layer = DecoderLayer.synthetic(Qwen2Shape(hidden=heads * dim, inter=INTER, kv=kv * dim), cuda,
                                   seed=3, std=0.05, **kw)
    lens = [53, 21]
    xs = [(torch.randn(n, heads * dim, generator=g) * size).to(dtype) for n in lens]
    want = [_whole(layer, x, heads, kv, dim, kw.get("bias"), 1e-6 if eps is None else eps)
            for x in xs]
    width = -(-max(lens) // PAGE)
    table = torch.randperm(2 * width, generator=g).int().view(2, width).to(cuda)
    pages = torch.zeros((2 * width, PAGE, kv, dim), dtype=dtype, device=cuda)
    held = torch.zeros(2, dtype=torch.int32, device=cuda)
    cache = kernels.PagedKV(pages, torch.zeros_like(pages), table, held)
    cos, sin = kernels.rope_table(max(lens), dim, BASE, cuda)
    at = [0, 0]
    for take in ((40, 9), (1, 1), (12, 11)):  # prompts, a token each, chunks
        held += torch.tensor(take, dtype=torch.int32, device=cuda)
        cu = torch.tensor([0, take[0], sum(take)], dtype=torch.int32, device=cuda)
        x = torch.cat([x[a:a + n] for x, a, n in zip(xs, at, take)]).to(cuda)
        outs = layer.step(x, cache, cos, sin, cu_q=cu).split(take)
        for b in range(2):
            _close(outs[b], want[b][at[b]:at[b] + take[b]], dtype)
            at[b] += take[b]


@pytest.mark.parametrize("dtype,heads,kv,dim,bias,eps", FORMS)
def test_layer_forms(cuda, dtype, heads, kv, dim, bias, eps):
    """Two sequences taken in as prompts, a token each and chunks: every output is the whole
    sequence's at that position."""
    banner("decoder layer form", dtype, heads, kv, dim, bias, eps)
    _run_form(cuda, dtype, heads, kv, dim, bias, eps)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_layer_epsilon(cuda, dtype):
    """A norm's epsilon that counts: residual streams of 0.01 (mean square 1e-4) and 1e-3."""
    banner("decoder layer epsilon", dtype)
    _run_form(cuda, dtype, 4, 2, 64, False, 1e-3, size=0.01)


@pytest.mark.parametrize("dtype,given", [(torch.float16, torch.float32),
                                         (torch.bfloat16, torch.float16)])
def test_layer_bias_of_another_type(cuda, dtype, given):
    """A bias in another type than the layer's, and one that is a view of every second number."""
    banner("decoder layer bias", dtype, given)
    g = torch.Generator().manual_seed(7)
    bias = torch.randn(2 * 8 * 64, generator=g).to(dtype).to(given).to(cuda)[::2]
    _run_form(cuda, dtype, 4, 2, 64, bias, None)


def test_layer_bias_of_another_length(cuda):
    """Refused: the projection would read past it."""
    banner("decoder layer bias, short")
    with pytest.raises(ValueError):
        _run_form(cuda, torch.float16, 4, 2, 64, torch.zeros(8 * 64 - 64, device=cuda), None)
