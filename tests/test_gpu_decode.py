"""A decoder layer served over the paged cache against the same layer in 64 bits on whole
sequences: prompts, chunks, single tokens, a shared prefix, and a decoding step in a graph."""

import math

import pytest
import torch

from tests.gpu_util import banner, oracle_w16

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PAGE = 4, 2, 64, 16


def _layer(cuda, **kw):
    from solution.decode import DecoderLayer
    from solution.stack import Qwen2Shape

    return DecoderLayer.synthetic(Qwen2Shape(hidden=HEADS * DIM, inter=512, kv=KV * DIM), cuda,
                                  seed=3, std=0.05, **kw)


def _whole(layer, x, window=0, sinks=0):
    """The layer on one whole sequence x [n, hidden] in float64, weights as dequantized to fp16."""
    w = {n: oracle_w16(*p).double() for n, p in
         zip(("q", "k", "v", "o", "gate", "up", "down"),
             (*layer.qkv, layer.o, layer.gate, layer.up, layer.down))}
    x, n = x.double(), x.shape[0]

    def norm(t):
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6)

    def rotate(t):
        ang = torch.arange(n).double()[:, None] * 1e4 ** (-torch.arange(0, DIM, 2).double() / DIM)
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        lo, hi = t[..., :DIM // 2], t[..., DIM // 2:]
        return torch.cat((lo * c - hi * s, hi * c + lo * s), -1)

    h = norm(x)
    q = rotate((h @ w["q"].t()).view(n, HEADS, DIM))
    k = rotate((h @ w["k"].t()).view(n, KV, DIM)).repeat_interleave(HEADS // KV, 1)
    v = (h @ w["v"].t()).view(n, KV, DIM).repeat_interleave(HEADS // KV, 1)
    s = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) / math.sqrt(DIM)
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    seen = j <= i
    if window:
        seen &= (j > i - window) | (j < sinks)
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    a = torch.matmul(p, v.transpose(0, 1).contiguous()).transpose(0, 1).reshape(n, -1)
    x = x + a @ w["o"].t()
    h = norm(x)
    return x + (torch.nn.functional.silu(h @ w["gate"].t()) * (h @ w["up"].t())) @ w["down"].t()


def _close(got, want):
    # fp16 throughout: some ten roundings of half a step (2^-11) on values of a few units, summed
    # over products of 256 and 512 terms whose errors are independent: 2^-6 holds them all
    off = (got.double().cpu() - want).abs().max()
    assert off <= 2.0 ** -6 * want.abs().max(), float(off)


class _Run:
    """A cache for `lens` positions a sequence, and the layer stepped over it."""

    def __init__(self, cuda, layer, lens, shared=0):
        from solution import kernels

        self.k, self.layer = kernels, layer
        g = torch.Generator().manual_seed(1)
        need = [-(-n // PAGE) for n in lens]
        common = shared // PAGE
        order = torch.randperm(common + sum(n - common for n in need), generator=g).int()
        table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
        at = common
        for b, n in enumerate(need):
            table[b, :common] = order[:common]
            table[b, common:n] = order[at:at + n - common]
            at += n - common
        pages = torch.zeros((order.numel(), PAGE, KV, DIM), dtype=torch.float16, device=cuda)
        self.lens = torch.zeros(len(lens), dtype=torch.int32, device=cuda)
        self.cache = kernels.PagedKV(pages, torch.zeros_like(pages), table.to(cuda), self.lens)
        self.cos, self.sin = kernels.rope_table(max(lens), DIM, 1e4, cuda)
        self.cuda = cuda

    def step(self, parts, **kw):
        """parts: the new tokens of every sequence (host tensors); their outputs."""
        n = [p.shape[0] for p in parts]
        self.lens += torch.tensor(n, dtype=torch.int32, device=self.cuda)
        cu = torch.tensor([0, *torch.tensor(n).cumsum(0).tolist()], dtype=torch.int32)
        out = self.layer.step(torch.cat(parts).half().to(self.cuda), self.cache, self.cos, self.sin,
                              cu_q=cu.to(self.cuda), **kw)
        return out.split(n)


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_prompt_chunk_and_tokens(cuda, window, sinks):
    """Two sequences taken in as a prompt, a chunk and single tokens: every output is the whole
    sequence's at that position."""
    banner("decoder layer", window, sinks)
    layer = _layer(cuda, window=window, sinks=sinks)
    g = torch.Generator().manual_seed(2)
    xs = [torch.randn(n, HEADS * DIM, generator=g).half() for n in (83, 47)]
    want = [_whole(layer, x, window, sinks) for x in xs]
    run, at = _Run(cuda, layer, [83, 47]), [0, 0]
    for take in ((40, 9), (30, 0), (1, 1), (1, 1), (3, 20)):
        outs = run.step([x[a:a + n] for x, a, n in zip(xs, at, take)])
        for b, (o, n) in enumerate(zip(outs, take)):
            if n:
                _close(o, want[b][at[b]:at[b] + n])
            at[b] += n


def test_shared_prefix_layer(cuda):
    """Three sequences behind 37 common positions (two whole pages and a copied tail): the prefix
    taken in by each, single tokens with the common keys read once."""
    banner("decoder layer, shared prefix")
    layer = _layer(cuda)
    g = torch.Generator().manual_seed(4)
    head = torch.randn(37, HEADS * DIM, generator=g).half()
    xs = [torch.cat((head, torch.randn(n, HEADS * DIM, generator=g).half())) for n in (12, 3, 30)]
    run = _Run(cuda, layer, [x.shape[0] for x in xs], shared=37)
    run.step([x[:-2] for x in xs])
    for i in (2, 1):
        outs = run.step([x[x.shape[0] - i:x.shape[0] - i + 1] for x in xs], shared=37, max_q=1)
        for x, o in zip(xs, outs):
            _close(o, _whole(layer, x)[x.shape[0] - i:x.shape[0] - i + 1])


def test_decoding_step_in_a_graph(cuda):
    """A decoding step captured once: each replay at grown lengths is the eager step, bit for
    bit."""
    from solution import kernels

    banner("decoder layer in a graph")
    layer, lens = _layer(cuda), [60, 33]
    run = _Run(cuda, layer, [n + 8 for n in lens])
    g = torch.Generator().manual_seed(5)
    run.step([torch.randn(n, HEADS * DIM, generator=g) for n in lens])
    x = torch.zeros(2, HEADS * DIM, dtype=torch.float16, device=cuda)
    run.lens += 1

    def step():
        return layer.step(x, run.cache, run.cos, run.sin)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        x.copy_(torch.randn(2, HEADS * DIM, generator=g).half())
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())
        run.lens += 1
