"""The training operators together: rotation, LoRA dropout in the projection, attention through autograd,
captured and on other streams, and a whole decoder layer against its fp32 composition."""

import pytest
import torch

from tests import train_ref as ref
from tests.gpu_util import banner, oracle_w16, random_weight

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def tables(positions, dim, dev):
    """cos, sin [tokens, dim] fp32 of the given positions, both halves alike."""
    inv = 1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    ang = torch.tensor(positions, dtype=torch.float64)[:, None] * inv
    ang = torch.cat((ang, ang), -1)
    return ang.cos().float().to(dev), ang.sin().float().to(dev)


def rotate(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos[:, None] + torch.cat((-x[..., half:], x[..., :half]), -1) * sin[:, None]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,heads,dim,pad", [(1, 1, 8, 0), (5, 3, 64, 8), (33, 36, 128, 256), (7, 2, 512, 4)])
def test_rope(cuda, dtype, tokens, heads, dim, pad):
    """Two products and a sum in fp32 (three roundings), one rounding to the type."""
    from solution import kernels

    g = torch.Generator().manual_seed(0)
    big = torch.randn(tokens, heads * dim + pad, generator=g).to(dtype).to(cuda)
    cos = torch.randn(tokens, dim, generator=g).to(cuda)
    sin = torch.randn(tokens, dim, generator=g).to(cuda)
    half = dim // 2
    x = big[:, :heads * dim].double().view(tokens, heads, dim)
    lo, hi = x[..., :half], x[..., half:]
    c, s = cos.double()[:, None], sin.double()[:, None]
    want = torch.cat((lo * c[..., :half] - hi * s[..., :half], hi * c[..., half:] + lo * s[..., half:]), -1)
    back = torch.cat((lo * c[..., :half] + hi * s[..., half:], hi * c[..., half:] - lo * s[..., :half]), -1)
    size = (lo.abs() + hi.abs()).repeat(1, 1, 2) * (c.abs() + s.abs()).amax()
    for inverse, w in ((False, want), (True, back)):
        got = kernels.rope(big, cos, sin, heads, dim, inverse=inverse)
        bound = ref.HALF[dtype] * w.abs() + 3 * ref.U32 * size + ref.TINY[dtype]
        ref.assert_within(got.view(tokens, heads, dim), (w.cpu(), 1.01 * bound.cpu()), "rope")
    rest = big[:, heads * dim:].clone()
    kernels.rope(big, cos, sin, heads, dim, inverse=True, out=big)
    assert torch.equal(big[:, :heads * dim], got) and torch.equal(big[:, heads * dim:], rest)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_projection_dropout_is_the_dropped_input(cuda, dtype):
    """An adapter's `dropout` is the adapter with its own, dropped input: y, dA and dB bit for bit, and dX
    the sum that dropout_bwd forms."""
    from solution import kernels
    from solution.layer import LoraAdapter, ProjectionSpec, project

    banner("projection dropout", dtype)
    m, k, r = 77, 256, 8
    segs = [random_weight(n, k, seed=20 + i, dev=cuda) for i, n in enumerate((256, 64, 64))]
    g = torch.Generator().manual_seed(21)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(cuda)  # noqa: E731
    x = rnd(m, k).to(dtype)
    params = [rnd(r, k, std=0.1), rnd(256, r, std=0.1), rnd(r, k, std=0.1), rnd(64, r, std=0.1)]
    dy = rnd(m, 384).to(dtype)
    seed = torch.tensor([77, 3], device=cuda)
    sites = (5, 9)

    def run(loras, extra, xin):
        ps = [t.clone().requires_grad_() for t in params]
        flat = ps if extra is None else [ps[0], ps[1], extra[0], ps[2], ps[3], extra[1]]
        y = project(xin, ProjectionSpec(segs, loras, seed), None, flat)
        y.backward(dy)
        return y, [t.grad for t in ps]

    x1 = x.clone().requires_grad_()
    y1, g1 = run([LoraAdapter(0, 2.0, dropout=0.2, site=5), LoraAdapter(2, 2.0, dropout=0.2, site=9)],
                 None, x1)
    xd = [t.requires_grad_() for t in kernels.dropout(x, 0.2, seed, sites)]
    x2 = x.clone().requires_grad_()
    y2, g2 = run([LoraAdapter(0, 2.0, own_input=True), LoraAdapter(2, 2.0, own_input=True)], xd, x2)
    assert torch.equal(y1, y2)
    assert all(torch.equal(a, b) for a, b in zip(g1, g2))
    want = kernels.dropout_bwd([t.grad for t in xd], 0.2, seed, sites, base=x2.grad)
    assert torch.equal(x1.grad, want)
    # two probabilities: the masks of each
    x3 = x.clone().requires_grad_()
    y3, g3 = run([LoraAdapter(0, 2.0, dropout=0.2, site=5), LoraAdapter(2, 2.0, dropout=0.5, site=9)],
                 None, x3)
    assert torch.equal(y3[:, :256], y1[:, :256]) and not torch.equal(y3[:, 320:], y1[:, 320:])


def test_a_seed_written_before_the_backward_pass_is_an_error(cuda):
    from solution.layer import LoraAdapter, ProjectionSpec, project

    w = random_weight(64, 64, seed=1, dev=cuda)
    x = torch.randn(4, 64, device=cuda).half().requires_grad_()
    a, b = torch.randn(4, 64, device=cuda).requires_grad_(), torch.randn(64, 4, device=cuda).requires_grad_()
    seed = torch.tensor([1, 1], device=cuda)
    y = project(x, ProjectionSpec([w], [LoraAdapter(0, 1.0, dropout=0.5)], seed), None, (a, b))
    seed[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(ValueError, match="seed"):
        project(x, ProjectionSpec([w], [LoraAdapter(0, 1.0, dropout=0.5)]), None, (a, b))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_autograd(cuda, dtype):
    """attention() and rope_attention() against the 64-bit definition, with an expanded gradient."""
    from solution.layer import attention, rope_attention

    heads, kv, dim, lens = 4, 2, 64, (70, 33)
    g = torch.Generator().manual_seed(31)
    qkv = torch.randn(110, (heads + 2 * kv) * dim, generator=g).to(dtype).to(cuda)
    cu = torch.tensor([0, 70, 103], dtype=torch.int32, device=cuda)
    q, k, v = (t.contiguous().requires_grad_() for t in
               qkv.view(110, heads + 2 * kv, dim).split((heads, kv, kv), 1))
    out = attention(q, k, v, cu, max_len=70)
    dout = torch.randn(dim, generator=g).to(dtype).to(cuda)
    (out * dout).sum().backward()
    want = ref.attention(q.detach(), k.detach(), v.detach(), [0, 70, 103], dout.expand(110, heads, dim))
    for name, got in (("out", out), ("dq", q.grad), ("dk", k.grad), ("dv", v.grad)):
        ref.assert_within(got, want[name], name)
    # the rotation before it and behind its gradients, as calls of their own
    from solution import kernels

    cos, sin = tables(list(range(70)) + list(range(33)) + [0] * 7, dim, cuda)
    leaf = qkv.clone().requires_grad_()
    out = rope_attention(leaf, cos, sin, heads, kv, cu)
    out.backward(torch.ones_like(out))
    qk = kernels.rope(qkv, cos, sin, heads + kv, dim).view(110, heads + kv, dim)
    v = qkv.view(110, -1, dim)[:, heads + kv:]
    o2, stats = kernels.attention_fwd(qk[:, :heads], qk[:, heads:], v, cu)
    assert torch.equal(out, o2)
    dq, dk, dv = kernels.attention_bwd(torch.ones_like(o2), qk[:, :heads], qk[:, heads:], v, o2, stats, cu)
    dqk = kernels.rope(torch.cat((dq, dk), 1).view(110, -1), cos, sin, heads + kv, dim, inverse=True)
    assert torch.equal(leaf.grad, torch.cat((dqk, dv.reshape(110, -1)), 1))


def test_captured_and_replayed(cuda):
    """One graph of dropout, attention and both gradients, replayed with new inputs, offsets and steps
    between eager calls, against the eager results."""
    from solution import kernels

    heads, kv, dim, tokens = 4, 2, 128, 700
    g = torch.Generator(device=cuda).manual_seed(41)
    new = lambda *s: torch.randn(*s, generator=g, device=cuda).to(BF16)  # noqa: E731
    x, q, k, v = new(tokens, 512), new(tokens, heads, dim), new(tokens, kv, dim), new(tokens, kv, dim)
    dout = new(tokens, heads, dim)
    cu = torch.tensor([0, 100, 700, 700], dtype=torch.int32, device=cuda)
    seed = torch.tensor([5, 0], device=cuda)

    def step():
        (xd,) = kernels.dropout(x, 0.1, seed, [2])
        out, stats = kernels.attention_fwd(q, k, v, cu)
        grads = kernels.attention_bwd(dout, q, k, v, out, stats, cu)
        return [xd, out, stats, *grads, kernels.dropout_bwd([xd], 0.1, seed, [2], base=x)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for i, offsets in enumerate(([0, 100, 700, 700], [0, 650, 651, 690], [0, 1, 2, 700], [3, 300, 300, 699])):
        for t in (x, q, k, v, dout):
            t.copy_(new(*t.shape))
        cu.copy_(torch.tensor(offsets, dtype=torch.int32))
        seed[1] = i
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in kept]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_two_streams_at_once(cuda):
    """Calls on two streams, each with its own workspace."""
    from solution import kernels

    g = torch.Generator(device=cuda).manual_seed(51)
    sets = []
    for n in (900, 400):
        q, k, v, do = (torch.randn(n, h, 64, generator=g, device=cuda).half() for h in (6, 2, 2, 6))
        sets.append((q, k, v, do))

    def both(q, k, v, do):
        out, stats = kernels.attention_fwd(q, k, v)
        return [out, *kernels.attention_bwd(do, q, k, v, out, stats)]

    want = [both(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(3):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i] = both(*s)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def _plain_layer(x, w, norm_in, norm_post, bias, lora, scale, masks, share, cos, sin, lens, heads, kv, eps,
                 window):
    """The layer in fp32 on the CPU."""
    def norm(t, n):
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps) * n

    def lin(t, name):
        return t @ w[name].t()

    tokens, dim = x.shape[0], w["q"].shape[0] // heads
    h = norm(x, norm_in)
    q, k, v = lin(h, "q"), lin(h, "k"), lin(h, "v")
    aq, bq, av, bv = lora
    hq, hv = (h * m * share for m in masks)
    q = q + scale * (hq @ aq.t()) @ bq.t()
    v = v + scale * (hv @ av.t()) @ bv.t()
    n_q, n_k = q.shape[1], k.shape[1]
    q, k, v = q + bias[:n_q], k + bias[n_q:n_q + n_k], v + bias[n_q + n_k:]
    q = rotate(q.view(tokens, heads, dim), cos, sin)
    k = rotate(k.view(tokens, kv, dim), cos, sin).repeat_interleave(heads // kv, 1)
    v = v.view(tokens, kv, dim).repeat_interleave(heads // kv, 1)
    outs, t0 = [], 0
    for n in lens:
        sl = slice(t0, t0 + n)
        s = torch.stack([q[sl, i] @ k[sl, i].t() for i in range(heads)]) * dim ** -0.5
        s = s.masked_fill(ref.hidden(n, window), float("-inf"))
        p = torch.softmax(s, -1)
        outs.append(torch.stack([p[i] @ v[sl, i] for i in range(heads)], 1))
        t0 += n
    x = x + lin(torch.cat(outs).reshape(tokens, -1), "o")
    h = norm(x, norm_post)
    return x + lin(torch.nn.functional.silu(lin(h, "gate")) * lin(h, "up"), "down")


@pytest.mark.parametrize("dtype,res", [(F16, torch.float32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("window", [0, 20])
def test_train_layer(cuda, dtype, res, window):
    """Output and every gradient of a layer.  About 12 roundings to the type lie between input and
    output, and about 24 to a gradient, each half a step: of the largest value at most, were all alike."""
    from solution.train import TrainLayer

    banner("train layer", dtype, res, window)
    heads, kv, dim, hidden, inter, rank, p = 4, 2, 64, 256, 512, 8, 0.2
    lens = (37, 90, 1, 20)
    tokens = sum(lens)
    names = {"q": (256, hidden), "k": (128, hidden), "v": (128, hidden), "o": (hidden, 256),
             "gate": (inter, hidden), "up": (inter, hidden), "down": (hidden, inter)}
    w = {n: random_weight(*s, seed=60 + i, dev=cuda, std=0.06) for i, (n, s) in enumerate(names.items())}
    w32 = {n: oracle_w16(*t, "bf16" if dtype == BF16 else "f16").float() for n, t in w.items()}
    g = torch.Generator().manual_seed(61)
    rnd = lambda *s, std=1.0: torch.randn(*s, generator=g) * std  # noqa: E731
    x, dy = rnd(tokens, hidden).to(res), rnd(tokens, hidden).to(res)
    lora = [rnd(rank, hidden, std=0.06), rnd(256, rank, std=0.06), rnd(rank, hidden, std=0.06), rnd(128, rank, std=0.06)]
    norm_in, norm_post = 1 + rnd(hidden, std=0.1), 1 + rnd(hidden, std=0.1)
    bias = rnd(512, std=0.2).to(dtype)
    cos, sin = tables([i for n in lens for i in range(n)], dim, cuda)
    seed, index = (0x1234567890ABC, 17), 5

    params = [t.to(cuda).requires_grad_() for t in lora]
    layer = TrainLayer(w, norm_in.to(cuda), norm_post.to(cuda), heads, kv, params, alpha=16.0, dropout=p,
                       index=index, bias=bias.to(cuda), window=window)
    xg = x.to(cuda).requires_grad_()
    cu = torch.tensor([0, 37, 127, 128, 148], dtype=torch.int32, device=cuda)
    y = layer.forward(xg, cos, sin, cu, max_len=90, seed=torch.tensor(seed, device=cuda), dtype=dtype)
    y.backward(dy.to(cuda))

    xr = x.float().requires_grad_()
    lr = [t.to(dtype).float().requires_grad_() for t in lora]
    masks = [ref.kept(*seed, 2 * index + i, tokens, hidden, p).float() for i in (0, 1)]
    yr = _plain_layer(xr, w32, norm_in, norm_post, bias.float(), lr, 2.0, masks, ref.drop_scale(p),
                      cos.cpu(), sin.cpu(), lens, heads, kv, 1e-6, window)
    yr.backward(dy.float())
    half = ref.HALF[dtype]
    assert y.dtype == res
    for name, got, want, n in [("y", y, yr, 12), ("dx", xg.grad, xr.grad, 24)] + \
            [(f"lora{i}", a.grad, b.grad, 24) for i, (a, b) in enumerate(zip(params, lr))]:
        off = (got.detach().float().cpu() - want.detach()).abs().max() / want.detach().abs().max()
        assert off <= n * half, (name, float(off), n * half)
    # evaluation: no dropout, no need of a seed
    with torch.no_grad():
        y0 = layer.forward(xg, cos, sin, cu, dtype=dtype)
        ones = [torch.ones(tokens, hidden)] * 2
        yr = _plain_layer(xr, w32, norm_in, norm_post, bias.float(), lr, 2.0, ones, 1.0, cos.cpu(),
                          sin.cpu(), lens, heads, kv, 1e-6, window)
    assert (y0.float().cpu() - yr).abs().max() <= 12 * half * yr.abs().max()
