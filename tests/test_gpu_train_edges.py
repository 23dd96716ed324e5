"""Calls of the training operators that lie at an edge: a spec that changes between the passes, views at any
address, empty batches, second derivatives, values that are not finite in a split launch."""

import copy
import ctypes
import math

import pytest
import torch

from tests import train_ref as ref
from tests.gpu_util import banner, oracle_w16, random_weight
from tests.test_gpu_attention import check, make, run
from tests.test_gpu_train import tables

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def offset(t):
    """t's values in a contiguous tensor whose start is not 16-byte aligned."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.detach().reshape(-1)
    return flat[1:].view(t.shape)


# ------------------------------------------------------------------ a spec that changes

@pytest.mark.parametrize("change", ["seed", "no seed", "site", "dropout", "scale", "adapters"])
def test_a_spec_changed_before_the_backward_pass(cuda, change):
    """The backward pass is that of its own forward pass, whatever the program does to the spec for the
    next one: a new seed tensor, None, another site, probability, scale or list of adapters."""
    from solution.layer import LoraAdapter, ProjectionSpec, project

    banner("spec", change)
    segs = [random_weight(n, 128, seed=70 + i, dev=cuda) for i, n in enumerate((128, 64))]
    g = torch.Generator().manual_seed(71)
    rnd = lambda *s: torch.randn(*s, generator=g).to(cuda)  # noqa: E731
    x, dy = rnd(33, 128).half(), rnd(33, 192).half()
    params = [rnd(8, 128), rnd(128, 8), rnd(8, 128), rnd(64, 8)]
    spec = ProjectionSpec(segs, [LoraAdapter(0, 2.0, dropout=0.3, site=1), LoraAdapter(1, 2.0, dropout=0.3, site=2)],
                          torch.tensor([9, 4], device=cuda))

    def forward(spec):
        leaves = [t.clone().requires_grad_() for t in (x, *params)]
        return leaves, project(leaves[0], spec, None, leaves[1:])

    def grads(leaves, y):
        y.backward(dy)
        return [t.grad for t in leaves]

    def mutate():
        if change in ("seed", "no seed"):
            spec.seed = torch.tensor([9, 5], device=cuda) if change == "seed" else None
        elif change == "adapters":
            spec.loras[:] = [LoraAdapter(0, 2.0), LoraAdapter(1, 2.0)]
        else:
            setattr(spec.loras[0], change, {"site": 3, "dropout": 0.5, "scale": 1.0}[change])

    want = [grads(*forward(copy.deepcopy(spec)))]
    first = forward(spec)
    mutate()
    if change == "no seed":
        got = [grads(*first)]
    else:  # two micro-batches' forward passes, then both backward passes
        want.append(grads(*forward(copy.deepcopy(spec))))
        second = forward(spec)
        got = [grads(*first), grads(*second)]
        assert not torch.equal(want[0][1], want[1][1])
    for a, b in zip(got, want):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


# -------------------------------------------------------------- views at any address

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
def test_attention_of_an_offset_view(cuda, dtype, which):
    from solution.layer import attention

    q, k, v, dout, cu = make(cuda, dtype, 4, 2, 64, (70, 9), seed=80, layout="plain")
    c = torch.tensor(cu, dtype=torch.int32, device=cuda)
    want = run(q, k, v, dout, cu)
    args = {"q": q, "k": k, "v": v, "dout": dout}
    args[which] = offset(args[which])
    assert args[which].data_ptr() % 16 and args[which].is_contiguous()
    leaves = [args[n].requires_grad_() for n in "qkv"]
    out = attention(*leaves, c)
    out.backward(args["dout"])
    assert torch.equal(out, want["out"])
    assert all(torch.equal(t.grad, want["d" + n]) for n, t in zip("qkv", leaves))


def test_attention_of_rows_far_apart(cuda):
    """More elements between two tokens than the kernels take."""
    from solution.layer import attention, rope_attention

    q, k, v, dout, cu = make(cuda, BF16, 4, 2, 64, (3,), seed=81, layout="plain")
    want = run(q, k, v, dout, cu)
    far = (1 << 23) + 8
    big = torch.zeros(2 * far + 4 * 64, dtype=BF16, device=cuda)

    def place(t):
        x = torch.as_strided(big, t.shape, (far, 64, 1) if t.dim() == 3 else (far, 1))
        x.copy_(t)
        return x

    for i in range(3):
        leaves = [t.clone() for t in (q, k, v)]
        leaves[i] = place(leaves[i])
        for t in leaves:
            t.requires_grad_()
        out = attention(*leaves)
        out.backward(dout)
        assert torch.equal(out, want["out"])
        assert all(torch.equal(t.grad, want["d" + n]) for n, t in zip("qkv", leaves))
    assert torch.equal(attention(q, k, v.requires_grad_()), want["out"])
    v.grad = None
    attention(q, k, v).backward(place(dout))
    assert torch.equal(v.grad, want["dv"])
    cos, sin = tables([0, 1, 2], 64, cuda)
    qkv = torch.cat([t.detach().flatten(1) for t in (q, k[:, :1], v[:, :1])], 1)  # 4 heads over 1
    a, b = qkv.clone().requires_grad_(), torch.as_strided(torch.zeros(2 * far + 384, dtype=BF16, device=cuda), (3, 384), (far, 1))
    b.copy_(qkv)
    b.requires_grad_()
    for t in (a, b):
        rope_attention(t, cos, sin, 4, 1).backward(dout)
    assert torch.equal(a.grad, b.grad)


def test_rope_attention_of_an_offset_view(cuda):
    from solution.layer import rope_attention

    g = torch.Generator().manual_seed(82)
    qkv = torch.randn(50, 8 * 64, generator=g).half().to(cuda)
    dout = torch.randn(50, 4, 64, generator=g).half().to(cuda)
    cos, sin = tables(range(50), 64, cuda)
    a, b = qkv.clone().requires_grad_(), offset(qkv).requires_grad_()
    ya, yb = (rope_attention(t, cos, sin, 4, 2) for t in (a, b))
    ya.backward(dout)
    yb.backward(offset(dout))
    assert torch.equal(ya, yb) and torch.equal(a.grad, b.grad)


@pytest.mark.parametrize("m", [1, 40, 200])
def test_projection_of_offset_views(cuda, m):
    """x, dY and adapters in the GEMM dtype that start anywhere; segments whose columns do."""
    from solution.layer import LoraAdapter, ProjectionSpec, project

    segs = [random_weight(n, 128, seed=83 + i, dev=cuda) for i, n in enumerate((64, 128))]
    g = torch.Generator().manual_seed(84)
    rnd = lambda *s: torch.randn(*s, generator=g).half().to(cuda)  # noqa: E731
    x, dy = rnd(m, 128), rnd(m, 192)
    params = [rnd(8, 128), rnd(64, 8), rnd(8, 128), rnd(128, 8)]
    spec = ProjectionSpec(segs, [LoraAdapter(0, 2.0, dropout=0.3, site=1), LoraAdapter(1, 1.0)],
                          torch.tensor([9, 4], device=cuda))
    got = []
    for place in (torch.clone, offset):
        leaves = [place(t).requires_grad_() for t in (x, *params)]
        y = project(leaves[0], spec, None, leaves[1:])
        y.backward(place(dy))
        got.append([y] + [t.grad for t in leaves])
    assert all(torch.equal(a, b) for a, b in zip(got[0][1:], got[1][1:]))
    # y: an adapter's B that is not 16-byte aligned may be summed in another order, each sum in fp32 and
    # rounded once.  A sum of n terms is off by n half steps of fp32 of what its terms' sizes add up to, and
    # the two results by half a step of fp16 each: |dy| <= 2 (2^-11 |y| + (128 + 8 + 2) 2^-24 size + 2^-25),
    # with t of at most its terms' sizes (1.01: its own rounding), scaled by the share kept.
    size = []
    for (w, qs), ad, a, b in zip(segs, spec.loras, params[::2], params[1::2]):
        t = 1.01 * ref.drop_scale(ad.dropout) * (x.double().abs() @ a.double().abs().t())
        w16 = oracle_w16(w, qs).double().to(cuda)
        size.append(x.double().abs() @ w16.abs().t() + ad.scale * t @ b.double().abs().t())
    bound = 2 * (ref.HALF[F16] * got[0][0].double().abs() + 138 * ref.U32 * torch.cat(size, 1) + ref.TINY[F16])
    assert ((got[0][0].double() - got[1][0].double()).abs() <= bound).all()


@pytest.mark.parametrize("m", [20, 100])
def test_mlp_of_offset_views(cuda, m):
    from solution.mlp import RecomputedMLP

    w = [random_weight(*s, seed=85 + i, dev=cuda) for i, s in enumerate(((256, 128), (256, 128), (128, 256)))]
    g = torch.Generator().manual_seed(86)
    x, dy = (torch.randn(m, 128, generator=g).half().to(cuda) for _ in range(2))
    got = []
    for place in (torch.clone, offset):
        leaf = place(x).requires_grad_()
        y = RecomputedMLP.apply(leaf, *w[0], *w[1], *w[2])
        y.backward(place(dy))
        got.append((y, leaf.grad))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("m", [20, 100])
def test_mlp_of_expanded_and_strided_tensors(cuda, m):
    """The gradient of a sum (one value, expanded), and every second column of a wider tensor."""
    from solution.mlp import RecomputedMLP

    w = [random_weight(*s, seed=87 + i, dev=cuda) for i, s in enumerate(((256, 128), (256, 128), (128, 256)))]
    x = torch.randn(m, 256, generator=torch.Generator().manual_seed(88)).half().to(cuda)[:, ::2]
    got = []
    for dense in (True, False):
        leaf = (x.clone(memory_format=torch.contiguous_format) if dense else x.detach()).requires_grad_()
        y = RecomputedMLP.apply(leaf, *w[0], *w[1], *w[2])
        one = torch.ones((), dtype=F16, device=cuda).expand(m, 128)
        y.backward(one.contiguous() if dense else one)
        got.append((y, leaf.grad))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def small_layer(dev, dropout=0.0):
    from solution.train import TrainLayer

    names = {"q": (128, 128), "k": (64, 128), "v": (64, 128), "o": (128, 128), "gate": (256, 128),
             "up": (256, 128), "down": (128, 256)}
    w = {n: random_weight(*s, seed=90 + i, dev=dev, std=0.06) for i, (n, s) in enumerate(names.items())}
    g = torch.Generator().manual_seed(91)
    lora = [(0.06 * torch.randn(*s, generator=g)).to(dev).requires_grad_()
            for s in ((8, 128), (128, 8), (8, 128), (64, 8))]
    one = torch.ones(128, device=dev)
    return TrainLayer(w, one, one, 2, 1, lora, dropout=dropout, index=3), lora


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
def test_train_layer_of_offset_views(cuda, dtype):
    layer, lora = small_layer(cuda, 0.2)
    g = torch.Generator().manual_seed(92)
    x, dy = (torch.randn(30, 128, generator=g).to(dtype).to(cuda) for _ in range(2))
    cos, sin = tables(range(30), 64, cuda)
    seed = torch.tensor([3, 1], device=cuda)
    got = []
    for place in (torch.clone, offset):
        leaf = place(x).requires_grad_()
        for t in lora:
            t.grad = None
        y = layer.forward(leaf, cos, sin, seed=seed)
        y.backward(place(dy))
        got.append([y, leaf.grad] + [t.grad for t in lora])
    assert all(torch.equal(a, b) for a, b in zip(*got))


# ----------------------------------------------------------------- nothing, and twice

def test_no_tokens(cuda):
    """An empty batch has empty results and gradients."""
    from solution.layer import attention, rope_attention

    for cu in (None, torch.zeros(1, dtype=torch.int32, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda)):
        q, k, v = (torch.empty(0, h, 64, dtype=F16, device=cuda, requires_grad=True) for h in (4, 2, 2))
        out = attention(q, k, v, cu)
        out.backward(torch.empty_like(out))
        assert out.shape == q.grad.shape == (0, 4, 64) and k.grad.shape == v.grad.shape == (0, 2, 64)
        qkv = torch.empty(0, 8 * 64, dtype=F16, device=cuda, requires_grad=True)
        table = torch.empty(0, 64, device=cuda)
        out = rope_attention(qkv, table, table, 4, 2, cu)
        out.backward(torch.empty_like(out))
        assert out.shape == (0, 4, 64) and qkv.grad.shape == (0, 512)


def test_second_derivatives_of_projection_and_mlp_raise(cuda):
    """A penalty on their gradients has no derivative here: it raises rather than being left out."""
    from solution.layer import LoraAdapter, ProjectionSpec, project
    from solution.mlp import RecomputedMLP

    w = [random_weight(*s, seed=95 + i, dev=cuda) for i, s in enumerate(((256, 128), (256, 128), (128, 256)))]
    x = torch.randn(20, 128, device=cuda).half().requires_grad_()
    a, b = torch.randn(8, 128, device=cuda).requires_grad_(), torch.randn(256, 8, device=cuda).requires_grad_()
    seed = torch.tensor([1, 1], device=cuda)
    for ad in (LoraAdapter(0, 1.0, dropout=0.5), LoraAdapter(0, 1.0)):
        y = project(x, ProjectionSpec(w[:1], [ad], seed), None, (a, b))
        for g in torch.autograd.grad(y.float().square().sum(), (x, a, b), create_graph=True):
            with pytest.raises(RuntimeError, match="once_differentiable"):
                g.float().square().sum().backward(retain_graph=True)
    y = RecomputedMLP.apply(x, *w[0], *w[1], *w[2])
    g, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().square().sum().backward()


# -------------------------------------------------------- launches of either kind

def workspaces(q, k, v, max_len=0, window=0):
    """(forward's, backward's) bytes: more of them where the work is in pieces or shares."""
    from solution import _lib, kernels

    c = torch.zeros(2, dtype=torch.int32, device=q.device)
    d = ctypes.byref(kernels._attn_desc(q, k, v, c, None, window, max_len))
    lib = _lib.load()
    return lib.nf4_attn_fwd_workspace(d), lib.nf4_attn_bwd_workspace(d)


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 64), (BF16, 128)])
def test_a_workgroup_a_tile_and_shares(cuda, dtype, dim):
    """`max_len` below the longest sequence: a workgroup takes a tile of any length; as it is: shares."""
    q, k, v, dout, cu = make(cuda, dtype, 16, 16, dim, (1100, 64, 964), seed=100)
    tiles, shares = (workspaces(q, k, v, n)[1] for n in (64, 2000))
    assert shares > tiles + (20 << 20)  # (2 * 16 slots a head of 64 KB and more, at the least)
    want = ref.attention(q, k, v, cu, dout)
    for n in (64, 2000):
        got = run(q, k, v, dout, cu, max_len=n)
        for name in got:
            ref.assert_within(got[name], want[name], (name, n))


def split(dev, dtype, seed):
    """A forward pass whose tiles are in several pieces."""
    q, k, v, dout, cu = make(dev, dtype, 4, 2, 64, (900,), seed=seed, layout="plain")
    assert workspaces(q, k, v)[0] >= 8 * 4 * 3 * 128 * 264  # 8 tiles of 4 heads, 3 pieces at least
    return q, k, v, dout, cu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("at", [3, 500, 800])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_values_that_are_not_finite_in_pieces(cuda, dtype, at, value):
    """A value of v that is not finite is in one channel of the rows that see it, and in nothing else."""
    banner("pieces", dtype, at, value)
    q, k, v, dout, cu = split(cuda, dtype, 101)
    want = ref.attention(q, k, v, cu, dout)
    v[at, 1, 5] = value  # of heads 2 and 3
    got = run(q, k, v, dout, cu)
    touched = torch.zeros(900, 4, 64, dtype=torch.bool)
    touched[at:, 2:, 5] = True
    there = got["out"].cpu()[touched].float()
    assert torch.isnan(there).all() if math.isnan(value) else (there == value).all()
    ref.assert_within(got["out"].cpu()[~touched], tuple(t[~touched] for t in want["out"]), "out")
    ref.assert_within(got["stats"], want["stats"], "stats")
    ref.assert_within(got["dq"][:at], tuple(t[:at] for t in want["dq"]), "dq")
    for name in ("dk", "dv"):
        ref.assert_within(got[name][:, 0], tuple(t[:, 0] for t in want[name]), name)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_keys_of_no_weight_in_pieces(cuda, dtype):
    """The first 300 keys have scores of -inf: rows before 300 are NaN, the others those of a sequence that
    begins there, though their first pieces saw nothing else."""
    q, k, v, dout, cu = split(cuda, dtype, 102)
    q[:, :, 0], k[:, :, 0] = 1.0, 0.0
    want = ref.attention(q[300:], k[300:], v[300:], [0, 600], dout[300:])
    k[:300, :, 0] = -math.inf
    got = run(q, k, v, dout, cu)
    for name in ("out", "dk", "dv"):
        ref.assert_within(got[name][300:], want[name], name)
        assert torch.isnan(got[name][:300]).all()
    ref.assert_within(got["stats"][300:], want["stats"], "stats")
    ref.assert_within(got["dq"][300:, :, 1:], tuple(t[..., 1:] for t in want["dq"]), "dq")
    assert torch.isnan(got["dq"][:300]).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("pieces", [False, True])
@pytest.mark.parametrize("value", [math.inf, math.nan, -math.inf])
def test_statistics_of_scores_that_are_not_finite(cuda, dtype, pieces, value):
    """A row that sees a score of NaN or +inf, or of -inf only, has NaN for its output and both statistics."""
    banner("statistics", dtype, pieces, value)
    if pieces:
        q, k, v, dout, cu = split(cuda, dtype, 103)
    else:
        q, k, v, dout, cu = make(cuda, dtype, 4, 2, 64, (100,), seed=103, layout="plain")
        assert workspaces(q, k, v)[0] == 0
    n = q.shape[0]
    q[:, :, 0], k[:, :, 0] = 1.0, 0.0
    want = ref.attention(q, k, v, cu)
    lo, hi = (0, 30) if value == -math.inf else (n - 30, n)  # the rows that are NaN
    at = range(30) if value == -math.inf else [n - 30]
    for i in at:
        k[i, :, 0] = value
    got = run(q, k, v, dout, cu)
    assert torch.isnan(got["out"][lo:hi]).all() and torch.isnan(got["stats"][lo:hi]).all()
    if value != -math.inf:
        for name in ("out", "stats"):
            ref.assert_within(got[name][:lo], tuple(t[:lo] for t in want[name]), name)
    else:
        assert not torch.isnan(got["out"][hi:]).any() and not torch.isnan(got["stats"][hi:]).any()


def test_the_generators_published_output(cuda):
    """Philox4x32-10 of counter and key 0 is 6627e8d5 e169c58d bc57ac4c 9b00dbd8: an element is kept up to its
    own number, and no further."""
    from solution import kernels

    numbers = [0xe8d5, 0x6627, 0xc58d, 0xe169, 0xac4c, 0xbc57, 0xdbd8, 0x9b00]
    x = torch.ones(1, 8, dtype=F16, device=cuda)
    seed = torch.zeros(2, dtype=torch.int64, device=cuda)
    for n in numbers:
        for cut in (n, n + 1):
            (y,) = kernels.dropout(x, cut / 65536, seed, [0])
            assert [bool(t) for t in y[0]] == [u >= cut for u in numbers]
            dx = kernels.dropout_bwd([x], cut / 65536, seed, [0])
            assert torch.equal(dx, y)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,lens,window,max_len", [
    (64, (300,), 0, 300), (128, (300, 7, 130), 0, 300), (64, (400, 90), 70, 400), (128, (700,), 33, 700),
    (128, (900, 60), 0, 900),
])
def test_values_that_are_not_finite_by_channel(cuda, dtype, dim, lens, window, max_len):
    """NaN and infinities here and there in v: NaN in the channels and rows that see a NaN, an infinity in those
    that see one and no NaN, and everything else as it is without them."""
    banner("channels", dtype, dim, lens, window)
    q, k, v, dout, cu = make(cuda, dtype, 4, 2, dim, lens, pad=5, seed=104, layout="plain")
    want = ref.attention(q, k, v, cu, window=window)
    n, g = sum(lens), torch.Generator().manual_seed(105)
    nan, inf = (torch.zeros(n + 5, 2, dim, dtype=torch.bool) for _ in range(2))
    for at in (2, 100, 129, 255, n - 3):
        nan[at, at % 2, torch.randint(dim, (2,), generator=g)] = True
    for at in (50, 140, n - 20):
        inf[at, :, torch.randint(dim, (1,), generator=g)] = True
    inf &= ~nan
    v[nan.to(cuda)], v[inf.to(cuda)] = math.nan, math.inf
    from solution import kernels

    c = torch.tensor(cu, dtype=torch.int32, device=cuda)
    out, stats = (t.cpu() for t in kernels.attention_fwd(q, k, v, c, window=window, max_len=max_len))
    sees = torch.zeros(n + 5, n + 5, dtype=torch.float64)
    for a, b in zip(cu, cu[1:]):
        sees[a:b, a:b] = (~ref.hidden(b - a, window)).double()
    sees_nan, sees_inf = (((sees @ t.double().flatten(1)) > 0).view(-1, 2, dim).repeat_interleave(2, 1) for t in (nan, inf))
    assert torch.equal(torch.isnan(out), sees_nan)
    assert torch.equal(torch.isinf(out), sees_inf & ~sees_nan)
    rest = ~(sees_nan | sees_inf)
    ref.assert_within(out[rest], tuple(t[rest] for t in want["out"]), "out")
    ref.assert_within(stats, want["stats"], "stats")


def test_an_early_nan_of_v_costs_little(cuda):
    """One pass over v says which rows see it: twice the time of finite values (formed again row by row, all
    rows behind it took 110 times as long)."""
    from solution import kernels

    q, k, v, dout, cu = make(cuda, BF16, 12, 2, 128, (2048,), seed=106, layout="plain")

    def us(v):
        times = []
        for _ in range(6):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            kernels.attention_fwd(q, k, v)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b) * 1e3)
        return sorted(times)[2]

    clean = us(v)
    v[3, 0, 5] = math.nan
    assert us(v) < 20 * clean + 100


# ------------------------------------------------------------- a layer's step, as it is used

def test_a_captured_step_that_adds_to_its_seed(cuda):
    """A layer's forward and backward pass and the step's increment in one graph: every replay has the next
    step's masks, and what the eager calls give with that seed."""
    layer, lora = small_layer(cuda, 0.3)
    g = torch.Generator(device=cuda).manual_seed(110)
    new = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    x, dy = new(50, 128).half().requires_grad_(), new(50, 128).half()
    cos, sin = tables([*range(30), *range(20)], 64, cuda)
    cu = torch.tensor([0, 30, 50], dtype=torch.int32, device=cuda)
    seed = torch.tensor([9, 4], device=cuda)

    def step(seed):
        y = layer.forward(x, cos, sin, cu, seed=seed)
        return [y.detach(), *torch.autograd.grad(y, [x, *lora], dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(seed)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step(seed)
        seed[1] += 1
    masks = set()
    for i in range(4):
        with torch.no_grad():
            x.copy_(new(50, 128).half())
        dy.copy_(new(50, 128).half())
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in kept]
        assert seed.tolist() == [9, 5 + i]
        want = step(torch.tensor([9, 4 + i], device=cuda))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        masks.add(float(got[2].double().sum()))
    assert len(masks) == 4


def test_a_layer_whose_input_needs_no_gradient(cuda):
    """The first layer behind frozen embeddings, and a second backward pass of the same graph: the adapters'
    gradients are the same."""
    layer, lora = small_layer(cuda, 0.2)
    g = torch.Generator().manual_seed(111)
    x, dy = (torch.randn(30, 128, generator=g).half().to(cuda) for _ in range(2))
    cos, sin = tables(range(30), 64, cuda)
    seed = torch.tensor([3, 1], device=cuda)
    got = []
    for leaf in (x.clone().requires_grad_(), x.clone()):
        y = layer.forward(leaf, cos, sin, seed=seed)
        for again in (True, False):
            got.append(torch.autograd.grad(y, lora, dy, retain_graph=again))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


def test_two_adapters_of_one_site(cuda):
    """Adapters that share a site have one mask."""
    from solution.layer import LoraAdapter, ProjectionSpec, project

    w = random_weight(64, 128, seed=112, dev=cuda)
    g = torch.Generator().manual_seed(113)
    x = torch.randn(20, 128, generator=g).half().to(cuda)
    a, b = torch.randn(8, 128, generator=g).to(cuda), torch.randn(64, 8, generator=g).to(cuda)
    seed = torch.tensor([2, 2], device=cuda)

    def forward(*sites):
        loras = [LoraAdapter(i, 1.0, dropout=0.4, site=s) for i, s in enumerate(sites)]
        return project(x, ProjectionSpec([w] * len(sites), loras, seed), None, [a, b] * len(sites))

    y = forward(7, 7)
    assert torch.equal(y[:, :64], y[:, 64:])
    y = forward(7, 8)
    assert not torch.equal(y[:, :64], y[:, 64:])


# --------------------------------------------- what lies beside a sequence costs nothing

def gpu_us(call):
    times = []
    for _ in range(6):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return sorted(times)[2]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_rows_before_the_first_sequence(cuda, dtype, dim, value):
    """Rows of no sequence in the first tile: results are the same bit for bit, and in about the same time
    (each row formed again on its own: 55 times as long)."""
    from solution import kernels

    q, k, v, dout, _ = make(cuda, dtype, 4, 2, dim, (2148,), seed=107, layout="plain")
    c = torch.tensor([101, 2148], dtype=torch.int32, device=cuda)

    def both():
        out, stats = kernels.attention_fwd(q, k, v, c)
        return [out, stats, *kernels.attention_bwd(dout, q, k, v, out, stats, c)]

    want, clean = both(), gpu_us(both)
    for t in (q, k, v, dout):
        t[:101] = value
    assert all(torch.equal(a, b) for a, b in zip(both(), want))
    assert gpu_us(both) < 5 * clean + 100


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_nan_of_v_beside_and_before(cuda, dtype, dim):
    """A NaN of v at the end of a short sequence leaves the long one behind it as it is, and the keys and rows
    before it have their gradients from the tiles: about the time of finite values (67 times as long before)."""
    from solution import kernels

    q, k, v, dout, cu = make(cuda, dtype, 4, 2, dim, (101, 2000), seed=108, layout="plain")
    c = torch.tensor(cu, dtype=torch.int32, device=cuda)
    out, stats = kernels.attention_fwd(q, k, v, c)
    want = ref.attention(q, k, v, cu, dout)
    clean = gpu_us(lambda: kernels.attention_bwd(dout, q, k, v, out, stats, c))
    v[98, :, 5] = math.nan
    out2, stats2 = kernels.attention_fwd(q, k, v, c)
    assert torch.equal(out2[128:], out[128:]) and torch.equal(stats2, stats)
    got = kernels.attention_bwd(dout, q, k, v, out2, stats2, c)
    assert gpu_us(lambda: kernels.attention_bwd(dout, q, k, v, out2, stats2, c)) < 5 * clean + 100
    # (not bit for bit: the outputs of rows 101 to 127, whose wave has rows that see it, are formed in fp32,
    # so their D differs by a rounding)
    for name, t in zip(("dq", "dk", "dv"), got):
        ref.assert_within(t[101:], tuple(x[101:] for x in want[name]), name)  # another sequence's
        assert torch.isnan(t[98:101]).all(), name
    ref.assert_within(got[0][:98], tuple(x[:98] for x in want["dq"]), "dq")  # rows that do not see it
    assert torch.isnan(got[1][:98]).all() and torch.isnan(got[2][:98]).all()  # keys that the NaN rows see


@pytest.mark.parametrize("widths", [(100,), (100, 64), (64, 100, 128)])
@pytest.mark.parametrize("m", [1, 40])
def test_projection_of_any_width(cuda, widths, m):
    """Rows of Y and dY that are no multiple of 8 apart: the gradients of x and of the adapters, against the
    products in 64 bits.  A sum of n terms is off by n half steps of fp32 of their sizes' sum, the operands that
    are rounded on the way (t, da) and the result by half a step of fp16 each, and so is d(xd)."""
    from solution import kernels
    from solution.layer import LoraAdapter, ProjectionSpec, project

    segs = [random_weight(n, 128, seed=120 + i, dev=cuda) for i, n in enumerate(widths)]
    g = torch.Generator().manual_seed(121)
    rnd = lambda *s: torch.randn(*s, generator=g).half().to(cuda)  # noqa: E731
    n, p = sum(widths), 0.25
    x, dy, a, b = rnd(m, 128).requires_grad_(), rnd(m, n), rnd(8, 128).requires_grad_(), rnd(widths[0], 8).requires_grad_()
    seed = torch.tensor([4, 4], device=cuda)
    project(x, ProjectionSpec(segs, [LoraAdapter(0, 2.0, dropout=p, site=3)], seed), None, (a, b)).backward(dy)
    w = torch.cat([oracle_w16(*s) for s in segs]).double()
    d0, d, a64, b64 = dy[:, :widths[0]].double().cpu(), dy.double().cpu(), a.detach().double().cpu(), b.detach().double().cpu()
    xd = kernels.dropout(x.detach(), p, seed, [3])[0].double().cpu()
    keep = ref.kept(4, 4, 3, m, 128, p).double() * ref.drop_scale(p)
    half, terms = ref.HALF[F16], (n + 128 + 16) * ref.U32

    def within(got, value, size, roundings):
        ref.assert_within(got, (value, 1.01 * (roundings * half + terms) * size + ref.TINY[F16]), "gradient")

    t, da = xd @ a64.t(), 2.0 * d0 @ b64
    t_size, da_size = xd.abs() @ a64.abs().t(), 2.0 * d0.abs() @ b64.abs()
    within(x.grad, d @ w + (da @ a64) * keep, d.abs() @ w.abs() + (da_size @ a64.abs()) * keep, 4)
    within(a.grad, da.t() @ xd, da_size.t() @ xd.abs(), 2)
    within(b.grad, 2.0 * d0.t() @ t, 2.0 * d0.abs().t() @ t_size, 2)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,value", [(64, math.inf), (128, -math.inf)])
def test_an_infinite_key_of_no_weight(cuda, dtype, dim, value):
    """The first key has a score of -inf with every later row, by an infinity in one channel: those rows are a
    sequence that begins behind it, but for 0 times that infinity in their dq (formed again one by one, 40 times
    as long for 2048 tokens)."""
    from solution import kernels

    q, k, v, dout, cu = make(cuda, dtype, 4, 2, dim, (1400,), seed=122, layout="plain")
    q[:, :2, 5] = -1.0 if value > 0 else 1.0  # the heads of key head 0
    k[:, 0, 5] = 0.25
    clean = run(q, k, v, dout, cu)
    want = ref.attention(q[1:], k[1:], v[1:], [0, 1399], dout[1:])
    whole = ref.attention(q, k, v, cu, dout)
    time = gpu_us(lambda: kernels.attention_bwd(dout, q, k, v, clean["out"], clean["stats"]))
    k[0, 0, 5] = value
    got = run(q, k, v, dout, cu)
    assert gpu_us(lambda: kernels.attention_bwd(dout, q, k, v, got["out"], got["stats"])) < 10 * time + 100
    other = [c for c in range(dim) if c != 5]
    for name, n in (("out", 2), ("stats", 2), ("dq", 2), ("dk", 1), ("dv", 1)):
        assert torch.isnan(got[name][0, :n]).all(), name
        x, (val, bound) = got[name].cpu(), want[name]
        if name == "dq":
            assert torch.isnan(x[1:, :2, 5]).all()
            ref.assert_within(x[1:, :2, other], (val[:, :2, other], bound[:, :2, other]), name)
        else:
            ref.assert_within(x[1:, :n], (val[:, :n], bound[:, :n]), name)
        ref.assert_within(x[:, n:], tuple(t[:, n:] for t in whole[name]), name)
