"""The paged-cache operators where numbers are at the ends of their ranges: infinities beside
missing pages, scores of any size, weights far below a row's largest, scales of nothing, values
at the type's end; and launches of unusual size."""

import math

import pytest
import torch

from tests import paged_ref as ref
from tests.gpu_util import banner
from tests.test_gpu_paged import _check, _run

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
EPS = ref.EPS


def _one(cuda, k, v, q, page=16, prefix=0, batch=1):
    """A Setup of `batch` sequences over the same keys k, values v [positions, dim] of one
    key/value head (float64), queries q [tokens, heads, dim] the last tokens of each; the first
    `prefix` positions' whole pages are shared."""
    s = ref.Setup(cuda, q.dtype, q.shape[1], 1, q.shape[2], page, [k.shape[0]] * batch,
                  [q.shape[0] // batch] * batch, shared=prefix)
    j = torch.arange(k.shape[0])
    for b in range(batch):
        at = s.table[b].long()[j // page].to(cuda)
        s.k[at, (j % page).to(cuda), 0] = k.to(s.k)
        s.v[at, (j % page).to(cuda), 0] = v.to(s.v)
    s.q = q
    return s


@pytest.mark.parametrize("new,page,shared", [(3, 16, 0), (40, 16, 0), (3, 8, 0), (40, 32, 0),
                                             (40, 8, 0), (3, 16, 96), (40, 16, 96)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_not_finite_beside_a_missing_page(cuda, new, page, shared, bad):
    """A table entry that names no page next to the page of an infinity or NaN, all of them before
    the new tokens: every row sees the value, in its channel and its key/value head, and nothing
    else changes."""
    from solution import kernels

    banner("not finite beside a missing page", new, page, shared, bad)
    lens = [200, 210]
    s = ref.Setup(cuda, F16, 4, 2, 64, page, lens, [new] * 2, seed=30, shared=shared)
    if shared:
        s.table[:, 32 // page] = -1
    else:
        s.table[0, 32 // page] = s.table[1, 32 // page] = -1
    want = ref.attention(s, shared=shared)
    j = 32 + page + 1 if page < 32 else 17  # in the slab of 32 keys, or tile of 64, of the missing page
    for b in range(2):
        s.v[int(s.table[b, j // page]), j % page, 1, 7] = bad
    o, l = _run(kernels, s, cuda, shared=shared)
    hit = torch.zeros(o.shape, dtype=torch.bool)
    hit[:, 2:, 7] = True
    got = o.cpu()[hit]
    assert got.isnan().all() if math.isnan(bad) else (got == bad).all()
    o = torch.where(hit.to(cuda), torch.zeros_like(o), o)
    want[0][hit] = 0
    _check((o, l), want, F16)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,prefix", [(1, 0), (40, 0), (40, 192)])
def test_largest_weight_is_exact(cuda, dtype, new, prefix):
    """One key ahead of the rest by 1 to 5, behind others that a running maximum met first, and the
    only one whose value is not 0.  Its weight is 2^0 over an unrounded sum, so what is off is the
    output's rounding, and 1e-4 for fp32's scores, exponentials and sums."""
    from solution import kernels

    banner("largest weight", dtype, new, prefix)
    g = torch.Generator().manual_seed(36)
    # (rows enough for 256 workgroups: the keys are not cut, one workgroup meets them in turn)
    n, dim, heads, at, batch = 260, 64, 128, 150, 8
    k = torch.randn(n, dim, generator=g) * 0.01
    k[:, 0] = 0.0
    k[at, 0] = 1.0
    v = torch.zeros(n, dim)
    v[at] = 1 + torch.rand(dim, generator=g)
    q = torch.randn(batch * new, heads, dim, generator=g)
    q[..., 0] = 1 + 4 * torch.rand(batch * new, heads, generator=g)
    q = q.to(dtype)
    s = _one(cuda, k, v, q, prefix=prefix, batch=batch)
    o, _ = _run(kernels, s, cuda, shared=prefix, scale=1.0)
    pos = n - new + torch.arange(new).repeat(batch)
    sc = (q.double() @ k.to(dtype).double().t().contiguous()).masked_fill(
        (torch.arange(n) > pos[:, None])[:, None], -math.inf)
    want = torch.softmax(sc, -1)[..., at:at + 1] * v[at].to(dtype).double()
    off = (o.double().cpu() - want).abs()
    assert (off <= want * (EPS[dtype] + 1e-4)).all(), f"relative {(off / want).max():.3e}"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,heads,prefix", [(1, 2, 0), (40, 4, 0), (1, 2, 16000), (2, 40, 16000)])
@pytest.mark.parametrize("lead", [12.0, 18.0])
def test_weights_far_below_the_largest(cuda, dtype, new, heads, prefix, lead):
    """A first key whose score leads all others by `lead`, its value 0: what is left of the output
    is the many small weights.  Each counts with its rounding to the 16-bit type (half a step,
    relative: exp(-18) = 2^-26 of the largest is above the type's smallest normal value where the
    largest is 2^15), the output with its own, the scores (about 20 units, fp32 sums of 64 terms)
    with 1e-5 of exp's relative error, the fp32 sums over 20000 weights with 1e-4."""
    from solution import kernels

    banner("small weights", dtype, new, heads, prefix, lead)
    g = torch.Generator().manual_seed(31)
    n, dim = 20000, 64
    k = torch.randn(n, dim, generator=g) * 0.01
    k[:, 0] = 0.0
    k[0] = 0.0
    k[0, 0] = lead / 2
    v = 1 + torch.rand(n, dim, generator=g)
    v[0] = 0.0
    batch = 2 if prefix else 1
    q = torch.randn(batch * new, heads, dim, generator=g)
    q[..., 0] = 2.0
    q = q.to(dtype)
    s = _one(cuda, k, v, q, prefix=prefix, batch=batch)
    ks, vs = k.to(dtype).double(), v.to(dtype).double()
    o, l = _run(kernels, s, cuda, shared=prefix, scale=1.0)
    pos = n - new + torch.arange(new).repeat(batch)
    sc = (q.double() @ ks.t().contiguous()).masked_fill(
        (torch.arange(n) > pos[:, None])[:, None], -math.inf)
    lse = torch.logsumexp(sc, -1)
    want = torch.exp(sc - lse[..., None]) @ vs
    bound = want * (2 * EPS[dtype] + 1.2e-4)
    off = (o.double().cpu() - want).abs()
    assert (off <= bound).all(), f"relative {(off / want).max():.3e}"
    torch.testing.assert_close(l.cpu().double(), lse, rtol=1e-5, atol=2e-5)


@pytest.mark.parametrize("dtype,size", [(F16, 1e4), (BF16, 1e6), (BF16, 1e12)])
@pytest.mark.parametrize("new,prefix", [(1, 0), (40, 0), (1, 160)])
def test_scores_of_any_size(cuda, dtype, size, new, prefix):
    """Queries and keys of 1e4 (fp16) and more: scores of 1e8 to 1e25, where one step of fp32 is
    many units.  A key that leads by more than their rounding (1e-4 of the largest) has all the
    weight, so the output is its value, bit for bit; every output is finite."""
    from solution import kernels

    banner("scores of any size", dtype, size, new, prefix)
    g = torch.Generator().manual_seed(32)
    n, dim, batch = 300, 128, 2 if prefix else 1
    k = (torch.randn(n, dim, generator=g) * size).clamp(-6e4 if dtype == F16 else -1e30,
                                                        6e4 if dtype == F16 else 1e30)
    v = torch.randn(n, dim, generator=g)
    q = (torch.randn(batch * new, 4, dim, generator=g) * size).clamp(-6e4 if dtype == F16 else -1e30,
                                                                     6e4 if dtype == F16 else 1e30)
    q[:, 3] = q[:, 3] / size / size  # a head of ordinary scores beside them
    q = q.to(dtype)
    s = _one(cuda, k, v, q, prefix=prefix, batch=batch)
    o, l = _run(kernels, s, cuda, shared=prefix)
    pos = n - new + torch.arange(new).repeat(batch)
    sc = (q.double() @ k.to(dtype).double().t().contiguous()).masked_fill(
        (torch.arange(n) > pos[:, None])[:, None], -math.inf) * dim ** -0.5
    two = sc.topk(2, -1)
    clear = two.values[..., 0] - two.values[..., 1] > 1e-4 * two.values[..., 0].abs() + 50
    assert clear[:, :3].double().mean() > 0.9
    assert torch.isfinite(o.float()).all()
    winner = v.to(dtype)[two.indices[..., 0]]
    assert torch.equal(o.cpu()[clear], winner[clear])
    torch.testing.assert_close(l.cpu().double(), torch.logsumexp(sc, -1), rtol=2e-5, atol=2e-4)


@pytest.mark.parametrize("new", [1, 40])
def test_scale_of_nothing(cuda, new):
    """A scale of 0 weighs every key alike, whatever its score (1e30 here)."""
    from solution import kernels

    banner("scale 0", new)
    g = torch.Generator().manual_seed(33)
    k = torch.randn(90, 64, generator=g) * 1e15
    v = torch.randn(90, 64, generator=g)
    q = (torch.randn(new, 4, 64, generator=g) * 1e15).to(BF16)
    s = _one(cuda, k, v, q)
    o, l = _run(kernels, s, cuda, scale=0.0)
    vs = v.to(BF16).double()
    want = torch.stack([vs[:91 - new + i].mean(0) for i in range(new)])[:, None].expand(-1, 4, -1)
    # weights of 1: no rounding but the output's, and fp32 sums
    assert ((o.double().cpu() - want).abs() <= want.abs() * EPS[BF16] + 1e-5).all()
    count = torch.arange(91 - new, 91).double()
    torch.testing.assert_close(l.cpu().double(), count.log()[:, None].expand(-1, 4).contiguous(),
                               rtol=1e-5, atol=1e-4)


@pytest.mark.parametrize("n,new,prefix", [(32, 1, 0), (60, 40, 0), (33, 1, 32), (100, 40, 32)])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_at_the_end_of_the_type(cuda, n, new, prefix, dim):
    """Values of +-65504: an output is their mean, so it is finite, and off by the rounding of the
    weights and its own, half a step each.  All weights but a first one are just above the middle
    between 0.5 and the next number, so that a tile's are rounded up together."""
    from solution import kernels

    banner("values of 65504", n, new, prefix, dim)
    batch, heads = 4, 8
    k = torch.zeros(n, dim)
    k[1:, 0] = -1.0
    v = torch.full((n, dim), 65504.0)
    v[:, 1::2] = -65504.0
    q = torch.zeros(batch * new, heads, dim, dtype=F16)
    q[..., 0] = 1.0
    s = _one(cuda, k, v, q, prefix=prefix, batch=batch)
    o, _ = _run(kernels, s, cuda, shared=prefix, scale=-math.log(0.5 + 1.02 * 2.0 ** -12))
    o = o.double().cpu()
    assert torch.isfinite(o).all()
    assert (o[..., 0::2] >= 65504 * (1 - 2 * EPS[F16])).all()
    assert (o[..., 1::2] <= -65504 * (1 - 2 * EPS[F16])).all()


@pytest.mark.parametrize("heads,kv,new", [(42, 6, 5), (33, 3, 4), (24, 12, 20)])
def test_three_row_blocks_of_many_heads(cuda, heads, kv, new):
    """33 to 48 rows a sequence, key/value heads whose number does not divide 256."""
    from solution import kernels

    banner("three row blocks of many heads", heads, kv, new)
    s = ref.Setup(cuda, BF16, heads, kv, 64, 16, [700, 90, new, 300], [new] * 4, seed=37,
                  extra_width=1000)
    for window, sinks in ((0, 0), (9000, 3)):
        _check(_run(kernels, s, cuda, window, sinks), ref.attention(s, window, sinks), BF16)


def test_three_row_blocks_in_a_window(cuda):
    """40 rows a sequence whose windows of 8300 keys end before some sequences begin."""
    from solution import kernels

    banner("three row blocks in a window")
    s = ref.Setup(cuda, F16, 40, 8, 64, 16, [9100, 300, 40, 8, 8500, 100], [8] * 6, seed=38)
    _check(_run(kernels, s, cuda, 8300, 3), ref.attention(s, 8300, 3), F16)


def test_more_rows_than_a_grid_dimension(cuda):
    """Tokens times heads past 2^20 with pieces to join: the rows on both sides of it."""
    from solution import kernels

    banner("rows past 2^20")
    heads, kv, dim, new, shared = 1024, 16, 64, 205, 20
    s = ref.Setup(cuda, F16, heads, kv, dim, 16, [shared + new] * 5, [new] * 5, seed=35,
                  shared=shared)
    assert s.q.shape[0] * heads > 1 << 20
    o, l = _run(kernels, s, cuda, shared=shared)
    k, v = s.k.double().cpu(), s.v.double().cpu()
    for t in (0, 1, 204, 205, 640, 1022, 1023, 1024):
        b, n = t // new, shared + t % new + 1
        j = torch.arange(n)
        at = s.table[b].long()[j // 16]
        ks, vs = (x[at, j % 16].repeat_interleave(heads // kv, 1) for x in (k, v))
        sc = (ks * s.q[t].double()).sum(-1) * dim ** -0.5  # [keys, heads]
        lse = torch.logsumexp(sc, 0)
        want = (torch.exp(sc - lse)[..., None] * vs).sum(0)
        _check((o[t], l[t]), (want, lse, vs.abs().amax((0, 2))), F16)
