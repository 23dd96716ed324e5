"""Dropout from the counter-based generator against its definition in whole numbers: the kernels make
the same fp32 operations, so results are equal, bit for bit."""

import pytest
import torch

from tests import train_ref as ref
from tests.gpu_util import banner

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
SEED = (-0x123456789ABCDEF, 0x7FFFFFFFFFFFFFF3)  # all four words used, the step's high one ignored


def seed_tensor(dev, seed=SEED):
    return torch.tensor(seed, dtype=torch.int64, device=dev)


def place(x, dev, layout):
    """x on the device; "wide": rows further apart, 16-byte aligned; "odd": rows and start at any
    place."""
    rows, cols = x.shape
    if layout == "plain":
        return x.to(dev)
    ld, at = ((cols + 7) // 8 * 8 + 16, 8) if layout == "wide" else (cols + 3, 1)
    big = torch.full((rows, ld + at), 9.0, dtype=x.dtype, device=dev)
    view = big[:, at:at + cols]
    view.copy_(x)
    return view


CASES = [
    # rows, cols, sites, p, dtype, layout
    (1, 1, 1, 0.5, F16, "plain"), (1, 8, 2, 0.3, BF16, "plain"), (3, 7, 3, 0.1, F16, "plain"),
    (5, 9, 1, 0.05, BF16, "odd"), (17, 64, 8, 0.5, F16, "plain"), (4, 1536, 2, 0.05, F16, "plain"),
    (9, 200, 4, 0.9, BF16, "wide"), (6, 333, 5, 0.25, F16, "wide"), (2, 1023, 6, 0.7, BF16, "odd"),
    (33, 72, 7, 0.05, F16, "odd"), (3, 40, 2, 0.0, F16, "plain"), (3, 40, 2, 1.0, BF16, "plain"),
    (3, 41, 2, 1e-6, F16, "plain"),
]


@pytest.mark.parametrize("rows,cols,sites,p,dtype,layout", CASES)
def test_definition(cuda, rows, cols, sites, p, dtype, layout):
    from solution import kernels

    banner("dropout", rows, cols, sites, p, dtype, layout)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(rows, cols, generator=g).to(dtype)
    grads = [torch.randn(rows, cols, generator=g).to(dtype) for _ in range(sites)]
    base = torch.randn(rows, cols, generator=g).to(dtype)
    where = [0xFFFFFFFF - 5 * i for i in range(sites)]
    masks = [ref.kept(*SEED, s, rows, cols, p) for s in where]
    scale = torch.tensor(ref.drop_scale(p))
    seed = seed_tensor(cuda)
    outs = kernels.dropout(place(x, cuda, layout), p, seed, where,
                           outs=[place(torch.zeros_like(x), cuda, layout) for _ in where])
    for got, m in zip(outs, masks):
        assert torch.equal(got.cpu(), torch.where(m, x.float() * scale, 0.0).to(dtype))
    for b in (None, base):
        want = torch.zeros(rows, cols) if b is None else b.float()
        for t, m in zip(grads, masks):
            want = want + torch.where(m, t.float() * scale, 0.0)
        got = kernels.dropout_bwd([place(t, cuda, layout) for t in grads], p, seed, where,
                                  base=None if b is None else place(b, cuda, layout),
                                  out=place(torch.zeros_like(x), cuda, layout))
        assert torch.equal(got.cpu(), want.to(dtype))


def test_a_dropped_infinity_is_zero(cuda):
    from solution import kernels

    x = torch.full((64, 64), float("inf"), dtype=F16, device=cuda)
    (y,) = kernels.dropout(x, 0.5, seed_tensor(cuda), [1])
    m = ref.kept(*SEED, 1, 64, 64, 0.5)
    assert torch.equal(torch.isinf(y.cpu()), m) and not torch.isnan(y).any()
    dx = kernels.dropout_bwd([x], 0.5, seed_tensor(cuda), [1])
    assert torch.equal(dx, y)


def test_in_place(cuda):
    from solution import kernels

    g = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn(100, 264, generator=g, device=cuda).to(BF16)
    base, grad = torch.randn_like(x), torch.randn_like(x)
    seed = seed_tensor(cuda)
    (want,) = kernels.dropout(x, 0.2, seed, [3])
    dx = kernels.dropout_bwd([grad], 0.2, seed, [3], base=base)
    (got,) = kernels.dropout(x, 0.2, seed, [3], outs=[x])
    assert got is x and torch.equal(x, want)
    assert torch.equal(kernels.dropout_bwd([grad], 0.2, seed, [3], base=base, out=base), dx)


def test_share_kept_and_independence(cuda):
    """Of n numbers each kept with probability q the share is q within six deviations; two sites, two
    steps and two seeds agree as often as independent ones do."""
    from solution import kernels

    n, p = 4096 * 1024, 0.3
    x = torch.ones(4096, 1024, dtype=F16, device=cuda)
    seeds = [(1, 0), (1, 1), (2, 0), (1 << 40, 0)]
    masks = []
    for s in seeds:
        masks += [t != 0 for t in kernels.dropout(x, p, seed_tensor(cuda, s), [0, 1])]
    q = 1 - ref.math.floor(65536 * p + 0.5) / 65536
    for m in masks:
        assert abs(float(m.double().mean()) - q) < 6 * (q * (1 - q) / n) ** 0.5
    both = q * q + (1 - q) ** 2
    for i in range(len(masks)):
        for j in range(i):
            same = float((masks[i] == masks[j]).double().mean())
            assert abs(same - both) < 6 * (both * (1 - both) / n) ** 0.5, (i, j)
