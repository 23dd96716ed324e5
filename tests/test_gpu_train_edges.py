"""Calls of the training operators that lie at an edge: a spec that changes between the passes, views at any
address, empty batches, second derivatives, values that are not finite in a split launch."""

import copy

import pytest
import torch

from tests.gpu_util import banner, random_weight

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


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
