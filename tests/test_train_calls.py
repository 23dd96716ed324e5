"""How the training operators' calls find their tensors' device, what they refuse and what they hand on,
and the generator's published outputs (no GPU needed)."""

import contextlib

import pytest
import torch

from tests import train_ref as ref


class Tensor:
    def __init__(self, index, is_cuda=True):
        self.index, self.is_cuda = index, is_cuda

    def get_device(self):
        return self.index


@pytest.fixture()
def two_devices(monkeypatch):
    """Two GPUs as the calls see them; [the current one]."""
    from solution import kernels

    at = [0]

    @contextlib.contextmanager
    def device(index):
        old, at[0] = at[0], index
        try:
            yield
        finally:
            at[0] = old

    monkeypatch.setattr(kernels, "_devices", lambda: 2)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: at[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    return at


def test_keywords_in_any_order(two_devices):
    """The first parameter's tensor decides, wherever the call names it."""
    from solution import kernels

    seen = kernels._on_its_device(lambda x, p=0.5, other=None: two_devices[0])
    assert seen(p=0.1, x=Tensor(1)) == 1 and seen(other=None, x=Tensor(1)) == 1
    assert seen(other=Tensor(0), x=Tensor(1)) == 1 and seen(p=[], x=[Tensor(1)]) == 1
    assert seen(p=0.1, x=Tensor(1, is_cuda=False)) == 0 and two_devices == [0]
    with pytest.raises(TypeError):
        seen(p=0.1)


def test_refusals_by_keyword_are_the_calls_own(two_devices):
    """What a call refuses it refuses with two devices as with one."""
    from solution import kernels

    x, seed = torch.zeros(3, 8).half(), torch.zeros(2, dtype=torch.int64)
    q = torch.zeros(4, 4, 64).half()
    with pytest.raises(ValueError, match="cuda"):
        kernels.dropout(p=0.5, seed=seed, sites=[0], x=x)
    with pytest.raises(ValueError, match="cuda"):
        kernels.attention_fwd(cu_seqlens=None, k=q, v=q, q=q)
    with pytest.raises(TypeError):
        kernels.attention_fwd(k=q, v=q)


@pytest.mark.parametrize("devices", [1, 2])
def test_no_gradients_are_refused(monkeypatch, devices):
    from solution import kernels

    monkeypatch.setattr(kernels, "_devices", lambda: devices)
    seed = torch.zeros(2, dtype=torch.int64)
    for grads, sites in (([], []), ([], [0])):
        with pytest.raises(ValueError, match="gradient"):
            kernels.dropout_bwd(grads, 0.5, seed, sites)


def test_the_mlp_hands_on_rows(monkeypatch):
    """An expanded gradient (a sum's: one value, strides of 0) and every second column of a wider tensor
    reach the products as rows of consecutive values, in memory of their own."""
    from solution import kernels, mlp

    class Stop(Exception):
        pass

    def product(t, *args, **kw):
        assert t.stride(1) == 1 and t.stride(0) == t.shape[1]
        assert t.untyped_storage().nbytes() == 2 * t.numel()
        raise Stop

    class State:
        shape = (256, 128)

    class Ctx:
        saved_tensors = (torch.zeros(100, 128).half(),) * 4
        qs, shape = (State,) * 3, (100, 128)

    for name in ("linear_fwd", "linear_swiglu_fwd", "linear_dx"):
        monkeypatch.setattr(kernels, name, product)
    w = torch.zeros(8, dtype=torch.uint8)
    for rows in (20, 100):
        wide = torch.zeros(rows, 256).half()[:, ::2]
        with pytest.raises(Stop):
            mlp.RecomputedMLP.forward(Ctx(), wide, w, State, w, State, w, State)
        for grad in (torch.ones((), dtype=torch.half).expand(rows, 128), wide):
            with pytest.raises(Stop):
                mlp.RecomputedMLP.backward(Ctx(), grad)


@pytest.mark.parametrize("counter,key,words", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_the_generators_published_outputs(counter, key, words):
    """Philox4x32-10's known answers, against which the tests' own definition stands."""
    got = ref.philox(key[0] | key[1] << 32, counter[2], counter[3], [counter[0] | counter[1] << 32])
    assert got[0].tolist() == [w >> s & 0xffff for w in words for s in (0, 16)]


def test_a_layers_calls_run_on_its_inputs_device(two_devices, monkeypatch):
    """project and TrainLayer.forward launch on the device of x, also where another is the current one."""
    from solution import layer, train

    class X(Tensor):
        shape = (3, 8)

        def reshape(self, *shape):
            return self

    seen = []

    class Stop(Exception):
        pass

    class Function:
        @staticmethod
        def apply(*args):
            seen.append(two_devices[0])
            raise Stop

    monkeypatch.setattr(layer, "NF4Projection", Function)
    monkeypatch.setattr(train, "AddNorm", Function)
    spec = layer.ProjectionSpec([])
    for call in (lambda: layer.project(X(1), spec), lambda: layer.project(spec=spec, x=X(1))):
        with pytest.raises(Stop):
            call()
    a, b = torch.zeros(2, 8), torch.zeros(8, 2)
    step = train.TrainLayer({n: None for n in ("q", "k", "v", "o", "gate", "up", "down")}, None, None, 1, 1, (a, b, a, b))
    for call in (lambda: step.forward(X(1), None, None, dtype=torch.float16),
                 lambda: step.forward(cos=None, sin=None, x=X(1), dtype=torch.float16)):
        with pytest.raises(Stop):
            call()
    assert seen == [1] * 4 and two_devices == [0]
