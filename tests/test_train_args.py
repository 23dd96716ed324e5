"""Refusals of the training attention's and the dropout's calls, answered on the host before any launch
(no GPU needed)."""

import ctypes

import pytest

OK, ARG, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4
P = 1 << 12  # an aligned address that no refused call reads


@pytest.fixture()
def lib():
    from solution import _lib

    return _lib.load()


def desc(**kw):
    from solution._lib import NF4Attn

    f = dict(q=P, k=P, v=P, q_tok=256, q_head=64, k_tok=128, k_head=64, v_tok=128, v_head=64, cu=P,
             tokens=9, window=0, max_len=0, batch=2, n_heads=4, n_kv=2, head_dim=64, scale=0.125,
             dtype=0)
    f.update(kw)
    return NF4Attn(**f)


def grad(p=P, tok=256, head=64):
    from solution._lib import NF4Grad

    return ctypes.byref(NF4Grad(p, tok, head))


def fwd(lib, a, out=P, stats=P, ws=None, nws=0):
    return lib.nf4_attn_fwd(ctypes.byref(a) if a else None, out, stats, ws, nws, None)


def bwd(lib, a, out=P, stats=P, dout=True, dq=True, dk=True, dv=True, ws=None, nws=0):
    g = [grad() if x is True else x for x in (dout, dq)]
    g += [grad(tok=128) if x is True else x for x in (dk, dv)]
    return lib.nf4_attn_bwd(ctypes.byref(a) if a else None, out, stats, *g, ws, nws, None)


BAD = [
    (dict(q=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG), (dict(tokens=-1), ARG),
    (dict(window=-1), ARG), (dict(max_len=-1), ARG), (dict(batch=-1), ARG), (dict(n_heads=0), ARG),
    (dict(n_kv=0), ARG), (dict(n_heads=5), ARG), (dict(dtype=2), ARG), (dict(dtype=-1), ARG),
    (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG), (dict(scale=-3e38), ARG),
    (dict(cu=None), ARG), (dict(cu=None, batch=0), ARG), (dict(q_tok=-256), ARG),
    (dict(k_head=-64), ARG),
    (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED),
    (dict(q=P + 8), UNSUPPORTED), (dict(k=P + 2), UNSUPPORTED), (dict(v=P + 4), UNSUPPORTED),
    (dict(cu=P + 2), UNSUPPORTED), (dict(q_tok=260), UNSUPPORTED), (dict(v_head=68), UNSUPPORTED),
    (dict(k_tok=(1 << 23) + 8), UNSUPPORTED), (dict(tokens=(1 << 23) + 1), UNSUPPORTED),
    (dict(n_heads=1026), UNSUPPORTED), (dict(batch=(1 << 20) + 1), UNSUPPORTED),
    (dict(tokens=1 << 23, n_heads=256), UNSUPPORTED),
]


@pytest.mark.parametrize("kw,status", BAD)
def test_attention_refusals(lib, kw, status):
    assert fwd(lib, desc(**kw)) == status
    assert bwd(lib, desc(**kw)) == status


def test_attention_pointers_and_gradients(lib):
    a = desc()
    assert fwd(lib, None) == ARG and bwd(lib, None) == ARG
    assert fwd(lib, a, out=None) == ARG and fwd(lib, a, stats=None) == ARG
    assert bwd(lib, a, out=None) == ARG and bwd(lib, a, stats=None) == ARG
    assert fwd(lib, a, out=P + 2) == UNSUPPORTED and fwd(lib, a, stats=P + 4) == UNSUPPORTED
    for name in ("dout", "dq", "dk", "dv"):
        assert bwd(lib, a, **{name: None}) == ARG
        assert bwd(lib, a, **{name: grad(p=None)}) == ARG
        assert bwd(lib, a, **{name: grad(p=P + 8)}) == UNSUPPORTED
        assert bwd(lib, a, **{name: grad(tok=260)}) == UNSUPPORTED
    for name in ("dq", "dk", "dv"):  # rows that overlap (a broadcast tensor)
        assert bwd(lib, a, **{name: grad(tok=0)}) == ARG
        assert bwd(lib, a, **{name: grad(head=0)}) == ARG
        assert bwd(lib, a, **{name: grad(tok=64, head=64)}) == ARG
    assert fwd(lib, desc(tokens=0, q=None, cu=None, batch=0), out=None, stats=None) == OK
    assert bwd(lib, desc(tokens=0, q=None), out=None, dout=None) == OK


def drop(lib, x=P, ld=16, outs=(P,), lds=None, rows=3, cols=16, p=0.5, seed=P, sites=(0,), n=None,
         dtype=0):
    k = len(outs)
    return lib.nf4_dropout(x, ld, (ctypes.c_void_p * k)(*outs), (ctypes.c_int64 * k)(*(lds or [16] * k)),
                           rows, cols, p, seed, (ctypes.c_uint32 * len(sites))(*sites),
                           len(sites) if n is None else n, dtype, None)


def drop_bwd(lib, dx=P, ld=16, grads=(P,), lds=None, rows=3, cols=16, p=0.5, seed=P, sites=(0,),
             n=None, dtype=0, base=None, ldb=16):
    k = len(grads)
    return lib.nf4_dropout_bwd((ctypes.c_void_p * k)(*grads), (ctypes.c_int64 * k)(*(lds or [16] * k)),
                               base, ldb, dx, ld, rows, cols, p, seed,
                               (ctypes.c_uint32 * len(sites))(*sites), len(sites) if n is None else n,
                               dtype, None)


@pytest.mark.parametrize("call", [drop, drop_bwd])
def test_dropout_refusals(lib, call):
    assert call(lib, rows=-1) == ARG and call(lib, cols=-1) == ARG
    assert call(lib, n=0) == ARG and call(lib, n=-3) == ARG
    assert call(lib, p=-1e-9) == ARG and call(lib, p=1.0000001) == ARG
    assert call(lib, p=float("nan")) == ARG and call(lib, dtype=2) == ARG
    assert call(lib, seed=None) == ARG and call(lib, seed=P + 4) == ARG
    assert call(lib, ld=8) == ARG and call(lib, lds=[15]) == ARG
    assert call(lib, n=9) == UNSUPPORTED
    assert call(lib, rows=1 << 31, ld=16) == UNSUPPORTED
    assert call(lib, rows=1 << 30, cols=24, ld=24, lds=[24]) == UNSUPPORTED
    assert call(lib, rows=1, cols=(1 << 31) - 1) == UNSUPPORTED
    assert call(lib, rows=0, seed=None) == OK and call(lib, cols=0, seed=None) == OK


def test_dropout_pointers(lib):
    assert drop(lib, x=None) == ARG and drop(lib, outs=(None,)) == ARG
    assert drop(lib, x=P + 1) == ARG and drop(lib, outs=(P, P + 1), sites=(0, 1)) == ARG
    assert drop_bwd(lib, dx=None) == ARG and drop_bwd(lib, grads=(None,)) == ARG
    assert drop_bwd(lib, base=P + 1) == ARG and drop_bwd(lib, base=P, ldb=8) == ARG


def test_python_refusals():
    import torch

    from solution import kernels

    q, k = torch.zeros(4, 4, 64).half(), torch.zeros(4, 2, 64).half()
    with pytest.raises(ValueError, match="cuda"):
        kernels.attention_fwd(q, k, k)
    with pytest.raises(ValueError):
        kernels.attention_fwd(q, k[:3], k[:3])
    with pytest.raises(ValueError):
        kernels.attention_fwd(q, k.bfloat16(), k)
    with pytest.raises(ValueError):
        kernels.attention_fwd(q.transpose(1, 2), k.transpose(1, 2), k.transpose(1, 2))
    x, seed = torch.zeros(3, 8).half(), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="cuda"):
        kernels.dropout(x, 0.5, seed, [0])
    with pytest.raises(ValueError):
        kernels.dropout(x, 0.5, seed, [0, 1], outs=[x])
    with pytest.raises(ValueError):
        kernels.dropout(x[0], 0.5, seed, [0])
    with pytest.raises(TypeError):
        kernels.dropout(x.float(), 0.5, seed, [0])
    with pytest.raises(ValueError):
        kernels.dropout_bwd([x, x], 0.5, seed, [0])


def test_rope_refusals(lib):
    def rope(x=P, ld=128, cos=P, sin=P, y=P, ldy=128, tokens=3, heads=2, dim=64, inverse=0, dtype=0):
        return lib.nf4_rope(x, ld, cos, sin, y, ldy, tokens, heads, dim, inverse, dtype, None)

    assert rope(x=None) == ARG and rope(y=None) == ARG and rope(cos=None) == ARG and rope(sin=None) == ARG
    assert rope(tokens=-1) == ARG and rope(heads=0) == ARG and rope(dtype=2) == ARG and rope(dim=7) == ARG
    assert rope(ld=120) == ARG and rope(ldy=120) == ARG
    assert rope(dim=4, heads=2) == UNSUPPORTED and rope(dim=520, ld=2080, ldy=2080) == UNSUPPORTED
    assert rope(x=P + 4) == UNSUPPORTED and rope(y=P + 2) == UNSUPPORTED and rope(cos=P + 8) == UNSUPPORTED
    assert rope(ld=130) == UNSUPPORTED and rope(ldy=130) == UNSUPPORTED
    assert rope(tokens=0, x=None) == OK


def test_workspaces(lib):
    a = desc(tokens=4096, batch=1)
    for call, need in ((fwd, lib.nf4_attn_fwd_workspace(ctypes.byref(a))),
                       (bwd, lib.nf4_attn_bwd_workspace(ctypes.byref(a)))):
        assert need > 0
        assert call(lib, a) == WORKSPACE
        assert call(lib, a, ws=P, nws=need - 1) == WORKSPACE
        assert call(lib, a, ws=P + 8, nws=need) == UNSUPPORTED
    for bad in (desc(tokens=-1), desc(head_dim=96), desc(tokens=0)):
        assert lib.nf4_attn_fwd_workspace(ctypes.byref(bad)) == 0
        assert lib.nf4_attn_bwd_workspace(ctypes.byref(bad)) == 0
    assert lib.nf4_attn_fwd_workspace(None) == 0 and lib.nf4_attn_bwd_workspace(None) == 0


@pytest.mark.parametrize("kw", [
    dict(tokens=1 << 23, n_heads=128, n_kv=128, head_dim=128),  # the largest calls
    dict(tokens=1 << 23, n_heads=128, n_kv=1, head_dim=64),
    dict(tokens=1 << 20, n_heads=1024, n_kv=1024, head_dim=64, batch=1 << 20),
    dict(tokens=1 << 20, n_heads=1024, n_kv=1, head_dim=128, window=1),
    dict(tokens=1, n_heads=1024, n_kv=1, head_dim=128), dict(tokens=8192, n_heads=28, n_kv=4, head_dim=128),
])
def test_workspace_of_the_largest_calls(lib, kw):
    """Whole numbers of 64 bits on the way, and a workspace that a call of that size can have: the rows'
    numbers (16 bytes a row and head) and at most 300 MB of parts."""
    for dtype in (0, 1):
        for max_len in (0, 100):
            a = desc(dtype=dtype, max_len=max_len, **kw)
            rows = (kw["tokens"] + 127) // 128 * 128 * kw["n_heads"]
            assert 16 * rows <= lib.nf4_attn_bwd_workspace(ctypes.byref(a)) <= 18 * rows + kw["tokens"] + (300 << 20)
            assert lib.nf4_attn_fwd_workspace(ctypes.byref(a)) <= 300 << 20


def test_structs_as_the_header_has_them():
    from solution._lib import NF4Attn, NF4Grad

    assert ctypes.sizeof(NF4Attn) == 128 and NF4Attn.scale.offset == 120
    assert ctypes.sizeof(NF4Grad) == 24


def test_calls_run_on_their_tensors_device(monkeypatch):
    import contextlib

    import torch

    from solution import kernels

    class Tensor:
        is_cuda = True

        def __init__(self, index):
            self.index = index

        def get_device(self):
            return self.index

    at = [0]

    @contextlib.contextmanager
    def device(index):
        old, at[0] = at[0], index
        yield
        at[0] = old

    monkeypatch.setattr(kernels, "_devices", lambda: 2)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: at[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    seen = kernels._on_its_device(lambda x, y=None: at[0])
    assert seen(Tensor(1)) == 1 and seen(Tensor(0)) == 0 and seen([Tensor(1)]) == 1
    assert seen(x=Tensor(1), y=3) == 1 and at == [0]
