"""Refusals of the paged-cache calls, answered on the host before any launch (no GPU needed)."""

import ctypes

import pytest
import torch


@pytest.fixture()
def lib():
    from solution import _lib

    return _lib.load()


def _kv(**kw):
    from solution._lib import NF4PagedKV

    f = dict(k=1 << 12, v=1 << 12, page_stride=2048, slot_stride=128, head_stride=64,
             table=1 << 12, ld_table=4, lens=1 << 12, pages=3, page_size=16, width=4, batch=2,
             n_kv=2, head_dim=64)
    f.update(kw)
    return NF4PagedKV(**f)


def _attn(lib, kv, q=1 << 12, out=1 << 12, tokens=2, heads=4, ld=256, ldh=64, cu=None, window=0,
          sinks=0, shared=0, dtype=0, lse=None, ws=None, nws=0):
    return lib.nf4_paged_attn(ctypes.byref(kv) if kv else None, q, ld, ldh, cu, out, lse, tokens,
                              heads, 0.125, window, sinks, shared, 0, 0, dtype, ws, nws, None)


def _append(lib, kv, qkv=1 << 12, ld=512, cos=1 << 12, sin=1 << 12, rows=9, cu=None, q=1 << 12,
            tokens=2, heads=4, dtype=0):
    return lib.nf4_paged_append(ctypes.byref(kv) if kv else None, qkv, ld, cos, sin, rows, cu, q,
                                tokens, heads, dtype, None)


ARG, UNSUPPORTED = 1, 2

BAD_KV = [
    (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED),
    (dict(page_size=24), UNSUPPORTED), (dict(page_size=0), ARG), (dict(n_kv=3), ARG),
    (dict(n_kv=0), ARG), (dict(batch=-1), ARG), (dict(width=-1), ARG), (dict(pages=-1), ARG),
    (dict(width=9), ARG),  # wider than its rows are apart
    (dict(k=None), ARG), (dict(v=None), ARG), (dict(table=None), ARG), (dict(lens=None), ARG),
    (dict(k=(1 << 12) + 8), UNSUPPORTED), (dict(page_stride=2044), UNSUPPORTED),
    (dict(head_stride=12), UNSUPPORTED), (dict(slot_stride=-8), ARG),
    (dict(width=1 << 27, ld_table=1 << 27), UNSUPPORTED), (dict(batch=0), ARG),
]


@pytest.mark.parametrize("kw,status", BAD_KV)
def test_cache_refusals(lib, kw, status):
    assert _attn(lib, _kv(**kw)) == status
    assert _append(lib, _kv(**kw)) == status


def test_attention_refusals(lib):
    ok = _kv()
    assert _attn(lib, None) == ARG
    assert _attn(lib, ok, q=None) == ARG and _attn(lib, ok, out=None) == ARG
    assert _attn(lib, ok, tokens=-1) == ARG and _attn(lib, ok, tokens=3) == ARG
    assert _attn(lib, ok, heads=3) == ARG and _attn(lib, ok, heads=0) == ARG
    assert _attn(lib, ok, dtype=2) == ARG and _attn(lib, ok, window=-1) == ARG
    assert _attn(lib, ok, sinks=-1) == ARG and _attn(lib, ok, shared=-1) == ARG
    assert _attn(lib, ok, q=(1 << 12) + 2) == UNSUPPORTED
    assert _attn(lib, ok, ld=252) == UNSUPPORTED and _attn(lib, ok, ldh=-8) == ARG
    assert _attn(lib, ok, cu=(1 << 12) + 2) == UNSUPPORTED
    assert _attn(lib, ok, tokens=1 << 28, cu=1 << 12) == UNSUPPORTED
    assert _attn(lib, ok, tokens=0) == 0


def test_append_refusals(lib):
    ok = _kv()
    assert _append(lib, None) == ARG and _append(lib, ok, qkv=None) == ARG
    assert _append(lib, ok, q=None) == ARG and _append(lib, ok, cos=None) == ARG
    assert _append(lib, ok, ld=504) == ARG and _append(lib, ok, ld=516) == UNSUPPORTED
    assert _append(lib, ok, rows=-1) == ARG and _append(lib, ok, sin=(1 << 12) + 4) == UNSUPPORTED
    assert _append(lib, ok, dtype=3) == ARG and _append(lib, ok, tokens=3) == ARG
    assert _append(lib, ok, tokens=0) == 0


def test_struct_layout():
    from solution._lib import NF4PagedKV

    assert ctypes.sizeof(NF4PagedKV) == 88
    assert NF4PagedKV.lens.offset == 56 and NF4PagedKV.head_dim.offset == 84


def test_wrappers_refuse_host_tensors():
    from solution import kernels

    k = torch.zeros(2, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        kernels.PagedKV(k, k, torch.zeros(1, 2, dtype=torch.int32),
                        torch.zeros(1, dtype=torch.int32))


def test_rope_table_far_positions():
    """Angles of far positions keep their fp32 rounding only: against the closed form in 64
    bits, half a step of fp32 of a value of at most 1."""
    from solution import kernels

    cos, sin = kernels.rope_table(131073, 64, 1e6, "cpu")
    assert cos.shape == (131073, 32) and cos.dtype == torch.float32
    ang = 131072 * 1e6 ** (-torch.arange(32, dtype=torch.float64) / 32)
    assert (cos[-1].double() - ang.cos()).abs().max() < 1e-7
    assert (sin[-1].double() - ang.sin()).abs().max() < 1e-7


def test_rows_past_32_bits_are_refused(lib):
    """Tokens times heads stay under 2^30: what counts rows is 32 bits wide."""
    kv = _kv(n_kv=1, batch=1)
    assert _attn(lib, kv, tokens=1 << 21, heads=1024, ld=1 << 16, cu=1 << 12) == UNSUPPORTED
    assert _attn(lib, kv, tokens=(1 << 23) + 1, heads=1, cu=1 << 12) == UNSUPPORTED


@pytest.mark.parametrize("batch,width,max_len", [(1, 64, 500), (1, 1 << 16, 0), (64, 1000, 16000)])
def test_workspace_is_bounded(lib, batch, width, max_len):
    """Decoding: no workspace where a workgroup takes each sequence whole; else pieces of at most
    one workgroup per CU and one per sequence, whatever the lengths."""
    kv = _kv(batch=batch, width=width, ld_table=width)
    n = lib.nf4_paged_attn_workspace(ctypes.byref(kv), None, batch, 4, 0, 0, 0, 1, max_len)
    if max_len == 500:
        assert n == 0
    else:
        # (workgroups of a key/value head + sequences) x 2 heads x 16 rows of 64 + 2 floats, and
        # a pair for each of the rows
        assert 0 < n <= (128 + 2 * batch) * 2 * 16 * (64 * 4 + 8) + batch * 2 * 8
