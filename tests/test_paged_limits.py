"""Arguments that the paged calls refuse on the host, before any launch (no GPU needed)."""

import ctypes
import math

import pytest

from tests.test_paged_args import ARG, UNSUPPORTED, _kv, lib  # noqa: F401 (lib is a fixture)


def _attn(lib, kv, scale=0.125, tokens=2, heads=4, cu=None, max_q=0, max_len=0):
    """Status of an attention call whose workspace is refused where it needs one."""
    return lib.nf4_paged_attn(ctypes.byref(kv), 1 << 12, 64 * heads, 64, cu, 1 << 12, None, tokens,
                              heads, scale, 0, 0, 0, max_q, max_len, 0, None, 0, None)


WORKSPACE = 4


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 3e38])
def test_scales_that_are_no_number(lib, scale):  # noqa: F811
    """NaN, infinities, and what is one times log2 e."""
    assert _attn(lib, _kv(width=1 << 16, ld_table=1 << 16), scale=scale) == ARG


@pytest.mark.parametrize("scale", [0.125, -2.0, 0.0, 1e-40, 2e38])
def test_scales_that_are(lib, scale):  # noqa: F811
    assert _attn(lib, _kv(width=1 << 16, ld_table=1 << 16), scale=scale) == WORKSPACE


@pytest.mark.parametrize("n_kv", [1, 3, 4, 6, 12, 100])
@pytest.mark.parametrize("dim", [64, 128])
def test_three_row_blocks_fit_the_card(lib, n_kv, dim):  # noqa: F811
    """33 to 48 rows a sequence over long contexts: a workgroup fills a CU then, so there are at
    most 256 (or one of each key/value head).  Their number is in the workspace: a slot of 48 rows
    for each workgroup and item of a key/value head, and a pair of words for each row."""
    batch, new, group = 32, 5, 7
    kv = _kv(batch=batch, width=1 << 14, ld_table=1 << 14, n_kv=n_kv, head_dim=dim,
             page_stride=1 << 20, slot_stride=n_kv * dim, head_stride=dim)
    rows = batch * new * group
    size = lib.nf4_paged_attn_workspace(ctypes.byref(kv), None, batch * new, group * n_kv, 0, 0, 0, 0,
                                        1 << 18)
    slots, left = divmod(size - rows * 8, n_kv * 48 * (4 * dim + 8))
    assert left == 0
    items = rows // 48 + batch
    assert 0 < (slots - items) * n_kv <= max(256, n_kv)


@pytest.mark.parametrize("batch,n_kv,width,max_len,window,few", [
    (64, 4, 1 << 14, 16000, 0, True), (16, 4, 1 << 14, 9000, 0, True),
    (8, 4, 1 << 14, 16000, 0, True), (64, 4, 1 << 14, 5000, 0, False),
    (16, 4, 1 << 14, 6000, 0, False), (1, 4, 1 << 14, 16000, 0, False),
    (4, 1, 1 << 14, 32000, 0, False), (64, 4, 1 << 14, 0, 1024, False),
    (64, 4, 1 << 14, 0, 0, True), (8, 4, 512, 0, 0, True), (8, 4, 256, 0, 0, False),
    (1, 4, 1 << 14, 0, 0, False),
])
def test_route_of_33_to_48_rows(lib, batch, n_kv, width, max_len, window, few):  # noqa: F811
    """Which kernel 35 rows a sequence go to, by what the host knows of their lengths: the
    workspace has slots of 48 rows of a key/value head for the one, whole pieces of the output for
    the other (or nothing)."""
    kv = _kv(batch=batch, width=width, ld_table=width, n_kv=n_kv, head_dim=64, slot_stride=n_kv * 64)
    tokens, heads = 5 * batch, 7 * n_kv
    size = lib.nf4_paged_attn_workspace(ctypes.byref(kv), None, tokens, heads, window, 0, 0, 0, max_len)
    rows = 35 * batch
    tiled = size % (tokens * heads * (4 * 64 + 8)) == 0
    slots = size > rows * 8 and (size - rows * 8) % (n_kv * 48 * (4 * 64 + 8)) == 0
    assert (slots and not tiled) if few else (tiled and not slots)


# (each accepted call is one that needs a workspace, and gets none: it ends there)
LIMITS = [  # cache, call, accepted
    (dict(), dict(heads=1024), True), (dict(), dict(heads=1026), False),
    (dict(batch=1 << 20), dict(tokens=1 << 20), True),
    (dict(batch=(1 << 20) + 1), dict(tokens=(1 << 20) + 1), False),
    (dict(slot_stride=1 << 26), dict(), True), (dict(slot_stride=(1 << 26) + 8), dict(), False),
    (dict(batch=1), dict(tokens=1 << 23, max_q=1, cu=1 << 12), True),
    (dict(batch=1), dict(tokens=(1 << 23) + 1, max_q=1, cu=1 << 12), False),
    (dict(n_kv=8, batch=2), dict(tokens=1 << 23, heads=128, cu=1 << 12), False),  # > 2^23 workgroups
    (dict(width=1 << 26, ld_table=1 << 26), dict(), True),
    (dict(width=(1 << 26) + 1, ld_table=1 << 27), dict(), False),
]


@pytest.mark.parametrize("cache,call,accepted", LIMITS)
def test_limits(lib, cache, call, accepted):  # noqa: F811
    kv = _kv(**{**dict(width=1 << 16, ld_table=1 << 16), **cache})
    assert _attn(lib, kv, **call) == (WORKSPACE if accepted else UNSUPPORTED)
