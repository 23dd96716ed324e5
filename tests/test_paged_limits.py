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
