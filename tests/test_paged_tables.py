"""Page tables whose rows are not a table's: refused when the cache is made, before anything could
read or write through them (no GPU needed: nothing is launched)."""

import pytest
import torch


@pytest.fixture()
def paged(monkeypatch):
    """PagedKV over host tensors, of which it takes the layout and the addresses only."""
    from solution import kernels

    monkeypatch.setattr(kernels, "_check_device", lambda *tensors: None)

    def make(table, batch=None):
        k = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
        lens = torch.zeros(table.shape[0] if batch is None else batch, dtype=torch.int32)
        return kernels.PagedKV(k, torch.zeros_like(k), table, lens)

    return make


def _overlapping(batch, width, apart):
    return torch.as_strided(torch.arange(batch * width, dtype=torch.int32), (batch, width), (apart, 1))


@pytest.mark.parametrize("table", [
    torch.arange(5, dtype=torch.int32)[None].expand(3, -1),  # one row for all
    _overlapping(3, 5, 4), _overlapping(2, 2, 1), _overlapping(64, 9, 0),
])
def test_rows_closer_than_they_are_long(paged, table):
    with pytest.raises(ValueError):
        paged(table)


def test_rows_apart_and_single_rows(paged):
    wide = torch.zeros(3, 9, dtype=torch.int32)
    assert paged(wide[:, :5]).desc.ld_table == 9
    assert paged(wide).desc.ld_table == 9
    # the stride of a dimension of size one says nothing
    for apart in (0, 2, 5, 70):
        one = torch.as_strided(torch.zeros(9, dtype=torch.int32), (1, 5), (apart, 1))
        assert paged(one).desc.ld_table == 5
    assert paged(torch.zeros(0, 5, dtype=torch.int32)).desc.ld_table == 5
    assert paged(torch.zeros(3, 0, dtype=torch.int32)).desc.width == 0
