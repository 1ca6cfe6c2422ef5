"""The level table of the group norm is read as int64: an address that is not on an 8-byte boundary is refused before any launch (no GPU
needed)."""
import pytest

from test_capi_row_ops import ENTRIES, call, lib, refused  # noqa: F401


@pytest.mark.parametrize("name", ["dfa3d_group_norm_forward", "dfa3d_group_norm_backward"])
@pytest.mark.parametrize("address", [20, 18, 17])
def test_tables_off_their_grid_are_refused(lib, name, address):  # noqa: F811
    # without images nothing else would stop the call, and nothing would be launched
    for table in ("shapes", "start"):
        refused(lib, call(lib, name, B=0, **{table: address}), b"8-byte aligned")


@pytest.mark.parametrize("name", ["dfa3d_group_norm_forward", "dfa3d_group_norm_backward"])
def test_tables_on_it_are_taken(lib, name):  # noqa: F811
    extra = dict(grad_weight=None, grad_bias=None) if name.endswith("backward") else {}
    assert call(lib, name, B=0, shapes=24, start=8, **extra) == 0
