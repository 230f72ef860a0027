"""CPU tests of what the serving operators' C entry points refuse beside tests/test_serve.py:
layouts and sizes that their kernels cannot serve."""
import pytest

from tests.test_serve import EINVAL, LAYOUT, PACKED, ROPE, Layout, Packed, Rope, call, lib, make  # noqa: F401  (lib: a fixture)


@pytest.mark.parametrize("stride", [0, 8, 56])
def test_values_that_overlap(lib, stride):   # noqa: F811
    """More than one row of V has to lie apart: a tile's rows behind the last key are outside the memory it reads."""
    rc, err = call(lib, "mi355_packed_fwd", make(Packed, PACKED, v_ts=stride))
    assert rc == EINVAL and "overlap" in err, (rc, err)


@pytest.mark.parametrize("stride", [0, 8, 56])
def test_outputs_that_overlap(lib, stride):   # noqa: F811
    """A wave stores 32 rows, those behind a sequence's last one outside the memory it may write."""
    rc, err = call(lib, "mi355_packed_fwd", make(Packed, PACKED, o_ts=stride))
    assert rc == EINVAL and "overlap" in err, (rc, err)


@pytest.mark.parametrize("cols", [2 ** 30 + 1, 2 ** 31 - 256, 2 ** 31 - 1])
def test_tables_too_wide(lib, cols):   # noqa: F811
    """Columns are counted in 32 bits, 256 at a step: near 2^31 the count would turn negative."""
    rc, err = call(lib, "mi355_paged_layout", make(Layout, LAYOUT, n=1, cols=cols))
    assert rc == EINVAL and "2^30 columns" in err, (rc, err)


@pytest.mark.parametrize("h,hk", [(2 ** 27, 1), (2 ** 31 - 1, 1), (2 ** 30, 2 ** 30)])
def test_too_many_heads_to_turn(lib, h, hk):   # noqa: F811
    """Units of 16 elements are counted in 32 bits: 8 a head of 128."""
    rc, err = call(lib, "mi355_rope_paged_store", make(Rope, ROPE, h=h, h_k=hk, d=128))
    assert rc == EINVAL and "heads" in err, (rc, err)
