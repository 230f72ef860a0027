"""CPU tests of the limits that launches set: calls past them ask for no workspace and are refused."""
import ctypes
import re

import pytest

from custom_ops_amd import build
from tests.test_beam import SELECT, SHARED, Select, Shared
from tests.test_serve import EINVAL, P, call, make


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(build.BEAM_LIB_PATH)


def size(lib, name, params):
    f = getattr(lib, name + "_workspace_bytes")
    f.argtypes, f.restype = [P], ctypes.c_size_t
    return f(ctypes.addressof(params))


@pytest.mark.parametrize("rows,beams", [(2 ** 24, 1), (2 ** 16, 256), (5592406, 3)])
def test_rows_of_a_selection(lib, rows, beams):
    over, under = make(Select, SELECT, groups=rows, beams=beams, vocab=7), make(Select, SELECT, groups=rows - 1, beams=beams, vocab=7)
    assert size(lib, "mi355_beam_select", over) == 0 and size(lib, "mi355_beam_select", under) > 0
    rc, err = call(lib, "mi355_beam_select", over)
    assert rc == EINVAL and re.search("2\\^24", err)
    assert call(lib, "mi355_beam_select", under)[0] != EINVAL


@pytest.mark.parametrize("h,h_k,b,groups,fits", [(64, 64, 1024, 1024, True), (2 ** 16, 2 ** 16, 1024, 1, False), (2 ** 14, 2 ** 14, 1000, 1024, False),
                                                 (2 ** 13, 2 ** 13, 1000, 1024, True), (2 ** 16, 1, 1024, 0, False), (2 ** 16, 1, 1023, 0, True)])
def test_heads_and_groups(lib, h, h_k, b, groups, fits):
    assert (size(lib, "mi355_shared_decode", make(Shared, SHARED, h=h, h_k=h_k, b=b, groups=groups)) > 0) == fits
