"""4-bit products and their weights' quantisation where values, arguments and
rows are out of the ordinary.

Tolerances: half(t) = eps(t) / 2 is the stored type's rounding, D(K) the bound
on the sums of tests/test_int4.py."""

import re

import pytest
import torch

from int8blockwisegemm_b200 import _lib, int4
from tests.conftest import ROOT
from tests.test_int4 import DEV, DTYPES, D, half, offsets, rows_of, tiny, values, weights

CSRC = ROOT / "int8blockwisegemm_b200" / "csrc"


@pytest.fixture(autouse=True)
def no_device_error(request):
    if "gpu" not in request.keywords:
        yield
        return
    _lib.device_error(0, clear=True)
    yield
    assert _lib.device_error(0, clear=True) == 0


def test_transposes_stay_where_all_lanes_are():
    """The transpose of a tile takes all lanes of a warp, and lanes without a
    row drop its result: an asm that the compiler may move would follow the
    result into the branch."""
    found = 0
    for source in sorted(CSRC.glob("*.cu")):
        for line in re.findall(r"[^\n]*movmatrix\.sync[^\n]*", source.read_text()):
            found += 1
            assert "asm volatile(" in line, (source.name, line)
    assert found >= 1
