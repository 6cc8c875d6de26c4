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


def close_to_formula(x, packed, scale, G):
    """One expert's products within the roundings of the sums of |x| |w| and of
    the result: nothing else may enter a sum."""
    w = values(packed, scale, G)[0]
    got = int4.int4_grouped_mv(x, packed, scale, offsets([x.size(0)]), G).double()
    y, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    off = (got - y).abs() - (y.abs() * half(x.dtype) + D(x.size(1)) * size + tiny(x.dtype))
    assert not (off > 0).any(), (int((off > 0).sum()), float(off.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("outlier", [1e2, 1e3, 1e4, 6e4])
def test_a_large_value_under_a_zero_weight(outlier, G, dt):
    """It adds nothing to a result, so it costs the result nothing."""
    N, K = 64, 512
    packed, scale = weights(1, N, K, G, dt, seed=7)
    packed[..., ::16] = (packed[..., ::16] & 0xf0) | 8  # every 32nd column's weight is 0
    x = rows_of(9, K, dt)
    x[:, ::32] = outlier
    close_to_formula(x, packed, scale, G)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("G", [32, 64, 128])
def test_small_weights_and_values_of_one_sign(G, dt):
    """Groups whose scale one weight has set: the others are 0 and +-1."""
    N, K = 96, 1024
    g = torch.Generator().manual_seed(G)
    u = torch.randint(7, 10, (1, N, K), generator=g, dtype=torch.uint8)
    u[..., 5::G] = 15
    packed = (u[..., 0::2] | u[..., 1::2] << 4).to(DEV)
    scale = torch.full((1, N, K // G), 0.03, dtype=dt, device=DEV)
    close_to_formula(rows_of(5, K, dt).abs() * 100, packed, scale, G)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_infinities_and_the_largest_values(dt):
    """An infinity gives what the formula says: infinities of the weights'
    signs, NaN where the weight is 0.  Values near the type's end stay finite
    where the result is."""
    N, K, G = 64, 256, 128
    packed, scale = weights(1, N, K, G, dt, seed=3)
    x = rows_of(3, K, dt)
    x[1, 70], x[2, 8] = float("inf"), float("-inf")
    got = int4.int4_grouped_mv(x, packed, scale, offsets([3]), G)
    q = values(packed, torch.ones_like(scale), G)[0]
    for row, k, sign in ((1, 70, 1), (2, 8, -1)):
        assert torch.equal(got[row].isnan(), q[:, k] == 0)
        finite_sign = torch.sign(q[:, k]) * sign
        on = q[:, k] != 0
        assert on.any() and torch.equal(got[row][on].double(), finite_sign[on] * float("inf"))
    big = 2.0 ** 115 if dt == torch.bfloat16 else 60000.0
    scale.fill_(2.0 ** -12)
    close_to_formula(torch.full((2, K), big, dtype=dt, device=DEV), packed, scale, G)
