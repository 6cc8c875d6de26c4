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


@pytest.mark.gpu
@pytest.mark.parametrize("wdt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dt", DTYPES)
def test_weights_that_are_not_finite_stay_visible(dt, wdt):
    """A NaN or an infinity makes its group's scale say so and the products by
    it NaN; every other group is as it would be without."""
    E, N, K, G = 2, 6, 256, 64
    w = (torch.randn(E, N, K, generator=torch.Generator().manual_seed(1)) * 0.05).to(wdt).to(DEV)
    want_p, want_s = int4.quantize_weights_int4(w, G, dt)
    bad = {(0, 1, 0): float("nan"), (0, 2, 1): float("inf"), (1, 0, 3): float("-inf"), (1, 5, 2): float("nan")}
    if wdt == torch.float32 and dt == torch.float16:
        bad[(1, 3, 1)] = 1e6  # a scale above fp16's range
    for (e, n, g), v in bad.items():
        w[e, n, g * G + 7 * g + 3] = v
    packed, scale = int4.quantize_weights_int4(w, G, dt)
    for (e, n, g), v in bad.items():
        s = float(scale[e, n, g])
        assert s != s if v != v else s == float("inf")
        assert (packed[e, n, g * G // 2:(g + 1) * G // 2] == 0x88).all()
        packed[e, n, g * G // 2:(g + 1) * G // 2] = want_p[e, n, g * G // 2:(g + 1) * G // 2]
    x = rows_of(3, K, dt)
    got = int4.int4_grouped_mv(x, want_p, scale, offsets([2, 1]), G)
    rows = torch.zeros(E, N, dtype=torch.bool)
    for e, n, _ in bad:
        rows[e, n] = True
    rows = rows.to(DEV)[torch.tensor([0, 0, 1], device=DEV)]
    assert torch.equal(packed, want_p) and torch.equal(got.isfinite(), ~rows)
    whole = int4.int4_grouped_mv(x, *int4.quantize_weights_int4(w, G, dt), offsets([2, 1]), G)
    assert torch.equal(whole.isnan(), rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_silu_of_very_negative_gates(dt):
    """A tiny silu times a large factor.  One column per row is not zero, so
    gates and factors are exact; the exponential, the quotient and the products
    are off by a few units of 2^-24, and the exponential by a rounding to fp32's
    smallest values (2^-150)."""
    gates = [-102.0, -95.0, -89.0, -88.0, -87.5, -87.0, -80.0, -20.0, -1.0, -0.0, 0.5, 20.0, 87.5, 100.0]
    N, K, G = 16, 64, 32
    up = 2.0 ** 110 if dt == torch.bfloat16 else 2.0 ** 12
    packed = torch.full((1, N, K // 2), 0x99, dtype=torch.uint8, device=DEV)  # every q is 1
    scale = torch.ones(1, N, K // G, dtype=dt, device=DEV)
    scale[:, N // 2:] = up
    x = torch.zeros(len(gates), K, dtype=dt, device=DEV)
    x[:, 5] = torch.tensor(gates, dtype=dt)
    got = int4.int4_grouped_mv(x, packed, scale, offsets([len(gates)]), G, silu=True).double()
    g = x[:, 5:6].double().expand(-1, N // 2)
    y = g * torch.sigmoid(g) * (g * up)
    tol = y.abs() * (half(dt) + 16 * 2.0 ** -24) + (g * g * up).abs() * 2.0 ** -149 + tiny(dt)
    over = y.abs() > 1.01 * torch.finfo(dt).max  # fp16's 65504 at the largest gates: rounded to an infinity
    assert (got[over] == float("inf")).all()
    assert ((got - y).abs() <= tol)[~over].all(), (got[:, 0], y[:, 0])


@pytest.mark.gpu
def test_scales_that_want_a_gradient_are_refused():
    """As rows that want one are: they would get none."""
    packed, scale = weights(1, 32, 64, 32, torch.bfloat16)
    x, eo = rows_of(2, 64, torch.bfloat16), offsets([2])
    want = int4.int4_grouped_mv(x, packed, scale, eo, 32)
    scale.requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        int4.int4_grouped_mv(x, packed, scale, eo, 32)
    with torch.no_grad():
        assert torch.equal(int4.int4_grouped_mv(x, packed, scale, eo, 32), want)


def layer(**change):
    """A call of the layer with small operands, some of them others."""
    E, K, N, T, topk = 2, 64, 32, 3, 1
    d = change.pop("device", DEV)
    x = torch.zeros(T, K, dtype=torch.bfloat16, device=d)
    a = dict(output=torch.empty_like(x), hidden_states=x,
             w1_packed=torch.full((E, 2 * N, K // 2), 0x88, dtype=torch.uint8, device=d),
             w1_scale=torch.ones(E, 2 * N, 2, dtype=torch.bfloat16, device=d),
             w2_packed=torch.full((E, K, N // 2), 0x88, dtype=torch.uint8, device=d),
             w2_scale=torch.ones(E, K, 1, dtype=torch.bfloat16, device=d),
             topk_ids=torch.zeros(T, topk, dtype=torch.int32, device=d), topk_weights=torch.ones(T, topk, device=d),
             global_num_experts=E, group_size=32)
    a.update(change)
    int4.run_int4_moe(**a)
    return a["output"]


def test_layer_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match="one CUDA device"):
        layer(device="cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["topk_ids", "topk_weights"])
def test_layer_refuses_routing_on_another_device(name):
    """Its kernels would read the host's memory."""
    assert not layer().any()
    other = dict(topk_ids=torch.zeros(3, 1, dtype=torch.int32), topk_weights=torch.ones(3, 1))[name]
    with pytest.raises(RuntimeError, match="one CUDA device"):
        layer(**{name: other})


@pytest.mark.gpu
def test_out_may_not_lie_in_what_is_read():
    """Also where the rows have gaps, in which it may lie."""
    T, N, K, G, gap = 3, 64, 64, 32, 256
    packed, scale = weights(1, N, K, G, torch.bfloat16)
    eo = offsets([T])
    x = rows_of(T, K, torch.bfloat16)
    want = int4.int4_grouped_mv(x, packed, scale, eo, G)

    def out_at(start):
        flat = torch.zeros(T * (K + gap) + T * N, dtype=torch.bfloat16, device=DEV)
        rows = flat[:T * (K + gap)].view(T, K + gap)[:, :K]
        rows.copy_(x)
        return int4.int4_grouped_mv(rows, packed, scale, eo, G, out=flat[start:start + T * N].view(T, N))

    step = K + gap
    for start in (0, 56, step - 8, step, step + 56, 2 * step - T * N + 8, 2 * step, 2 * step + 56):
        with pytest.raises(RuntimeError, match="single memory location"):
            out_at(start)
    for start in (K, step - T * N, step + K, 2 * step - T * N, 2 * step + K, 3 * step):
        assert torch.equal(out_at(start), want), start
    one = torch.zeros(K + N, dtype=torch.bfloat16, device=DEV)  # a single row, whose stride says nothing
    one[:K] = x[0]
    row = one[:K].as_strided((1, K), (8, 1))
    assert torch.equal(int4.int4_grouped_mv(row, packed, scale, offsets([1]), G, out=one[K:].view(1, N)), want[:1])
    with pytest.raises(RuntimeError, match="single memory location"):
        int4.int4_grouped_mv(row, packed, scale, offsets([1]), G, out=one[K - 8:K + N - 8].view(1, N))
    into_scales = scale.view(-1)[:1 * N].view(1, N)
    with pytest.raises(RuntimeError, match="single memory location"):
        int4.int4_grouped_mv(x[:1], packed, scale, offsets([1]), G, out=into_scales)
