"""4-bit weights with group scales: the quantisation bit for bit, the experts'
products and the decoding layer against their formulas in 64 bits.

Tolerances: half(t) = eps(t) / 2 is the stored type's rounding.  A product
over K columns is added up in chunks of at least 8 columns whose sums the
tensor cores may truncate (2^-22 of the chunk's absolute values), so it is off
by at most D(K) = (K / 8 + 32) 2^-22 of the sum of absolute values."""

import ctypes

import numpy as np
import pytest
import torch

from int8blockwisegemm_b200 import _lib, int4, permute

DTYPES = [torch.bfloat16, torch.float16]
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def no_device_error(request):
    if "gpu" not in request.keywords:
        yield
        return
    _lib.device_error(0, clear=True)
    yield
    assert _lib.device_error(0, clear=True) == 0


def half(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def D(K):
    return (K / 8 + 32) * 2.0 ** -22


def weights(E, N, K, G, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    packed = torch.randint(0, 256, (E, N, K // 2), generator=g, dtype=torch.uint8)
    scale = (torch.randn(E, N, -(-K // G), generator=g) * 0.5 - 4).exp().to(dt)
    return packed.to(DEV), scale.to(DEV)


def values(packed, scale, G):
    """The weights in 64 bits."""
    E, N, b = packed.shape
    q = torch.stack([packed & 15, packed >> 4], -1).reshape(E, N, 2 * b).double() - 8
    return q * scale.double().repeat_interleave(G, 2)[..., :2 * b]


def offsets(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=DEV)


def check(got, x, packed, scale, G, counts, silu):
    """x: the sorted rows."""
    w, dt, K = values(packed, scale, G), x.dtype, x.size(1)
    r = 0
    for e, n in enumerate(counts):
        rows = x[r:r + n].double()
        y, size = rows @ w[e].T, rows.abs() @ w[e].abs().T
        err = D(K) * size
        if silu:
            h = w.size(1) // 2
            (g, u), (eg, eu) = y.split(h, 1), err.split(h, 1)
            s = g * torch.sigmoid(g)
            y = s * u
            # |silu'| < 1.1; expf, the quotient and the product: a few units of 2^-24
            err = 1.1 * eg * u.abs() + (s.abs() + 1.1 * eg) * eu + 16 * 2.0 ** -24 * y.abs()
        tol = y.abs() * half(dt) + err + tiny(dt)
        bad = (got[r:r + n].double() - y).abs() > tol
        assert not bad.any(), (e, int(bad.sum()), float((got[r:r + n].double() - y).abs().max()))
        r += n


def rows_of(R, K, dt, seed=1):
    return torch.randn(R, K, generator=torch.Generator().manual_seed(seed)).to(dt).to(DEV)


SHAPES = [  # counts, N, K
    ([1], 1, 32), ([1], 16, 64), ([3], 17, 96), ([0, 1, 0], 64, 128), ([8], 40, 160), ([9], 130, 224),
    ([2, 0, 5, 17], 96, 512), ([1, 2, 3, 4, 5, 6, 7, 8], 64, 1536), ([33], 48, 2048), ([70, 1], 34, 1056),
    ([4] * 40, 128, 256), ([1, 1], 2048, 544), ([2], 66, 4128), ([1], 8, 14336)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("counts,N,K", SHAPES, ids=lambda v: str(v)[:24])
def test_products(counts, N, K, G, dt):
    packed, scale = weights(len(counts), N, K, G, dt, seed=N + K)
    x = rows_of(sum(counts), K, dt)
    got = int4.int4_grouped_mv(x, packed, scale, offsets(counts), G)
    check(got, x, packed, scale, G, counts, False)
    if N % 2 == 0:
        got = int4.int4_grouped_mv(x, packed, scale, offsets(counts), G, silu=True)
        check(got, x, packed, scale, G, counts, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_gathered_rows_layouts_and_untouched_rows(dt):
    E, N, K, G, topk, T = 6, 48, 256, 64, 3, 9
    packed, scale = weights(E, N, K, G, dt)
    g = torch.Generator().manual_seed(0)
    ids = torch.stack([torch.randperm(E, generator=g)[:topk] for _ in range(T)])
    pidx = torch.sort(ids.reshape(-1), stable=True).indices.to(torch.int32).to(DEV)
    counts = torch.bincount(ids.reshape(-1), minlength=E).tolist()
    x = rows_of(T, K, dt)
    sorted_rows = x[pidx.long() // topk]
    got = int4.int4_grouped_mv(x, packed, scale, offsets(counts), G, permuted_idx=pidx, topk=topk, silu=True)
    check(got, sorted_rows, packed, scale, G, counts, True)
    assert torch.equal(got, int4.int4_grouped_mv(sorted_rows, packed, scale, offsets(counts), G, silu=True))
    wide = torch.zeros(T, K + 24, dtype=dt, device=DEV)
    for lo in (8, 3):  # aligned rows are read in place, others are copied
        wide[:, lo:lo + K] = x
        assert torch.equal(got, int4.int4_grouped_mv(wide[:, lo:lo + K], packed, scale, offsets(counts), G,
                                                     permuted_idx=pidx, topk=topk, silu=True))
    assert torch.equal(got, int4.int4_grouped_mv(x.t().contiguous().t(), packed, scale, offsets(counts), G,
                                                 permuted_idx=pidx, topk=topk, silu=True))
    # rows behind the last expert keep what they held
    more = torch.cat([pidx, pidx.new_full((5,), T * topk)])
    out = torch.full((T * topk + 5, N // 2), 7.0, dtype=dt, device=DEV)
    ret = int4.int4_grouped_mv(x, packed, scale, offsets(counts), G, permuted_idx=more, topk=topk, silu=True, out=out)
    assert ret is out and torch.equal(out[:T * topk], got) and (out[T * topk:] == 7).all()
    # one expert for all rows, one row at the last one, and no row at all
    for counts in ([7, 0, 0, 0, 0, 0], [0, 0, 0, 0, 0, 1], [0] * 6):
        r = rows_of(sum(counts), K, dt)
        check(int4.int4_grouped_mv(r, packed, scale, offsets(counts), G), r, packed, scale, G, counts, False)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_values_at_the_edges(dt):
    """A NaN or infinity in a row stays in that row's outputs; scales of zero
    and of infinity act as the formula says."""
    E, N, K, G = 2, 32, 256, 128
    packed, scale = weights(E, N, K, G, dt)
    x = rows_of(12, K, dt)
    eo = offsets([8, 4])
    want = int4.int4_grouped_mv(x, packed, scale, eo, G)
    y = x.clone()
    y[2, 100], y[9, 3] = float("nan"), float("inf")
    got = int4.int4_grouped_mv(y, packed, scale, eo, G)
    clean = [i for i in range(12) if i not in (2, 9)]
    assert torch.equal(got[clean], want[clean]) and got[2].isnan().all()
    assert not got[9].isfinite().any()
    scale[0, 5] = 0
    assert not int4.int4_grouped_mv(x, packed, scale, eo, G)[:8, 5].any()
    big = torch.full_like(x, 30000.0)  # sums above fp16's range, not above fp32's
    got = int4.int4_grouped_mv(big, packed, scale, eo, G)
    ref = (big[:8].double() @ values(packed, scale, G)[0].T).to(dt)
    assert torch.equal(got[:8].isinf(), ref.isinf())
    # silu of very negative and very large gates
    packed.fill_(0x99)  # every q is 1
    scale.fill_(1)
    for v in (-1000.0, 1000.0):
        got = int4.int4_grouped_mv(torch.full_like(x, v / K), packed, scale, eo, G, silu=True)
        assert (got == 0).all() if v < 0 else got.isfinite().all() or dt == torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("wdt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("sdt", [None, torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("E,N,K,G", [(1, 1, 32, 32), (3, 20, 160, 64), (2, 7, 224, 128), (2, 64, 1024, 128)])
def test_quantisation_bit_for_bit(E, N, K, G, wdt, sdt):
    g = torch.Generator().manual_seed(K)
    w = (torch.randn(E, N, K, generator=g) * 0.05).to(wdt)
    w[0, 0, :32] = 0  # a group of zeros (its first 32 columns at least)
    w[-1, -1, -32:] *= 1e-5
    packed, scale = int4.quantize_weights_int4(w.to(DEV), G, sdt)
    sdt = sdt or wdt
    groups = -(-K // G)
    f = torch.zeros(E, N, groups * G)
    f[..., :K] = w.float()
    f = f.reshape(E, N, groups, G)
    s = (f.abs().amax(-1) / 7).to(sdt)  # one fp32 division, one rounding
    sf = s.float()[..., None]
    q = torch.where(sf > 0, torch.round(f / sf), torch.zeros(())).clamp(-8, 7) + 8
    u = q.reshape(E, N, -1)[..., :K].to(torch.uint8)
    assert scale.dtype == sdt and torch.equal(scale.cpu(), s)
    assert torch.equal(packed.cpu(), u[..., 0::2] | u[..., 1::2] << 4)


def layer64(x, w1, w2, ids, weights):
    """The layer in 64 bits, in the kernels' steps: (out, bound on its error
    from the rounding of the activation, the rows' rounding and the sums)."""
    dt, K, N = x.dtype, x.size(1), w2.size(2)
    out, tol = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64)
    for t in range(x.size(0)):
        for j in range(ids.size(1)):
            e = int(ids[t, j])
            if e < 0:
                continue
            y, err = w1[e] @ x[t].double(), D(K) * (w1[e].abs() @ x[t].double().abs())
            g, u, eg, eu = y[:N], y[N:], err[:N], err[N:]
            s = g * torch.sigmoid(g)
            a = s * u
            ea = 1.1 * eg * u.abs() + (s.abs() + 1.1 * eg) * eu + a.abs() * (half(dt) + 16 * 2.0 ** -24) + tiny(dt)
            z = w2[e] @ a
            ez = w2[e].abs() @ ea + D(N) * (w2[e].abs() @ (a.abs() + ea))
            ez = ez + (z.abs() + ez) * half(dt) + tiny(dt)
            wt = float(weights[t, j])
            out[t] += wt * z
            tol[t] += abs(wt) * (ez + 2 * ids.size(1) * 2.0 ** -24 * z.abs())
    return out, tol + (out.abs() + tol) * half(dt) + tiny(dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,local", [(1, 8), (13, 8), (13, 3)])
def test_decoding_layer(T, local, dt):
    """Norm, router and the 4-bit layer together, captured and replayed with
    other tokens."""
    from int8blockwisegemm_b200 import norm
    E, K, N, topk, G = 8, 256, 96, 2, 32
    g = torch.Generator().manual_seed(3)
    w1 = int4.quantize_weights_int4((torch.randn(local, 2 * N, K, generator=g) * 0.05).to(dt).to(DEV), G)
    w2 = int4.quantize_weights_int4((torch.randn(local, K, N, generator=g) * 0.05).to(dt).to(DEV), G)
    wr = torch.randn(E, K, generator=g).to(DEV)
    wn = torch.ones(K, dtype=dt, device=DEV)
    x, r = (torch.randn(T, K, generator=g).to(dt).to(DEV) for _ in range(2))
    emap = None
    if local < E:
        emap = torch.full((E,), -1, dtype=torch.int32, device=DEV)
        emap[2:2 + local] = torch.arange(local, dtype=torch.int32, device=DEV)
    out = torch.zeros(T, K, dtype=dt, device=DEV)

    def step():
        y, h = norm.rms_norm(x, wn, 1e-6, r)
        w, ids = permute.router_topk((y.float() @ wr.T).contiguous(), topk)
        int4.run_int4_moe(out, y, *w1, *w2, ids, w, E, emap, G)
        return y, w, ids

    def verify(y, w, ids):
        lid = ids if emap is None else emap[ids.long()]
        ref, tol = layer64(y, values(*w1, G), values(*w2, G), lid, w)
        bad = (out.double() - ref).abs() > tol
        assert not bad.any(), int(bad.sum())

    verify(*step())
    first = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    x.copy_(x.flip(1))
    graph.replay()
    verify(*kept)


@pytest.mark.gpu
def test_bad_indices_are_reported():
    E, N, K, G = 2, 16, 64, 32
    packed, scale = weights(E, N, K, G, torch.bfloat16)
    x = rows_of(3, K, torch.bfloat16)
    pidx = torch.tensor([0, 99, 2, -1], dtype=torch.int32, device=DEV)
    got = int4.int4_grouped_mv(x, packed, scale, offsets([2, 2]), G, permuted_idx=pidx)
    assert _lib.device_error(0, clear=True) == 1 << 5
    assert not got[1].any() and not got[3].any()  # rows of zeros
    for eo in ([0, 3, 2], [0, 2, 9], [-1, 2, 3]):  # out of order, behind the rows, before them
        out = torch.full((3, N), 5.0, dtype=torch.bfloat16, device=DEV)
        int4.int4_grouped_mv(x, packed, scale, torch.tensor(eo, dtype=torch.int32, device=DEV), G, out=out)
        assert _lib.device_error(0, clear=True) == 1 << 4, eo
        assert (out == 5).all()


@pytest.mark.gpu
def test_refusals():
    E, N, K, G = 2, 16, 64, 32
    packed, scale = weights(E, N, K, G, torch.bfloat16)
    x, eo = rows_of(4, K, torch.bfloat16), offsets([2, 2])
    good = dict(x=x, w_packed=packed, w_scale=scale, expert_offsets=eo, group_size=G)
    pidx = torch.arange(4, dtype=torch.int32, device=DEV)
    for change, message in [
            (dict(x=x.float()), "bfloat16 or float16"), (dict(x=x[:, :32]), "twice"), (dict(x=x[0]), "rows, K"),
            (dict(w_packed=packed.to(torch.int8)), "uint8"), (dict(w_packed=packed.transpose(0, 1)), "contiguous"),
            (dict(w_scale=scale.float()), "x's dtype"), (dict(w_scale=scale[..., :1]), "ceil"),
            (dict(group_size=16), "32, 64 or 128"), (dict(group_size=64), "ceil"),
            (dict(expert_offsets=eo.long()), "int32"), (dict(expert_offsets=eo[:2]), "E \\+ 1"),
            (dict(expert_offsets=eo.cpu()), "device"), (dict(permuted_idx=pidx.long()), "permuted_idx"),
            (dict(permuted_idx=pidx, topk=0), "topk"), (dict(out=torch.empty(4, N, device=DEV)), "out"),
            (dict(out=torch.empty(3, N, dtype=torch.bfloat16, device=DEV)), "out"),
            (dict(w_packed=packed[:, :15].contiguous(), w_scale=scale[:, :15].contiguous(), silu=True), "even"),
            (dict(x=x[:, :48], w_packed=packed[..., :24].contiguous()), "divisible by 32")]:
        with pytest.raises(RuntimeError, match=message):
            int4.int4_grouped_mv(**{**good, **change})
    w = torch.zeros(2, 4, 64, device=DEV)
    for args, message in [((w[0],), "E, N, K"), ((w.double(),), "dtype"), ((w, 48), "32, 64 or 128"),
                          ((w[..., :40],), "divisible by 32"), ((w, 32, torch.int8), "dtype")]:
        with pytest.raises(RuntimeError, match=message):
            int4.quantize_weights_int4(*args)
    square = weights(E, K, K, G, torch.bfloat16)
    with pytest.raises(RuntimeError, match="single memory location"):
        int4.int4_grouped_mv(x, *square, eo, G, out=x)
    with pytest.raises(RuntimeError, match="no gradient"):
        int4.int4_grouped_mv(x.clone().requires_grad_(), packed, scale, eo, G)
    odd = torch.empty(4 * N + 1, dtype=torch.bfloat16, device=DEV)[1:].view(4, N)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        int4.int4_grouped_mv(x, packed, scale, eo, G, out=odd)
    ids, wt = torch.zeros(4, 1, dtype=torch.int32, device=DEV), torch.ones(4, 1, device=DEV)
    w1, w2 = weights(E, 64, K, G, torch.bfloat16), weights(E, K, 32, G, torch.bfloat16)
    for out, a, message in [(x[:2], (*w1, *w2), "output"), (x, (*w2, *w2), "w1 must")]:
        with pytest.raises(RuntimeError, match=message):
            int4.run_int4_moe(out, x, *a, ids, wt, E, None, G)
    with pytest.raises(RuntimeError, match="expert_map"):
        int4.run_int4_moe(x.clone(), x, *w1, *w2, ids, wt, E, torch.zeros(E, device=DEV), G)
    int4.run_int4_moe(x[:0].clone(), x[:0], *w1, *w2, ids[:0], wt[:0], E, None, G)  # no tokens: nothing to do


def test_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match="CUDA"):
        int4.quantize_weights_int4(torch.zeros(1, 2, 32))
    with pytest.raises(RuntimeError, match="CUDA"):
        int4.int4_grouped_mv(torch.zeros(1, 32, dtype=torch.bfloat16), torch.zeros(1, 2, 16, dtype=torch.uint8),
                             torch.zeros(1, 2, 1), torch.zeros(2, dtype=torch.int32))


def test_c_argument_errors_before_any_cuda_call():
    lib = _lib.LIB
    one = ctypes.c_void_p(256)  # never read: every call below is refused first

    def mv(x=one, stride=64, x_rows=4, dtype=0, pidx=None, topk=1, G=32, E=2, rows=4, n=16, k=64, silu=0):
        return lib.i8moe_int4_grouped_mv(x, stride, x_rows, dtype, pidx, topk, one, one, G, one, E, rows, n, k, silu,
                                         one, None)

    for kw, message in [(dict(dtype=2), "bfloat16"), (dict(G=16), "group_size"),
                        (dict(k=0), "K must"), (dict(k=48), "K must"), (dict(n=-1), "bad N"),
                        (dict(n=15, silu=1), "bad N"), (dict(E=-1), "n_expert"), (dict(E=4096), "n_expert"),
                        (dict(rows=-1), "n_rows"), (dict(rows=5), "fewer rows"), (dict(topk=0, pidx=one), "topk"),
                        (dict(stride=32), "aligned"), (dict(stride=65), "aligned"),
                        (dict(x=ctypes.c_void_p(8)), "aligned"), (dict(x=None), "must be given")]:
        assert mv(**kw) == -1 and message in _lib.last_error(), kw
    assert mv(rows=0) == 0 and mv(n=0) == 0 and mv(E=0) == 0

    def quantize(dtype=0, E=1, n=2, k=64, G=32, sdtype=0):
        return lib.i8moe_quantize_weights_int4(one, dtype, E, n, k, G, one, one, sdtype, None)

    for kw, message in [(dict(dtype=3), "dtype"), (dict(sdtype=4), "dtype"), (dict(k=40), "divisible"),
                        (dict(G=48), "group_size"), (dict(E=-1), "shape")]:
        assert quantize(**kw) == -1 and message in _lib.last_error(), kw
    assert quantize(E=0) == 0
