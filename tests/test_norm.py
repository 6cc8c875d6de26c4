"""The RMS norm with residual, int8 output and gradients against its formulas
in 64 bits.

Tolerances: u = 2^-24 is fp32's rounding, half(t) = eps(t) / 2 that of the
stored type.  A sum over K columns adds at most K / 32 + 16 terms one after
the other (32 threads share a row at least, then trees), so a sum's relative
error against the sum of absolute values is at most (K / 32 + 16) u; rstd
carries half of that.  C(K) = K / 32 + 24 covers the sum, the square root and
the products."""

import ctypes

import pytest
import torch

from int8blockwisegemm_b200 import _lib, norm

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DEV = "cuda:0"


def C(K):
    return K / 32 + 24


def half(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):  # half of the smallest subnormal: a rounding near zero
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def close(got, ref, tol, what):
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - ref).abs() - tol).max()))


def make(T, K, dt, wdt, residual, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, K, generator=g) * std).to(dt)
    w = (1 + 0.3 * torch.randn(K, generator=g)).to(wdt)
    r = (torch.randn(T, K, generator=g) * 3 * std).to(dt) if residual else None
    return x.to(DEV), w.to(DEV), r.to(DEV) if residual else None


def formula(x, w, r, eps):
    h = x.double() if r is None else x.double() + r.double()
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    return h, rstd, h * rstd * w.double()


def check_forward(x, w, r, eps):
    dt, K = x.dtype, x.size(-1)
    h, rstd, y = formula(x, w, r, eps)
    tol = y.abs() * (half(dt) + C(K) * U) + tiny(dt)
    got = norm.rms_norm(x, w, eps, r)
    gh = None
    if r is not None:
        got, gh = got
        close(gh, h, h.abs() * (half(dt) + U) + tiny(dt), "h")
    close(got, y, tol, "y")
    for keep in (False, True):
        q, s, y2, h2 = norm.rms_norm_quant_int8(x, w, eps, r, return_norm=keep)
        assert q.dtype == torch.int8 and s.shape == x.shape[:-1]
        if keep:
            assert torch.equal(y2, got)
        else:
            assert y2 is None
        assert (h2 is None) == (r is None) and (r is None or torch.equal(h2, gh))
        amax = y.abs().amax(-1)
        ref = amax.clamp_min(1e-10) / 127
        close(s, ref, ref * (C(K) + 2) * U, "scale")
        # a quotient of at most 127 may be off by 2 (C + 2) u of itself before it is rounded
        far = (y / ref[..., None] - q.double()).abs()
        assert float(far.max()) <= 0.5 + 127 * 2 * (C(K) + 2) * U


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,K", [(1, 1), (1, 2048), (3, 7), (5, 64), (17, 160), (64, 256), (33, 1001),
                                 (9, 2047), (300, 2048), (7, 4096), (130, 4100), (2, 8192),
                                 (3, 12289), (2, 20000), (2, 40961)])
def test_norm(T, K, dt):
    for residual in (False, True):
        for wdt in {dt, torch.float32}:
            check_forward(*make(T, K, dt, wdt, residual, seed=T + K), 1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_shapes_strides_and_alignment(dt):
    K = 256
    x, w, r = make(24, K + 8, dt, dt, True, seed=3)
    check_forward(x[:, :K], w[:K], r[:, :K], 1e-5)  # row stride above K
    check_forward(x[:, 1:K + 1], w[1:K + 1], r[:, 3:K + 3], 1e-5)  # rows off the 16-byte grid
    check_forward(x[::2, :K], w[:K], r[1::2, :K], 1e-5)
    check_forward(x[:1, :K].expand(9, K), w[:K], r[:9, :K], 1e-5)  # one row for all
    check_forward(x[:, :K].t().contiguous().t(), w[:K], r[:, :K], 1e-5)  # columns first
    check_forward(x[:, :K].reshape(2, 3, 4, K), w[:K], r[:, :K].reshape(2, 3, 4, K), 1e-5)
    check_forward(x[0, :K], w[:K], r[0, :K], 1e-5)  # a single row without a batch
    check_forward(x[:, :K], torch.stack([w[:K], w[:K]], 1)[:, 0], r[:, :K], 1e-5)  # strided weight


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_values_at_the_edges(dt):
    K = 512
    w = torch.ones(K, dtype=dt, device=DEV)
    x = torch.zeros(4, K, dtype=dt, device=DEV)
    q, s, y, _ = norm.rms_norm_quant_int8(x, w, 1e-6, return_norm=True)  # rows of zeros
    assert not q.any() and not y.any() and (s.double() - 1e-10 / 127).abs().max() < 1e-17
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    x[3] = torch.finfo(dt).smallest_normal
    q, s, y, _ = norm.rms_norm_quant_int8(x, w, 1e-6, return_norm=True)
    assert s[1].isnan() and s[2].isnan() and not q[1].any() and not q[2].any()
    assert y[1, 3].isnan() and y[2].isnan().all()
    assert s[0].isfinite() and s[3].isfinite() and y[0].isfinite().all() and y[3].isfinite().all()
    x = torch.zeros(1, K, dtype=dt, device=DEV)
    x[0, 7] = 3.0  # one value carries the row: the largest y there is, sqrt(K)
    q, s, y, _ = norm.rms_norm_quant_int8(x, w, 0.0, return_norm=True)
    assert int(q[0, 7]) == 127 and int(q.abs().sum()) == 127
    for T in (0,):
        y, h = norm.rms_norm(x[:T], w, 1e-6, x[:T])
        assert y.shape == (T, K) and h.shape == (T, K)
        q, s, _, _ = norm.rms_norm_quant_int8(x[:T], w)
        assert q.shape == (T, K) and s.shape == (T,)


@pytest.mark.gpu
def test_int8_of_the_largest_values():
    """Rows up to the last binade of fp32: q is 127 where |y| is largest."""
    x, _, _ = make(6, 256, torch.float32, torch.float32, False, seed=8)
    w = torch.full((256,), 5e37, device=DEV)
    for s in (1.0, 2.0 ** -20, 2.0 ** -120):
        check_forward(x, w * s, None, 1e-6)
    q, scale, _, _ = norm.rms_norm_quant_int8(x, w)
    assert float(scale.max()) * 127 > 2.0 ** 126 and (q.abs().amax(1) == 127).all()


def check_grad(x, w, r, eps, dy, dh):
    dt, K = x.dtype, x.size(-1)
    leaves = [t.detach().clone().requires_grad_() for t in ([x, w] if r is None else [x, w, r])]
    out = norm.rms_norm(leaves[0], leaves[1], eps, leaves[2] if r is not None else None)
    outs, grads = ([out], [dy]) if r is None else (list(out), [dy, dh])
    got = torch.autograd.grad(outs, leaves, grads)
    h, rstd, _ = formula(x, w, r, eps)
    n, a = h * rstd, dy.double() * w.double()
    mean = (a * n).mean(-1, keepdim=True)
    dx = rstd * (a - n * mean)
    if r is not None:
        dx = dx + dh.double()
    size = rstd * (a.abs() + n.abs() * (a * n).abs().mean(-1, keepdim=True))
    if r is not None:
        size = size + dh.double().abs()
    tol = dx.abs() * half(dt) + 2 * C(K) * U * size + tiny(dt)
    close(got[0], dx, tol, "dx")
    if r is not None:
        assert torch.equal(got[2], got[0])
    rows = x.numel() // K
    dw = (dy.double() * n).reshape(rows, K).sum(0)
    # at most rows + 300 additions in a row, and rstd's error
    tol = dw.abs() * half(w.dtype) + tiny(w.dtype) + \
        (rows + 300 + C(K)) * U * (dy.double() * n).abs().reshape(rows, K).sum(0)
    close(got[1], dw, tol, "dweight")
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,K", [(1, 1), (1, 2048), (3, 7), (17, 160), (64, 256), (333, 1001), (301, 2047),
                                 (1500, 2048), (97, 4096), (5, 8192), (3, 12289), (2, 40961)])
def test_gradients(T, K, dt):
    for residual in (False, True):
        for wdt in {dt, torch.float32}:
            x, w, r = make(T, K, dt, wdt, residual, seed=T + K)
            g = torch.Generator().manual_seed(9)
            dy = torch.randn(T, K, generator=g).to(dt).to(DEV)
            dh = torch.randn(T, K, generator=g).to(dt).to(DEV)
            first = check_grad(x, w, r, 1e-6, dy, dh)
            again = check_grad(x, w, r, 1e-6, dy, dh)
            assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("K,gap", [(1001, 8), (1001, 5), (67, 16), (2047, 8), (5003, 16), (9, 8)])
def test_odd_rows_keep_to_themselves(K, gap, dt):
    """Widths that no vector divides, alone and as the middle of wider rows:
    what stands before, behind and in the rows beside reaches no row."""
    T = 83
    x, w, r = make(T, K, dt, dt, True, seed=K)
    dy, dh = make(T, K, dt, dt, True, seed=K + 1)[::2]

    def wide(t):  # the same rows with NaN between them
        b = torch.full((T, K + gap), float("nan"), dtype=dt, device=DEV)
        b[:, :K] = t
        return b[:, :K]

    def run(x, w, r, dy, dh):
        leaves = [t.detach().requires_grad_() for t in (x, w, r)]
        y, h = norm.rms_norm(leaves[0], leaves[1], 1e-6, leaves[2])
        g = torch.autograd.grad([y, h], leaves, [dy, dh])
        return [y.detach(), h.detach(), g[0], g[2], *norm.rms_norm_quant_int8(x, w, 1e-6, r)[:2], g[1]]

    check_forward(x, w, r, 1e-6)
    check_grad(x, w, r, 1e-6, dy, dh)
    want = run(x, w, r, dy, dh)
    check_forward(wide(x), w, wide(r), 1e-6)
    check_grad(wide(x), w, wide(r), 1e-6, wide(dy), wide(dh))
    if gap % 8 == 0:  # the same kernel, so the same bits
        got = run(wide(x), w, wide(r), wide(dy), wide(dh))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    bad = torch.arange(T, device=DEV) % 3 == 1
    for t in (x, r, dy, dh):
        t[bad] = float("nan")
        got = run(x, w, r, dy, dh)
        for a, b in zip(got[:-1], want[:-1]):
            assert torch.equal(a[~bad], b[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_one_tensor_off_the_grid(dt):
    """Each tensor alone where no vector reaches it, or with a stride of its own."""
    T, K = 70, 200
    x, w, r = make(T, K + 8, dt, dt, True, seed=2)
    dy, dh = make(T, K + 8, dt, dt, True, seed=3)[::2]
    on = dict(x=x[:, :K], w=w[:K], r=r[:, :K], dy=dy[:, :K], dh=dh[:, :K])
    for name, t in dict(x=x, r=r, dy=dy, dh=dh).items():
        args = {**on, name: t[:, 1:K + 1]}
        check_grad(args["x"], args["w"], args["r"], 1e-6, args["dy"], args["dh"])
        odd = torch.cat([t, t[:, :3]], 1)[:, :K]  # rows K + 11 apart
        args = {**on, name: odd}
        check_grad(args["x"], args["w"], args["r"], 1e-6, args["dy"], args["dh"])
        if name in "xr":
            check_forward(args["x"], args["w"], args["r"], 1e-6)
    for k in (K, K - 1):
        check_forward(x[:, :k].contiguous(), w[1:k + 1], r[:, :k].contiguous(), 1e-6)
        check_grad(x[:, :k].contiguous(), w[3:k + 3], r[:, :k].contiguous(), 1e-6,
                   dy[:, :k].contiguous(), dh[:, :k].contiguous())


@pytest.mark.gpu
def test_gradient_against_differences():
    """Directional derivatives of the formula in 64 bits, by central
    differences (error about 1e-9 at this step), against the fp32 gradients."""
    T, K, eps = 6, 96, 1e-3
    x, w, r = make(T, K, torch.float32, torch.float32, True, seed=4)
    dy, dh = torch.randn(2, T, K, generator=torch.Generator().manual_seed(1)).to(DEV)
    got = check_grad(x, w, r, eps, dy, dh)

    def loss(x, w, r):
        h, _, y = formula(x, w, r, eps)
        return (y * dy.double()).sum() + (h * dh.double()).sum()

    for i, t in enumerate((x, w, r)):
        v = torch.randn(t.shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).to(DEV)
        step = 1e-5
        args = [[a.double() for a in (x, w, r)] for _ in range(2)]
        args[0][i] += step * v
        args[1][i] -= step * v
        diff = (loss(*args[0]) - loss(*args[1])) / (2 * step)
        dot = (got[i].double() * v).sum()
        size = (got[i].double() * v).abs().sum()
        assert abs(float(diff - dot)) <= float(size) * 1e-5 + 1e-6


@pytest.mark.gpu
def test_partial_gradients_and_unused_outputs():
    x, w, r = make(9, 64, torch.float32, torch.float32, True)
    r.requires_grad_()
    y, h = norm.rms_norm(x, w, 1e-6, r)
    one = torch.ones_like(h)
    assert torch.equal(torch.autograd.grad(h, r, one, retain_graph=True)[0], one)  # y unused
    both = torch.autograd.grad([y, h], r, [one, torch.zeros_like(h)], retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(y, r, one)[0], both)  # h unused
    w.requires_grad_()
    y = norm.rms_norm(x, w, 1e-6)
    y.sum().backward()  # an expanded gradient, weight alone
    assert x.grad is None and w.grad is not None
    w.grad = None
    one_row = torch.randn(64, device=DEV, requires_grad=True)  # no batch dimension
    norm.rms_norm(one_row, w, 1e-6, one_row).__getitem__(0).sum().backward()  # its own residual
    assert one_row.grad.shape == (64,) and w.grad.shape == (64,)
    y = norm.rms_norm(r, w)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y.sum(), r, create_graph=True)
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    w.grad = None
    norm.rms_norm(x, w).sum().backward()
    assert x.grad.shape == (0, 64) and not w.grad.any()
    with torch.no_grad():
        assert not norm.rms_norm(x, w).requires_grad
    z = r.detach().clone()
    y, h = norm.rms_norm(r, w, 1e-6, z)
    h.add_(1)  # the next block may go on in place
    y.sum().backward(retain_graph=True)
    z.add_(1)  # what the backward pass needs may not change
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.gpu
def test_streams_and_graph_capture():
    x, w, r = make(64, 2048, torch.bfloat16, torch.bfloat16, True)
    dy, dh = torch.randn_like(x), torch.randn_like(x)
    leaves = [t.clone().requires_grad_() for t in (x, w, r)]

    def step():
        y, h = norm.rms_norm(leaves[0], leaves[1], 1e-6, leaves[2])
        g = torch.autograd.grad([y, h], leaves, [dy, dh])
        with torch.no_grad():
            return (y.detach(), h.detach(), *g, *norm.rms_norm_quant_int8(x, w, 1e-6, r)[:2])

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, want))
    del on_side
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    with torch.no_grad():
        leaves[0].neg_()
        leaves[2].neg_()
        x.neg_()
        r.neg_()
    for g in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    fresh = step()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, fresh))
    assert torch.equal(fresh[0], -want[0])


@pytest.mark.gpu
def test_capture_beside_an_eager_graph_is_refused():
    """The captured backward pass would end the process; the call that would
    lead to it raises, and the device goes on working."""
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV)
    eager = norm.rms_norm(x, w)
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            norm.rms_norm(x, w)
    want = eager.detach().clone()
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = norm.rms_norm(x, w)
        y.backward(torch.ones_like(y))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y.detach(), want) and x.grad.isfinite().all()


@pytest.mark.gpu
def test_refusals():
    x, w, r = make(4, 64, torch.bfloat16, torch.bfloat16, True)
    cases = [(dict(x=x.to(torch.float64)), "bfloat16, float16 or float32"),
             (dict(weight=w[:32]), r"shape \[K\]"), (dict(weight=w.half()), "dtype or float32"),
             (dict(weight=w.cpu()), "device"), (dict(residual=r.float()), "x's dtype"),
             (dict(residual=r[:2]), "x's shape"), (dict(residual=r.cpu()), "device"),
             (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
             (dict(x=x[:, :0], weight=w[:0], residual=None), "K >= 1"),
             (dict(x=torch.zeros((), device=DEV), residual=None), "K >= 1")]
    for change, message in cases:
        args = {**dict(x=x, weight=w, eps=1e-6, residual=r), **change}
        for f in (norm.rms_norm, norm.rms_norm_quant_int8):
            with pytest.raises(RuntimeError, match=message):
                f(**args)
    with pytest.raises(RuntimeError, match="no gradient"):
        norm.rms_norm_quant_int8(x, w.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="x's shape"):
        norm.rms_norm_backward(x[:2], x, w, torch.ones(4, device=DEV))
    with pytest.raises(RuntimeError, match="rstd"):
        norm.rms_norm_backward(x, x, w, torch.ones(3, device=DEV))
    one = torch.ones(4, device=DEV)
    for args, message in [((x, x, w, one, r[:2]), "residual must"), ((x, x, w, one, r, r.float()), "residual_grad")]:
        with pytest.raises(RuntimeError, match=message):
            norm.rms_norm_backward(*args)


def test_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match="CUDA"):
        norm.rms_norm(torch.zeros(2, 8), torch.ones(8))
    with pytest.raises(RuntimeError, match="CUDA"):
        norm.rms_norm_quant_int8(torch.zeros(2, 8), torch.ones(8))


def test_c_argument_errors_before_any_cuda_call():
    lib = _lib.LIB
    one = ctypes.c_void_p(256)  # never read: every call below is refused first

    def forward(dtype=0, wdtype=0, rows=1, k=8, eps=1e-6, res=None, h=None, y=one, q=None, s=None, x=one):
        return lib.i8moe_rms_norm(x, k, res, k, dtype, one, wdtype, rows, k, eps, h, y, None, q, s, None)

    for kw, message in [(dict(dtype=3, wdtype=3), "dtype"), (dict(wdtype=1), "weight"), (dict(rows=-1), "n_rows"),
                        (dict(k=0), "n_hidden"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                        (dict(res=one), "residual"), (dict(h=one), "residual"), (dict(q=one), "q_scale"),
                        (dict(y=None), "no output"), (dict(x=None), "must be given")]:
        assert forward(**kw) == -1 and message in _lib.last_error(), kw
    assert forward(rows=0, x=None) == 0

    assert lib.i8moe_rms_norm_backward_workspace_size(0, 8) == 0
    assert lib.i8moe_rms_norm_backward_workspace_size(1, 8) >= 32
    big = lib.i8moe_rms_norm_backward_workspace_size(1 << 20, 2048)
    assert big == lib.i8moe_rms_norm_backward_workspace_size(1 << 30, 2048)

    def backward(dtype=0, wdtype=0, rows=4, k=8, dy=one, dw=None, ws=None, nbytes=0):
        return lib.i8moe_rms_norm_backward(dy, k, None, 0, one, k, None, 0, dtype, one, wdtype, one, rows, k, one, dw,
                                           ws, nbytes, None)

    for kw, message in [(dict(dtype=5, wdtype=5), "dtype"), (dict(wdtype=1), "weight"), (dict(rows=-1), "n_rows"),
                        (dict(k=0), "n_hidden"), (dict(dy=None), "must be given"), (dict(dw=one), "workspace"),
                        (dict(dw=one, ws=one, nbytes=8), "workspace")]:
        assert backward(**kw) == -1 and message in _lib.last_error(), kw
    assert backward(rows=0) == 0
