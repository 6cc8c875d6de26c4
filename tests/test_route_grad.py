"""The differentiable sort of tokens by expert and their weighted return
against the formulas in 64 bits.

Tolerances: copies are exact.  u = 2^-24 is fp32's rounding, half(t) the
stored type's.  A sum over topk rows is off by topk u of the sum of absolute
values, a dot product over K columns by (K / 32 + 16) u (32 lanes share a row,
then a tree)."""

import ctypes

import pytest
import torch

from int8blockwisegemm_b200 import _lib, int4, norm, ops, permute

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
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


def close(got, ref, tol, what):
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - ref).abs() - tol).max()))


def case(T, K, E, local, topk, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:topk] for _ in range(T)]) if T else \
        torch.zeros(0, topk)
    c = dict(ids=ids.to(torch.int32), x=torch.randn(T, K, generator=g).to(dt),
             y=torch.randn(T * topk, K, generator=g).to(dt), w=torch.rand(T, topk, generator=g),
             dout=torch.randn(T, K, generator=g).to(dt), drows=torch.randn(T * topk, K, generator=g).to(dt))
    emap = None
    if local < E:
        emap = torch.full((E,), -1, dtype=torch.int32)
        emap[E - local:] = torch.arange(local, dtype=torch.int32)
    c["map"] = emap
    return {k: None if v is None else v.to(DEV) for k, v in c.items()}


def plain_maps(ids, E, local, emap):
    """(order of the expanded rows, number of rows of local experts)."""
    flat = ids.reshape(-1).long().cpu()
    key = flat if emap is None else torch.where(emap.cpu().long()[flat] < 0, flat + E, emap.cpu().long()[flat])
    order = torch.sort(key, stable=True).indices
    return order.to(ids.device), int((key < local).sum())


def run(c, E, local):
    x, y, w = (c[k].clone().requires_grad_() for k in ("x", "y", "w"))
    rows, eft, inv, pidx = permute.moe_permute_train(x, c["ids"], E, local, c["map"])
    out = permute.moe_unpermute_train(y, w, inv, eft)
    dx, dy, dw = torch.autograd.grad([rows, out], [x, y, w], [c["drows"], c["dout"]])
    return [t.detach() for t in (rows, eft, inv, pidx, out, dx, dy, dw)]


def check(T, K, E, local, topk, dt, seed=0):
    c = case(T, K, E, local, topk, dt, seed)
    rows, eft, inv, pidx, out, dx, dy, dw = run(c, E, local)
    order, n = plain_maps(c["ids"], E, local, c["map"])
    place = torch.empty_like(order)
    place[order] = torch.arange(T * topk, device=DEV)
    assert torch.equal(inv.long(), place) and int(eft[-1]) == n and eft.numel() == local + 1
    assert torch.equal(pidx[:n].long(), order[:n])
    assert torch.equal(rows[:n], c["x"][order[:n] // topk]) and not rows[n:].any()
    on = (place < n).reshape(T, topk, 1)
    at = place.reshape(T, topk)
    y = torch.where(on, c["y"][at].double(), 0.0)
    g = torch.where(on, c["drows"][at].double(), 0.0)
    w = torch.where(on[..., 0], c["w"].double(), 0.0)[..., None]
    d = c["dout"].double()[:, None]
    for got, terms in ((out, w * y), (dx, g)):
        ref = terms.sum(1)
        close(got, ref, ref.abs() * half(dt) + topk * U * terms.abs().sum(1) + tiny(dt), "sum of rows")
    ref = torch.zeros(T * topk, K, dtype=torch.float64, device=DEV)
    ref[place] = (w * d).reshape(T * topk, K)
    close(dy, ref, ref.abs() * (half(dt) + U) + tiny(dt), "dy")
    assert not dy[n:].any()
    ref = (y * d).sum(2)
    close(dw, ref, (K / 32 + 16) * U * (y * d).abs().sum(2), "dw")
    assert not dw[~on[..., 0]].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,K,E,local,topk", [(1, 8, 1, 1, 1), (1, 2048, 256, 256, 8), (0, 64, 4, 4, 2),
                                              (64, 256, 8, 8, 2), (48, 160, 6, 3, 2), (37, 1000, 60, 60, 6),
                                              (500, 2048, 256, 128, 8), (129, 4096, 128, 1, 8), (5, 72, 4, 2, 4),
                                              (33, 40, 64, 64, 33), (3, 8200, 9, 9, 3), (2500, 512, 16, 16, 1)])
def test_sort_and_return(T, K, E, local, topk, dt):
    check(T, K, E, local, topk, dt, seed=T + K)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_behind_the_local_experts_nothing_is_read(dt):
    """NaN in the rows of other ranks' experts, and in their gradients, reaches
    no output."""
    c = case(50, 64, 8, 4, 2, dt, seed=5)
    _, n = plain_maps(c["ids"], 8, 4, c["map"])
    want = run(c, 8, 4)
    c["y"][n:] = float("nan")
    c["drows"][n:] = float("inf")
    assert n < 100 and all(torch.equal(a, b) for a, b in zip(run(c, 8, 4), want))


@pytest.mark.gpu
def test_same_expert_twice_and_padded_tokens():
    """A token may name an expert twice; ids of -1 (a padded batch) belong to
    no expert."""
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    ids = torch.tensor([[1, 1], [-1, -1], [0, 1], [0, 0]], dtype=torch.int32, device=DEV)
    rows, eft, inv, _ = permute.moe_permute_train(x, ids, 2)
    assert eft.tolist() == [0, 3, 6] and not rows[6:].any()
    w = torch.ones(4, 2, device=DEV, requires_grad=True)
    out = permute.moe_unpermute_train(rows, w, inv, eft)
    assert torch.equal(out[0], 2 * x[0]) and not out[1].any() and torch.equal(out[3], 2 * x[3])
    dx, dw = torch.autograd.grad(out, [x, w], torch.ones_like(out))
    assert dx[:, 0].tolist() == [2.0, 0.0, 2.0, 2.0] and not dw[1].any()


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of out in 64 bits (out is bilinear in rows and
    weights, so they are exact but for rounding)."""
    T, K, E, topk = 7, 16, 5, 3
    c = case(T, K, E, E, topk, torch.float32, seed=2)
    x, w = c["x"].clone().requires_grad_(), c["w"].clone().requires_grad_()
    rows, eft, inv, _ = permute.moe_permute_train(x, c["ids"], E)
    out = permute.moe_unpermute_train(rows * 2 + 1, w, inv, eft)
    got = torch.autograd.grad(out, [x, w], c["dout"])

    def loss(x, w):
        return ((2 * x[:, None] + 1) * w[..., None]).sum(1).mul(c["dout"].double()).sum()

    for i, t in enumerate((x, w)):
        v = torch.randn(t.shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).to(DEV)
        args = [[x.detach().double(), w.detach().double()] for _ in range(2)]
        args[0][i] += v
        args[1][i] -= v
        diff = (loss(*args[0]) - loss(*args[1])) / 2
        size = (got[i].double() * v).abs().sum()
        assert abs(float(diff - (got[i].double() * v).sum())) <= 1e-5 * float(size)


@pytest.mark.gpu
def test_layouts_and_partial_gradients():
    T, K, E, topk = 21, 64, 8, 2
    c = case(T, K, E, E, topk, torch.bfloat16)
    want = run(c, E, E)
    wide = torch.zeros(T, K + 4, dtype=torch.bfloat16, device=DEV)
    wide[:, 4:] = c["x"]
    d = dict(c, x=wide[:, 4:], dout=c["dout"].t().contiguous().t(), ids=c["ids"].long())
    x = wide[:, 4:].requires_grad_()
    rows, eft, inv, _ = permute.moe_permute_train(x, d["ids"], E)
    w16 = c["w"].to(torch.bfloat16).requires_grad_()
    out = permute.moe_unpermute_train(c["y"], w16, inv, eft)
    dw = torch.autograd.grad(out, w16, d["dout"])[0]  # the weights' alone, in their own type
    assert torch.equal(rows, want[0]) and dw.dtype == torch.bfloat16
    assert torch.equal(dw, want[7].to(torch.bfloat16))
    assert torch.equal(torch.autograd.grad(rows, x, c["drows"])[0], want[5])
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(permute.moe_permute_train(x, d["ids"], E)[0].sum(), x, create_graph=True)
    rows, *_ = permute.moe_permute_train(c["x"], c["ids"], E)
    assert not rows.requires_grad
    out = permute.moe_unpermute_train(c["y"], c["w"], inv)  # no offsets: every row counts
    assert torch.equal(out, want[4])


@pytest.mark.gpu
def test_agrees_with_the_inference_calls():
    c = case(333, 512, 32, 16, 4, torch.float16)
    rows, eft, inv, pidx, out, *_ = run(c, 32, 16)
    p, _, eft2, inv2, pidx2 = permute.moe_permute(c["x"], None, c["ids"], 32, 16, c["map"])
    n = int(eft[-1])
    assert torch.equal(rows[:n], p[:n]) and torch.equal(eft, eft2) and torch.equal(inv, inv2)
    assert torch.equal(pidx, pidx2)
    o = torch.empty_like(out)
    permute.moe_unpermute(o, c["y"], c["w"], inv, eft)
    assert torch.equal(o, out)


@pytest.mark.gpu
def test_streams_and_graph_capture():
    c = case(64, 256, 8, 4, 2, torch.bfloat16)
    x, y, w = (c[k].clone().requires_grad_() for k in ("x", "y", "w"))

    def step():
        rows, eft, inv, pidx = permute.moe_permute_train(x, c["ids"], 8, 4, c["map"])
        out = permute.moe_unpermute_train(y, w, inv, eft)
        return [t.detach() for t in (rows, eft, inv, out, *torch.autograd.grad(
            [rows, out], [x, y, w], [c["drows"], c["dout"]]))]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    c["ids"].copy_(c["ids"].flip(0))
    for g in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    want = step()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_capture_beside_an_eager_graph_is_refused():
    c = case(8, 64, 4, 4, 2, torch.float32)
    x, y = c["x"].requires_grad_(), c["y"].requires_grad_()
    rows, eft, inv, _ = permute.moe_permute_train(x, c["ids"], 4)
    out = permute.moe_unpermute_train(y, c["w"], inv, eft)
    for call in (lambda: permute.moe_permute_train(x, c["ids"], 4),
                 lambda: permute.moe_unpermute_train(y, c["w"], inv, eft)):
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    assert rows.isfinite().all() and out.isfinite().all()


@pytest.mark.gpu
def test_bad_maps_are_reported():
    """Entries outside the rows are skipped and set the error bit."""
    c = case(4, 64, 4, 4, 2, torch.float32)
    inv = torch.tensor([0, 1, 2, 99, 4, -5, 6, 7], dtype=torch.int32, device=DEV)
    eft = torch.tensor([0, 2, 4, 6, 8], device=DEV)
    dx = permute.moe_permute_backward(c["drows"], inv, eft, 4, 2)
    assert torch.equal(dx[1], c["drows"][2]) and torch.equal(dx[2], c["drows"][4])
    assert _lib.device_error(0, clear=True) == 1 << 5
    for offsets in (eft, None, eft * 100):  # rows past the tensor are not read
        out = torch.empty(4, 64, device=DEV)
        permute.moe_unpermute(out, c["y"], c["w"], inv, offsets)
        assert torch.equal(out[1], c["w"][1, 0] * c["y"][2])
    _, dw = permute.moe_unpermute_backward(c["dout"], c["y"], c["w"], inv, eft)
    assert float(dw[1, 1]) == 0.0 and float(dw[2, 1]) == 0.0
    assert _lib.device_error(0, clear=True) == 1 << 5


@pytest.mark.gpu
def test_refusals():
    c = case(8, 64, 4, 4, 2, torch.float16)
    x, ids, w, y = c["x"], c["ids"], c["w"], c["y"]
    emap = torch.zeros(4, dtype=torch.int32, device=DEV)
    for args, message in [((x.double(), ids, 4), "bfloat16, float16 or float32"), ((x[:, :63], ids, 4), "16 bytes"),
                          ((x, ids[:4], 4), "topk_ids"), ((x, ids.float(), 4), "integers"), ((x, ids[:, :0], 4), "topk"),
                          ((x, ids, 0), "n_expert"), ((x, ids, 4, 5), "n_expert"), ((x, ids, 3000), "n_expert"),
                          ((x, ids.cpu(), 4), "device"), ((x, ids, 4, 4, emap.long()), "expert_map"),
                          ((x, ids, 4, 4, emap[:3]), "expert_map"), ((x[0], ids, 4), "rows, hidden")]:
        with pytest.raises(RuntimeError, match=message):
            permute.moe_permute_train(*args)
    inv, eft = torch.arange(16, dtype=torch.int32, device=DEV), torch.tensor([0, 4, 8, 12, 16], device=DEV)
    for args, message in [((y[:15], w, inv, eft), "one row per element"), ((y, w, inv.long(), eft), "inv_permuted_idx"),
                          ((y, w, inv[:15], eft), "inv_permuted_idx"), ((y, w, inv, eft.int()), "expert_first"),
                          ((y, w.cpu(), inv, eft), "topk_weights"), ((y.long(), w, inv, eft), "bfloat16")]:
        with pytest.raises(RuntimeError, match=message):
            permute.moe_unpermute_train(*args)
    with pytest.raises(RuntimeError, match="out_grad"):
        permute.moe_unpermute_backward(c["dout"][:7], y, w, inv, eft)
    with pytest.raises(RuntimeError, match="n_token"):
        permute.moe_permute_backward(y, inv, eft, 9, 2)


def test_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match="CUDA"):
        permute.moe_permute_train(torch.zeros(2, 8), torch.zeros(2, 1, dtype=torch.int32), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        permute.moe_unpermute_train(torch.zeros(2, 8), torch.zeros(2, 1), torch.zeros(2, dtype=torch.int32))


def test_c_argument_errors_before_any_cuda_call():
    lib = _lib.LIB
    one = ctypes.c_void_p(256)  # never read: every call below is refused first

    def calls(dtype=0, n_local=4, n_token=2, topk=2, k=64, p=one):
        return [lib.i8moe_moe_scatter_rows(p, dtype, one, one, n_local, n_token, topk, k, one, None),
                lib.i8moe_moe_permute_backward(p, dtype, one, one, n_local, n_token, topk, k, one, None),
                lib.i8moe_moe_unpermute_backward(p, one, dtype, one, one, one, n_local, n_token, topk, k, one, one,
                                                 None)]

    for kw, message in [(dict(dtype=3), "dtype"), (dict(n_local=-1), "n_local"), (dict(n_token=-1), "int32"),
                        (dict(n_token=1 << 40), "int32"), (dict(topk=0), "topk"), (dict(k=63), "16 bytes"),
                        (dict(k=-8), "n_hidden"), (dict(p=ctypes.c_void_p(8)), "aligned")]:
        assert calls(**kw) == [-1] * 3 and message in _lib.last_error(), kw
    assert calls(p=None) == [-1] * 3 and "must be given" in _lib.last_error()
    assert calls(n_token=0) == [0] * 3


@pytest.mark.gpu
def test_training_step_of_a_layer():
    """Norm, router weights, sort, the experts' products, return: outputs and
    every gradient against the same layer in 64 bits."""
    T, K, N, E, topk = 40, 64, 32, 6, 2
    g = torch.Generator().manual_seed(0)
    leaves = [torch.randn(s, generator=g) * f for s, f in (((T, K), 1), ((T, K), 1), ((K,), 0.1), ((E, K), 0.2),
                                                          ((E, N, K), 0.2), ((E, K, N), 0.2))]
    leaves[2] += 1
    dout = torch.randn(T, K, generator=g).to(DEV)

    def layer(leaves, own):
        x, r, wn, wr, w1, w2 = leaves
        if own:
            y, h = norm.rms_norm(x, wn, 1e-6, r)
        else:
            h = x + r
            y = h * (h.square().mean(1, keepdim=True) + 1e-6).rsqrt() * wn
        logits = y @ wr.T
        if own:
            ids = permute.router_topk(logits.detach(), topk)[1]
        else:
            ids = picked[0]
        w = torch.softmax(logits.gather(1, ids.long()), 1)
        if own:
            picked.append(ids)
            rows, eft, inv, _ = permute.moe_permute_train(y, ids, E)
            at = eft.tolist()
            out = torch.cat([torch.tanh(rows[at[e]:at[e + 1]] @ w1[e].T) @ w2[e].T for e in range(E)])
            return permute.moe_unpermute_train(out, w, inv, eft) + h
        each = torch.einsum("eth,ekh->tek", torch.tanh(torch.einsum("tk,enk->etn", y, w1)), w2)
        return (each.gather(1, ids.long()[..., None].expand(-1, -1, K)) * w[..., None]).sum(1) + h

    picked, results = [], []
    for own, dt in ((True, torch.float32), (False, torch.float64)):
        at = [t.to(DEV, dt).requires_grad_() for t in leaves]
        out = layer(at, own)
        results.append([out, *torch.autograd.grad(out, at, dout.to(dt))])
    for i, (a, b) in enumerate(zip(*results)):
        # fp32 products of up to 64 terms in a chain of five: 1e-4 of the largest value is a wide bound
        a, b = a.detach().double(), b.detach()
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max()), i


@pytest.mark.gpu
def test_serving_step_with_int8_rows():
    """Norm to int8, router on the norm, rows and scales sorted by expert, the
    scaled grouped product, return."""
    T, K, N, E, topk = 64, 256, 128, 8, 2
    g = torch.Generator().manual_seed(0)
    x, r = (torch.randn(T, K, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    wn = torch.ones(K, dtype=torch.bfloat16, device=DEV)
    wr = torch.randn(E, K, generator=g).to(DEV)
    b = torch.randint(-127, 128, (E, N, K), generator=g, dtype=torch.int8).to(DEV)
    sb = torch.rand(E, generator=g).to(DEV) * 1e-3
    q, s, y, h = norm.rms_norm_quant_int8(x, wn, 1e-6, r, return_norm=True)
    w, ids = permute.router_topk(y.float() @ wr.T, topk)
    eft, inv, pidx = permute.moe_permute_metadata(x, ids, E)
    eo = eft.to(torch.int32)
    ps = torch.stack([eo[1:] - eo[:-1], torch.full_like(eo[1:], N), torch.full_like(eo[1:], K)], 1)
    src = pidx.long() // topk
    mm = torch.empty(T * topk, N, dtype=torch.bfloat16, device=DEV)
    ops.int8_grouped_mm_scaled(q[src], b, mm, s[src].contiguous(), sb, eo, ps.contiguous())
    out = torch.empty(T, N, dtype=torch.bfloat16, device=DEV)
    permute.moe_unpermute(out, mm, w, inv, eft)
    val = (q.double() * s.double()[:, None])
    each = torch.einsum("tk,enk->ten", val, b.double()) * sb.double()[None, :, None]
    picked = each.gather(1, ids.long()[..., None].expand(-1, -1, N))
    terms = picked * w.double()[..., None]
    # the int32 sums are exact: two roundings to bf16 (product, return) of each term and a few of fp32
    tol = (2.0 ** -8 * 2 + 16 * U) * terms.abs().sum(1) + 1e-30
    close(out, terms.sum(1), tol, "out")
