"""Cases that measure the framework's operators around the experts of an MoE layer:

- ``norm``: the residual's addition and the RMS norm in front of the layer, also with an int8 output and a scale per
  token (what ``int8_grouped_mm_scaled`` takes), and with its gradients;
- ``sort``: tokens sorted by expert and brought back with their weights, with the gradients of both;
- ``mv``: the experts' products of a few tokens with 4-bit weights and group scales.

``run`` computes a case in elementary torch operations, or, with ``own`` set, by the framework's own entry points.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one token of a decoding step, through the norm in front of its expert layer: latency
        dict(name="norm, 1 token", op="norm", T=1, K=2048, dtype="bf16", residual=True),
        # a prefill at the benchmark's default size: the norm feeds the router (bf16) and int8 experts
        dict(name="norm to int8, default", op="norm_int8", T=8192, K=2048, dtype="bf16", residual=True, keep=True),
        # a ragged batch at the large configuration's width and type, int8 output alone
        dict(name="norm to int8, ragged", op="norm_int8", T=4097, K=4096, dtype="fp16", residual=False, keep=False),
        # a training step's norm at the default size, forward and backward
        dict(name="norm with gradients, default", op="norm_train", T=8192, K=2048, dtype="bf16", residual=True),
        # a small model in 32 bits with sizes that no tile divides
        dict(name="norm with gradients, odd", op="norm_train", T=1021, K=1001, dtype="fp32", residual=False),
        # the tiny configuration: a training step on a handful of tokens, where launches count
        dict(name="sort and back, tiny", op="sort", T=64, K=256, E=8, local=8, topk=2, dtype="bf16"),
        # a training step's routing at the default size
        dict(name="sort and back, default", op="sort", T=8192, K=2048, E=256, local=256, topk=8, dtype="bf16"),
        # one of two ranks of expert parallelism at the large width: half of the rows belong to other ranks
        dict(name="sort and back, half the experts", op="sort", T=5001, K=4096, E=128, local=64, topk=8, dtype="fp16"),
        # one decoding token through its 8 experts' first product and activation
        dict(name="4-bit first product, 1 token", op="mv", T=1, K=2048, N=1024, E=256, topk=8, group=128,
             dtype="bf16", silu=True),
        # the decode configuration (128 tokens, 256 experts): all experts' weights are read
        dict(name="4-bit first product, decode", op="mv", T=128, K=2048, N=1024, E=256, topk=8, group=128,
             dtype="bf16", silu=True),
        # the same layer's second product
        dict(name="4-bit second product, decode", op="mv", T=128, K=512, N=2048, E=256, topk=8, group=128,
             dtype="bf16", silu=False),
        # the large configuration's second product for a few tokens, finer groups
        dict(name="4-bit second product, large", op="mv", T=45, K=1536, N=4096, E=128, topk=8, group=64,
             dtype="fp16", silu=False),
    ]


def draw(rng):
    def size(lo, hi):  # spread over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "norm_int8", "norm_train", "sort", "sort", "mv", "mv", "mv"])
    if op.startswith("norm"):
        K = size(64, 8192)
        if rng.random() < 0.6:  # most models' widths fill whole vectors
            K = max(64, K // 64 * 64)
        T = size(1, max(1, min(16384, (1 << 24) // K)))
        c = dict(op=op, T=T, K=K, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), residual=rng.random() < 0.6)
        if op == "norm_int8":
            c["keep"] = rng.random() < 0.5
        return c
    if op == "sort":
        E = size(4, 256)
        topk = rng.randint(1, min(8, E))
        K = size(64, 4096) // 8 * 8
        T = size(1, max(1, min(16384, (1 << 26) // (K * topk))))
        return dict(op=op, T=T, K=K, E=E, local=E if rng.random() < 0.7 else max(1, E // 2), topk=topk,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    E = size(1, 256)
    topk = rng.randint(1, min(8, E))
    K = size(64, 4096) // 32 * 32
    silu = rng.random() < 0.5
    N = size(32, 4096) // (32 if silu else 16) * (32 if silu else 16)
    E = max(topk, min(E, (1 << 28) // (K * N)))
    return dict(op=op, T=size(1, max(1, min(128, 16 * E // topk))), K=K, N=N, E=E, topk=topk,
                group=rng.choice([32, 64, 128, 128]), dtype=rng.choice(["bf16", "bf16", "fp16"]), silu=silu)


def routing(g, T, E, topk):
    """Every token's experts, as a router picks them: distinct, by the largest of T x E values."""
    dev = g.device
    return torch.topk(torch.randn(T, E, generator=g, device=dev), topk, dim=1).indices.to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    T, K = case["T"], case["K"]

    def normal(*shape, dtype=dt, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)

    s = {"case": case}
    if case["op"].startswith("norm"):
        s["x"] = normal(T, K)
        s["residual"] = normal(T, K, std=4.0) if case["residual"] else None
        s["weight"] = (1 + 0.1 * torch.randn(K, generator=g, device=dev)).to(dt)
        if case["op"] == "norm_train":
            s["dy"] = normal(T, K)
            s["dh"] = normal(T, K) if case["residual"] else None
            for k in ("x", "residual", "weight"):
                if s[k] is not None:
                    s[k].requires_grad_()
        return s
    E, topk = case["E"], case["topk"]
    s["ids"] = routing(g, T, E, topk)
    if case["op"] == "sort":
        s["x"] = normal(T, K).requires_grad_()
        s["y"] = normal(T * topk, K).requires_grad_()  # what the experts made of the sorted rows
        s["w"] = torch.softmax(torch.randn(T, topk, generator=g, device=dev), 1).requires_grad_()
        s["dout"] = normal(T, K)
        s["drows"] = normal(T * topk, K)  # what reaches the sorted rows from the experts
        s["map"] = None
        if case["local"] < E:  # this rank's experts are the last ones
            s["map"] = torch.full((E,), -1, dtype=torch.int32, device=dev)
            s["map"][E - case["local"]:] = torch.arange(case["local"], dtype=torch.int32, device=dev)
        return s
    N, G = case["N"], case["group"]
    flat = s["ids"].reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    s["pidx"] = order.to(torch.int32)
    counts = torch.bincount(flat, minlength=E)
    s["eo"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    # a first product gathers its rows from the tokens, a second one has them sorted already
    s["gather"] = bool(case["silu"])
    s["x"] = normal(T if s["gather"] else T * topk, K)
    s["packed"] = torch.randint(0, 256, (E, N, K // 2), generator=g, device=dev, dtype=torch.uint8)
    s["scale"] = (torch.randn(E, N, -(-K // G), generator=g, device=dev) * 0.4 - 5).exp().to(dt)
    s["most"] = int(counts.max())  # the plain form's padding
    s["active"] = int((counts > 0).sum())
    return s


def values(q, scale):
    """What int8 values with a scale per row stand for; bf16 has the 8 bits that they carry."""
    return torch.mul(q, scale[:, None], out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device))


# ---------------------------------------------------------------- plain forms

def plain_norm(s):
    """h = x + residual; y = h * rsqrt(mean(h^2) + eps) * weight."""
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    h = x if s["residual"] is None else x + s["residual"].detach().float()
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    n = h * rstd
    y = n * w
    out = {}
    if c["op"] == "norm_int8":
        scale = y.abs().amax(1).clamp_min(1e-10) / 127
        q = torch.round(y / scale[:, None]).clamp(-127, 127)
        out["q"], out["scale"] = values(q, scale), scale
        if c["keep"]:
            out["y"] = y.to(dt)
    else:
        out["y"] = y.to(dt)
    if s["residual"] is not None:
        out["h"] = h.to(dt)
    if c["op"] == "norm_train":
        dy = s["dy"].float()
        out["dweight"] = (dy * n).sum(0).to(dt)
        dn = dy * w
        dx = rstd * (dn - n * (dn * n).mean(1, keepdim=True))
        if s["dh"] is not None:
            dx = dx + s["dh"].float()
        out["dx"] = dx.to(dt)
        if s["residual"] is not None:
            out["dresidual"] = dx.to(dt)
    return out


def plain_sort(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    topk, local = c["topk"], c["local"]
    ids = s["ids"].reshape(-1)
    key = ids if s["map"] is None else s["map"][ids.long()]
    key = torch.where(key < 0, ids + c["E"], key)  # other ranks' rows come last, by expert
    order = torch.sort(key, stable=True).indices
    inv = torch.empty_like(order)
    inv[order] = torch.arange(order.numel(), device=order.device)
    experts = torch.arange(local + 1, device=order.device, dtype=key.dtype)
    offsets = (key[:, None] < experts[None, :]).sum(0)
    n = offsets[local]  # the rows behind belong to other ranks and are zero
    behind = torch.arange(order.numel(), device=order.device) >= n
    rows = s["x"].detach()[order // topk].masked_fill(behind[:, None], 0)
    mine = (inv < n).reshape(-1, topk)
    at = torch.where(mine, inv.reshape(-1, topk), 0)
    w, dout = s["w"].detach(), s["dout"].float()
    y = s["y"].detach()[at].float() * mine[..., None]
    out = (y * w[..., None]).sum(1).to(dt)
    dw = (y * dout[:, None, :]).sum(2)
    dy = torch.zeros_like(s["y"])
    dy[inv] = ((mine * w)[..., None] * dout[:, None, :]).reshape(-1, c["K"]).to(dt)
    dx = (s["drows"][at].float() * mine[..., None]).sum(1).to(dt)
    return {"rows": rows, "offsets": offsets, "inv": inv.to(torch.int32), "out": out, "dw": dw, "dy": dy, "dx": dx}


def plain_mv(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    R, G, K = s["pidx"].numel(), c["group"], c["K"]
    row = torch.arange(R, device=s["x"].device)
    expert = torch.searchsorted(s["eo"], row, right=True, out_int32=True).long() - 1
    new = torch.cat([expert.new_zeros(1), (expert[1:] != expert[:-1]).long()]).cumsum(0)  # which active expert
    active = torch.zeros(s["active"], dtype=torch.long, device=row.device).index_copy_(0, new, expert)
    p = s["packed"][active]
    q = torch.stack([p & 15, p >> 4], -1).reshape(*p.shape[:2], K).float() - 8
    w = q * s["scale"][active].float().repeat_interleave(G, 2)[..., :K]
    x = s["x"].float()
    if s["gather"]:
        x = x[s["pidx"].long() // c["topk"]]
    at = row - s["eo"][expert]
    pad = x.new_zeros(s["active"], s["most"], K)
    pad[new, at] = x
    y = torch.bmm(pad, w.transpose(1, 2))[new, at]
    if c["silu"]:
        gate, up = y.chunk(2, 1)
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(dt)


# ------------------------------------------------- the framework's entry points

def own_norm(s):
    from int8blockwisegemm_b200 import norm
    c = s["case"]
    if c["op"] == "norm_int8":
        q, scale, y, h = norm.rms_norm_quant_int8(s["x"], s["weight"], EPS, s["residual"], return_norm=c["keep"])
        out = {"q": values(q, scale), "scale": scale}
        if c["keep"]:
            out["y"] = y
        if h is not None:
            out["h"] = h
        return out
    if s["residual"] is None:
        y = norm.rms_norm(s["x"], s["weight"], EPS)
        out, ends, grads, leaves, names = {"y": y}, [y], [s.get("dy")], [s["x"], s["weight"]], ["dx", "dweight"]
    else:
        y, h = norm.rms_norm(s["x"], s["weight"], EPS, s["residual"])
        out, ends, grads = {"y": y, "h": h}, [y, h], [s.get("dy"), s.get("dh")]
        leaves, names = [s["x"], s["weight"], s["residual"]], ["dx", "dweight", "dresidual"]
    if c["op"] == "norm_train":
        out.update(zip(names, torch.autograd.grad(ends, leaves, grads)))
    return out


def own_sort(s):
    from int8blockwisegemm_b200 import permute
    c = s["case"]
    rows, offsets, inv, _ = permute.moe_permute_train(s["x"], s["ids"], c["E"], c["local"], s["map"])
    out = permute.moe_unpermute_train(s["y"], s["w"], inv, offsets)
    dx, dy, dw = torch.autograd.grad([rows, out], [s["x"], s["y"], s["w"]], [s["drows"], s["dout"]])
    return {"rows": rows, "offsets": offsets, "inv": inv, "out": out, "dw": dw, "dy": dy, "dx": dx}


def own_mv(s):
    from int8blockwisegemm_b200 import int4
    c = s["case"]
    if s["gather"]:
        return int4.int4_grouped_mv(s["x"], s["packed"], s["scale"], s["eo"], c["group"], permuted_idx=s["pidx"],
                                    topk=c["topk"], silu=c["silu"])
    return int4.int4_grouped_mv(s["x"], s["packed"], s["scale"], s["eo"], c["group"], silu=c["silu"])


def run(state):
    op = state["case"]["op"]
    if own:
        return own_sort(state) if op == "sort" else own_mv(state) if op == "mv" else own_norm(state)
    return plain_sort(state) if op == "sort" else plain_mv(state) if op == "mv" else plain_norm(state)


def work(case):
    T, K = case["T"], case["K"]
    b = DTYPES[case["dtype"]].itemsize
    op = case["op"]
    if op.startswith("norm"):
        rows = 1 + 2 * case["residual"]  # x; the residual and the sum
        if op != "norm_int8" or case["keep"]:
            rows += 1
        n, flops = T * K * b * rows + K * b, 5 * T * K
        if op == "norm_int8":  # the int8 values are handed over as the numbers that they stand for
            n, flops = n + T * K * 2 + 4 * T, flops + 3 * T * K
        if op == "norm_train":  # dy (and the sum's gradient), the gradients of x and residual (one tensor), dweight
            n, flops = n + T * K * b * (2 + case["residual"]) + K * b, flops + 10 * T * K
        return {"bytes": n, "flops": flops}
    topk, E = case["topk"], case["E"]
    if op == "sort":
        R = T * topk * case["local"] / E  # the rank's own rows, on average
        rows = R * (1 + 1 + 1 + 1) + 2 * (T * topk - R)  # sorted rows, y, drows and dy; other ranks' zeros in two of them
        return {"bytes": (rows + T * 4) * K * b + T * topk * (4 + 4 + 4 + 4) + (E + 1) * 8, "flops": 6 * R * K}
    N, R = case["N"], T * topk
    active = E * (1 - (1 - topk / E) ** T)  # experts that a token reaches, on average
    weights = active * N * (K / 2 + -(-K // case["group"]) * b)
    io = (T if case["silu"] else R) * K * b + R * (N // 2 if case["silu"] else N) * b
    return {"bytes": weights + io + 4 * (E + 1 + R), "flops": 2 * R * N * K}


# ------------------------------------------------------- definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    op, K = case["op"], case["K"]
    if op.startswith("norm"):
        h = d["x"].clone()
        if d["residual"] is not None:
            h += d["residual"]
        size = torch.sqrt(torch.linalg.vector_norm(h, dim=1) ** 2 / K + EPS)[:, None]
        y = h / size * d["weight"]
        out = {}
        if op == "norm_int8":
            scale = torch.clamp_min(torch.amax(torch.abs(y), 1), 1e-10) / 127
            out = {"q": torch.round(y / scale[:, None]) * scale[:, None], "scale": scale}
        if op != "norm_int8" or case["keep"]:
            out["y"] = y
        if d["residual"] is not None:
            out["h"] = h
        if op == "norm_train":
            out["dweight"] = torch.einsum("tk,tk->k", d["dy"], h / size)
            a = d["dy"] * d["weight"]
            dx = a / size - h * torch.einsum("tk,tk->t", a, h)[:, None] / (K * size ** 3)
            if d["dh"] is not None:
                dx = dx + d["dh"]
            out["dx"] = dx
            if d["residual"] is not None:
                out["dresidual"] = dx
        return out
    topk, E = case["topk"], case["E"]
    if op == "sort":
        T, first = case["T"], E - case["local"]
        chosen = s["ids"].reshape(-1).tolist()
        order = sorted(range(T * topk), key=lambda i: ((chosen[i] < first), chosen[i], i))
        place = torch.empty(T * topk, dtype=torch.long)
        place[torch.tensor(order)] = torch.arange(T * topk)
        place = place.to(s["x"].device)
        n = sum(e >= first for e in chosen)
        out, dx = torch.zeros_like(d["dout"]), torch.zeros_like(d["dout"])
        dw, dy = torch.zeros_like(d["w"]), torch.zeros_like(d["y"])
        for j in range(topk):
            here = place[j::topk]
            t = torch.nonzero(here < n)[:, 0]
            r = here[t]
            out[t] += d["w"][t, j, None] * d["y"][r]
            dx[t] += d["drows"][r]
            dw[t, j] = torch.einsum("tk,tk->t", d["y"][r], d["dout"][t])
            dy[r] = d["w"][t, j, None] * d["dout"][t]
        return {"rows": None, "offsets": None, "inv": None, "out": out, "dw": dw, "dy": dy, "dx": dx}
    eo, G = s["eo"].tolist(), case["group"]
    src = (s["pidx"] // topk).long() if s["gather"] else torch.arange(eo[-1], device=s["x"].device)
    y = torch.empty(eo[-1], case["N"], dtype=torch.float64, device=s["x"].device)
    for e in range(E):
        if eo[e] < eo[e + 1]:
            w = torch.empty(case["N"], K, dtype=torch.float64, device=y.device)
            w[:, 0::2] = s["packed"][e].bitwise_and(15).double() - 8
            w[:, 1::2] = s["packed"][e].bitwise_right_shift(4).double() - 8
            w *= d["scale"][e][:, torch.arange(K, device=y.device) // G]
            y[eo[e]:eo[e + 1]] = d["x"][src[eo[e]:eo[e + 1]]] @ w.T
    if case["silu"]:
        half = case["N"] // 2
        y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
    return y
