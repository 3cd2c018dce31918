"""The expert-layer operators in 8 bits, as cases to be timed and compared.

``own`` False computes each operator in elementary torch operations in 32 bits; ``own`` True makes the
calls a user makes of ``rwkv_mlx_b200``.  Four operators:

  route    routing from logits: sigmoid or softmax scores, a bias for balance, groups, top-k,
           renormalised weights; with ``grad`` the gradient of the logits too;
  quant    rows to e4m3 with one fp32 scale for each block of 128 values of a row;
  linear   y = x W^T with x quantised in the call and W held in e4m3 with a scale for each
           128 x 128 block; with ``grad`` dx = q(dy) W too (W frozen);
  experts  rows sorted by expert through each expert's squared-ReLU layer: key product, relu^2,
           quantisation of the hidden rows, value product.
"""

import math

import torch

own = False

E4M3_MAX = 448.0
BLOCK = 128
TINY = 1e-30  # an all-zero block quantises with this maximum
DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one token of a single stream: latency
        dict(name="route one token", op="route", n=1, E=64, k=6, score="softmax", bias=False, groups=8, keep=3,
             by="max", renorm=False, dtype="float32", grad=False),
        # a decode batch of 256 sequences (the batched decode step's size) over many experts
        dict(name="route decode 256", op="route", n=256, E=256, k=8, score="sigmoid", bias=True, groups=8, keep=4,
             by="top2", renorm=True, dtype="float32", grad=False),
        # a prefill of 8 x 4096 tokens, the same router
        dict(name="route prefill 32768", op="route", n=32768, E=256, k=8, score="sigmoid", bias=True, groups=8, keep=4,
             by="top2", renorm=True, dtype="float32", grad=False),
        # a training step's router: 16-bit logits (many exact ties), forward and gradient, odd token count
        dict(name="route train 16381", op="route", n=16381, E=96, k=4, score="softmax", bias=False, groups=1, keep=1,
             by="max", renorm=True, dtype="bfloat16", grad=True),
        # activations of a prefill before an 8-bit product
        dict(name="quant prefill", op="quant", n=32768, K=1024, dtype="bfloat16"),
        # odd rows, the last block of each row ragged
        dict(name="quant ragged", op="quant", n=1021, K=776, dtype="float16"),
        # decode: four tokens through the key projection of the D=1024 model
        dict(name="linear decode 4", op="linear", n=4, N=4096, K=1024, dtype="bfloat16", grad=False),
        # nothing a multiple of a tile, the last K block ragged
        dict(name="linear ragged", op="linear", n=1531, N=1000, K=1096, dtype="float16", grad=False),
        # frozen projection in a fine-tuning step: product and gradient of its input
        dict(name="linear tune", op="linear", n=8192, N=4096, K=1024, dtype="bfloat16", grad=True),
        # the largest: a long-K product of a prefill
        dict(name="linear large", op="linear", n=16384, N=8192, K=4096, dtype="bfloat16", grad=False),
        # decode batch through 64 experts: most experts get no or a few rows
        dict(name="experts decode", op="experts", n=64, E=64, C=1024, D=2048, dtype="bfloat16"),
        # prefill through 32 experts, skewed load
        dict(name="experts prefill", op="experts", n=32768, E=32, C=1024, D=4096, dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route", "quant", "linear", "linear", "experts"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = rng.randint(max(2, 16 // groups), 256 // groups)
        keep = rng.randint(1, groups)
        score = rng.choice(["softmax", "sigmoid"])
        k = rng.randint(1, min(8, keep * per))
        # one expert a token has the constant weight 1 when renormalised: no gradient to compare
        return dict(op=op, n=_log_int(rng, 1, 32768), E=groups * per, k=k, score=score,
                    bias=score == "sigmoid" and rng.random() < 0.7, groups=groups, keep=keep,
                    by="top2" if score == "sigmoid" else "max", renorm=k > 1 and rng.random() < 0.6, dtype=dtype,
                    grad=rng.random() < 0.5)
    if op == "quant":
        return dict(op=op, n=_log_int(rng, 1, 32768), K=8 * _log_int(rng, 8, 512), dtype=dtype)
    if op == "linear":
        return dict(op=op, n=_log_int(rng, 1, 16384), N=8 * _log_int(rng, 4, 1024), K=8 * _log_int(rng, 4, 512),
                    dtype=rng.choice(["float16", "bfloat16"]), grad=rng.random() < 0.4)
    return dict(op=op, n=_log_int(rng, 8, 16384), E=rng.randint(2, 64), C=128 * rng.randint(2, 8),
                D=8 * rng.randint(32, 256), dtype=rng.choice(["float16", "bfloat16"]))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, n, K, dtype):
    """Activations: unit rows with a few channels of larger size, as after a layer norm's weight."""
    ch = 1.0 + 3.0 * (torch.rand(K, device="cuda", generator=g) < 0.02)
    return (torch.randn(n, K, device="cuda", generator=g) * ch).to(DT[dtype])


def _weights(g, G, N, K):
    """(G, N, K) e4m3 with a row pitch of a multiple of 16 bytes, and the scales of its 128 x 128 blocks."""
    w = torch.randn(G, N, K, device="cuda", generator=g) / math.sqrt(K)
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    wp = torch.zeros(G, nb * BLOCK, kb * BLOCK, device="cuda")
    wp[:, :N, :K] = w
    wb = wp.view(G, nb, BLOCK, kb, BLOCK)
    a = wb.abs().amax((2, 4)).clamp(min=TINY)
    q = (wb * (torch.reciprocal(a) * E4M3_MAX)[:, :, None, :, None]).reshape(G, nb * BLOCK, kb * BLOCK)[:, :N, :K].to(torch.float8_e4m3fn)
    return _pitched(q), a * (1.0 / E4M3_MAX)


def _pitched(q):
    G, N, K = q.shape
    out = torch.zeros(G, N, -(-K // 16) * 16, device="cuda", dtype=torch.uint8)
    out[:, :, :K] = q.contiguous().view(torch.uint8)
    return out.view(torch.float8_e4m3fn)[:, :, :K]


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "route":
        n, E = case["n"], case["E"]
        skew = torch.randn(E, device="cuda", generator=g) * 0.5
        s["logits"] = (torch.randn(n, E, device="cuda", generator=g) * 1.5 + skew).to(DT[case["dtype"]])
        s["bias_t"] = torch.randn(E, device="cuda", generator=g) * 0.1 if case["bias"] else None
        s["dweights"] = torch.randn(n, case["k"], device="cuda", generator=g) if case["grad"] else None
    elif case["op"] == "quant":
        s["x"] = _rows(g, case["n"], case["K"], case["dtype"])
    elif case["op"] == "linear":
        s["x"] = _rows(g, case["n"], case["K"], case["dtype"])
        q, sc = _weights(g, 1, case["N"], case["K"])
        s["wq"], s["ws"] = q[0], sc[0]
        if case["grad"]:
            s["dy"] = _rows(g, case["n"], case["N"], case["dtype"]) * 1e-2
            # the transposed layout that the gradient reads, kept like the weight itself
            s["wqt"] = _pitched(q.contiguous().view(torch.uint8).transpose(1, 2).contiguous().view(torch.float8_e4m3fn))[0]
            s["wst"] = s["ws"].t().contiguous()
    else:
        n, E = case["n"], case["E"]
        load = torch.softmax(torch.randn(E, device="cuda", generator=g), 0)
        who = torch.multinomial(load, n, replacement=True, generator=g)
        sizes = torch.bincount(who, minlength=E)
        s["offsets"] = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).to(torch.int32)
        s["cap"] = int(sizes.max())
        s["x"] = _rows(g, n, case["C"], case["dtype"])
        s["kq"], s["ks"] = _weights(g, E, case["D"], case["C"])
        s["vq"], s["vs"] = _weights(g, E, case["C"], case["D"])
    return s


# ---------------------------------------------------------------- plain forms


def _plain_route(s):
    l = s["logits"].float()
    n, E, k = s["n"], s["E"], s["k"]
    if s["score"] == "sigmoid":
        p = torch.reciprocal(1.0 + torch.exp(-l))
    else:
        e = torch.exp(l - l.max(-1, keepdim=True).values)
        p = e / e.sum(-1, keepdim=True)
    # softmax keeps the logits' order: without a bias the logits themselves are compared
    key = p if s["bias_t"] is None else p + s["bias_t"]
    if s["score"] == "softmax" and s["bias_t"] is None:
        key = l
    if s["groups"] > 1:
        kg = torch.sort(key.view(n, s["groups"], -1), dim=-1, descending=True, stable=True).values
        gs = kg[..., 0] if s["by"] == "max" else kg[..., 0] + kg[..., 1]
        best = torch.sort(gs, dim=-1, descending=True, stable=True).indices[:, : s["keep"]]
        stay = torch.zeros_like(gs, dtype=torch.bool).scatter(1, best, True)
        key = torch.where(stay[..., None], key.view(n, s["groups"], -1), -math.inf).view(n, E)
    inds = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :k]
    sel = p.gather(1, inds)
    total = sel.sum(-1, keepdim=True)
    w = sel / total if s["renorm"] else sel
    counts = torch.zeros(E, device=l.device, dtype=torch.int32)
    counts.scatter_add_(0, inds.reshape(-1), torch.ones_like(inds.reshape(-1), dtype=torch.int32))
    out = {"inds": inds.to(torch.int32), "weights": w, "counts": counts}
    if s["grad"]:
        gw = s["dweights"]
        ds = (gw - (gw * w).sum(-1, keepdim=True)) / total if s["renorm"] else gw
        d = torch.zeros_like(p).scatter(1, inds, ds)
        d = d * p * (1.0 - p) if s["score"] == "sigmoid" else p * (d - (d * p).sum(-1, keepdim=True))
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _plain_quant(x):
    n, K = x.shape
    kb = -(-K // BLOCK)
    xp = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - K)).view(n, kb, BLOCK)
    a = xp.abs().amax(-1).clamp(min=TINY)
    q = (xp * (torch.reciprocal(a) * E4M3_MAX)[..., None]).view(n, kb * BLOCK)[:, :K].to(torch.float8_e4m3fn)
    return q, a * (1.0 / E4M3_MAX)


def _spread_rows(q, sc):
    return q.float() * sc.repeat_interleave(BLOCK, -1)[..., : q.shape[-1]]


def _spread_blocks(q, sc):
    return q.float() * sc.repeat_interleave(BLOCK, -2)[..., : q.shape[-2], :].repeat_interleave(BLOCK, -1)[..., : q.shape[-1]]


def _plain_linear(x, wq, ws):
    return (_spread_rows(*_plain_quant(x)) @ _spread_blocks(wq, ws).mT).to(x.dtype)


def _plain_experts(s):
    n, E, cap = s["n"], s["E"], s["cap"]
    row = torch.arange(n, device="cuda")
    e = torch.searchsorted(s["offsets"][1:].long(), row, right=True)
    at = e * cap + row - s["offsets"].long()[e]  # the row's place when every expert has room for `cap` rows
    x = torch.zeros(E * cap, s["C"], device="cuda").index_copy(0, at, _spread_rows(*_plain_quant(s["x"])))
    h = torch.bmm(x.view(E, cap, -1), _spread_blocks(s["kq"], s["ks"]).mT)
    h = _spread_rows(*_plain_quant(torch.relu(h).square().view(E * cap, -1)))
    y = torch.bmm(h.view(E, cap, -1), _spread_blocks(s["vq"], s["vs"]).mT)
    return y.view(E * cap, -1)[at].to(s["x"].dtype)


# ---------------------------------------------------------------- one pass


def run(s):
    op = s["op"]
    if not own:
        if op == "route":
            return _plain_route(s)
        if op == "quant":
            q, sc = _plain_quant(s["x"])
            return {"q": q, "scale": sc}
        if op == "linear":
            out = {"y": _plain_linear(s["x"], s["wq"], s["ws"])}
            if s["grad"]:
                out["dx"] = _plain_linear(s["dy"], s["wqt"], s["wst"])
            return out
        return {"y": _plain_experts(s)}
    from rwkv_mlx_b200 import fp8, route

    if op == "route":
        logits = s["logits"].detach().requires_grad_(True) if s["grad"] else s["logits"]
        inds, w, counts = route.route_experts(logits, s["k"], score=s["score"], bias=s["bias_t"], n_groups=s["groups"],
                                              topk_groups=s["keep"], group_score=s["by"], renormalize=s["renorm"],
                                              return_counts=True)
        out = {"inds": inds, "weights": w.detach(), "counts": counts}
        if s["grad"]:
            out["dlogits"], = torch.autograd.grad(w, logits, s["dweights"])
        return out
    if op == "quant":
        q, sc = fp8.quantize_fp8_rows(s["x"])
        return {"q": q, "scale": sc}
    if op == "linear":
        if not s["grad"]:
            return {"y": fp8.fp8_linear(s["x"], s["wq"], s["ws"])}
        x = s["x"].detach().requires_grad_(True)
        y = fp8.fp8_linear(x, s["wq"], s["ws"], s["wqt"], s["wst"])
        dx, = torch.autograd.grad(y, x, s["dy"])
        return {"y": y.detach(), "dx": dx}
    return {"y": fp8.fp8_experts(s["x"], s["kq"], s["ks"], s["vq"], s["vs"], s["offsets"])}


def work(case):
    b = DT[case.get("dtype", "float32")].itemsize
    op = case["op"]
    if op == "route":
        n, E, k = case["n"], case["E"], case["k"]
        grad = n * E * b + 4 * n * k if case["grad"] else 0
        return {"bytes": n * E * b + 8 * n * k + 4 * E + grad, "flops": 0}
    if op == "quant":
        n, K = case["n"], case["K"]
        return {"bytes": n * K * (b + 1) + 4 * n * -(-K // BLOCK), "flops": 0}
    if op == "linear":
        n, N, K = case["n"], case["N"], case["K"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (n * (N + K) * b + N * K), "flops": passes * 2 * n * N * K}
    n, E, C, D = case["n"], case["E"], case["C"], case["D"]
    return {"bytes": 2 * n * C * b + 2 * min(n, E) * C * D, "flops": 4 * n * C * D}


# ---------------------------------------------------------------- 64 bits, from the definitions


def _exact_rows(x):
    """Values that the rows stand for after quantisation, their e4m3 values and scales."""
    n, K = x.shape
    v = x.double()
    q, v8, sc = torch.empty_like(v), torch.empty(n, K, device=x.device, dtype=torch.float8_e4m3fn), []
    for k0 in range(0, K, BLOCK):
        part = v[:, k0:k0 + BLOCK]
        top = part.abs().max(dim=1).values.clamp(min=TINY)
        v8[:, k0:k0 + BLOCK] = (part * E4M3_MAX / top[:, None]).to(torch.float8_e4m3fn)
        q[:, k0:k0 + BLOCK] = v8[:, k0:k0 + BLOCK].double() * (top / E4M3_MAX)[:, None]
        sc.append(top / E4M3_MAX)
    return q, v8, torch.stack(sc, 1)


def _exact_weight(wq, ws):
    w = wq.double()
    for i in range(ws.shape[0]):
        for j in range(ws.shape[1]):
            w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= ws[i, j].double()
    return w


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        l = s["logits"].double()
        p = torch.sigmoid(l) if case["score"] == "sigmoid" else torch.softmax(l, -1)
        key = l if s["bias_t"] is None and case["score"] == "softmax" else p
        key = key if s["bias_t"] is None else key + s["bias_t"].double()
        if case["groups"] > 1:
            gk = key.unflatten(1, (case["groups"], -1))
            gs = gk.amax(-1) if case["by"] == "max" else gk.topk(2, -1).values.sum(-1)
            order = torch.argsort(gs, dim=-1, descending=True, stable=True)
            rank = torch.argsort(order, dim=-1)
            key = key.masked_fill((rank >= case["keep"]).repeat_interleave(case["E"] // case["groups"], 1), -math.inf)
        inds = torch.argsort(key, dim=-1, descending=True, stable=True)[:, : case["k"]]
        leaf = l.clone().requires_grad_(True)
        pl = torch.sigmoid(leaf) if case["score"] == "sigmoid" else torch.softmax(leaf, -1)
        w = pl.gather(1, inds)
        if case["renorm"]:
            w = w / w.sum(-1, keepdim=True)
        out = {"inds": None, "weights": w.detach(), "counts": None}
        if case["grad"]:
            out["dlogits"], = torch.autograd.grad(w, leaf, s["dweights"].double())
        return out
    if case["op"] == "quant":
        _, v8, sc = _exact_rows(s["x"])
        return {"q": v8.double(), "scale": sc}
    if case["op"] == "linear":
        out = {"y": _exact_rows(s["x"])[0] @ _exact_weight(s["wq"], s["ws"]).T}
        if case["grad"]:
            out["dx"] = _exact_rows(s["dy"])[0] @ _exact_weight(s["wq"], s["ws"])
        return out
    y = torch.zeros(case["n"], case["C"], device="cuda", dtype=torch.float64)
    offs, x = s["offsets"].tolist(), _exact_rows(s["x"])[0]
    for e in range(case["E"]):
        lo, hi = offs[e], offs[e + 1]
        if hi > lo:
            h = (x[lo:hi] @ _exact_weight(s["kq"][e], s["ks"][e]).T).clamp(min=0) ** 2
            y[lo:hi] = _exact_rows(h)[0] @ _exact_weight(s["vq"][e], s["vs"][e]).T
    return {"y": y}
