"""Routing to experts from logits (csrc/route.cu) against the definition in float64.

Indices: where keys are logits (softmax without a bias, largest-key groups) the comparison is
exact.  Where keys are computed scores, fp32 keys carry an error below 4e-7 (a few roundings of values
up to 2), so the chosen experts' float64 keys, in order, must match the reference's within 2e-6, and
tokens whose float64 keys are all further apart than that must match exactly.
Weights: expf within 2 ulp, a sum of at most 32 terms and a division: 5e-6 relative.
Gradients in fp32: three more products of such terms, 2e-5 relative to the row's largest entry; 16-bit
logits add one rounding (2^-11 / 2^-8).
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(l, k, score, bias, groups, keep, by, renorm, scale):
    """(keys with excluded experts at nan, order-defining keys, weights, p) in float64; l (n, E) float64."""
    n, E = l.shape
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            p = 1.0 / (1.0 + np.exp(-l))
    else:
        m = l.max(1, keepdims=True)
        e = np.exp(l - np.where(np.isfinite(m), m, 0.0))
        z = e.sum(1, keepdims=True)
        p = np.where(z == 0, 0.0, e / np.where(z == 0, 1.0, z))
    key = p if bias is None else p + bias
    if score == "softmax" and bias is None and not (groups > 1 and by == "top2"):
        key = l
    key = key.copy()
    if groups > 1:
        kg = -np.sort(-key.reshape(n, groups, -1), axis=2)
        gs = kg[:, :, 0] if by == "max" or kg.shape[2] == 1 else kg[:, :, 0] + kg[:, :, 1]
        order = np.argsort(-gs, axis=1, kind="stable")
        stay = np.zeros((n, groups), bool)
        np.put_along_axis(stay, order[:, :keep], True, 1)
        out = ~np.repeat(stay, E // groups, axis=1)
    else:
        gs, out = np.zeros((n, 1)), np.zeros((n, E), bool)
    rank = np.where(out, np.inf, -key)
    inds = np.argsort(rank, axis=1, kind="stable")[:, :k]
    return key, gs, inds, p


def weights_of(p, inds, renorm, scale):
    s = np.take_along_axis(p, inds, 1)
    t = s.sum(1, keepdims=True)
    return scale * (np.where(t == 0, 0.0, s / np.where(t == 0, 1.0, t)) if renorm else s)


def separated(v, keep, tol):
    """Rows of v whose first keep + 1 largest values are all further apart than tol."""
    s = -np.sort(-v, axis=1)[:, : keep + 1]
    return (np.abs(np.diff(s, axis=1)) > tol).all(1)


CASES = [
    # n, E, k, score, bias, groups, keep, by, renorm, scale
    (1, 64, 6, "softmax", False, 8, 3, "max", False, 16.0),
    (257, 256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5),
    (300, 96, 4, "softmax", False, 1, 1, "max", True, 1.0),
    (33, 81, 8, "sigmoid", True, 1, 1, "max", False, 1.0),
    (65, 512, 32, "sigmoid", False, 32, 9, "top2", True, 1.0),
    (40, 60, 5, "sigmoid", True, 4, 2, "top2", True, 1.0),       # groups of 15: not whole lanes
    (40, 48, 3, "softmax", False, 6, 2, "max", True, 1.0),       # groups of 8 over 2 logits a lane
    (17, 8, 8, "softmax", True, 1, 1, "max", False, 1.0),        # every expert chosen
    (9, 1, 1, "sigmoid", False, 1, 1, "max", True, 1.0),
    (50, 32, 2, "softmax", False, 32, 5, "top2", True, 1.0),     # groups of one expert
    (128, 160, 6, "softmax", False, 8, 3, "max", False, 1.0),    # 160 = 20 lanes of 8, groups of 20
]


def run(l, k, score, bias, groups, keep, by, renorm, scale, **kw):
    from rwkv_mlx_b200.route import route_experts

    return route_experts(l, k, score=score, bias=bias, n_groups=groups, topk_groups=keep, group_score=by,
                         renormalize=renorm, scale=scale, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
def test_forward_matches_the_definition(case, dtype):
    n, E, k, score, bias, groups, keep, by, renorm, scale = case
    g = torch.Generator(device="cuda").manual_seed(n + E)
    l = (torch.randn(n, E, device="cuda", generator=g) * 2).to(dtype)
    b = torch.randn(E, device="cuda", generator=g) * 0.1 if bias else None
    inds, w, counts = run(l, k, score, b, groups, keep, by, renorm, scale, return_counts=True)
    torch.cuda.synchronize()
    assert inds.dtype == torch.int32 and w.dtype == torch.float32 and counts.dtype == torch.int32
    ln, bn = l.double().cpu().numpy(), None if b is None else b.double().cpu().numpy()
    key, gs, ref, p = reference(ln, k, score, bn, groups, keep, by, renorm, scale)
    got = inds.cpu().numpy().astype(np.int64)
    assert all(len(set(r)) == k for r in got) and got.min() >= 0 and got.max() < E
    exact_keys = score == "softmax" and b is None and not (groups > 1 and by == "top2")
    if exact_keys:
        np.testing.assert_array_equal(got, ref)
    else:
        clear = separated(key, E - 1, 2e-6) & separated(gs, groups - 1, 4e-6)
        clear |= (ln[:, :1] == ln).all(1)
        np.testing.assert_array_equal(got[clear], ref[clear])
        # ties in the logits (16-bit types have many) resolve exactly when the bias is absent
        same = np.sort(np.take_along_axis(key, got, 1), 1) - np.sort(np.take_along_axis(key, ref, 1), 1)
        assert (np.abs(same[separated(gs, groups - 1, 4e-6)]) < 2e-6).all()
    np.testing.assert_allclose(w.cpu().numpy(), weights_of(p, got, renorm, scale), rtol=5e-6, atol=1e-30)
    np.testing.assert_array_equal(counts.cpu().numpy(), np.bincount(got.reshape(-1), minlength=E))


def test_ties_go_to_the_lower_index():
    """Equal logits have equal keys, so every choice is decided by the index."""
    for E, groups, keep, k in ((64, 8, 3, 12), (60, 4, 2, 9), (256, 1, 1, 8)):
        l = torch.zeros(5, E, device="cuda")
        for score, by in (("softmax", "max"), ("sigmoid", "top2")):
            inds, w = run(l, k, score, None, groups, keep, by, True, 1.0)
            assert (inds.cpu() == torch.arange(k, dtype=torch.int32)).all()
            torch.testing.assert_close(w.cpu(), torch.full((5, k), 1.0 / k))


def test_few_distinct_logits():
    """Integer logits: long runs of exact ties between and inside groups."""
    g = torch.Generator(device="cuda").manual_seed(3)
    l = torch.randint(-2, 3, (200, 128), device="cuda", generator=g).float()
    for score, groups, keep, by in (("sigmoid", 8, 3, "max"), ("softmax", 4, 2, "max"), ("sigmoid", 16, 5, "top2"),
                                    ("sigmoid", 1, 1, "max")):
        inds, _ = run(l, 7, score, None, groups, keep, by, True, 1.0)
        # equal logits give equal fp32 keys and equal float64 keys, distinct ones keep their order
        _, _, ref, _ = reference(l.double().cpu().numpy(), 7, score, None, groups, keep, by, True, 1.0)
        np.testing.assert_array_equal(inds.cpu().numpy(), ref)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep,by", [(1, 1, "max"), (4, 2, "max"), (4, 2, "top2")])
def test_masked_saturated_and_nan_logits(score, groups, keep, by):
    inf, nan = math.inf, math.nan
    E, k = 64, 4
    l = torch.randn(6, E, device="cuda")
    l[0] = -inf                          # nothing to choose from
    l[1] = -inf
    l[1, 37] = 0.5                       # one expert left
    l[2] = torch.finfo(torch.float32).min
    l[3, ::2], l[3, 1::2] = 300.0, -300.0  # scores of exactly 1 and 0 or less than fp32 has
    l[4, 9] = nan
    inds, w, counts = run(l, k, score, None, groups, keep, by, True, 1.0, return_counts=True)
    i, w = inds.cpu(), w.cpu()
    for r in range(6):
        assert len(set(i[r].tolist())) == k and 0 <= int(i[r].min()) and int(i[r].max()) < E
    assert (w[0] == 0).all()
    assert i[1, 0] == 37 and w[1, 0] == 1 and (w[1, 1:] == 0).all()
    if score == "softmax":
        assert torch.allclose(w[2], torch.full((k,), 0.25)) and (i[2] == torch.arange(k)).all()
    else:
        assert (w[2] == 0).all()         # sigmoid of the lowest value is 0
    assert (i[3] % 2 == 0).all() and torch.allclose(w[3], torch.full((k,), 0.25))
    # (softmax scores of that row are all NaN, so top2 groups choose by index there)
    assert 9 in i[4].tolist() or (score == "softmax" and by == "top2")
    assert torch.isnan(w[4]).any()
    assert torch.isfinite(w[5]).all() and abs(float(w[5].sum()) - 1) < 1e-6
    assert int(counts.sum()) == 6 * k


def test_strided_offset_leading_dims_empty_and_streams():
    g = torch.Generator(device="cuda").manual_seed(1)
    big = torch.randn(40, 131, device="cuda", generator=g)
    view = big[3:33, 1:97]               # row pitch 131, base off the 16-byte grid
    for kw in (dict(score="softmax"), dict(score="sigmoid")):
        from rwkv_mlx_b200.route import route_experts

        a, b = route_experts(view, 5, **kw), route_experts(view.contiguous(), 5, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        t = route_experts(view.contiguous().view(5, 6, 96), 5, **kw)
        assert t[0].shape == (5, 6, 5) and torch.equal(t[0].view(30, 5), b[0])
        tr = route_experts(big[:33, :40].t(), 3, **kw)       # columns contiguous: copied
        tb = route_experts(big[:33, :40].t().contiguous(), 3, **kw)
        assert torch.equal(tr[0], tb[0]) and torch.equal(tr[1], tb[1])
        e = route_experts(view[:0], 5, return_counts=True, **kw)
        assert e[0].shape == (0, 5) and (e[2] == 0).all()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            c = route_experts(view, 5, return_counts=True, **kw)
        s.synchronize()
        assert torch.equal(c[0], a[0]) and torch.equal(c[1], a[1])


GRAD = [c for c in CASES if not (c[2] == 1 and c[8])]


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.float16, 2.0 ** -11 + 2e-5),
                                       (torch.bfloat16, 2.0 ** -8 + 2e-5)])
@pytest.mark.parametrize("case", GRAD)
def test_gradient_matches_the_formula(case, dtype, tol):
    n, E, k, score, bias, groups, keep, by, renorm, scale = case
    g = torch.Generator(device="cuda").manual_seed(n * E)
    l = (torch.randn(n, E, device="cuda", generator=g) * 2).to(dtype).requires_grad_(True)
    b = torch.randn(E, device="cuda", generator=g) * 0.1 if bias else None
    inds, w = run(l, k, score, b, groups, keep, by, renorm, scale)
    dw = torch.randn(n, k, device="cuda", generator=g)
    (got,) = torch.autograd.grad(w, l, dw)
    assert got.dtype == dtype and got.shape == l.shape
    leaf = l.detach().double().requires_grad_(True)
    p = torch.sigmoid(leaf) if score == "sigmoid" else torch.softmax(leaf, -1)
    s = p.gather(1, inds.long())
    (ref,) = torch.autograd.grad(scale * (s / s.sum(1, keepdim=True) if renorm else s), leaf, dw.double())
    err = (got.double() - ref).abs()
    # renormalised: t_j = w_j (g_j - sum g w): relative to the terms, not to their difference
    terms = scale * dw.double().abs().amax(1, keepdim=True)
    assert (err <= tol * ref.abs() + 2e-5 * terms * p.detach().amax(1, keepdim=True).clamp(min=1e-3)
            + (2.0 ** -24 if dtype == torch.float16 else 0)).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_matches_differences(score, renorm):
    """Central differences of the float64 weights at the kernel's selection: step 1e-5, so an error of
    about 1e-10, far below the kernel's 1e-6."""
    n, E, k = 5, 24, 4
    g = torch.Generator(device="cuda").manual_seed(8)
    l = torch.randn(n, E, device="cuda", generator=g).requires_grad_(True)
    inds, w = run(l, k, score, None, 4, 2, "max", renorm, 1.5)
    dw = torch.randn(n, k, device="cuda", generator=g)
    (got,) = torch.autograd.grad(w, l, dw)
    ln, iv, dn = l.detach().double().cpu().numpy(), inds.cpu().numpy().astype(np.int64), dw.double().cpu().numpy()

    def loss(x):
        _, _, _, p = reference(x, k, score, None, 1, 1, "max", renorm, 1.5)
        return (weights_of(p, iv, renorm, 1.5) * dn).sum(1)

    h = 1e-5
    for e in range(E):
        step = np.zeros_like(ln)
        step[:, e] = h
        d = (loss(ln + step) - loss(ln - step)) / (2 * h)
        np.testing.assert_allclose(got[:, e].cpu().numpy(), d, atol=5e-6, rtol=2e-5)


def test_gradient_of_rows_without_scores_is_zero():
    l = torch.randn(3, 32, device="cuda")
    l[1] = -math.inf
    l.requires_grad_(True)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            _, w = run(l, 4, score, None, 1, 1, "max", renorm, 1.0)
            (d,) = torch.autograd.grad(w, l, torch.ones_like(w))
            assert torch.isfinite(d).all() and (d[1] == 0).all()


def test_refusals():
    from rwkv_mlx_b200 import RwkvNativeError
    from rwkv_mlx_b200.route import route_experts

    l = torch.zeros(4, 64, device="cuda")
    for kw in (dict(top_k=0), dict(top_k=33), dict(top_k=17, n_groups=8, topk_groups=2), dict(top_k=2, n_groups=7),
               dict(top_k=2, n_groups=8, topk_groups=9), dict(top_k=2, score="tanh"), dict(top_k=2, group_score="mean"),
               dict(top_k=2, n_groups=64, topk_groups=4), dict(top_k=2, bias=torch.zeros(63, device="cuda")),
               dict(top_k=2, bias=torch.zeros(64))):
        with pytest.raises(ValueError):
            route_experts(l, **kw)
    with pytest.raises(ValueError):
        route_experts(torch.zeros(4, 513, device="cuda"), 2)
    with pytest.raises(RwkvNativeError):
        route_experts(l.double(), 2)
    with pytest.raises(ValueError):
        route_experts(l.cpu(), 2)


def test_balance_bias_evens_the_load():
    """A skewed router: updating the bias from the counts brings the largest load down."""
    from rwkv_mlx_b200.moe import GroupRouter

    torch.manual_seed(0)
    r = GroupRouter(64, 32, 4, n_groups=4, topk_groups=2).cuda()
    with torch.no_grad():
        r.gate.weight[:4] *= 4
    x = torch.randn(4096, 64, device="cuda")
    loads = []
    for _ in range(150):
        with torch.no_grad():
            _, w, counts = r(x)
        assert int(counts.sum()) == 4096 * 4
        loads.append(int(counts.max()))
        r.update_balance(counts, 5e-3)
    assert loads[-1] < 0.6 * loads[0]
    y = r(x)[1].square().sum()
    y.backward()
    assert torch.isfinite(r.gate.weight.grad).all() and r.gate.weight.grad.abs().sum() > 0
