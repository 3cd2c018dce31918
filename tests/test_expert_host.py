"""The host module of the expert-layer operators: what it refuses without a GPU, and on the GPU its
errors from backward passes, its launch count, its stream and its calls from several threads."""

import threading

import pytest
import torch

from rwkv_mlx_b200 import _native, fp8, route

DEV = "cuda"


def test_bad_arguments_raise_before_the_device_is_needed():
    x = torch.zeros(4, 16)
    for kw in ({"top_k": 17}, {"top_k": 0}, {"top_k": 2, "n_groups": 3}, {"top_k": 2, "n_groups": 0}, {"top_k": 2, "score": "tanh"},
               {"top_k": 2, "group_score": "sum"}, {"top_k": 2, "bias": torch.zeros(15)}, {"top_k": 5, "n_groups": 4}):
        with pytest.raises(ValueError, match="route_experts: "):
            route.route_experts(x, **kw)
    with pytest.raises(ValueError, match="1 to 512 experts, not 513"):
        route.route_experts(torch.zeros(2, 513), 2)
    with pytest.raises(ValueError, match="logits must be"):
        route.route_experts(torch.tensor(1.0), 1)
    with pytest.raises(ValueError, match="K >= 1"):
        fp8.quantize_fp8_rows(torch.zeros(4, 0))
    with pytest.raises(ValueError, match=r"x \[4, 16\] and w \[8, 32\] do not fit"):
        fp8.fp8_linear(x, torch.zeros(8, 32), torch.zeros(1, 1))
    with pytest.raises(ValueError, match="do not fit"):
        fp8.fp8_experts(x, torch.zeros(2, 8, 15), x, x, x, x)
    for call in (lambda: route.route_experts(x.double(), 2), lambda: fp8.quantize_fp8_rows(x.double()),
                 lambda: fp8.fp8_linear(x.double(), torch.zeros(8, 16), torch.zeros(1, 1))):
        with pytest.raises(_native.RwkvNativeError, match="unsupported dtype"):
            call()


def test_cpu_tensors_are_refused():
    """ValueError beside a GPU, RwkvNativeError without one: never a result from elsewhere."""
    x = torch.zeros(4, 16)
    for call in (lambda: route.route_experts(x, 2), lambda: fp8.quantize_fp8_rows(x),
                 lambda: fp8.fp8_linear(x, torch.zeros(8, 16), torch.zeros(1, 1))):
        with pytest.raises((ValueError, _native.RwkvNativeError), match="CUDA device"):
            call()


@pytest.mark.gpu
def test_launch_count_includes_both_sides():
    x = torch.randn(3, 256, device=DEV)
    w, s = fp8.quantize_fp8_weight(torch.randn(128, 256, device=DEV))
    n0 = _native.launch_count
    route.route_experts(x, 2)
    fp8.fp8_matmul(*fp8.quantize_fp8_rows(x), w, s)
    assert _native.launch_count - n0 == 3
    with pytest.raises(AttributeError):
        _native.no_such_name


@pytest.mark.gpu
def test_runs_on_the_callers_stream():
    side = torch.cuda.Stream()
    x = torch.randn(64, 128, device=DEV)
    want = route.route_experts(x * 2, 4)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)  # a call on another stream would read y before it is written
        y = x * 2
        got = route.route_experts(y, 4)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_gradients_from_several_threads():
    logits = torch.randn(33, 64, device=DEV)
    dw = torch.randn(33, 4, device=DEV)

    def grad():
        z = logits.clone().requires_grad_()
        route.route_experts(z, 4)[1].backward(dw)
        return z.grad

    want, got = grad(), [None] * 4
    torch.cuda.synchronize()

    def work(i):
        for _ in range(25):
            got[i] = grad()
        torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.gpu
def test_no_gradient_asked_for_the_weights():
    """Only the indices and counts used: the logits get no gradient, and nothing fails."""
    z = torch.randn(5, 16, device=DEV, requires_grad=True)
    inds, weights, counts = route.route_experts(z, 2, return_counts=True)
    assert not inds.requires_grad and not counts.requires_grad and weights.requires_grad
    (z.sum() + weights.detach().sum()).backward()
    assert torch.equal(z.grad, torch.ones_like(z))


@pytest.mark.gpu
def test_gradient_of_a_gradient_raises():
    z = torch.randn(5, 16, device=DEV, requires_grad=True)
    w = route.route_experts(z, 2)[1]
    (g,) = torch.autograd.grad(w.square().sum(), z, create_graph=True)
    with pytest.raises(RuntimeError, match="only once"):
        g.sum().backward()
