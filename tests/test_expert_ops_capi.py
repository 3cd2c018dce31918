"""C entry points of routing and the e4m3 products: argument checks that come before any GPU work, and the
workspace sizes (CPU only)."""

import ctypes

import pytest

OK, SHAPE, DTYPE, ALIGN, ARG, WORKSPACE = 0, 1, 2, 5, 6, 7
N = None


@pytest.fixture(scope="module")
def lib():
    from rwkv_mlx_b200 import _native

    return _native.load()


@pytest.fixture(scope="module")
def p():
    """A host buffer with a 256-byte aligned address: never read, only its alignment is looked at."""
    buf = ctypes.create_string_buffer(1024)
    a = ctypes.addressof(buf)
    return buf, a + (-a) % 256


def route(lib, logits, ld=64, inds=N, weights=N, counts=N, n=4, E=64, k=4, groups=1, keep=1, dtype=0):
    return lib.rwkv_route_experts(logits, ld, N, inds, weights, counts, n, E, k, groups, keep, 0, 0, 1, 1.0, dtype, N)


def test_route_checks(lib, p):
    a = p[1]
    assert route(lib, a, dtype=9) == DTYPE
    for kw in (dict(n=-1), dict(E=0), dict(E=513, ld=513), dict(k=0), dict(k=33), dict(ld=63), dict(groups=7), dict(groups=0),
               dict(groups=64, keep=4), dict(groups=8, keep=9), dict(groups=8, keep=0), dict(groups=16, keep=2, k=9)):
        assert route(lib, a, **kw) == SHAPE, kw
    assert route(lib, N) == ARG and route(lib, a, inds=a) == ARG
    assert route(lib, N, n=0) == OK
    assert lib.rwkv_route_experts_backward(N, 64, N, N, N, N, 4, 64, 65, 0, 1, 1.0, 0, N) == SHAPE
    assert lib.rwkv_route_experts_backward(N, 64, N, N, N, N, 4, 64, 4, 0, 1, 1.0, 3, N) == DTYPE
    assert lib.rwkv_route_experts_backward(N, 64, N, N, N, N, 4, 64, 4, 0, 1, 1.0, 0, N) == ARG
    assert lib.rwkv_route_experts_backward(N, 64, N, N, N, N, 0, 64, 4, 0, 1, 1.0, 0, N) == OK


def test_quantise_checks(lib, p):
    a = p[1]
    q = lib.rwkv_quantize_fp8_rows
    assert q(a, 16, a, 16, a, 2, 16, 7, N) == DTYPE
    assert q(a, 15, a, 16, a, 2, 16, 0, N) == SHAPE and q(a, 16, a, 15, a, 2, 16, 0, N) == SHAPE
    assert q(a, 16, a, 16, a, -1, 16, 0, N) == SHAPE and q(a, 16, a, 16, a, 2, 0, 0, N) == SHAPE
    assert q(N, 16, a, 16, a, 2, 16, 0, N) == ARG and q(a, 16, a, 16, N, 2, 16, 0, N) == ARG
    assert q(a, 16, a + 4, 16, a, 2, 16, 0, N) == ALIGN and q(a, 16, a, 20, a, 2, 16, 0, N) == ALIGN
    assert q(N, 16, N, 16, N, 0, 16, 0, N) == OK
    assert lib.rwkv_quantize_fp8_relu_sq_grad(a, N, 16, a, 16, a, 2, 16, 0, N) == ARG
    w = lib.rwkv_quantize_fp8_weight
    assert w(a, a, 16, a, 1, 4, 16, 9, N) == DTYPE and w(a, a, 16, a, 0, 4, 16, 0, N) == SHAPE
    assert w(N, a, 16, a, 1, 4, 16, 0, N) == ARG and w(a, a, 24, a, 1, 4, 16, 0, N) == ALIGN


def gemm(lib, a, w, lda=32, ldw=32, gs=0, ws=1, offs=N, out=1, ldo=16, os=N, M=4, n=16, K=32, G=1, epi=0, dtype=2, asc=1):
    return lib.rwkv_fp8_gemm(a, lda, a if asc else N, w, ldw, gs, w if ws else N, offs, a if out else N, ldo, os, M, n, K, G,
                             epi, dtype, N)


def test_product_checks(lib, p):
    a = p[1]
    assert gemm(lib, a, a, dtype=5) == DTYPE and gemm(lib, a, a, epi=3) == ARG
    for kw in (dict(M=-1), dict(n=0), dict(K=0), dict(G=257), dict(lda=31), dict(ldw=31), dict(ldo=15), dict(G=2, gs=16)):
        assert gemm(lib, a, a, **kw) == SHAPE, kw
    assert gemm(lib, a, a, G=2, gs=512) == ARG                    # groups without offsets
    assert gemm(lib, N, a) == ARG and gemm(lib, a, N) == ARG and gemm(lib, a, a, out=0) == ARG
    assert gemm(lib, a, a, epi=2) == ARG                          # no place for the output's scales
    assert gemm(lib, a + 8, a) == ALIGN and gemm(lib, a, a + 8) == ALIGN and gemm(lib, a, a, ldw=40) == ALIGN
    assert gemm(lib, N, a, M=0) == OK
    assert lib.rwkv_fp8_set_gemm_impl(4) == ARG and lib.rwkv_fp8_set_gemm_impl(-1) == ARG


def test_linear_and_experts_workspace(lib, p):
    a = p[1]
    size = lib.rwkv_fp8_linear_workspace_size
    assert size(8, 1024) == 0                                     # quantised inside the product
    assert size(9, 1024) >= 9 * 1024 + 9 * 8 * 4 and size(8, 1000) >= 8 * 1008 + 8 * 8 * 4
    assert size(0, 64) == 0 and size(4, 0) == 0
    lin = lib.rwkv_fp8_linear
    assert lin(a, 64, a, 64, a, a, 16, a, 16, 100, 16, 64, 2, N) == WORKSPACE
    assert lin(a, 64, a, 64, a, a, 16, N, 0, 100, 16, 64, 2, N) == ARG
    assert lin(a, 64, a, 64, a, a, 16, a + 8, 1 << 20, 100, 16, 64, 2, N) == ALIGN
    assert lin(a, 63, a, 64, a, a, 16, a, 1 << 20, 100, 16, 64, 2, N) == SHAPE
    assert lin(N, 64, a, 64, a, N, 16, N, 0, 0, 16, 64, 2, N) == OK
    esize = lib.rwkv_fp8_experts_workspace_size
    M, C, D, E = 1000, 256, 512, 4
    assert esize(M, C, D, E) >= M * (C + D) + 4 * M * (C + D) // 128
    assert esize(4, C, D, E) >= 4 * D * 4 and esize(0, C, D, E) == 0
    ex = lib.rwkv_fp8_experts
    args = lambda ws, n, m=M, e=E: (a, C, a, C, D * C, a, a, D, D * C, a, a, a, C, ws, n, m, C, D, e, 2, N)  # noqa: E731
    assert ex(*args(a, 16)) == WORKSPACE and ex(*args(N, 0)) == ARG and ex(*args(a, 16, m=0)) == OK
    assert ex(*args(a, 16, e=300)) == SHAPE
