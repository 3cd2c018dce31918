// e4m3 products for few rows, and the entry point of all e4m3 products:
//
//   out[m, n] = epi( sum_kb as[kb, m] ws[g, n / 128, kb] sum_{k in block kb} a[m, k] w[g, n, k] )
//
// over the rows m in [offs[g], offs[g + 1]) of group g.  With few rows the product is bound
// by reading the weights once, so this kernel streams them: a CTA owns 16 rows of W, its 8
// warps take the 128-blocks of K in turn, and every lane reads 16 consecutive bytes of a
// weight row at a time straight into the operand registers of mma.sync m16n8k32 (weights as
// the 16-row operand, tokens as the 8-column one).  The order of K inside a 64-byte piece
// is the same permutation for both operands, so no shuffle is needed.  A block's partial
// sums are scaled in fp32, the warps' sums meet in shared memory in a fixed order.
#include "fp8_gemm.cuh"

namespace rwkv {
namespace fp8 {

constexpr int SNT = 256, SNW = SNT / 32, SROWS = 16;

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 bytes of a row from k on; bytes past K are 0 (never read).
__device__ __forceinline__ uint4 load16(const uint8_t* row, int k, int K, bool on) {
    uint4 r = make_uint4(0u, 0u, 0u, 0u);
    if (!on || k >= K) return r;
    if (k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
    uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (k + i < K) v[i >> 2] |= (uint32_t)row[k + i] << (8 * (i & 3));
    return make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename TO, int NT8, bool RELU2>
__global__ void __launch_bounds__(SNT) gemm_stream_kernel(const GemmArgs p) {
    constexpr int TP = 8 * NT8;
    __shared__ float red[SNW][SROWS][TP + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t = lane & 3;
    const int g = blockIdx.y, n0 = blockIdx.x * SROWS;
    const int r0 = p.offs ? max(p.offs[g], 0) : 0, r1 = p.offs ? min(p.offs[g + 1], p.M) : p.M;
    const int nkb = (p.K + BLK - 1) / BLK;
    const float* wsb = p.ws + ((long long)g * ((p.N + BLK - 1) / BLK) + n0 / BLK) * nkb;
    const uint8_t* w0 = p.w + (long long)g * p.gsw + (long long)(n0 + gr) * p.ldw;
    const uint8_t* w1 = w0 + 8 * p.ldw;
    const bool on0 = n0 + gr < p.N, on1 = n0 + gr + 8 < p.N;
    for (int m0 = r0; m0 < r1; m0 += TP) {
        float acc[NT8][4];
#pragma unroll
        for (int j = 0; j < NT8; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) acc[j][c] = 0.f;
        for (int kb = warp; kb < nkb; kb += SNW) {
            const float sb = wsb[kb];
            float part[NT8][4];
#pragma unroll
            for (int j = 0; j < NT8; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) part[j][c] = 0.f;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int k = kb * BLK + h * 64 + t * 16;
                const uint4 a0 = load16(w0, k, p.K, on0), a1 = load16(w1, k, p.K, on1);
#pragma unroll
                for (int j = 0; j < NT8; j++) {
                    const int m = m0 + 8 * j + gr;
                    const uint4 b = load16(p.a + (long long)m * p.lda, k, p.K, m < r1);
                    mma_e4m3(part[j], a0.x, a1.x, a0.y, a1.y, b.x, b.y);
                    mma_e4m3(part[j], a0.z, a1.z, a0.w, a1.w, b.z, b.w);
                }
            }
#pragma unroll
            for (int j = 0; j < NT8; j++) {
                const int m = m0 + 8 * j + 2 * t;
                const float s0 = m < r1 ? p.as[(long long)kb * p.M + m] * sb : 0.f;
                const float s1 = m + 1 < r1 ? p.as[(long long)kb * p.M + m + 1] * sb : 0.f;
                acc[j][0] += part[j][0] * s0, acc[j][1] += part[j][1] * s1;
                acc[j][2] += part[j][2] * s0, acc[j][3] += part[j][3] * s1;
            }
        }
#pragma unroll
        for (int j = 0; j < NT8; j++) {
            red[warp][gr][8 * j + 2 * t] = acc[j][0], red[warp][gr][8 * j + 2 * t + 1] = acc[j][1];
            red[warp][gr + 8][8 * j + 2 * t] = acc[j][2], red[warp][gr + 8][8 * j + 2 * t + 1] = acc[j][3];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < SROWS * TP; i += SNT) {
            const int m = m0 + i / SROWS, n = i % SROWS;
            if (m < r1 && n0 + n < p.N) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < SNW; w++) v += red[w][n][i / SROWS];
                if (RELU2) v = relu_sq(v);
                reinterpret_cast<TO*>(p.out)[(long long)m * p.ldo + n0 + n] = from_f32<TO>(v);
            }
        }
        __syncthreads();
    }
}

template <typename TO, bool RELU2>
static int stream_launch(const GemmArgs& p, cudaStream_t st) {
    const dim3 grid((p.N + SROWS - 1) / SROWS, p.G);
    // 8 tokens a pass when a group has at most about that many rows, else 32
    if ((long long)p.M <= 8LL * p.G) gemm_stream_kernel<TO, 1, RELU2><<<grid, SNT, 0, st>>>(p);
    else gemm_stream_kernel<TO, 4, RELU2><<<grid, SNT, 0, st>>>(p);
    return check_launch();
}

int gemm_stream(const GemmArgs& p, int epi, int out_dtype, cudaStream_t st) {
    if (epi == RELU2_Q) return RWKV_ERR_ARG;
    RWKV_DISPATCH_DTYPE(out_dtype, TO, {
        return epi == RELU2 ? stream_launch<TO, true>(p, st) : stream_launch<TO, false>(p, st);
    });
    return RWKV_ERR_DTYPE;
}

static int g_gemm_impl = 0;

// Few rows: the weights are read once for every 32 rows of a group at most, and 16-row tiles of
// W keep the SMs busy where 128 x 128 output tiles would not.  Measured, us, this kernel / tcgen05:
// N = 4096, K = 1024, M = 16 4.7 / 6.2, 32 5.5 / 6.5, 64 9.3 / 6.6; 64 groups of N = 2048, K = 1024,
// one row a group 19.3 / 19.4, four 35 / 32.
static bool prefers_stream(int M, int G) { return M <= 32 || (G > 1 && M <= 2LL * G); }

}  // namespace fp8
}  // namespace rwkv

using namespace rwkv;

namespace {

using fp8::GemmArgs;

size_t align256(size_t n) { return (n + 255) / 256 * 256; }
long long pitch16(long long k) { return (k + 15) / 16 * 16; }
size_t rows_bytes(int M, int K) { return align256((size_t)M * pitch16(K)); }
size_t scale_bytes(int M, int K) { return align256((size_t)M * ((K + fp8::BLK - 1) / fp8::BLK) * sizeof(float)); }

int check_weight(const void* w, long long ldw, long long gs, const float* ws, int G, int N, int K) {
    if (N <= 0 || K <= 0 || G <= 0 || G > 256) return RWKV_ERR_SHAPE;
    if (ldw < K || (G > 1 && gs < (long long)(N - 1) * ldw + K)) return RWKV_ERR_SHAPE;
    if (!w || !ws) return RWKV_ERR_ARG;
    if (!aligned(w, 16) || ldw % 16 || (G > 1 && gs % 16)) return RWKV_ERR_ALIGN;
    return RWKV_OK;
}
bool known(int dtype) { return dtype == RWKV_F32 || dtype == RWKV_F16 || dtype == RWKV_BF16; }

int gemm(const GemmArgs& p, int epi, int out_dtype, cudaStream_t st) {
    const bool few = epi != fp8::RELU2_Q && (fp8::g_gemm_impl ? fp8::g_gemm_impl == 1 : fp8::prefers_stream(p.M, p.G));
    return few ? fp8::gemm_stream(p, epi, out_dtype, st) : fp8::gemm_tc(p, epi, out_dtype, fp8::g_gemm_impl == 1 ? 0 : fp8::g_gemm_impl, st);
}

}  // namespace

extern "C" int rwkv_fp8_gemm(const void* a, long long lda, const float* a_scale, const void* w, long long ldw,
                             long long w_group_stride, const float* w_scale, const int32_t* offs, void* out,
                             long long ldo, float* out_scale, int M, int N, int K, int G, int epi, int out_dtype,
                             void* stream) {
    if (epi != fp8::STORE && epi != fp8::RELU2 && epi != fp8::RELU2_Q) return RWKV_ERR_ARG;
    if (epi != fp8::RELU2_Q && !known(out_dtype)) return RWKV_ERR_DTYPE;
    if (M < 0 || lda < K || ldo < N) return RWKV_ERR_SHAPE;
    const int rc = check_weight(w, ldw, w_group_stride, w_scale, G, N, K);
    if (rc) return rc;
    if (G > 1 && !offs) return RWKV_ERR_ARG;
    if (M == 0) return RWKV_OK;
    if (!a || !a_scale || !out || (epi == fp8::RELU2_Q && !out_scale)) return RWKV_ERR_ARG;
    if (!aligned(a, 16) || lda % 16) return RWKV_ERR_ALIGN;
    return gemm({(const uint8_t*)a, lda, a_scale, (const uint8_t*)w, ldw, w_group_stride, w_scale, offs, out, ldo,
                 out_scale, M, N, K, G},
                epi, out_dtype, (cudaStream_t)stream);
}

extern "C" size_t rwkv_fp8_linear_workspace_size(int M, int K) {
    return M <= 0 || K <= 0 ? 0 : rows_bytes(M, K) + scale_bytes(M, K);
}

extern "C" int rwkv_fp8_linear(const void* x, long long ldx, const void* w, long long ldw, const float* w_scale,
                               void* out, long long ldo, void* workspace, size_t workspace_bytes, int M, int N, int K,
                               int dtype, void* stream) {
    if (!known(dtype)) return RWKV_ERR_DTYPE;
    if (M < 0 || ldx < K || ldo < N) return RWKV_ERR_SHAPE;
    int rc = check_weight(w, ldw, 0, w_scale, 1, N, K);
    if (rc) return rc;
    if (M == 0) return RWKV_OK;
    if (!x || !out || !workspace) return RWKV_ERR_ARG;
    if (!aligned(workspace, 256)) return RWKV_ERR_ALIGN;
    if (workspace_bytes < rwkv_fp8_linear_workspace_size(M, K)) return RWKV_ERR_WORKSPACE;
    uint8_t* q = (uint8_t*)workspace;
    float* qs = (float*)(q + rows_bytes(M, K));
    rc = rwkv_quantize_fp8_rows(x, ldx, q, pitch16(K), qs, M, K, dtype, stream);
    if (rc) return rc;
    return gemm({q, pitch16(K), qs, (const uint8_t*)w, ldw, 0, w_scale, nullptr, out, ldo, nullptr, M, N, K, 1},
                fp8::STORE, dtype, (cudaStream_t)stream);
}

extern "C" size_t rwkv_fp8_experts_workspace_size(int M, int C, int D, int E) {
    if (M <= 0 || C <= 0 || D <= 0 || E <= 0) return 0;
    const size_t h = fp8::prefers_stream(M, E) || fp8::g_gemm_impl == 1 ? align256((size_t)M * D * sizeof(float)) : 0;
    return rows_bytes(M, C) + scale_bytes(M, C) + rows_bytes(M, D) + scale_bytes(M, D) + h;
}

extern "C" int rwkv_fp8_experts(const void* x, long long ldx, const void* key, long long ldk, long long key_gs,
                                const float* key_scale, const void* val, long long ldv, long long val_gs,
                                const float* val_scale, const int32_t* offs, void* out, long long ldo, void* workspace,
                                size_t workspace_bytes, int M, int C, int D, int E, int dtype, void* stream) {
    if (!known(dtype)) return RWKV_ERR_DTYPE;
    if (M < 0 || ldx < C || ldo < C) return RWKV_ERR_SHAPE;
    int rc = check_weight(key, ldk, key_gs, key_scale, E, D, C);
    if (!rc) rc = check_weight(val, ldv, val_gs, val_scale, E, C, D);
    if (rc) return rc;
    if (E > 1 && !offs) return RWKV_ERR_ARG;
    if (M == 0) return RWKV_OK;
    if (!x || !out || !workspace) return RWKV_ERR_ARG;
    if (!aligned(workspace, 256)) return RWKV_ERR_ALIGN;
    if (workspace_bytes < rwkv_fp8_experts_workspace_size(M, C, D, E)) return RWKV_ERR_WORKSPACE;
    uint8_t* at = (uint8_t*)workspace;
    auto take = [&](size_t n) { return at += n, at - n; };
    uint8_t* q = take(rows_bytes(M, C));
    float* qs = (float*)take(scale_bytes(M, C));
    uint8_t* hq = take(rows_bytes(M, D));
    float* hs = (float*)take(scale_bytes(M, D));
    cudaStream_t st = (cudaStream_t)stream;
    const bool few = fp8::g_gemm_impl ? fp8::g_gemm_impl == 1 : fp8::prefers_stream(M, E);
    rc = rwkv_quantize_fp8_rows(x, ldx, q, pitch16(C), qs, M, C, dtype, stream);
    if (rc) return rc;
    GemmArgs p{q, pitch16(C), qs, (const uint8_t*)key, ldk, key_gs, key_scale, offs, hq, pitch16(D), hs, M, D, C, E};
    if (few) {  // 16 columns a CTA: a block's maximum is not in one place, so the hidden rows pass through fp32
        p.out = at, p.ldo = D, p.os = nullptr;
        rc = gemm(p, fp8::RELU2, RWKV_F32, st);
        if (!rc) rc = rwkv_quantize_fp8_rows(at, D, hq, pitch16(D), hs, M, D, RWKV_F32, stream);
    } else {
        rc = gemm(p, fp8::RELU2_Q, dtype, st);
    }
    if (rc) return rc;
    return gemm({hq, pitch16(D), hs, (const uint8_t*)val, ldv, val_gs, val_scale, offs, out, ldo, nullptr, M, C, D, E},
                fp8::STORE, dtype, st);
}

extern "C" int rwkv_fp8_set_gemm_impl(int impl) {
    if (impl < 0 || impl > 3) return RWKV_ERR_ARG;
    fp8::g_gemm_impl = impl;
    return RWKV_OK;
}
