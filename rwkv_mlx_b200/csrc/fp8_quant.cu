// e4m3 quantisation: activations with an fp32 scale for each 128 values of a row, weights
// with one for each 128 x 128 block (fp8_common.cuh has the formulas).
//
// Rows: bound by HBM (each value read once, one byte written).  16 lanes hold a block, 8
// values each in one or two 16-byte loads, so the maximum is four shuffles and the values
// stay in registers between the two uses.  A CTA owns 16 rows and walks the blocks of the
// rows; the scales go out as (blocks of K, rows), rows contiguous, which is the order in
// which the product's epilogue (one thread per row) reads them.
#include "fp8_common.cuh"

namespace rwkv {
namespace fp8 {

constexpr int QT = 256, QROWS = QT / 16;

template <typename T>
__global__ void __launch_bounds__(QT)
    quant_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq,
                      float* __restrict__ scale, int M, int K, int kb_per, int vec) {
    const int row = blockIdx.x * QROWS + (threadIdx.x >> 4), l = threadIdx.x & 15;
    const int nkb = (K + BLK - 1) / BLK;
    const int kb0 = blockIdx.y * kb_per, kb1 = min(nkb, kb0 + kb_per);
    const bool on = row < M;
    const T* xr = x + (long long)row * ldx;
    uint8_t* qr = q + (long long)row * ldq;
    constexpr int U = 4;  // blocks in flight
    for (int kb = kb0; kb < kb1; kb += U) {
        float v[U][8];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = (kb + u) * BLK + l * 8;
#pragma unroll
            for (int e = 0; e < 8; e++) v[u][e] = 0.f;
            if (on && kb + u < kb1) {
                if (vec && k + 8 <= K) {
                    load8(xr + k, v[u]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (k + e < K) v[u][e] = to_f32(xr[k + e]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float a = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) a = fmaxf(a, fabsf(v[u][e]));
#pragma unroll
            for (int o = 8; o; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
            a = clamp_amax(a);
            const float mul = quant_mul(a);
            uint2 r;
            r.x = pack4(v[u][0] * mul, v[u][1] * mul, v[u][2] * mul, v[u][3] * mul);
            r.y = pack4(v[u][4] * mul, v[u][5] * mul, v[u][6] * mul, v[u][7] * mul);
            if (on && kb + u < kb1) {
                const int k = (kb + u) * BLK + l * 8;
                if (k + 8 <= K) {
                    *reinterpret_cast<uint2*>(qr + k) = r;
                } else {
                    const uint8_t* b = reinterpret_cast<const uint8_t*>(&r);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (k + e < K) qr[k + e] = b[e];
                }
                if (l == 0) scale[(long long)(kb + u) * M + row] = dequant_scale(a);
            }
        }
    }
}

// One CTA per 128 x 128 block; each thread keeps 64 values (half a row of the block).
template <typename T>
__global__ void __launch_bounds__(256)
    quant_weight_kernel(const T* __restrict__ w, uint8_t* __restrict__ q, long long ldq, float* __restrict__ scale,
                        int N, int K) {
    const int kb = blockIdx.x, nb = blockIdx.y, g = blockIdx.z;
    const int n = nb * BLK + (threadIdx.x >> 1), k0 = kb * BLK + (threadIdx.x & 1) * 64;
    const T* wr = w + ((long long)g * N + n) * K;
    uint8_t* qr = q + ((long long)g * N + n) * ldq;
    float a = 0.f;
    if (n < N)
        for (int e = 0; e < 64; e++)
            if (k0 + e < K) a = fmaxf(a, fabsf(to_f32(wr[k0 + e])));
    __shared__ float part[8];
#pragma unroll
    for (int o = 16; o; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) a = fmaxf(a, part[i]);
    a = clamp_amax(a);
    const float mul = quant_mul(a);
    if (n < N)
        for (int e = 0; e < 64; e += 2) {
            if (k0 + e + 1 < K)
                *reinterpret_cast<uint16_t*>(qr + k0 + e) =
                    (uint16_t)pack2(to_f32(wr[k0 + e]) * mul, to_f32(wr[k0 + e + 1]) * mul);
            else if (k0 + e < K)
                qr[k0 + e] = (uint8_t)pack2(to_f32(wr[k0 + e]) * mul, 0.f);
        }
    if (threadIdx.x == 0) scale[((long long)g * gridDim.y + nb) * gridDim.x + kb] = dequant_scale(a);
}

}  // namespace fp8
}  // namespace rwkv

using namespace rwkv;

extern "C" int rwkv_quantize_fp8_rows(const void* x, long long ldx, void* q, long long ldq, float* scale, int M, int K,
                                      int dtype, void* stream) {
    if (dtype != RWKV_F32 && dtype != RWKV_F16 && dtype != RWKV_BF16) return RWKV_ERR_DTYPE;
    if (M < 0 || K <= 0 || ldx < K || ldq < K) return RWKV_ERR_SHAPE;
    if (M == 0) return RWKV_OK;
    if (!x || !q || !scale) return RWKV_ERR_ARG;
    if (!aligned(q, 8) || ldq % 8) return RWKV_ERR_ALIGN;
    const int es = dtype == RWKV_F32 ? 4 : 2;
    const int vec = aligned(x, 16) && (ldx * es) % 16 == 0;
    const int nkb = (K + fp8::BLK - 1) / fp8::BLK, gx = (M + fp8::QROWS - 1) / fp8::QROWS;
    // few rows: the blocks of a row are spread over CTAs (4 at a time), else one CTA walks them
    const int kb_per = gx >= 1184 ? nkb : 4;
    const dim3 grid(gx, (nkb + kb_per - 1) / kb_per);
    if (grid.y > 65535) return RWKV_ERR_SHAPE;
    RWKV_DISPATCH_DTYPE(dtype, T, {
        fp8::quant_rows_kernel<T><<<grid, fp8::QT, 0, (cudaStream_t)stream>>>((const T*)x, ldx, (uint8_t*)q, ldq, scale,
                                                                             M, K, kb_per, vec);
    });
    return check_launch();
}

extern "C" int rwkv_quantize_fp8_weight(const void* w, void* q, long long ldq, float* scale, int G, int N, int K,
                                        int dtype, void* stream) {
    if (dtype != RWKV_F32 && dtype != RWKV_F16 && dtype != RWKV_BF16) return RWKV_ERR_DTYPE;
    if (G <= 0 || N <= 0 || K <= 0 || ldq < K) return RWKV_ERR_SHAPE;
    if (!w || !q || !scale) return RWKV_ERR_ARG;
    if (!aligned(q, 16) || ldq % 16) return RWKV_ERR_ALIGN;
    const dim3 grid((K + fp8::BLK - 1) / fp8::BLK, (N + fp8::BLK - 1) / fp8::BLK, G);
    if (grid.y > 65535 || grid.z > 65535) return RWKV_ERR_SHAPE;
    RWKV_DISPATCH_DTYPE(dtype, T, {
        fp8::quant_weight_kernel<T>
            <<<grid, 256, 0, (cudaStream_t)stream>>>((const T*)w, (uint8_t*)q, ldq, scale, N, K);
    });
    return check_launch();
}
