// Arguments of the e4m3 products (fp8_gemm.cu: few rows, fp8_gemm_tc.cu: tcgen05).
#pragma once
#include "fp8_common.cuh"

namespace rwkv {
namespace fp8 {

enum Epi { STORE = 0, RELU2 = 1, RELU2_Q = 2 };

struct GemmArgs {
    const uint8_t* a;   // (M, K), row pitch lda
    long long lda;
    const float* as;    // (ceil(K / 128), M)
    const uint8_t* w;   // (G, N, K), row pitch ldw, group pitch gsw
    long long ldw, gsw;
    const float* ws;    // (G, ceil(N / 128), ceil(K / 128))
    const int32_t* offs;
    void* out;          // (M, N), row pitch ldo (elements of the output type)
    long long ldo;
    float* os;          // RELU2_Q: (ceil(N / 128), M) scales of the output rows
    int M, N, K, G;
    const void* x = nullptr;  // gemm_stream: rows of the output's type, still to be quantised, instead of a and as
    long long ldx = 0;
};

// gemm_stream quantises x itself (in every CTA) for at most this many rows and K up to SELF_K, a
// multiple of 16.
constexpr int SELF_ROWS = 8, SELF_K = 8192;

int gemm_stream(const GemmArgs& p, int epi, int out_dtype, cudaStream_t st);
int gemm_tc(const GemmArgs& p, int epi, int out_dtype, int impl, cudaStream_t st);

}  // namespace fp8
}  // namespace rwkv
