// Shared by the tcgen05 e4m3 products (fp8_gemm_tc.cu: one CTA a tile, fp8_gemm_pair.cuh: a
// CTA pair a tile; both are one translation unit with one device error word): sizes, the group
// table, packed adds and output packing.
#pragma once
#include "fp8_gemm.cuh"
#include "tma_common.cuh"
#include "wkv7.cuh"

namespace rwkv {

__device__ int g_device_error_fp8;
// Test hook (rwkv_debug_force_wait_timeout): every bounded wait gives up at once.
static __constant__ int c_force_wait_timeout_fp8;

namespace fp8 {
using namespace tcc;
using namespace tma;

constexpr int BM = 128, NDRAIN = 256, NTH = NDRAIN + 128, MAXG = 256;
// A pair kernel's drain thread keeps 128 sums and 32 loaded values, more than the 168 registers that
// 384 threads can have: the drain warpgroups take them from the third (setmaxnreg).
constexpr int REG_LAUNCH = 168, REG_DRAIN = 216, REG_ISSUE = 72;
static_assert(REG_DRAIN * NDRAIN + REG_ISSUE * (NTH - NDRAIN) <= REG_LAUNCH * NTH, "register split");

__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int Nn) {  // fp32 accumulate, both e4m3, K-major
    return (1u << 4) | ((uint32_t)(Nn >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// Bounded wait; the first look is a bare try_wait, since the issuing thread's own instructions
// are what bounds short blocks.
__device__ __forceinline__ bool wait_f(unsigned long long* b, uint32_t parity, volatile int* abort) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok)
                 : "r"(ck::smem_u32(b)), "r"(parity)
                 : "memory");
    return ok || ck::mbar_wait(b, parity, abort, &g_device_error_fp8);
}

// One lane of a converged warp.  The issuing warps run their loops as a whole and only the
// asynchronous instructions under this predicate: descriptors and addresses then stay in uniform
// registers (issued from a one-lane branch, four MMAs took 260 cycles instead of 50).
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(ok));
    return ok != 0;
}
// wait_f by a whole warp, with the same answer for all lanes.
__device__ __forceinline__ bool wait_w(unsigned long long* b, uint32_t parity, volatile int* abort) {
    return __all_sync(0xffffffffu, wait_f(b, parity, abort));
}

// a0 += s * v[0], a1 += s * v[1] in one packed instruction (same roundings as two fmaf).
__device__ __forceinline__ void fma2(float& a0, float& a1, const float* v, float s) {
    asm("{ .reg .b64 a, b, c; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %4}; mov.b64 c, {%0, %1}; "
        "fma.rn.f32x2 c, a, b, c; mov.b64 {%0, %1}, c; }"
        : "+f"(a0), "+f"(a1)
        : "f"(v[0]), "f"(v[1]), "f"(s));
}

// Row offsets and the first unit (output tile) of every group, built once per CTA.
struct Groups {
    int off[MAXG + 1], unit[MAXG + 1];  // unit[G] = number of units
};
// Offsets are clamped to [0, M]: rows outside the matrix belong to no tile.
__device__ __forceinline__ void load_offsets(Groups& gs, const GemmArgs& p, int tid) {
    if (tid <= p.G) gs.off[tid] = p.offs ? min(max(p.offs[tid], 0), p.M) : (tid == 0 ? 0 : p.M);
}
// One warp: units of `rows` rows x ntn column tiles per group (empty or negative groups: none).
__device__ __forceinline__ void scan_units(Groups& gs, int G, int rows_per, int ntn, int lane) {
    constexpr int PER = (MAXG + 31) / 32;
    int loc[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int g = lane * PER + i;
        const int rows = g < G ? gs.off[g + 1] - gs.off[g] : 0;
        loc[i] = sum;
        sum += rows > 0 ? (rows + rows_per - 1) / rows_per * ntn : 0;
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int g = lane * PER + i;
        if (g < G) gs.unit[g] = incl - sum + loc[i];
    }
    if (lane == 31) gs.unit[G] = incl;
}

struct Unit {
    int g, row0, rend, nt;
};
__device__ __forceinline__ Unit unit_of(const Groups& gs, int G, int rows_per, int ntn, int u) {
    int lo = 0, hi = G;  // largest g with unit[g] <= u (empty groups repeat a value)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (gs.unit[mid] <= u) lo = mid;
        else hi = mid;
    }
    const int l = u - gs.unit[lo];
    return {lo, gs.off[lo] + l / ntn * rows_per, gs.off[lo + 1], l % ntn};
}

// 16 bytes of outputs from PER sums.
template <int EPI, typename TO, int PER>
__device__ __forceinline__ uint4 pack_out(const float* v, float mul) {
    uint4 r;
    if constexpr (EPI == RELU2_Q) {
        r.x = pack4(v[0] * mul, v[1] * mul, v[2] * mul, v[3] * mul);
        r.y = pack4(v[4] * mul, v[5] * mul, v[6] * mul, v[7] * mul);
        r.z = pack4(v[8] * mul, v[9] * mul, v[10] * mul, v[11] * mul);
        r.w = pack4(v[12] * mul, v[13] * mul, v[14] * mul, v[15] * mul);
    } else {
        TO* o = reinterpret_cast<TO*>(&r);
#pragma unroll
        for (int e = 0; e < PER; e++) o[e] = from_f32<TO>(v[e]);
    }
    return r;
}

// Tensor maps: A (M, K) in boxes of `rows` x 128 bytes, W (G, N, K) likewise, 128-byte swizzle.
inline int map_a(CUtensorMap* m, const GemmArgs& p, int rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)p.K, (cuuint64_t)p.M}, strides[1] = {(cuuint64_t)p.lda};
    const cuuint32_t box[2] = {(cuuint32_t)BLK, (cuuint32_t)rows};
    return make_map_dt(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.a, 2, dims, strides, box, true) ? RWKV_ERR_CUDA : RWKV_OK;
}
inline int map_w(CUtensorMap* m, const GemmArgs& p, int rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)p.K, (cuuint64_t)p.N, (cuuint64_t)p.G};
    const cuuint64_t strides[2] = {(cuuint64_t)p.ldw, (cuuint64_t)(p.G > 1 ? p.gsw : (long long)p.N * p.ldw)};
    const cuuint32_t box[3] = {(cuuint32_t)BLK, (cuuint32_t)rows, 1};
    return make_map_dt(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.w, 3, dims, strides, box, true) ? RWKV_ERR_CUDA : RWKV_OK;
}

// An upper bound of the tiles of `rows` rows of all groups that needs no offsets.
inline long long row_tiles(int M, int G, int rows) {
    const long long most = (M + rows - 1) / rows + (G > 1 ? G - 1 : 0);
    return most < M ? most : M;
}

}  // namespace fp8
}  // namespace rwkv
