// W8A8 matrix product on the gfx950 integer matrix cores:
//   out[m][n] = act(a_scale[m] * w_scale[n] * sum_k A[m][k] W[n][k] + bias[n]) + residual[m][n]
// A, W int8 rows, one fp32 scale per row of A (token) and per row of W (channel).  The sum is an exact int32 for K <= 131071
// (|a * w| <= 2^14), whatever order it is taken in: every tile shape and every split of K gives the same bits.  The epilogue is fp32,
// rounded once on the way out.
//
// Fragments (v_mfma_i32_16x16x64_i8): lane l holds 16 bytes of row l % 16 at k = 16 * (l / 16); the WEIGHT fragment is the first operand,
// so a lane's accumulator quad is one output row (l % 16) and 4 consecutive columns (4 * (l / 16)).
#include "common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// the same 16 bytes at any address (global memory accepts them unaligned)
typedef u32x4 __attribute__((aligned(1))) u32x4_u;
typedef f16x8 __attribute__((aligned(2))) f16x8_u;
typedef f16x4 __attribute__((aligned(2))) f16x4_u;
typedef f32x4 __attribute__((aligned(4))) f32x4_u;

struct I8Args {
    const int8_t* A; const int8_t* W; const float* a_scale; const float* w_scale; const float* bias; const void* residual; void* out;
    long lda, ldw, ldr, ldc;
    int M, N, K, epilogue, tiles_m, tiles_n;
};

constexpr int BKB = 128;   // bytes (= values of k) of a K-step: 8 chunks of 16 bytes

// 16 bytes of a row from byte `k` on, zeros behind the row's end
__device__ __forceinline__ u32x4 load_chunk(const int8_t* row, int k, int K) {
    u32x4 v = {0, 0, 0, 0};
    if (k + 16 <= K) {
        v = *reinterpret_cast<const u32x4_u*>(row + k);
    } else {
        for (int j = 0; k + j < K; ++j) v[j >> 2] |= (unsigned)(uint8_t)row[k + j] << (8 * (j & 3));
    }
    return v;
}

__device__ __forceinline__ float silu_f(float v) { return v / (1.0f + expf(-v)); }
__device__ __forceinline__ float gelu_f(float g) { return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f)); }

// one output value before the residual (the accumulators of a GEGLU pair come together)
__device__ __forceinline__ float scaled(int acc, float sa, float sw, float b) { return (float)acc * sa * sw + b; }

__device__ __forceinline__ float residual_at(const I8Args& p, int m, int n) {
    if (!p.residual) return 0.0f;
    const long at = (long)m * p.ldr + n;
    return (p.epilogue & DS_EPI_RES_F32) ? reinterpret_cast<const float*>(p.residual)[at] : (float)reinterpret_cast<const f16*>(p.residual)[at];
}

__device__ __forceinline__ void store_at(const I8Args& p, int m, int n, float v) {
    const long at = (long)m * p.ldc + n;
    if (p.epilogue & DS_EPI_OUT_F32) reinterpret_cast<float*>(p.out)[at] = v;
    else reinterpret_cast<f16*>(p.out)[at] = (f16)v;
}

// Any sizes, strides and alignments: 128 x 64 tiles, 4 waves of 32 x 64 (a wave's 64 columns hold whole GEGLU groups), operands through
// registers (unaligned 16-byte global loads, byte loads in a row's last chunk) into two LDS stages, 16-byte chunks XOR-swizzled by
// (row >> 1) & 7 so that a fragment read and a staging write each touch every bank once.
template <bool GEGLU>
__global__ void __launch_bounds__(256, 2) gemm_i8_any_kernel(I8Args p) {
    constexpr int BM = 128, BN = 64;
    __shared__ __attribute__((aligned(16))) int8_t sm[2][(BM + BN) * BKB];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m0 = (blockIdx.x / p.tiles_n) * BM, n0 = (blockIdx.x % p.tiles_n) * BN;
    const int l15 = lane & 15, l4 = lane >> 4;
    const int row = tid >> 3, chunk = tid & 7;      // staging: 32 rows per sweep, 8 lanes per row
    u32x4 r[6];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < 6; ++i) {
            const int rr = row + 32 * (i < 4 ? i : i - 4);
            const bool in = i < 4 ? m0 + rr < p.M : n0 + rr < p.N;
            const int8_t* src = i < 4 ? p.A + (long)(m0 + rr) * p.lda : p.W + (long)(n0 + rr) * p.ldw;
            r[i] = in ? load_chunk(src, k0 + 16 * chunk, p.K) : u32x4{0, 0, 0, 0};
        }
    };
    auto store = [&](int s) {
#pragma unroll
        for (int i = 0; i < 6; ++i) {
            const int rr = row + 32 * i;
            *reinterpret_cast<u32x4*>(&sm[s][rr * BKB + (chunk ^ ((rr >> 1) & 7)) * 16]) = r[i];
        }
    };
    i32x4 acc[4][2];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) acc[t][u] = i32x4{0, 0, 0, 0};
    const int nk = (p.K + BKB - 1) / BKB;
    if (nk > 0) load(0);
    for (int kt = 0; kt < nk; ++kt) {
        store(kt & 1);
        __syncthreads();       // stage kt & 1 is whole; the other one was last read before the previous barrier's successor store
        if (kt + 1 < nk) load((kt + 1) * BKB);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            auto frag = [&](int rr) { return *reinterpret_cast<const i32x4*>(&sm[kt & 1][rr * BKB + ((4 * ks + l4) ^ ((rr >> 1) & 7)) * 16]); };
            i32x4 a[2], w[4];
#pragma unroll
            for (int u = 0; u < 2; ++u) a[u] = frag(wave * 32 + u * 16 + l15);
#pragma unroll
            for (int t = 0; t < 4; ++t) w[t] = frag(BM + t * 16 + l15);
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int u = 0; u < 2; ++u) acc[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[t], a[u], acc[t][u], 0, 0, 0);
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int m = m0 + wave * 32 + u * 16 + l15;
        if (m >= p.M) continue;
        const float sa = p.a_scale[m];
#pragma unroll
        for (int t = 0; t < (GEGLU ? 2 : 4); ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = n0 + t * 16 + 4 * l4 + j;
                if (n >= p.N) continue;
                float v = scaled(acc[t][u][j], sa, p.w_scale[n], p.bias ? p.bias[n] : 0.0f);
                int col = n;
                if constexpr (GEGLU) {
                    v *= gelu_f(scaled(acc[t + 2][u][j], sa, p.w_scale[n + 32], p.bias ? p.bias[n + 32] : 0.0f));
                    col = n0 / 2 + t * 16 + 4 * l4 + j;
                } else if (p.epilogue & DS_EPI_SILU) {
                    v = silu_f(v);
                }
                store_at(p, m, col, v + residual_at(p, m, col));
            }
    }
}

}  // namespace

extern "C" int ds_gemm_i8(const int8_t* A, const int8_t* W, const float* a_scale, const float* w_scale, const float* bias, const void* residual,
                          void* out, const ds_gemm_i8_desc* desc, void* stream) {
    DS_CHECK_ARG(desc, "ds_gemm_i8: desc is NULL");
    const ds_gemm_i8_desc d = *desc;
    DS_CHECK_ARG(d.M >= 0 && d.N >= 0 && d.K >= 0, "ds_gemm_i8: negative size (M %d, N %d, K %d)", d.M, d.N, d.K);
    DS_CHECK_ARG(d.K <= 131071, "ds_gemm_i8: K %d: the 32-bit sums hold K <= 131071", d.K);
    DS_CHECK_ARG((d.epilogue & ~(DS_EPI_GEGLU | DS_EPI_SILU | DS_EPI_OUT_F32 | DS_EPI_RES_F32)) == 0, "ds_gemm_i8: epilogue %d", d.epilogue);
    const bool geglu = d.epilogue & DS_EPI_GEGLU;
    DS_CHECK_ARG(!(geglu && (d.epilogue & DS_EPI_SILU)), "ds_gemm_i8: GEGLU and SiLU exclude each other");
    DS_CHECK_ARG(!geglu || d.N % 64 == 0, "ds_gemm_i8: GEGLU needs N %% 64 == 0 (32-row groups of values and gates), N %d", d.N);
    DS_CHECK_ARG(!(geglu && residual), "ds_gemm_i8: GEGLU takes no residual");
    if (d.M == 0 || d.N == 0) return DS_OK;
    const int cols = geglu ? d.N / 2 : d.N;
    DS_CHECK_ARG((A && W) || d.K == 0, "ds_gemm_i8: A or W is NULL");
    DS_CHECK_ARG(a_scale && w_scale && out, "ds_gemm_i8: a_scale, w_scale or out is NULL");
    DS_CHECK_ARG(d.lda >= d.K && d.ldw >= d.K && d.ldc >= cols && (!residual || d.ldr >= cols),
                 "ds_gemm_i8: a row stride is shorter than its row (lda %ld, ldw %ld, ldc %ld, ldr %ld)", (long)d.lda, (long)d.ldw, (long)d.ldc, (long)d.ldr);
    const int osz = (d.epilogue & DS_EPI_OUT_F32) ? 4 : 2, rsz = (d.epilogue & DS_EPI_RES_F32) ? 4 : 2;
    DS_CHECK_ARG((((uintptr_t)a_scale | (uintptr_t)w_scale | (uintptr_t)bias) & 3) == 0 && ((uintptr_t)out & (osz - 1)) == 0 && ((uintptr_t)residual & (rsz - 1)) == 0,
                 "ds_gemm_i8: a pointer is not aligned to its element");
    I8Args p{A, W, a_scale, w_scale, bias, residual, out, d.lda, d.ldw, d.ldr, d.ldc, d.M, d.N, d.K, d.epilogue, 0, 0};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    p.tiles_m = ds_cdiv(d.M, 128);
    p.tiles_n = ds_cdiv(d.N, 64);
    DS_CHECK_ARG((long)p.tiles_m * p.tiles_n <= 0xffffff, "ds_gemm_i8: M %d x N %d has too many tiles for one launch", d.M, d.N);
    const dim3 grid(p.tiles_m * p.tiles_n);
    if (geglu) gemm_i8_any_kernel<true><<<grid, 256, 0, st>>>(p);
    else gemm_i8_any_kernel<false><<<grid, 256, 0, st>>>(p);
    DS_CHECK_LAUNCH("ds_gemm_i8");
    return DS_OK;
}
