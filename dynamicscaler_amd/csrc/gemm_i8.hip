// W8A8 matrix product on the gfx950 integer matrix cores:
//   out[m][n] = act(a_scale[m] * w_scale[n] * sum_k A[m][k] W[n][k] + bias[n]) + residual[m][n]
// A, W int8 rows, one fp32 scale per row of A (token) and per row of W (channel).  The sum is an exact int32 for K <= 131071
// (|a * w| <= 2^14), whatever order it is taken in: every tile shape and every split of K gives the same bits.  The epilogue is fp32,
// rounded once on the way out.
//
// Fragments (v_mfma_i32_16x16x64_i8): lane l holds 16 bytes of row l % 16 at k = 16 * (l / 16); the WEIGHT fragment is the first operand,
// so a lane's accumulator quad is one output row (l % 16) and 4 consecutive columns (4 * (l / 16)).
//
// Two kernels: a few rows (bound by what a CU fetches) and tiles (bound by the matrix cores and, by a third at K = 1280, by what stands before and behind
// the K loop -- 8192^3 433 us, 2.54 POP/s; 40960 x 10240 x 1280 with GEGLU 550 us, 1.95 POP/s -- or, for short K, by memory: 655360 x 320 x 320
// onto an fp32 residual 396 us, 4.77 TB/s).
#include "common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// the same 16 bytes at any address (global memory accepts them unaligned)
typedef u32x4 __attribute__((aligned(1))) u32x4_u;
typedef f16x8 __attribute__((aligned(2))) f16x8_u;
typedef f16x4 __attribute__((aligned(2))) f16x4_u;
typedef f32x4 __attribute__((aligned(4))) f32x4_u;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 __attribute__((aligned(4))) u32x4_4;
typedef u32x2 __attribute__((aligned(2))) u32x2_2;

struct I8Args {
    const int8_t* A; const int8_t* W; const float* a_scale; const float* w_scale; const float* bias; const void* residual; void* out;
    long lda, ldw, ldr, ldc;
    int M, N, K, epilogue, tiles_m, tiles_n, group_m;
};

constexpr int BKB = 128;   // bytes (= values of k) of a K-step: 8 chunks of 16 bytes

// 16 bytes of a row from byte `k` on, zeros behind the row's end, in two halves so that several loads can be on their way: fetch() and, when they
// have come, bytes().  The last bytes are fetched as the 16 that end with the row (rows of at least 16 bytes) and moved down afterwards.
// ODD: addresses that are no multiple of 4 are read as the aligned dwords that hold the 16 bytes, five where they straddle -- each holds at
// least one of them, so nothing outside the row's own dwords is touched -- and shifted into place: loads from odd addresses as such
// take up to five times as long (16 x 4097 x 4095: 23 us; with K = 4092 6.8 us).
template <bool ODD> struct Fetched {
    u32x4 v;
    unsigned e;
    __device__ __forceinline__ void fetch(const int8_t* from) {
        if constexpr (ODD) {
            const unsigned s = (unsigned)(uintptr_t)from & 3;
            const unsigned* at = reinterpret_cast<const unsigned*>(from - s);
            v = *reinterpret_cast<const u32x4_4*>(at);
            e = at[s ? 4 : 3];
        } else {
            v = *reinterpret_cast<const u32x4_u*>(from);
        }
    }
    __device__ __forceinline__ u32x4 bytes(const int8_t* from) const {
        if constexpr (!ODD) return v;
        const unsigned s = (unsigned)(uintptr_t)from & 3;
        return u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], s), __builtin_amdgcn_alignbyte(v[2], v[1], s), __builtin_amdgcn_alignbyte(v[3], v[2], s),
                     __builtin_amdgcn_alignbyte(e, v[3], s)};
    }
};
// the same where the row may end
template <bool ODD> __device__ __forceinline__ void fetch_end(Fetched<ODD>& f, const int8_t* row, int k, int K) {
    if (K >= 16) {
        f.fetch(row + min(k, K - 16));
        return;
    }
    f.v = u32x4{0, 0, 0, 0};
    for (int j = 0; k + j < K; ++j) f.v[j >> 2] |= (unsigned)(uint8_t)row[k + j] << (8 * (j & 3));
}
__device__ __forceinline__ u32x4 end_chunk(u32x4 v, int k, int K);
template <bool ODD> __device__ __forceinline__ u32x4 bytes_end(const Fetched<ODD>& f, const int8_t* row, int k, int K) {
    return K >= 16 ? end_chunk(f.bytes(row + min(k, K - 16)), k, K) : f.v;
}
__device__ __forceinline__ u32x4 end_chunk(u32x4 v, int k, int K) {
    const int bytes = k + 16 - K;
    if (K < 16 || bytes <= 0) return v;
    unsigned long long lo = v[0] | (unsigned long long)v[1] << 32, hi = v[2] | (unsigned long long)v[3] << 32;
    if (bytes >= 8) { lo = hi; hi = 0; }
    const int s = 8 * (bytes & 7);
    lo = (lo >> s) | ((hi << 1) << (63 - s));
    hi >>= s;
    if (bytes >= 16) lo = hi = 0;
    return u32x4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
}

// x / (1 + e^-x) without the divide's ~10 instructions: the hardware's reciprocal (1 ulp) and a Newton step; an infinite denominator gives zero.  For
// fp16 results the hardware's 2^x and reciprocal as they are (2^-22 and |x| 2^-23 of the value)
__device__ __forceinline__ float silu_f(float v) {
    const float d = 1.0f + expf(-v), r = __builtin_amdgcn_rcpf(d);
    return v * (d < __builtin_huge_valf() ? fmaf(r, fmaf(-d, r, 1.0f), r) : 0.0f);
}
__device__ __forceinline__ float silu_f16(float v) { return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * v)); }

// gelu(g) = g / 2 * erfc(-g / sqrt 2) for fp32 results: E(a) = erfc(a / sqrt 2), a = |g|, is relative to itself what E(a) for g < 0 and 2 - E(a) otherwise need
// (1 + erf(g / sqrt 2) cancels: at g = -4 a thousandth of it is wrong, at -6 all).  E = e^(-a^2 / 2) F(a), F(a) (a + 4.75) = P((a - 4.75) / (a + 4.75)) with a
// polynomial P of degree 8 (least maximum on [0, 13.6], 1.3e-8 off); the exponent keeps what a^2 and its factor round away.  Within
// 8 2^-24 of itself in exact reciprocals and powers of two, 12 2^-24 with the hardware's.  Behind 13.2 E < 2^-125 counts as zero.  97866 x 8704
// x 464 870 us (1 + erff 907, erfcf 1045).
__device__ __forceinline__ float gelu_f(float g) {
    const float a = fabsf(g), d = a + 4.75f, r0 = __builtin_amdgcn_rcpf(d), r = fmaf(r0, fmaf(-d, r0, 1.0f), r0), t = (a - 4.75f) * r;
    float p = -0.0026136799715459347f;
    p = fmaf(p, t, 0.00045183568727225065f);
    p = fmaf(p, t, 0.02308657020330429f);
    p = fmaf(p, t, -0.10125736147165298f);
    p = fmaf(p, t, 0.27621373534202576f);
    p = fmaf(p, t, -0.5683676600456238f);
    p = fmaf(p, t, 0.9441288709640503f);
    p = fmaf(p, t, -1.3071787357330322f);
    p = fmaf(p, t, 1.5328326225280762f);
    const float s = a * a, x = s * -0.7213475108146667f;           // e^(-a^2 / 2) = 2^x 2^y
    const float y = fmaf(s, -9.629815167500055e-09f, fmaf(fmaf(a, a, -s), -0.7213475108146667f, fmaf(s, -0.7213475108146667f, -x)));
    const float w = __builtin_amdgcn_exp2f(x), e = a < 13.2f ? fmaf(w, y * 0.69314718f, w) * (r * p) : 0.0f;
    return 0.5f * g * (g < 0.0f ? e : 2.0f - e);
}

// The same for fp16 results: E(a) = 2^-q(a) with a polynomial q of degree 8 (least maximum on [0, 9]; 1.2e-5 off with its coefficients in 32 bits, E 1.3e-5 of
// itself evaluated in them, 2e-5 with the hardware's 2^x, and gelu 2e-6 absolute: a twenty-fifth and less of an fp16 rounding); behind 9 E < 2.3e-19
// counts as zero.  12 vector instructions where erff takes ~40: the GEGLU epilogue is bound by them.
__device__ __forceinline__ float gelu_f16(float g) {
    const float a = fabsf(g);
    float q = -7.463252416073374e-08f;
    q = fmaf(q, a, 3.6557733983055757e-06f);
    q = fmaf(q, a, -7.943754462758079e-05f);
    q = fmaf(q, a, 0.001020048395730555f);
    q = fmaf(q, a, -0.008750868029892445f);
    q = fmaf(q, a, 0.054304663091897964f);
    q = fmaf(q, a, 0.4582415223121643f);
    q = fmaf(q, a, 1.1512949466705322f);
    q = fmaf(q, a, -3.414401817281032e-06f);
    const float e = a < 9.0f ? __builtin_amdgcn_exp2f(-q) : 0.0f;
    return 0.5f * g * (g < 0.0f ? e : 2.0f - e);
}

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

// ------------------------------------------------------------------------------------------------ few rows
// M <= 16 MT: the weights are read once and that is the time.  A workgroup owns 16 columns (GEGLU: 16 values and their 16 gates); its waves
// split K and read both operands straight from memory in fragment order (a wave's load covers 64 contiguous bytes of 16 rows; W is used once,
// A sits in L2), then add their exact integer partial sums through LDS.  Rows past M / N repeat the last one and
// are not stored.
// waves of a workgroup: at most 16, and 64 KiB of partial sums
template <int MT, bool GEGLU> struct Few {
    static constexpr int FIT = 64 / (MT * (GEGLU ? 2 : 1)), WAVES = FIT > 16 ? 16 : FIT;
    static constexpr int U = MT == 1 ? (GEGLU ? 4 : 8) : MT == 2 && !GEGLU ? 4 : 2;      // blocks of 64 bytes whose loads a wave sends out together
};

template <int MT, bool GEGLU, bool ODD>
__global__ void __launch_bounds__((64 * Few<MT, GEGLU>::WAVES)) gemm_i8_few_kernel(I8Args p) {
    constexpr int NT = GEGLU ? 2 : 1, U = Few<MT, GEGLU>::U;
    extern __shared__ __attribute__((aligned(16))) i32x4 red[];      // [waves][NT][MT][64 lanes]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
    const int l15 = lane & 15, l4 = lane >> 4;
    const int n0 = GEGLU ? (blockIdx.x >> 1) * 64 + (blockIdx.x & 1) * 16 : blockIdx.x * 16;
    const int8_t* w[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) w[t] = p.W + (long)min(n0 + 32 * t + l15, p.N - 1) * p.ldw;
    const int8_t* a[MT];
#pragma unroll
    for (int u = 0; u < MT; ++u) a[u] = p.A + (long)min(16 * u + l15, p.M - 1) * p.lda;
    i32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[t][u] = i32x4{0, 0, 0, 0};
    const int whole = p.K / 64, per = (whole + waves - 1) / waves;
    const int end = min(whole, (wave + 1) * per);
    // What the epilogue needs is on its way while the product is formed -- as it lies in memory, since a conversion would wait for it -- and in
    // whole fours where the 16 columns are all there: the instructions fetched are a large part of so short a kernel's time.
    const int col = GEGLU ? (blockIdx.x >> 1) * 32 + (blockIdx.x & 1) * 16 + 4 * l4 : n0 + 4 * l4, cols = GEGLU ? p.N / 2 : p.N;
    const bool full = GEGLU || n0 + 16 <= p.N, res32 = p.epilogue & DS_EPI_RES_F32;
    f32x4 sw[NT], bw[NT];
    float sa = 0.0f;
    u32x4 res = {0, 0, 0, 0};
    auto row_data = [&](int u) {
        const int m = min(16 * u + l15, p.M - 1);
        sa = p.a_scale[m];
        if (!p.residual) return;
        const long at = (long)m * p.ldr + col;
        if (full && res32) res = *reinterpret_cast<const u32x4_4*>(reinterpret_cast<const float*>(p.residual) + at);
        else if (full) {
            const u32x2_2 h = *reinterpret_cast<const u32x2_2*>(reinterpret_cast<const f16*>(p.residual) + at);
            res[0] = h[0];
            res[1] = h[1];
        }
    };
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int n = n0 + 32 * t + 4 * l4;
        bw[t] = f32x4{0, 0, 0, 0};
        if (full) {
            sw[t] = *reinterpret_cast<const f32x4_u*>(p.w_scale + n);
            if (p.bias) bw[t] = *reinterpret_cast<const f32x4_u*>(p.bias + n);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sw[t][j] = p.w_scale[min(n + j, p.N - 1)];
                if (p.bias) bw[t][j] = p.bias[min(n + j, p.N - 1)];
            }
        }
    }
    if (wave < MT) row_data(wave);
    for (int b = wave * per; b < end; b += U) {
        Fetched<ODD> fw[U][NT], fa[U][MT];
        const int k = b * 64 + 16 * l4;
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (b + i < end) {
#pragma unroll
                for (int t = 0; t < NT; ++t) fw[i][t].fetch(w[t] + k + 64 * i);
#pragma unroll
                for (int u = 0; u < MT; ++u) fa[i][u].fetch(a[u] + k + 64 * i);
            }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (b + i < end) {
#pragma unroll
                for (int u = 0; u < MT; ++u) {
                    const i32x4 av = (i32x4)fa[i][u].bytes(a[u]);
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8((i32x4)fw[i][t].bytes(w[t]), av, acc[t][u], 0, 0, 0);
                }
            }
    }
    if (p.K % 64 != 0 && wave == waves - 1) {
        const int k = whole * 64 + 16 * l4;
        Fetched<ODD> fw[NT], fa[MT];
#pragma unroll
        for (int t = 0; t < NT; ++t) fetch_end(fw[t], w[t], k, p.K);
#pragma unroll
        for (int u = 0; u < MT; ++u) fetch_end(fa[u], a[u], k, p.K);
#pragma unroll
        for (int u = 0; u < MT; ++u) {
            const i32x4 av = (i32x4)bytes_end(fa[u], a[u], k, p.K);
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8((i32x4)bytes_end(fw[t], w[t], k, p.K), av, acc[t][u], 0, 0, 0);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) red[((wave * NT + t) * MT + u) * 64 + lane] = acc[t][u];
    __syncthreads();
    for (int u = wave; u < MT; u += waves) {
        if (u != wave) row_data(u);
        i32x4 sum[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            sum[t] = red[(t * MT + u) * 64 + lane];
#pragma unroll 4
            for (int v = 1; v < waves; ++v) sum[t] += red[((v * NT + t) * MT + u) * 64 + lane];
        }
        const int m = 16 * u + l15;
        if (m >= p.M) continue;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = scaled(sum[0][j], sa, sw[0][j], bw[0][j]);
            if constexpr (GEGLU) {
                const float gate = scaled(sum[NT - 1][j], sa, sw[NT - 1][j], bw[NT - 1][j]);
                v[j] *= p.epilogue & DS_EPI_OUT_F32 ? gelu_f(gate) : gelu_f16(gate);
            }
        }
        if (!GEGLU && (p.epilogue & DS_EPI_SILU)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = p.epilogue & DS_EPI_OUT_F32 ? silu_f(v[j]) : silu_f16(v[j]);
        }
        if (full) {
            if (p.residual) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += res32 ? __uint_as_float(res[j]) : (float)__builtin_bit_cast(f16x2, (unsigned)res[j / 2])[j % 2];
            }
            const long at = (long)m * p.ldc + col;
            if (p.epilogue & DS_EPI_OUT_F32) *reinterpret_cast<f32x4_u*>(reinterpret_cast<float*>(p.out) + at) = f32x4{v[0], v[1], v[2], v[3]};
            else *reinterpret_cast<f16x4_u*>(reinterpret_cast<f16*>(p.out) + at) = f16x4{(f16)v[0], (f16)v[1], (f16)v[2], (f16)v[3]};
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < cols) store_at(p, m, col + j, v[j] + residual_at(p, m, col + j));
        }
    }
}

// ------------------------------------------------------------------------------------------------ many rows
typedef __attribute__((address_space(3))) void lds_void;
// LDS-DMA: lane l's 16 bytes land at dst + 16 l (dst wave-uniform); offsets past the buffer's end bring zeros
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, int8_t* dst, unsigned voff, unsigned soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)dst, 16, voff, soff, 0, 0);
}
constexpr unsigned OOB = 0x80000000u;    // past every buffer (all are < 2 GiB)

template <int BM, int BN, int WGM, int WGN, int NS> struct I8Tile {
    static constexpr int NT = 64 * WGM * WGN;
    static constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
    static constexpr int LROWS = NT / 8, AR = BM / LROWS, BR = BN / LROWS;
    static constexpr size_t STAGE = (size_t)(BM + BN) * BKB, LDS = NS * STAGE;
    static constexpr int PER_CU = (int)(163840 / LDS) * (NT / 64) > 16 ? 16 / (NT / 64) : (int)(163840 / LDS);
    static_assert(BM % (16 * WGM) == 0 && WN % 64 == 0 && BM % LROWS == 0 && BN % LROWS == 0 && LROWS % 32 == 0, "tile shape");
};

// DMA (K % 16 == 0 and 16-byte aligned rows): both operands by LDS-DMA into NS stages, the pieces of K-step k + NS - 1 issued between the MFMAs
// of k.  Otherwise (any size, stride and alignment) through registers into two stages, loaded D + 1 K-steps ahead by unaligned 16-byte loads,
// rows past M / N repeating the last one.  A stage holds BM rows of A, then BN rows of W, 128 bytes each, the 16-byte chunks XOR-swizzled through the SOURCE address so that a fragment
// read touches every bank once.  fp16 results: the wave's W rows are dealt to its MFMA tiles so that a lane ends up with 8 consecutive columns
// (tile t, row i <-> column 32 (t / 2) + 8 (i / 4) + 4 (t % 2) + i % 4) as it does with 4 and the natural
// order in fp32.
template <int BM, int BN, int WGM, int WGN, int NS, bool DMA, bool STREAM, bool OUT32, bool GEGLU>
__global__ void __launch_bounds__((I8Tile<BM, BN, WGM, WGN, NS>::NT), (DMA || BM * BN > 64 * 64 ? I8Tile<BM, BN, WGM, WGN, NS>::PER_CU * I8Tile<BM, BN, WGM, WGN, NS>::NT / 256 : 3)) gemm_i8_tile_kernel(I8Args p) {
    using T = I8Tile<BM, BN, WGM, WGN, NS>;
    constexpr int TM = T::TM, TN = T::TN;
    extern __shared__ __attribute__((aligned(256))) int8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WGN, wn = wave % WGN;
    const int l15 = lane & 15, l4 = lane >> 4;
    // workgroups that share an XCD (blockIdx % 8) take consecutive tiles; within them group_m row panels walk the columns together
    int tile_m, tile_n;
    {
        const int nwg = p.tiles_m * p.tiles_n, xcd = blockIdx.x & 7, q = nwg >> 3, r = nwg & 7;
        const int id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (blockIdx.x >> 3);
        const int per = p.group_m * p.tiles_n, first = (id / per) * p.group_m, in = id % per;
        const int size = min(p.tiles_m - first, p.group_m);
        tile_m = first + in % size;
        tile_n = in / size;
    }
    const int m0 = tile_m * BM, n0 = tile_n * BN;
    const int rows_a = min(BM, p.M - m0), rows_w = min(BN, p.N - n0);
    // staging: lane -> row tid / 8 (+ LROWS per piece), physical chunk tid % 8, whose source is the chunk that the swizzle puts there
    const int srow = tid >> 3;
    auto swz_a = [](int row) { return (row >> 1) & 7; };
    auto swz_w = [](int row) { return OUT32 ? (row >> 1) & 7 : ((row >> 1) & 1) | (((row >> 3) & 3) << 1); };
    const int ca = (tid & 7) ^ swz_a(srow), cw = (tid & 7) ^ swz_w(srow);
    const int nk = (p.K + BKB - 1) / BKB;
    constexpr int PIECES = T::AR + T::BR;
    // DMA: byte offsets inside the tile's rows (its operands as buffers that end with its last row), registers: addresses
    const int8_t* a_tile = p.A + (long)m0 * p.lda;
    const int8_t* w_tile = p.W + (long)n0 * p.ldw;
    const __amdgpu_buffer_rsrc_t rsA = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a_tile), 0, DMA ? (rows_a - 1) * (int)p.lda + p.K : 0, 0x00020000);
    const __amdgpu_buffer_rsrc_t rsW = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(w_tile), 0, DMA ? (rows_w - 1) * (int)p.ldw + p.K : 0, 0x00020000);
    unsigned voff[PIECES];
    const int8_t* src[PIECES];
    constexpr int D = !DMA && BM * BN <= 64 * 64 ? 2 : 1;       // K-steps held in registers on their way
    Fetched<false> reg[D][PIECES];              // (reading aligned dwords gains nothing here: 129 x 4097 x 4095 35 us against 21)
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        const bool of_a = j < T::AR;
        const int row = srow + T::LROWS * (of_a ? j : j - T::AR), rows = of_a ? rows_a : rows_w;
        if constexpr (DMA) voff[j] = row < rows ? (unsigned)row * (unsigned)(of_a ? p.lda : p.ldw) + 16u * (of_a ? ca : cw) : OOB;
        else src[j] = (of_a ? a_tile : w_tile) + (long)min(row, rows - 1) * (of_a ? p.lda : p.ldw);
    }
    const int last = p.K - (nk - 1) * BKB;      // bytes of the last K-step; chunks behind them bring zeros
    const unsigned cut_a = 16 * ca >= last ? OOB : 0u, cut_w = 16 * cw >= last ? OOB : 0u;
    auto stage_row = [&](int j, int kt) { return smem + (kt % NS) * T::STAGE + (j < T::AR ? T::LROWS * j : BM + T::LROWS * (j - T::AR)) * BKB; };
    auto piece = [&](int j, int kt) {
        const bool tail = kt == nk - 1;
        dma16(j < T::AR ? rsA : rsW, stage_row(j, kt) + 8 * wave * BKB, voff[j] | (tail ? (j < T::AR ? cut_a : cut_w) : 0u), (unsigned)kt * BKB);
    };
    auto load_regs = [&](int kt, int set) {
        if (kt + 1 < nk || last == BKB) {
#pragma unroll
            for (int j = 0; j < PIECES; ++j) reg[set][j].fetch(src[j] + kt * BKB + 16 * (j < T::AR ? ca : cw));
        } else {
#pragma unroll
            for (int j = 0; j < PIECES; ++j) fetch_end(reg[set][j], src[j], kt * BKB + 16 * (j < T::AR ? ca : cw), p.K);
        }
    };
    auto store_regs = [&](int kt, int set) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const bool whole = kt + 1 < nk || last == BKB;
            const u32x4 v = whole ? reg[set][j].bytes(src[j]) : bytes_end(reg[set][j], src[j], kt * BKB + 16 * (j < T::AR ? ca : cw), p.K);
            *reinterpret_cast<u32x4*>(stage_row(j, kt) + srow * BKB + (tid & 7) * 16) = v;
        }
    };
    i32x4 acc[TN][TM];
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int u = 0; u < TM; ++u) acc[t][u] = i32x4{0, 0, 0, 0};
    constexpr int G = OUT32 ? 1 : 2, CW = 4 * G;               // a lane's consecutive columns on the way out, and their fours
    // on the way out (GEGLU apart): lane -> row lane / LANES (+ 64 / LANES a turn) of a block of 16 RB rows, CW columns
    constexpr int RB = TM < 2 || TM * TN > 16 || (size_t)T::NT / 2 * (T::WN + 4) * sizeof(float) > T::LDS ? 1 : 2, BLOCKS = TM / RB, LANES = T::WN / CW, TURNS = 16 * RB * LANES / 64;
    const int mw = m0 + wm * T::WM, nw = n0 + wn * T::WN;
    const int out_row = lane / LANES, out_col = nw + lane % LANES * CW;
    constexpr int SETS = TM * TN > 16 && !OUT32 ? 1 : 2;       // (the 256 x 256 tile has no registers for a second set of fp16 results' residual)
    u32x4 res[SETS][TURNS][G];
    auto load_residual = [&](int m, int col, u32x4* to) {
        const long at = (long)m * p.ldr + col;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            if (p.epilogue & DS_EPI_RES_F32) {
                to[i] = *reinterpret_cast<const u32x4_4*>(reinterpret_cast<const float*>(p.residual) + at + 4 * i);
            } else {
                const u32x2_2 h = *reinterpret_cast<const u32x2_2*>(reinterpret_cast<const f16*>(p.residual) + at + 4 * i);
                to[i][0] = h[0];
                to[i][1] = h[1];
            }
        }
    };
    auto load_block = [&](int b) {
        if (!GEGLU && p.residual && out_col + CW <= p.N) {
#pragma unroll
            for (int i = 0; i < TURNS; ++i) load_residual(min(mw + 16 * RB * b + out_row + 64 / LANES * i, p.M - 1), out_col, res[b % SETS][i]);
        }
    };
    constexpr bool EARLY = TM * TN <= 8;           // a small wave tile's residual is on its way while the product is formed
    if (EARLY) load_block(0);
    // the next K-step's pieces have landed for every wave (those of the NS - 2 steps behind it may be on their way) and every wave is through with
    // the stage that is written next (lgkmcnt: its fragment reads)
    auto sync = [&](bool all) {
        if constexpr (!DMA) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        else if (all || NS == 2) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PIECES * (NS - 2)) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    if constexpr (DMA) {
#pragma unroll
        for (int k = 0; k < NS - 1; ++k)
            if (k < nk) {
#pragma unroll
                for (int j = 0; j < PIECES; ++j) piece(j, k);
            }
    } else if (nk > 0) {
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (d < nk) load_regs(d, d);
        store_regs(0, 0);
        if (D < nk) load_regs(D, 0);
    }
    sync(nk < NS - 1);
    auto kstep = [&](int kt, int set) {
        const bool more = DMA ? kt + NS - 1 < nk : kt + 1 < nk;
        if constexpr (!DMA) {        // K-step kt + 1 into the stage that every wave has left, the ones behind it on their way
            if (more) store_regs(kt + 1, set);
            if (kt + 1 + D < nk) load_regs(kt + 1 + D, set);
        }
        const int8_t* sa = smem + (kt % NS) * T::STAGE + wm * T::WM * BKB;
        const int8_t* sw = smem + (kt % NS) * T::STAGE + (BM + wn * T::WN) * BKB;
        auto read_a = [&](int ks, int u) {
            const int row = u * 16 + l15;
            return *reinterpret_cast<const i32x4*>(sa + row * BKB + ((4 * ks + l4) ^ swz_a(row)) * 16);
        };
        auto read_w = [&](int ks, int t) {
            const int row = OUT32 ? t * 16 + l15 : 32 * (t >> 1) + 8 * (l15 >> 2) + 4 * (t & 1) + (l15 & 3);
            return *reinterpret_cast<const i32x4*>(sw + row * BKB + ((4 * ks + l4) ^ swz_w(row)) * 16);
        };
        // the short side's fragments of a 64-deep slice are held (two sets), the long side streams through a ring of three
        constexpr bool STREAM_A = TM >= TN;
        constexpr int L = STREAM_A ? TM : TN, S = STREAM_A ? TN : TM, NF = 2 * L, SLOTS = NF * S, SPAN = SLOTS / 2;
        static_assert(SPAN >= PIECES, "the next K-step's pieces fit the first half of this one");
        i32x4 held[2][S], ring[3];
        auto read_s = [&](int ks, int t) { return STREAM_A ? read_w(ks, t) : read_a(ks, t); };
        auto read_l = [&](int f) { return STREAM_A ? read_a(f / L, f % L) : read_w(f / L, f % L); };
#pragma unroll
        for (int t = 0; t < S; ++t) held[0][t] = read_s(0, t);
        ring[0] = read_l(0);
        ring[1] = read_l(1);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int ks = f / L, li = f % L;
            __builtin_amdgcn_sched_barrier(0);
            if (f + 2 < NF) ring[(f + 2) % 3] = read_l(f + 2);
            if (ks == 0 && li < S) held[1][li] = read_s(1, li);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int si = 0; si < S; ++si) {
                const int u = STREAM_A ? li : si, t = STREAM_A ? si : li;
                acc[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(STREAM_A ? held[ks][si] : ring[f % 3], STREAM_A ? ring[f % 3] : held[ks][si], acc[t][u], 0, 0, 0);
                const int slot = f * S + si;
#pragma unroll
                for (int j = 0; j < PIECES; ++j)
                    if (slot == ((j + 1) * SPAN) / PIECES - 1) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (DMA && more) piece(j, kt + NS - 1);
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
        }
        sync(!more);
    };
    for (int k0 = 0; k0 < nk; k0 += D)
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (k0 + d < nk) kstep(k0 + d, (d + 1) % D);

    auto add_residual = [&](float* v, const u32x4* r) {
#pragma unroll
        for (int j = 0; j < CW; ++j) {
            if (p.epilogue & DS_EPI_RES_F32) v[j] += __uint_as_float(r[j / 4][j % 4]);
            else v[j] += (float)__builtin_bit_cast(f16x2, (unsigned)r[j / 4][(j % 4) / 2])[j % 2];
        }
    };
    // STREAM (results that L2 does not hold): past the cache, A rows and W panels stay (16384 x 2560 x 1280 in fp16: 85 -> 66 us).  The pointers say
    // that a row may begin at any element.
    auto store_columns = [&](int m, int col, const float* v) {
        const long at = (long)m * p.ldc + col;
        if constexpr (OUT32) {
            const f32x4 o = {v[0], v[1], v[2], v[3]};
            f32x4_u* to = reinterpret_cast<f32x4_u*>(reinterpret_cast<float*>(p.out) + at);
            if constexpr (STREAM) __builtin_nontemporal_store(o, to);
            else *to = o;
        } else {
            f16x8 h;
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = (f16)v[j];
            f16x8_u* to = reinterpret_cast<f16x8_u*>(reinterpret_cast<f16*>(p.out) + at);
            if constexpr (STREAM) __builtin_nontemporal_store(h, to);
            else *to = h;
        }
    };
    float sa[TM];
#pragma unroll
    for (int u = 0; u < TM; ++u) sa[u] = p.a_scale[min(mw + 16 * u + l15, p.M - 1)];
    // a large wave tile's fp16 results without a residual go straight out (40960 x 1280 x 1280: 85 us against 102) where its 64-byte pieces are whole
    // ones (100001 x 2008 x 1008: 392 us straight)
    const bool turned = !GEGLU && (OUT32 || TM * TN <= 16 || p.residual || (p.ldc & 31) || ((uintptr_t)p.out & 63));
    if (turned) {
        // a wave turns its tile through a strip of LDS that is its own, 16 RB rows at a time: 256 (fp32) or 128 (fp16) contiguous bytes of a row
        // go out together (655360 x 320 x 320 on fp32 rows: 495 -> 416 us); a block's residual is on its way while the one before it is stored
        constexpr int LD = T::WN + 4;
        static_assert((size_t)T::NT / 64 * 16 * RB * LD * sizeof(float) <= T::LDS, "strips");
        float* strip = reinterpret_cast<float*>(smem) + wave * 16 * RB * LD;
        if (!EARLY) load_block(0);
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            if (SETS == 2 && b + 1 < BLOCKS) load_block(b + 1);
            if (SETS == 1 && b > 0) load_block(b);
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                f32x4 sw, bw;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = min(nw + (OUT32 ? 16 * t + 4 * l4 : 32 * (t >> 1) + 8 * l4 + 4 * (t & 1)) + j, p.N - 1);
                    sw[j] = p.w_scale[n];
                    bw[j] = p.bias ? p.bias[n] : 0.0f;
                }
#pragma unroll
                for (int u = 0; u < RB; ++u) {
                    f32x4 v;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[j] = scaled(acc[t][RB * b + u][j], sa[RB * b + u], sw[j], bw[j]);
                        if (p.epilogue & DS_EPI_SILU) v[j] = OUT32 ? silu_f(v[j]) : silu_f16(v[j]);
                    }
                    *reinterpret_cast<f32x4*>(strip + (16 * u + l15) * LD + (OUT32 ? 16 * t + 4 * l4 : 32 * (t >> 1) + 8 * l4 + 4 * (t & 1))) = v;
                }
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < TURNS; ++i) {
                const int row = out_row + 64 / LANES * i, m = mw + 16 * RB * b + row;
                float v[CW];
#pragma unroll
                for (int j = 0; j < CW; j += 4) *reinterpret_cast<f32x4*>(v + j) = *reinterpret_cast<const f32x4*>(strip + row * LD + lane % LANES * CW + j);
                if (m >= p.M) continue;
                if (out_col + CW <= p.N) {
                    if (p.residual) add_residual(v, res[b % SETS][i]);
                    store_columns(m, out_col, v);
                } else {
#pragma unroll
                    for (int j = 0; j < CW; ++j)
                        if (out_col + j < p.N) store_at(p, m, out_col + j, v[j] + residual_at(p, m, out_col + j));
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
        return;
    }
    // straight from the accumulators, 8 (fp16) or 4 (fp32) consecutive columns a lane; GEGLU: of every 64 columns 32 values, then their 32 gates
    constexpr int GB = GEGLU ? 32 / (16 * G) : 1;              // a lane's value groups in a block of 64 columns
    constexpr int GROUPS = (GEGLU ? TN / 2 : TN) / G;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        const int t0 = GEGLU ? g / GB * 4 + g % GB * G : g * G;        // first MFMA tile of the values; the gates' are two further
        const int n = nw + 16 * t0 + CW * l4, col = GEGLU ? (nw + 64 * (g / GB)) / 2 + g % GB * 16 * G + CW * l4 : n;
        if (n >= p.N) continue;
        float sw[CW], bw[CW], sg[CW], bg[CW];
#pragma unroll
        for (int j = 0; j < CW; ++j) {
            const int c = min(n + j, p.N - 1);
            sw[j] = p.w_scale[c];
            bw[j] = p.bias ? p.bias[c] : 0.0f;
            if constexpr (GEGLU) {
                sg[j] = p.w_scale[c + 32];
                bg[j] = p.bias ? p.bias[c + 32] : 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < TM; ++u) {
            const int m = mw + 16 * u + l15;
            if (m >= p.M) continue;
            float v[CW];
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                v[j] = scaled(acc[t0 + j / 4][u][j % 4], sa[u], sw[j], bw[j]);
                if constexpr (GEGLU) {
                    const float gate = scaled(acc[t0 + 2 + j / 4][u][j % 4], sa[u], sg[j], bg[j]);
                    v[j] *= OUT32 ? gelu_f(gate) : gelu_f16(gate);
                } else if (p.epilogue & DS_EPI_SILU) {
                    v[j] = OUT32 ? silu_f(v[j]) : silu_f16(v[j]);
                }
            }
            if (GEGLU || col + CW <= p.N) {
                store_columns(m, col, v);
            } else {
#pragma unroll
                for (int j = 0; j < CW; ++j)
                    if (col + j < p.N) store_at(p, m, col + j, v[j]);
            }
        }
    }
}

// Rows of K bytes at any address into rows of K rounded up to 16, zeros behind, which is what LDS-DMA takes: both operands in one launch, A's rows
// first.  Teams of 1 << shift lanes a row, 16 bytes a lane and turn.
struct AlignArgs { const int8_t* A; const int8_t* W; int8_t* to_a; int8_t* to_w; long lda, ldw; int M, N, K, stride, shift; };
__global__ void __launch_bounds__(256) align_rows_kernel(AlignArgs p) {
    const int team = 256 >> p.shift, lane = threadIdx.x & ((1 << p.shift) - 1);
    const long rows_a = p.to_a ? p.M : 0, rows = rows_a + (p.to_w ? p.N : 0);
    for (long row = (long)blockIdx.x * team + (threadIdx.x >> p.shift); row < rows; row += (long)gridDim.x * team) {
        const bool of_a = row < rows_a;
        const long at = of_a ? row : row - rows_a;
        const int8_t* src = of_a ? p.A + at * p.lda : p.W + at * p.ldw;
        int8_t* dst = (of_a ? p.to_a : p.to_w) + at * p.stride;
        for (int k = 16 * lane; k < p.stride; k += 16 << p.shift) {
            Fetched<true> f;
            fetch_end(f, src, k, p.K);
            *reinterpret_cast<u32x4*>(dst + k) = bytes_end(f, src, k, p.K);
        }
    }
}

template <int BM, int BN, int WGM, int WGN, int NS, bool DMA, bool STREAM, bool OUT32, bool GEGLU>
int launch_tile(I8Args p, hipStream_t st) {
    using T = I8Tile<BM, BN, WGM, WGN, NS>;
    p.tiles_m = ds_cdiv(p.M, BM);
    p.tiles_n = ds_cdiv(p.N, BN);
    const long tiles = (long)p.tiles_m * p.tiles_n;
    DS_CHECK_ARG(tiles * T::NT <= 0xffffffffL, "ds_gemm_i8: M %d x N %d has too many tiles for one launch", p.M, p.N);
    p.group_m = p.tiles_n > 8 ? 8 : 1;
    auto kernel = gemm_i8_tile_kernel<BM, BN, WGM, WGN, NS, DMA, STREAM, OUT32, GEGLU>;
    if (T::LDS > 65536) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)T::LDS);
        if (e != hipSuccess) { ds_set_error("ds_gemm_i8: %s", hipGetErrorString(e)); return DS_ELAUNCH; }
    }
    kernel<<<(int)tiles, T::NT, T::LDS, st>>>(p);
    return DS_OK;
}

template <int BM, int BN, int WGM, int WGN, bool DMA, bool STREAM, int NS>
int launch_tile(const I8Args& p, hipStream_t st) {
    const bool f32 = p.epilogue & DS_EPI_OUT_F32;
    if (p.epilogue & DS_EPI_GEGLU)
        return f32 ? launch_tile<BM, BN, WGM, WGN, NS, DMA, STREAM, true, true>(p, st) : launch_tile<BM, BN, WGM, WGN, NS, DMA, STREAM, false, true>(p, st);
    return f32 ? launch_tile<BM, BN, WGM, WGN, NS, DMA, STREAM, true, false>(p, st) : launch_tile<BM, BN, WGM, WGN, NS, DMA, STREAM, false, false>(p, st);
}

template <int BM, int BN, int WGM, int WGN, bool DMA>
int launch_large(const I8Args& p, bool stream_out, hipStream_t st) {
    return stream_out ? launch_tile<BM, BN, WGM, WGN, DMA, true, 2>(p, st) : launch_tile<BM, BN, WGM, WGN, DMA, false, 2>(p, st);
}

// Which tile: the one whose estimate is the shortest.  Microseconds of a round (every workgroup that fits on the chip at once does one tile) =
// start and end + (bytes per accumulator that go in and out with it) * b + K / 1024 * g, fitted to measurements of M = 300 ... 655360,
// N = 320 ... 10240, K = 320 ... 8192, fp16 and fp32 results with and without a residual (within 20 %).  On either side of the choices: 8192^3 in
// fp16 256 x 256 460 us, 128 x 128 582, 256 x 64 629, 128 x 64 688; 655360 x 320 x 320 on fp32 rows 553, 411, 387, 412; 2048 x 1280 x 1280
// 64 x 64 9.9, 128 x 64 11.3, 256 x 256 20.5; 4096 x 1280 x 1280 64 x 64 16.8, 128 x 64 14.7, 128 x 128 16.4, 256 x 256 22.4.
enum { TILE_256x256, TILE_128x128, TILE_256x64, TILE_128x64, TILE_64x64 };
int choose_tile(const I8Args& p) {
    struct Cost { int m, n, slots; double f, b, g; };
    static const Cost cost[] = {{256, 256, 256, 5.2, 2.35, 11.6}, {128, 128, 512, 5.2, 0.72, 8.8}, {256, 64, 512, 5.0, 0.94, 9.6}, {128, 64, 768, 4.7, 0.68, 7.0}, {64, 64, 768, 4.0, 0.4, 4.3}};
    double bytes = p.epilogue & DS_EPI_OUT_F32 ? 4 : 2;
    if (p.epilogue & DS_EPI_GEGLU) bytes /= 2;
    if (p.residual) bytes += p.epilogue & DS_EPI_RES_F32 ? 4 : 2;
    int best = 0;
    double least = 0;
    for (int t = 0; t < 5; ++t) {
        const Cost& c = cost[t];
        const long tiles = (long)ds_cdiv(p.M, c.m) * ds_cdiv(p.N, c.n), rounds = (tiles + c.slots - 1) / c.slots;
        const double part = (double)tiles / c.slots;          // several workgroups a CU: the next tiles begin before a round is over
        const double us = (c.slots == 256 || rounds == 1 ? rounds : 0.5 * (rounds + part)) * (c.f + bytes * c.b + p.K / 1024.0 * c.g);
        if (t == 0 || us < least) { best = t; least = us; }
    }
    const int forced = (int)DS_TUNE_INT("DS_I8_TILE", -1);     // (the "tune" build variant)
    return forced >= 0 ? forced : best;
}

int launch_tiles(const I8Args& p, bool dma, hipStream_t st) {
    // results that are more than L2 holds (32 MiB)
    const bool stream_out = (long)p.M * p.N * (p.epilogue & DS_EPI_OUT_F32 ? 4 : 2) / (p.epilogue & DS_EPI_GEGLU ? 2 : 1) > (32 << 20);
    if (!dma) {
        // 64 x 64 up to one round of them (2057 x 997 x 1273: 19 us against 23), 128 x 128 behind (20057 x 1997 x 1273: 129 us against 186)
        if ((long)ds_cdiv(p.M, 64) * ds_cdiv(p.N, 64) <= 768) return launch_tile<64, 64, 4, 1, false, false, 2>(p, st);
        return launch_large<128, 128, 2, 2, false>(p, stream_out, st);
    }
    switch (choose_tile(p)) {
        case TILE_256x256: return launch_large<256, 256, 2, 4, true>(p, stream_out, st);
        case TILE_128x128: return launch_large<128, 128, 2, 2, true>(p, stream_out, st);
        case TILE_256x64: return launch_large<256, 64, 8, 1, true>(p, stream_out, st);
        case TILE_128x64: return launch_tile<128, 64, 4, 1, true, false, 2>(p, st);
        default: return launch_tile<64, 64, 4, 1, true, false, 3>(p, st);
    }
}

template <int MT, bool GEGLU>
void launch_few(const I8Args& p, bool odd, hipStream_t st) {
    using F = Few<MT, GEGLU>;
    int waves = 1;                         // as many as let each have all its loads in flight at once
    while (waves * 2 <= F::WAVES && waves * 64 * F::U < p.K) waves *= 2;
    const size_t lds = (size_t)waves * MT * (GEGLU ? 2 : 1) * 1024;
    const int grid = GEGLU ? p.N / 32 : ds_cdiv(p.N, 16);
    if (odd) gemm_i8_few_kernel<MT, GEGLU, true><<<grid, waves * 64, lds, st>>>(p);
    else gemm_i8_few_kernel<MT, GEGLU, false><<<grid, waves * 64, lds, st>>>(p);
}

// At most 64 rows: every workgroup of 16 columns reads all of A, so the few-rows kernel's time goes with (16 + M) N K at ~8.5 TB/s (a workgroup alone, by
// the same fit: 34 GB/s; odd addresses and GEGLU's two weight rows 40 % of that); the 64 x 64 tiles take about as long for one row as for 64, by K,
// while there are no more of them than CUs.  Microseconds of both, within 20 % at 1 ... 64 rows, N = 320 ... 40960, K = 320 ... 4096:
// 16 x 1280 x 1280 3.3 against 6.0, 64 x 4096 x 4096 12.0 / 12.7, 32 x 10240 x 1280 8.6 / 7.1 (GEGLU 10.3 / 6.4), 48 x 40960 x 1280 26.9 / 12.5,
// 32 x 4097 x 4095 18.2 / 21, 64 x 4097 x 4095 29.9 / 21.
bool few_rows(const I8Args& p, bool dma, bool odd) {
    if (p.M > 64) return false;
    const bool geglu = p.epilogue & DS_EPI_GEGLU;
    const double k = p.K / 1024.0, rows = 16.0 * ds_cdiv(p.M, 16), groups = geglu ? p.N / 32 : ds_cdiv(p.N, 16);
    const double mine = ((geglu ? 32 : 16) + rows) * k * 1024;          // bytes of a workgroup
    const double all = groups * mine / 8.5e6 * (geglu ? 2.4 : 1.0), one = mine / 34e3, tiles = ds_cdiv(p.N, 64) / 256.0;
    return 2.0 + (all > one ? all : one) * (odd ? 2.6 : 1.0) < (3.3 + (dma ? 2.3 : odd ? 4.4 : 3.5) * k) * (tiles > 1 ? 0.6 + 0.4 * tiles : 1.0);
}

struct Aligned { bool a, w; size_t bytes_a, bytes_w; int stride; };      // which operands to lay out anew, and where that ends
bool dma_rows(const int8_t* p, int64_t ld, int K) { return ((uintptr_t)p & 15) == 0 && (ld & 15) == 0 && (K & 15) == 0 && 256 * ld < (int64_t)OOB; }

// Operands that LDS-DMA does not take are worth a copy for it where the copy (a launch of ~2 us, in and out at ~4.5 TB/s) costs less than the
// unaligned loads of the product, 0.75 us a K-step for every round of 768 64 x 64 tiles.  With and without: 2057 x 997 x 1273 17.7 and 19.6 us,
// 20057 x 1997 x 1273 97 and 126, 100001 x 2001 x 1001 337 and 488, 1000 x 4097 x 4095 42 and 63; not worth it: 1000 x 997 x 1273 12.6 and
// 10.4, 129 x 4097 x 4095 24.8 and 21.9.
Aligned aligned_copies(const ds_gemm_i8_desc& d, const int8_t* A, const int8_t* W) {
    Aligned c{false, false, 0, 0, (d.K + 15) / 16 * 16};
    if (d.M <= 64 || d.N <= 0 || d.K < 16) return c;
    const bool a = !dma_rows(A, d.lda, d.K), w = !dma_rows(W, d.ldw, d.K);
    const double rounds = (double)ds_cdiv(d.M, 64) * ds_cdiv(d.N, 64) / 768;
    const double moved = 2.0 * d.K * ((a ? d.M : 0.0) + (w ? d.N : 0.0));
    if (!(a || w) || 2.2 + moved / 4.5e6 > 0.75 * d.K / BKB * rounds) return c;
    c.a = a;
    c.w = w;
    c.bytes_a = a ? (size_t)d.M * c.stride : 0;                          // (rows of whole 16s: W's copy begins at a multiple of 16)
    c.bytes_w = w ? (size_t)d.N * c.stride : 0;
    return c;
}

void align_operands(I8Args& p, const Aligned& c, void* workspace, hipStream_t st) {
    AlignArgs q{p.A, p.W, c.a ? static_cast<int8_t*>(workspace) : nullptr, c.w ? static_cast<int8_t*>(workspace) + c.bytes_a : nullptr, p.lda, p.ldw, p.M, p.N, p.K, c.stride, 3};
    while (q.shift < 8 && (16 << q.shift) < c.stride) ++q.shift;
    const long rows = (c.a ? p.M : 0L) + (c.w ? p.N : 0L);
    const long groups = (rows + (256 >> q.shift) - 1) / (256 >> q.shift);
    align_rows_kernel<<<(int)(groups < (1 << 20) ? groups : 1 << 20), 256, 0, st>>>(q);
    if (c.a) { p.A = q.to_a; p.lda = c.stride; }
    if (c.w) { p.W = q.to_w; p.ldw = c.stride; }
    p.K = c.stride;                                                       // one side of every product behind K is a zero
}

int launch_i8(const I8Args& p, bool dma, bool odd, hipStream_t st) {
    if (!few_rows(p, dma, odd)) return launch_tiles(p, dma, st);
    const int tiles = ds_cdiv(p.M, 16);
    if (p.epilogue & DS_EPI_GEGLU) {
        if (tiles == 1) launch_few<1, true>(p, odd, st);
        else if (tiles == 2) launch_few<2, true>(p, odd, st);
        else launch_few<4, true>(p, odd, st);
    } else {
        if (tiles == 1) launch_few<1, false>(p, odd, st);
        else if (tiles == 2) launch_few<2, false>(p, odd, st);
        else if (tiles == 3) launch_few<3, false>(p, odd, st);
        else launch_few<4, false>(p, odd, st);
    }
    return DS_OK;
}

}  // namespace

// what makes a product of these sizes illegal whatever its operands
static int check_desc(const ds_gemm_i8_desc& d) {
    DS_CHECK_ARG(d.M >= 0 && d.N >= 0 && d.K >= 0, "ds_gemm_i8: negative size (M %d, N %d, K %d)", d.M, d.N, d.K);
    DS_CHECK_ARG(d.K <= 131071, "ds_gemm_i8: K %d: the 32-bit sums hold K <= 131071", d.K);
    DS_CHECK_ARG((d.epilogue & ~(DS_EPI_GEGLU | DS_EPI_SILU | DS_EPI_OUT_F32 | DS_EPI_RES_F32)) == 0, "ds_gemm_i8: epilogue %d", d.epilogue);
    const bool geglu = d.epilogue & DS_EPI_GEGLU;
    DS_CHECK_ARG(!(geglu && (d.epilogue & DS_EPI_SILU)), "ds_gemm_i8: GEGLU and SiLU exclude each other");
    DS_CHECK_ARG(!geglu || d.N % 64 == 0, "ds_gemm_i8: GEGLU needs N %% 64 == 0 (32-row groups of values and gates), N %d", d.N);
    return DS_OK;
}

extern "C" size_t ds_gemm_i8_workspace_bytes(const int8_t* A, const int8_t* W, const ds_gemm_i8_desc* desc) {
    if (!desc || check_desc(*desc) != DS_OK) return 0;
    const Aligned c = aligned_copies(*desc, A, W);
    return c.bytes_a + c.bytes_w;
}

extern "C" int ds_gemm_i8(const int8_t* A, const int8_t* W, const float* a_scale, const float* w_scale, const float* bias, const void* residual,
                          void* out, const ds_gemm_i8_desc* desc, void* workspace, size_t workspace_bytes, void* stream) {
    DS_CHECK_ARG(desc, "ds_gemm_i8: desc is NULL");
    const ds_gemm_i8_desc d = *desc;
    const int legal = check_desc(d);
    if (legal != DS_OK) return legal;
    const bool geglu = d.epilogue & DS_EPI_GEGLU;
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
    I8Args p{A, W, a_scale, w_scale, bias, residual, out, d.lda, d.ldw, d.ldr, d.ldc, d.M, d.N, d.K, d.epilogue, 0, 0, 1};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const Aligned copies = aligned_copies(d, A, W);
    if (workspace && copies.bytes_a + copies.bytes_w) {
        DS_CHECK_ARG(((uintptr_t)workspace & 15) == 0 && workspace_bytes >= copies.bytes_a + copies.bytes_w,
                     "ds_gemm_i8: workspace of %zu bytes: %zu at a multiple of 16 are needed", workspace_bytes, copies.bytes_a + copies.bytes_w);
        align_operands(p, copies, workspace, st);
    }
    const bool dma = p.K > 0 && dma_rows(p.A, p.lda, p.K) && dma_rows(p.W, p.ldw, p.K);
    const int rc = launch_i8(p, dma, (((uintptr_t)p.A | (uintptr_t)p.W | p.lda | p.ldw) & 3) != 0, st);
    if (rc != DS_OK) return rc;
    DS_CHECK_LAUNCH("ds_gemm_i8");
    return DS_OK;
}
