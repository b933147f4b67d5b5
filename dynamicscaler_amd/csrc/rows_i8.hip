// Rows in 8 bits: the root-mean-square norm with the residual's addition (8-bit, fp16 or fp32 result), the quantisation of rows with one
// scale each, and the way back.
//
//   norm      h = x + r;  t = h g;  root = 1 / sqrt(mean(h^2) + eps);  y = t root
//   8 bits    top = max |t|;  q = rint(127 t / top)  (the root cancels);  scale = top root / 127
//   quantize  the same with t = x, root = 1
// t is formed and compared in 64 bits and the sums are 64-bit, so q is the correctly rounded quotient (halves to even) of the inputs as
// they are given: it does not depend on the order of a reduction.  A row without a largest value (all zeros) has q = 0, scale = 0; a row that
// holds a NaN or an infinity (in x, r or t) has q = 0, scale = NaN: it stands for NaN throughout.
// fp16 results are rounded once, from the 64-bit value (by way of a rounding to odd: fp16 rows of 655360 x 320 164 us a call, 159 with two roundings).
#include "common.h"

namespace {

struct RowsArgs {
    const void* x; const void* r; const float* g; void* h; void* y; float* scale;
    long ldx, ldr, ldh, ldy;
    int C;
    float eps;
    double inv_C;
};

template <typename T> __device__ __forceinline__ double as_f64(T v) { return (double)(float)v; }

// rint(127 t / top), exactly, from an estimate v of 127 |t| / top that is off by less than a quarter: 254 |t| against the odd multiple of top that
// is the half above floor(v) (both exact for fp16 / fp32 t)
__device__ __forceinline__ int quantum(double t, double top, double v) {
    const double k = floor(v), d = fma(-fma(2.0, k, 1.0), top, 254.0 * fabs(t));
    const int i = (int)k, q = i + (d > 0.0 || (d == 0.0 && (i & 1)) ? 1 : 0);
    return t < 0.0 ? -q : q;
}

// 1 / sqrt(s) for s > 0: the hardware's 2^-23 and one Newton step (2^-44); 0 for an infinite s
__device__ __forceinline__ double inverse_root(double s) {
    const double y = __builtin_amdgcn_rsq(s);
    return s < __builtin_huge_val() ? y * fma(-0.5 * s * y, y, 1.5) : s != s ? s : 0.0;
}

// Sum / maximum over the T lanes of a team (a power of two, at most a wave), the same bits in every lane: two quad permutes, two mirrors,
// two swaps of 16 and 32 lanes -- no trip through LDS.
__device__ __forceinline__ void swap16(double v, double& a, double& b) {
    const unsigned long long u = __double_as_longlong(v);
    const auto lo = __builtin_amdgcn_permlane16_swap((unsigned)u, (unsigned)u, false, false), hi = __builtin_amdgcn_permlane16_swap((unsigned)(u >> 32), (unsigned)(u >> 32), false, false);
    a = __longlong_as_double(lo[0] | (unsigned long long)hi[0] << 32);
    b = __longlong_as_double(lo[1] | (unsigned long long)hi[1] << 32);
}
__device__ __forceinline__ void swap32(double v, double& a, double& b) {
    const unsigned long long u = __double_as_longlong(v);
    const auto lo = __builtin_amdgcn_permlane32_swap((unsigned)u, (unsigned)u, false, false), hi = __builtin_amdgcn_permlane32_swap((unsigned)(u >> 32), (unsigned)(u >> 32), false, false);
    a = __longlong_as_double(lo[0] | (unsigned long long)hi[0] << 32);
    b = __longlong_as_double(lo[1] | (unsigned long long)hi[1] << 32);
}
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
    const unsigned long long u = __double_as_longlong(v);
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (unsigned)u, CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_update_dpp(0, (unsigned)(u >> 32), CTRL, 0xf, 0xf, true);
    return __longlong_as_double(lo | (unsigned long long)hi << 32);
}
template <int T, typename F> __device__ __forceinline__ double team_reduce(double v, F&& op) {
    if constexpr (T >= 2) v = op(v, dpp<0xB1>(v));        // lane ^ 1
    if constexpr (T >= 4) v = op(v, dpp<0x4E>(v));        // lane ^ 2
    if constexpr (T >= 8) v = op(v, dpp<0x141>(v));       // 7 - lane of 8
    if constexpr (T >= 16) v = op(v, dpp<0x140>(v));      // 15 - lane of 16
    double a, b;
    if constexpr (T >= 32) { swap16(v, a, b); v = op(a, b); }
    if constexpr (T >= 64) { swap32(v, a, b); v = op(a, b); }
    return v;
}
template <int T> __device__ __forceinline__ double team_sum(double v) { return team_reduce<T>(v, [](double a, double b) { return a + b; }); }
template <int T> __device__ __forceinline__ double team_max(double v) { return team_reduce<T>(v, [](double a, double b) { return fmax(a, b); }); }

// 8 values of a row as they lie in memory (any address that is a multiple of the element's size), as fp32 (exact for fp16), and back
typedef f16x8 __attribute__((aligned(2))) f16x8_u;
typedef f32x4 __attribute__((aligned(4))) f32x4_u;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 __attribute__((aligned(1))) u32x2_u;

// v + lost (v rounded to nearest, `lost` what the rounding took away) rounded to odd: towards zero, and the last bit set where that lost anything.  What
// goes on to fp16 from there is rounded once in effect (von Neumann's rounding: fp32 has the two spare bits that it needs).
__device__ __forceinline__ float to_odd(float v, float lost) {
    const unsigned u = __float_as_uint(v), towards_zero = (int)(__float_as_uint(lost) ^ u) >> 31;
    return fabsf(lost) > 0.0f ? __uint_as_float((u + towards_zero) | 1) : v;        // (no for the NaN that an infinite v leaves)
}
// the same for 64 bits, to the 21 that the upper word holds (and fp32 takes as they are)
__device__ __forceinline__ double to_odd(double v) {
    const unsigned long long u = __double_as_longlong(v);
    return __longlong_as_double((unsigned long long)((unsigned)(u >> 32) | min((unsigned)u, 1u)) << 32);
}

template <typename T> struct Chunk;
template <> struct Chunk<f16> {
    f16x8 v;
    __device__ __forceinline__ void zero() { v = f16x8{0, 0, 0, 0, 0, 0, 0, 0}; }
    __device__ __forceinline__ void load(const f16* p) { v = *reinterpret_cast<const f16x8_u*>(p); }
    __device__ __forceinline__ void hold() { asm volatile("" : "+v"(v)); }
    __device__ __forceinline__ float at(int j) const { return (float)v[j]; }
    __device__ __forceinline__ void set(int j, float x) { v[j] = (f16)x; }
    __device__ __forceinline__ void set(int j, double x) { set(j, (float)to_odd(x)); }
    __device__ __forceinline__ void store(f16* p) const { *reinterpret_cast<f16x8_u*>(p) = v; }
};
template <> struct Chunk<float> {
    f32x4 v[2];
    __device__ __forceinline__ void zero() { v[0] = v[1] = f32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void hold() { asm volatile("" : "+v"(v[0]), "+v"(v[1])); }
    __device__ __forceinline__ void load(const float* p) {
        v[0] = *reinterpret_cast<const f32x4_u*>(p);
        v[1] = *reinterpret_cast<const f32x4_u*>(p + 4);
    }
    __device__ __forceinline__ float at(int j) const { return v[j >> 2][j & 3]; }
    __device__ __forceinline__ void set(int j, float x) { v[j >> 2][j & 3] = x; }
    __device__ __forceinline__ void set(int j, double x) { set(j, (float)x); }
    __device__ __forceinline__ void store(float* p) const {
        *reinterpret_cast<f32x4_u*>(p) = v[0];
        *reinterpret_cast<f32x4_u*>(p + 4) = v[1];
    }
};
template <> struct Chunk<int8_t> {
    u32x2 v;
    __device__ __forceinline__ void zero() { v = u32x2{0, 0}; }
    __device__ __forceinline__ void put(int j, int q) { v[j >> 2] |= (unsigned)(q & 255) << (8 * (j & 3)); }
    __device__ __forceinline__ void store(int8_t* p) const { *reinterpret_cast<u32x2_u*>(p) = v; }
};

// Rows of 8 ... 8 T V values: a team of T lanes (of one wave for T <= 64, a whole workgroup above) keeps a row in registers -- read once,
// reduced twice, written once; lane i of the team holds chunks i, i + T, ... of 8 values, so a load covers 16 T contiguous bytes (fp16).
// A row's last chunk always ends at the row's end: where C % 8 != 0 it overlaps the one before, counts its own values only in the sum, and
// stores the same bits over the shared ones (every load of a row comes before its first store, also where sum / y lie over an input).
// A team walks rows `grid` apart and keeps its part of gamma.  Bound by memory: 655360 x 320 with an fp32 residual (11 bytes a value) 472 us = 4.9 TB/s,
// the quantisation of 40960 x 5120 (3 bytes) 134 us = 4.7 TB/s, where a copy of 4 GiB reaches 4.75.  A few rows are bound by instruction
// fetch: one row of 1280 takes 3.5 us, of which the launch alone is 1.8, and took 4.9 with an exact branch at every value.
template <typename X, typename R, typename Y, bool NORM, bool RES, int T, int V>
__global__ void __launch_bounds__(T > 256 ? T : 256) rows_team_kernel(RowsArgs p, int rows) {
    constexpr int TEAMS = T > 256 ? 1 : 256 / T, WAVES = T / 64;
    constexpr bool I8 = sizeof(Y) == 1;
    __shared__ double s_sum[2][WAVES > 1 ? WAVES : 1], s_top[2][WAVES > 1 ? WAVES : 1];
    const int tid = threadIdx.x, lane = tid % T, team = tid / T;
    const int C = p.C;
    auto chunk = [&](int v) { return (v * T + lane) * 8; };            // where the lane's chunk v would begin: it has one if that is < C,
    auto at = [&](int v) { return min(chunk(v), C - 8); };              // and it begins here
    Chunk<float> g[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if constexpr (NORM) {
            g[v].zero();
            if (chunk(v) < C) g[v].load(p.g + at(v));
        }
    }
    int turn = 0;
    for (long row0 = (long)blockIdx.x * TEAMS; row0 < rows; row0 += (long)gridDim.x * TEAMS, turn ^= 1) {
        const long row = row0 + team;
        const bool live = row < rows;          // teams of one wave: the reductions below need every lane
        const long rr = live ? row : rows - 1;
        const X* x = reinterpret_cast<const X*>(p.x) + rr * p.ldx;
        const R* r = reinterpret_cast<const R*>(p.r) + rr * p.ldr;
        Chunk<X> cx[V];
        Chunk<R> cr[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (v * T * 8 >= C) break;
            cx[v].zero();
            if constexpr (RES) cr[v].zero();
            if (chunk(v) < C) {
                cx[v].load(x + at(v));
                if constexpr (RES) cr[v].load(r + at(v));
            }
        }
        auto h_of = [&](int v, int j) {
            double h = (double)cx[v].at(j);
            if constexpr (RES) h += (double)cr[v].at(j);
            return h;
        };
        auto t_of = [&](int v, int j) { return NORM ? h_of(v, j) * (double)g[v].at(j) : h_of(v, j); };
        if constexpr (NORM) {
#pragma unroll
            for (int v = 0; v < V; ++v) g[v].hold();      // gamma stays in 32 bits between the rows
        }
        double sum = 0.0, top = 0.0;
        float topf = 0.0f, bad = 0.0f;                    // NaN or infinite where a value of the row (a gamma) is
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (v * T * 8 >= C) break;
            if constexpr (NORM) {
                const int shared = chunk(v) < C ? chunk(v) - at(v) : 0;       // values that belong to the chunk before
                if (shared == 0) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) { const double h = h_of(v, j); sum = fma(h, h, sum); }
                } else {
#pragma unroll
                    for (int j = 1; j < 8; ++j) { const double h = j < shared ? 0.0 : h_of(v, j); sum = fma(h, h, sum); }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (NORM) {
                    if constexpr (I8) {
                        top = fmax(top, fabs(t_of(v, j)));
                        bad = fmaf(0.0f, g[v].at(j), bad);
                    }
                } else {
                    topf = fmaxf(topf, fabsf(cx[v].at(j)));
                    bad = fmaf(0.0f, cx[v].at(j), bad);
                }
            }
        }
        if constexpr (!NORM) top = topf;
        if (I8 && bad != 0.0f) top = __builtin_huge_val();     // fmax passes NaN over: an infinity stands for it from here on
        if constexpr (NORM) sum = team_sum<(T < 64 ? T : 64)>(sum);
        if constexpr (I8) top = team_max<(T < 64 ? T : 64)>(top);
        if constexpr (T > 64) {
            if ((tid & 63) == 0) { s_sum[turn][tid >> 6] = sum; s_top[turn][tid >> 6] = top; }
            __syncthreads();                    // two copies in turn: the next row's stores come a barrier after this row's loads
            sum = s_sum[turn][0];
            top = s_top[turn][0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) {
                sum += s_sum[turn][w];
                top = fmax(top, s_top[turn][w]);
            }
        }
        const double root = NORM ? inverse_root(sum * p.inv_C + (double)p.eps) : 1.0;
        const bool off = I8 && (!(sum < __builtin_huge_val()) || !(top < __builtin_huge_val()));
        const bool none = off || top == 0.0;              // every q is 0
        // 32-bit quotients v = t (127 / top): t carries two roundings of 2^-24, 127 / top two, v one -- within 3.8e-5 of the quotient, |v| <= 127 --
        // decide all but the values within 2^-14 of a half (one in 8000); rows whose h, t or 127 / top are no ordinary fp32 numbers are done exactly
        // (a small gamma hides an x + r beyond fp32 from top; h^2 <= sum < 1e76 does not)
        const bool in32 = none || (top < 1e36 && top > 1e-30 && (!RES || sum < 1e76));
        const float inv32 = none || !in32 ? 0.0f : 127.0f / (float)top;
        double inv = 0.0;
        if (I8 && !in32) inv = 127.0 / top;
        if (I8 && live && lane == 0) p.scale[row] = off ? __builtin_nanf("") : (float)(top * root * (1.0 / 127.0));
        Y* y = reinterpret_cast<Y*>(p.y) + rr * p.ldy;
        R* hs = reinterpret_cast<R*>(p.h) + rr * p.ldh;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (v * T * 8 >= C) break;
            cx[v].hold();                    // the raw values stay in registers, their 64-bit forms are made again (half the registers)
            if constexpr (RES) cr[v].hold();
            if constexpr (NORM) g[v].hold();
            const bool mine = live && chunk(v) < C;
            Chunk<Y> cy;
            cy.zero();
            if constexpr (I8) {
                int q[8];
                bool near = !in32;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float t = cx[v].at(j);
                    if constexpr (RES) t += cr[v].at(j);
                    if constexpr (NORM) t *= g[v].at(j);
                    const float w = none ? 0.0f : t * inv32, n = rintf(w);
                    q[j] = (int)n;
                    near |= fabsf(w - n) > 0.5f - 0x1p-14f;
                }
                if (near) {                  // once for the chunk, so that the way past it is short
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const double t = t_of(v, j);
                        q[j] = quantum(t, top, in32 ? fabs((double)((float)t * inv32)) : fabs(t) * inv);
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) cy.put(j, q[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) cy.set(j, t_of(v, j) * root);
            }
            if (mine) cy.store(y + at(v));
            if constexpr (RES) {
                Chunk<R> ch;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // (the fp32 sum of two fp16 values is exact wherever it is near a half of fp16)
                    if constexpr (sizeof(X) == 4 && sizeof(R) == 2) ch.set(j, h_of(v, j));
                    else ch.set(j, cx[v].at(j) + cr[v].at(j));
                }
                if (mine && p.h) ch.store(hs + at(v));
            }
        }
    }
}

// Longer rows, and rows of less than 8 values: one workgroup per row and turn, the row read for the sums and again for the result.
template <typename X, typename R, typename Y, bool NORM>
__global__ void __launch_bounds__(1024) rows_long_kernel(RowsArgs p, int rows) {
    __shared__ double s_sum[16], s_top[16];
    const int tid = threadIdx.x;
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
        const X* x = reinterpret_cast<const X*>(p.x) + row * p.ldx;
        const R* r = p.r ? reinterpret_cast<const R*>(p.r) + row * p.ldr : nullptr;
        auto h_of = [&](int c) { return r ? as_f64(x[c]) + as_f64(r[c]) : as_f64(x[c]); };
        double sum = 0.0, top = 0.0;
        for (int c = tid; c < p.C; c += blockDim.x) {
            const double h = h_of(c);
            sum += h * h;
            const double t = fabs(NORM ? h * (double)p.g[c] : h);
            top = fmax(top, t < __builtin_huge_val() ? t : __builtin_huge_val());        // an infinity stands for NaN too
        }
        sum = team_sum<64>(sum);
        top = team_max<64>(top);
        __syncthreads();                     // the row before has been read
        if ((tid & 63) == 0) { s_sum[tid >> 6] = sum; s_top[tid >> 6] = top; }
        __syncthreads();
        sum = 0.0;
        for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
            sum += s_sum[w];
            top = fmax(top, s_top[w]);
        }
        const double root = NORM ? inverse_root(sum * p.inv_C + (double)p.eps) : 1.0;
        if constexpr (sizeof(Y) == 1) {
            const bool bad = !(sum < __builtin_huge_val()) || !(top < __builtin_huge_val());
            const double inv = top > 0.0 && !bad ? 127.0 / top : 0.0;
            int8_t* q = reinterpret_cast<int8_t*>(p.y) + row * p.ldy;
            if (tid == 0) p.scale[row] = bad ? __builtin_nanf("") : (float)(top * root * (1.0 / 127.0));
            for (int c = tid; c < p.C; c += blockDim.x) {
                const double h = h_of(c), t = NORM ? h * (double)p.g[c] : h;
                q[c] = (int8_t)(inv > 0.0 ? quantum(t, top, fabs(t) * inv) : 0);
                if constexpr (NORM) {
                    if (p.h) reinterpret_cast<R*>(p.h)[row * p.ldh + c] = (R)h;
                }
            }
        } else {
            Y* y = reinterpret_cast<Y*>(p.y) + row * p.ldy;
            for (int c = tid; c < p.C; c += blockDim.x) {
                const double h = h_of(c);
                y[c] = (Y)(h * (double)p.g[c] * root);
                if (p.h) reinterpret_cast<R*>(p.h)[row * p.ldh + c] = (R)h;
            }
        }
    }
}

// The chunks of 8 values of all rows in one sequence, `span` of them a workgroup (per_row of them a row; magic: i / per_row = i * magic >> 40 for
// i < per_row + span, both < 2^16): every lane has work whatever the row's length, and its loads are all on their way before the first product.  C >= 8;
// a row's last chunk ends at the row's end.  655360 x 320 to fp16 105 us a call (6.0 TB/s; 113 with each product rounded to odd), to fp32 208 (270 with
// the loads a turn apart); 3001 x 1283, in the cache, 3.8 us (4.2).
template <typename Y>
__global__ void __launch_bounds__(256) dequant_kernel(const int8_t* __restrict__ q8, long ldq, const float* __restrict__ scale, Y* __restrict__ y, long ldy, int rows, int C,
                                                      unsigned per_row, unsigned long long magic, int span) {
    const unsigned long long first = (unsigned long long)blockIdx.x * span;
    const long row0 = first / per_row;
    const unsigned in0 = (unsigned)(first - row0 * per_row);
    constexpr int TURNS = 4;
    long row[TURNS];
    int c[TURNS];
    float s[TURNS];
    u32x2 v[TURNS];
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
        if (256 * t >= span) break;
        const unsigned i = in0 + threadIdx.x + 256 * t, r = (unsigned)((i * magic) >> 40);
        row[t] = row0 + r;
        c[t] = min((int)(i - r * per_row) * 8, C - 8);
        if (row[t] < rows) {
            s[t] = scale[row[t]];
            v[t] = *reinterpret_cast<const u32x2_u*>(q8 + row[t] * ldq + c[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
        if (256 * t >= span || row[t] >= rows) break;
        auto q = [&](int j) { return (float)((int)(v[t][j >> 2] << (24 - 8 * (j & 3))) >> 24); };
        Chunk<Y> cy;
        // fp16: a product whose fp32 rounding lies halfway between two results (one in 8192; anything of a row with subnormal ones) is rounded to odd
        bool again = sizeof(Y) == 2 && !(fabsf(s[t]) >= 0x1p-14f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float p = q(j) * s[t];
            cy.set(j, p);
            again |= sizeof(Y) == 2 && (__float_as_uint(p) & 0x1fff) == 0x1000;
        }
        if (sizeof(Y) == 2 && again) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = q(j) * s[t];
                cy.set(j, to_odd(p, fmaf(q(j), s[t], -p)));
            }
        }
        cy.store(y + row[t] * ldy + c[t]);
    }
}

// ... and value by value: rows of less than 8 values, or of more chunks than `magic` takes
template <typename Y>
__global__ void __launch_bounds__(256) dequant_any_kernel(const int8_t* __restrict__ q, long ldq, const float* __restrict__ scale, Y* __restrict__ y, long ldy, int rows, int C) {
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
        const float s = scale[row];
        for (int c = threadIdx.x; c < C; c += blockDim.x) y[row * ldy + c] = (Y)((double)q[row * ldq + c] * (double)s);
    }
}

template <typename Y>
void launch_dequant(const int8_t* q, long ldq, const float* scale, Y* y, long ldy, int rows, int C, hipStream_t st) {
    const unsigned per_row = ds_cdiv(C, 8);
    const long chunks = (long)per_row * rows;
    const int span = chunks >= 1024 * 1024 ? 1024 : 256;        // four chunks a lane once they fill the chip
    if (C < 8 || per_row + span >= 65536 || ds_cdiv(chunks, span) > 0xffffff) {
        dequant_any_kernel<Y><<<rows < (1 << 20) ? rows : 1 << 20, C < 64 ? 64 : 256, 0, st>>>(q, ldq, scale, y, ldy, rows, C);
        return;
    }
    const unsigned long long magic = ((1ull << 40) + per_row - 1) / per_row;
    dequant_kernel<Y><<<ds_cdiv(chunks, span), 256, 0, st>>>(q, ldq, scale, y, ldy, rows, C, per_row, magic, span);
}

bool rows_dtype(int t) { return t == DS_F16 || t == DS_F32; }
bool aligned(const void* p, int dtype) { return ((uintptr_t)p & (dtype == DS_I8 ? 0 : dtype == DS_F32 ? 3 : 1)) == 0; }

template <typename X, typename R, typename Y, bool NORM, bool RES>
void launch_rows(const RowsArgs& p, int rows, hipStream_t st) {
    // the smallest team whose four chunks a lane hold the row; a norm's teams walk several rows, with gamma in registers, once the chip is
    // full (16 waves a CU)
    constexpr int V = 4;
    constexpr int MOST = 1 << 20;        // workgroups of a launch: every kernel walks what is left
    auto grid = [&](int teams) { const int n = ds_cdiv(rows, teams), most = NORM ? 256 * 4 : MOST; return n < most ? n : most; };
    if (p.C < 8) rows_long_kernel<X, R, Y, NORM><<<rows < MOST ? rows : MOST, 64, 0, st>>>(p, rows);
    else if (p.C <= 8 * 8 * V) rows_team_kernel<X, R, Y, NORM, RES, 8, V><<<grid(32), 256, 0, st>>>(p, rows);
    else if (p.C <= 16 * 8 * V) rows_team_kernel<X, R, Y, NORM, RES, 16, V><<<grid(16), 256, 0, st>>>(p, rows);
    else if (p.C <= 32 * 8 * V) rows_team_kernel<X, R, Y, NORM, RES, 32, V><<<grid(8), 256, 0, st>>>(p, rows);
    else if (p.C <= 64 * 8 * V) rows_team_kernel<X, R, Y, NORM, RES, 64, V><<<grid(4), 256, 0, st>>>(p, rows);
    else if (p.C <= 256 * 8 * V) rows_team_kernel<X, R, Y, NORM, RES, 256, V><<<grid(1), 256, 0, st>>>(p, rows);
    else if (p.C <= 512 * 8 * V) rows_team_kernel<X, R, Y, NORM, RES, 512, V><<<grid(1), 512, 0, st>>>(p, rows);
    else {
        if constexpr (!NORM) {         // (a norm's registers do not fit 1024 threads)
            if (p.C <= 1024 * 8 * V) {
                rows_team_kernel<X, R, Y, NORM, RES, 1024, V><<<grid(1), 1024, 0, st>>>(p, rows);
                return;
            }
        }
        rows_long_kernel<X, R, Y, NORM><<<rows < MOST ? rows : MOST, 1024, 0, st>>>(p, rows);
    }
}

template <typename X, typename R, bool RES>
void launch_norm(const RowsArgs& p, int y_dtype, int rows, hipStream_t st) {
    if (y_dtype == DS_I8) launch_rows<X, R, int8_t, true, RES>(p, rows, st);
    else if (y_dtype == DS_F16) launch_rows<X, R, f16, true, RES>(p, rows, st);
    else launch_rows<X, R, float, true, RES>(p, rows, st);
}

}  // namespace

extern "C" int ds_rmsnorm_rows(const void* x, const void* residual, const float* gamma, void* sum, void* y, float* scale, const ds_rmsnorm_desc* desc, void* stream) {
    DS_CHECK_ARG(desc, "ds_rmsnorm_rows: desc is NULL");
    const int64_t ldx = desc->ldx, ldr = desc->ldr, lds = desc->lds, ldy = desc->ldy;
    const int rows = desc->rows, C = desc->C, x_dtype = desc->x_dtype, r_dtype = desc->r_dtype, y_dtype = desc->y_dtype;
    const float eps = desc->eps;
    DS_CHECK_ARG(rows >= 0 && C >= 1, "ds_rmsnorm_rows: rows %d, C %d", rows, C);
    DS_CHECK_ARG(rows_dtype(x_dtype) && (!residual || rows_dtype(r_dtype)), "ds_rmsnorm_rows: x / residual type %d / %d", x_dtype, r_dtype);
    DS_CHECK_ARG(y_dtype == DS_I8 || rows_dtype(y_dtype), "ds_rmsnorm_rows: result type %d", y_dtype);
    DS_CHECK_ARG(eps > 0.0f && eps < __builtin_huge_valf(), "ds_rmsnorm_rows: eps has to be positive");
    if (rows == 0) return DS_OK;
    DS_CHECK_ARG(x && gamma && y && (scale || y_dtype != DS_I8), "ds_rmsnorm_rows: a pointer is NULL");
    DS_CHECK_ARG(!sum || residual, "ds_rmsnorm_rows: a sum without a residual");
    DS_CHECK_ARG(ldx >= C && ldy >= C && (!residual || ldr >= C) && (!sum || lds >= C), "ds_rmsnorm_rows: a row stride is shorter than C %d", C);
    DS_CHECK_ARG(aligned(x, x_dtype) && aligned(residual, r_dtype) && aligned(sum, r_dtype) && aligned(y, y_dtype) && aligned(gamma, DS_F32) && aligned(scale, DS_F32),
                 "ds_rmsnorm_rows: a pointer is not aligned to its element");
    const RowsArgs p{x, residual, gamma, sum, y, scale, ldx, ldr, lds, ldy, C, eps, 1.0 / C};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const bool xf = x_dtype == DS_F32, rf = r_dtype == DS_F32;
    if (!residual) {
        if (xf) launch_norm<float, f16, false>(p, y_dtype, rows, st);
        else launch_norm<f16, f16, false>(p, y_dtype, rows, st);
    } else if (rf) {
        if (xf) launch_norm<float, float, true>(p, y_dtype, rows, st);
        else launch_norm<f16, float, true>(p, y_dtype, rows, st);
    } else {
        if (xf) launch_norm<float, f16, true>(p, y_dtype, rows, st);
        else launch_norm<f16, f16, true>(p, y_dtype, rows, st);
    }
    DS_CHECK_LAUNCH("ds_rmsnorm_rows");
    return DS_OK;
}

extern "C" int ds_quantize_rows_i8(const void* x, int x_dtype, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int rows, int C, void* stream) {
    DS_CHECK_ARG(rows >= 0 && C >= 1, "ds_quantize_rows_i8: rows %d, C %d", rows, C);
    DS_CHECK_ARG(rows_dtype(x_dtype), "ds_quantize_rows_i8: x type %d", x_dtype);
    if (rows == 0) return DS_OK;
    DS_CHECK_ARG(x && q && scale, "ds_quantize_rows_i8: a pointer is NULL");
    DS_CHECK_ARG(ldx >= C && ldq >= C, "ds_quantize_rows_i8: a row stride is shorter than C %d", C);
    DS_CHECK_ARG(aligned(x, x_dtype) && aligned(scale, DS_F32), "ds_quantize_rows_i8: a pointer is not aligned to its element");
    const RowsArgs p{x, nullptr, nullptr, nullptr, q, scale, ldx, 0, 0, ldq, C, 0.0f, 1.0 / C};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (x_dtype == DS_F32) launch_rows<float, f16, int8_t, false, false>(p, rows, st);
    else launch_rows<f16, f16, int8_t, false, false>(p, rows, st);
    DS_CHECK_LAUNCH("ds_quantize_rows_i8");
    return DS_OK;
}

extern "C" int ds_dequantize_rows_i8(const int8_t* q, int64_t ldq, const float* scale, void* y, int y_dtype, int64_t ldy, int rows, int C, void* stream) {
    DS_CHECK_ARG(rows >= 0 && C >= 1, "ds_dequantize_rows_i8: rows %d, C %d", rows, C);
    DS_CHECK_ARG(rows_dtype(y_dtype), "ds_dequantize_rows_i8: result type %d", y_dtype);
    if (rows == 0) return DS_OK;
    DS_CHECK_ARG(q && scale && y, "ds_dequantize_rows_i8: a pointer is NULL");
    DS_CHECK_ARG(ldq >= C && ldy >= C, "ds_dequantize_rows_i8: a row stride is shorter than C %d", C);
    DS_CHECK_ARG(aligned(y, y_dtype) && aligned(scale, DS_F32), "ds_dequantize_rows_i8: a pointer is not aligned to its element");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (y_dtype == DS_F32) launch_dequant<float>(q, ldq, scale, (float*)y, ldy, rows, C, st);
    else launch_dequant<f16>(q, ldq, scale, (f16*)y, ldy, rows, C, st);
    DS_CHECK_LAUNCH("ds_dequantize_rows_i8");
    return DS_OK;
}
