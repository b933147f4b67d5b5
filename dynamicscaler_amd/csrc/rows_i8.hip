// Rows in 8 bits: the root-mean-square norm with the residual's addition (8-bit, fp16 or fp32 result), the quantisation of rows with one
// scale each, and the way back.
//
//   norm      h = x + r;  t = h g;  root = 1 / sqrt(mean(h^2) + eps);  y = t root
//   8 bits    top = max |t|;  q = rint(127 t / top)  (the root cancels);  scale = top root / 127
//   quantize  the same with t = x, root = 1
// t is formed and compared in 64 bits and the sums are 64-bit, so q is the correctly rounded quotient (halves to even) of the inputs as
// they are given: it does not depend on the order of a reduction.  A row without a largest value (all zeros) has q = 0, scale = 0; a row that
// holds a NaN or an infinity (in x, r or t) has q = 0, scale = NaN: it stands for NaN throughout.
#include "common.h"

namespace {

struct RowsArgs {
    const void* x; const void* r; const float* g; void* h; void* y; float* scale;
    long ldx, ldr, ldh, ldy;
    int C;
    float eps;
};

template <typename T> __device__ __forceinline__ double as_f64(T v) { return (double)(float)v; }

// rint(127 t / top), exactly: the quotient in 64 bits decides unless it is next to a half, where 254 |t| is compared with an odd multiple of
// top (both exact for fp16 / fp32 t)
__device__ __forceinline__ int quantum(double t, double top, double inv) {
    const double v = fabs(t) * inv;
    double q = rint(v);
    if (fabs(fabs(v - q) - 0.5) < 1e-9) {
        const double k = floor(v);                   // the half is k + 0.5
        const double d = fma(-(2.0 * k + 1.0), top, 254.0 * fabs(t));
        q = d > 0.0 ? k + 1.0 : d < 0.0 ? k : 2.0 * rint(0.5 * k + 0.25);
    }
    return t < 0.0 ? -(int)q : (int)q;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ unsigned long long wave_max(unsigned long long v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long u = __shfl_xor(v, o);
        v = u > v ? u : v;
    }
    return v;
}

// One workgroup per row, the row read once for the sums and once for the result.
template <typename X, typename R, typename Y, bool NORM>
__global__ void __launch_bounds__(256) rows_kernel(RowsArgs p) {
    __shared__ double s_sum[4];
    __shared__ unsigned long long s_top[4];
    const long row = blockIdx.x;
    const int tid = threadIdx.x;
    const X* x = reinterpret_cast<const X*>(p.x) + row * p.ldx;
    const R* r = p.r ? reinterpret_cast<const R*>(p.r) + row * p.ldr : nullptr;
    auto h_of = [&](int c) { return r ? as_f64(x[c]) + as_f64(r[c]) : as_f64(x[c]); };
    double sum = 0.0;
    unsigned long long top = 0;       // bit patterns of non-negative doubles order like the values, infinities and NaN above them
    for (int c = tid; c < p.C; c += 256) {
        const double h = h_of(c);
        sum += h * h;
        const double t = NORM ? h * (double)p.g[c] : h;
        const unsigned long long b = __double_as_longlong(fabs(t));
        top = b > top ? b : top;
    }
    sum = wave_sum(sum);
    top = wave_max(top);
    if ((tid & 63) == 0) { s_sum[tid >> 6] = sum; s_top[tid >> 6] = top; }
    __syncthreads();
    sum = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    top = s_top[0];
    for (int w = 1; w < 4; ++w) top = s_top[w] > top ? s_top[w] : top;
    const double root = NORM ? 1.0 / sqrt(sum / p.C + (double)p.eps) : 1.0;
    const double dtop = __longlong_as_double(top);
    if constexpr (sizeof(Y) == 1) {
        const bool bad = !(sum < __builtin_huge_val()) || !(dtop < __builtin_huge_val());
        const double inv = dtop > 0.0 && !bad ? 127.0 / dtop : 0.0;
        int8_t* q = reinterpret_cast<int8_t*>(p.y) + row * p.ldy;
        if (tid == 0) p.scale[row] = bad ? __builtin_nanf("") : (float)(dtop * root / 127.0);
        for (int c = tid; c < p.C; c += 256) {
            const double h = h_of(c);
            q[c] = (int8_t)(inv > 0.0 ? quantum(NORM ? h * (double)p.g[c] : h, dtop, inv) : 0);
            if constexpr (NORM) {
                if (p.h) reinterpret_cast<R*>(p.h)[row * p.ldh + c] = (R)h;
            }
        }
    } else {
        Y* y = reinterpret_cast<Y*>(p.y) + row * p.ldy;
        for (int c = tid; c < p.C; c += 256) {
            const double h = h_of(c);
            y[c] = (Y)(float)(h * root * (double)p.g[c]);
            if (p.h) reinterpret_cast<R*>(p.h)[row * p.ldh + c] = (R)h;
        }
    }
}

template <typename Y>
__global__ void __launch_bounds__(256) dequant_kernel(const int8_t* q, long ldq, const float* scale, Y* y, long ldy, int C) {
    const long row = blockIdx.x;
    const float s = scale[row];
    for (int c = threadIdx.x; c < C; c += 256) y[row * ldy + c] = (Y)((float)q[row * ldq + c] * s);
}

bool rows_dtype(int t) { return t == DS_F16 || t == DS_F32; }
bool aligned(const void* p, int dtype) { return ((uintptr_t)p & (dtype == DS_I8 ? 0 : dtype == DS_F32 ? 3 : 1)) == 0; }

template <typename X, typename R, bool NORM>
void launch_y(const RowsArgs& p, int y_dtype, int rows, hipStream_t st) {
    if (y_dtype == DS_I8) rows_kernel<X, R, int8_t, NORM><<<rows, 256, 0, st>>>(p);
    else if constexpr (NORM) {
        if (y_dtype == DS_F16) rows_kernel<X, R, f16, NORM><<<rows, 256, 0, st>>>(p);
        else rows_kernel<X, R, float, NORM><<<rows, 256, 0, st>>>(p);
    }
}

}  // namespace

extern "C" int ds_rmsnorm_rows(const void* x, int x_dtype, int64_t ldx, const void* residual, int r_dtype, int64_t ldr, const float* gamma,
                               void* sum, int64_t lds, void* y, int y_dtype, int64_t ldy, float* scale, int rows, int C, float eps, void* stream) {
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
    const RowsArgs p{x, residual, gamma, sum, y, scale, ldx, ldr, lds, ldy, C, eps};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const bool xf = x_dtype == DS_F32, rf = residual && r_dtype == DS_F32;
    if (xf && rf) launch_y<float, float, true>(p, y_dtype, rows, st);
    else if (xf) launch_y<float, f16, true>(p, y_dtype, rows, st);
    else if (rf) launch_y<f16, float, true>(p, y_dtype, rows, st);
    else launch_y<f16, f16, true>(p, y_dtype, rows, st);
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
    const RowsArgs p{x, nullptr, nullptr, nullptr, q, scale, ldx, 0, 0, ldq, C, 0.0f};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (x_dtype == DS_F32) launch_y<float, float, false>(p, DS_I8, rows, st);
    else launch_y<f16, f16, false>(p, DS_I8, rows, st);
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
    if (y_dtype == DS_F32) dequant_kernel<float><<<rows, 256, 0, st>>>(q, ldq, scale, (float*)y, ldy, C);
    else dequant_kernel<f16><<<rows, 256, 0, st>>>(q, ldq, scale, (f16*)y, ldy, C);
    DS_CHECK_LAUNCH("ds_dequantize_rows_i8");
    return DS_OK;
}
