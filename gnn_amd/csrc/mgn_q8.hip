// Rows of activations in 8 bits with one scale per row, for the backward pass: code = nearest whole number (ties to even) of
// x * factor with factor = fl(127 / m), scale = fl(m / 127), m = the row's largest magnitude.  The product is rounded once
// (a fused multiply-add onto 1.5 * 2^23, whose last place is one), so a code never depends on how x * factor rounds in fp32.
//
// Memory bound: 4 (2) bytes read and 1 written per element and 4 per row.  32 lanes share a row, each with 16-byte pieces,
// so a row of 128 fp32 values is one load per lane; several rows per lane are requested before the first is reduced.
// Measured at 1 498 001 x 128 fp32: kept in 202 us, restored in 159 us, 0.97 GB each: 4.8 and 6.1 TB/s (a large copy 4.8).
#include "mgn_device.h"

namespace {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr float SMALLEST = 0x1p-119f;          // rows below this keep no codes: 127 / m would overflow

template <int DT> struct Elem;                  // MGN_F32 0, MGN_BF16 1, MGN_F16 2
template <> struct Elem<0> { using T = float; using V = f32x4; };
template <> struct Elem<1> { using T = __bf16; using V = bf16x4; };
template <> struct Elem<2> { using T = _Float16; using V = f16x4; };

// four elements of a row from column c; without VEC (odd widths) one by one, zeros past the end
template <int DT, bool VEC>
__device__ __forceinline__ f32x4 load4(const void* base, long long row, int width, int c) {
    using T = typename Elem<DT>::T;
    const T* p = (const T*)base + row * width + c;
    if constexpr (VEC) return __builtin_convertvector(*(const typename Elem<DT>::V*)p, f32x4);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e < width) v[e] = (float)p[e];
    return v;
}

template <int DT, int NCH, int U, bool VEC>
__global__ __launch_bounds__(256) void q8_rows_kernel(const void* __restrict__ x, signed char* __restrict__ codes, float* __restrict__ scale,
                                                      long long rows, int width, int keep) {
    const int l = threadIdx.x & 31, r = threadIdx.x >> 5;
    const long long row0 = (long long)blockIdx.x * (8 * U) + r;
    f32x4 v[U][NCH];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < NCH; ++n) {
            const int c = 4 * (l + 32 * n);
            const long long row = row0 + 8 * u;
            v[u][n] = row < rows && c < width ? load4<DT, VEC>(x, row, width, c) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long row = row0 + 8 * u;
        unsigned top = 0;                       // magnitudes compare as whole numbers; a NaN is above every other
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[u][n][e]) & 0x7fffffffu);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
        const float m = __uint_as_float(top);
        const bool finite = top < 0x7f800000u;  // a row that holds an infinity or a NaN comes back as NaN
        const float by = finite && m >= SMALLEST ? 127.0f / m : 0.f;
        if (row >= rows) continue;
        if (l == 0) scale[row] = finite ? m / 127.0f : __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int n = 0; n < NCH; ++n) {
            const int c = 4 * (l + 32 * n);
            if (c >= width) continue;
            int q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float k = finite ? __builtin_fmaf(v[u][n][e], by, 12582912.0f) - 12582912.0f : 0.f;
                q[e] = (int)fminf(fmaxf(k, -127.f), 127.f);
                if (keep && q[e] == 0 && v[u][n][e] != 0.f) q[e] = v[u][n][e] > 0.f ? 1 : -1;
            }
            signed char* p = codes + row * width + c;
            if constexpr (VEC) {
                *(unsigned*)p = (unsigned)(q[0] & 255) | (unsigned)(q[1] & 255) << 8 | (unsigned)(q[2] & 255) << 16 | (unsigned)(q[3] & 255) << 24;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < width) p[e] = (signed char)q[e];
            }
        }
    }
}

// x = code * scale, four elements per thread and step
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void q8_restore_kernel(const signed char* __restrict__ codes, const float* __restrict__ scale, void* __restrict__ x,
                                                         long long rows, int width) {
    using T = typename Elem<DT>::T;
    const int per = (width + 3) / 4;
    const long long n = rows * per;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long row = per == 32 ? i >> 5 : i / per;
        const int c = 4 * (int)(i - row * per);
        const float s = scale[row];
        const signed char* p = codes + row * width + c;
        T* o = (T*)x + row * width + c;
        if constexpr (VEC) {
            const unsigned w = *(const unsigned*)p;
            const f32x4 v = {(float)(int)(signed char)w * s, (float)(int)(signed char)(w >> 8) * s, (float)(int)(signed char)(w >> 16) * s,
                             (float)((int)w >> 24) * s};
            *(typename Elem<DT>::V*)o = __builtin_convertvector(v, typename Elem<DT>::V);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < width) o[e] = (T)((float)p[e] * s);
        }
    }
}

constexpr long long LAUNCH_ROWS = 1 << 26;      // a launch has fewer than 2^32 threads, 32 (or 8) of them for a row

template <int DT, int NCH, int U>
void rows_vec(bool vec, const void* x, signed char* codes, float* scale, long long rows, int width, int keep, hipStream_t st) {
    for (long long at = 0; at < rows; at += LAUNCH_ROWS) {
        const long long n = rows - at < LAUNCH_ROWS ? rows - at : LAUNCH_ROWS;
        const void* xs = (const typename Elem<DT>::T*)x + at * width;
        signed char* cs = codes + at * width;
        const dim3 grid((unsigned)((n + 8 * U - 1) / (8 * U)));
        if (vec) hipLaunchKernelGGL((q8_rows_kernel<DT, NCH, U, true>), grid, dim3(256), 0, st, xs, cs, scale + at, n, width, keep);
        else hipLaunchKernelGGL((q8_rows_kernel<DT, NCH, U, false>), grid, dim3(256), 0, st, xs, cs, scale + at, n, width, keep);
    }
}
template <int DT>
void rows_dt(bool vec, const void* x, signed char* codes, float* scale, long long rows, int width, int keep, hipStream_t st) {
    if (width <= 128) rows_vec<DT, 1, 4>(vec, x, codes, scale, rows, width, keep, st);
    else if (width <= 256) rows_vec<DT, 2, 2>(vec, x, codes, scale, rows, width, keep, st);
    else if (width <= 512) rows_vec<DT, 4, 1>(vec, x, codes, scale, rows, width, keep, st);
    else rows_vec<DT, 8, 1>(vec, x, codes, scale, rows, width, keep, st);
}
template <int DT>
void restore_dt(bool vec, const signed char* codes, const float* scale, void* x, long long rows, int width, hipStream_t st) {
    const long long n = rows * ((width + 3) / 4);
    long long g = (n + 255) / 256;
    if (g > 65536) g = 65536;
    if (vec) hipLaunchKernelGGL((q8_restore_kernel<DT, true>), dim3((unsigned)g), dim3(256), 0, st, codes, scale, x, rows, width);
    else hipLaunchKernelGGL((q8_restore_kernel<DT, false>), dim3((unsigned)g), dim3(256), 0, st, codes, scale, x, rows, width);
}

int q8_check(const void* x, const void* codes, const void* scale, int64_t rows, int32_t width, int32_t dtype, const char* name) {
    const char* bad = nullptr;
    if (dtype < 0 || dtype > 2) bad = "unknown type";
    else if (rows < 0 || rows >= (1ll << 31)) bad = "row count out of range";
    else if (width < 1 || width > 1024) bad = "width must be 1 .. 1024";
    else if (rows > 0 && (!x || !codes || !scale)) bad = "null pointer";
    else if (rows > 0 && (((uintptr_t)x & (dtype == MGN_F32 ? 3 : 1)) || ((uintptr_t)scale & 3))) bad = "misaligned pointer";
    if (bad) { mgn_set_error("%s: %s", name, bad); return MGN_E_ARG; }
    return 0;
}

bool q8_vec(const void* x, const void* codes, int32_t width, int32_t dtype) {
    return width % 4 == 0 && ((uintptr_t)codes & 3) == 0 && ((uintptr_t)x & (dtype == MGN_F32 ? 15 : 7)) == 0;
}

}  // namespace

extern "C" int mgn_q8_rows(const void* x, int32_t dtype, int64_t rows, int32_t width, int32_t keep_nonzero, int8_t* codes, float* scale, void* stream) {
    if (const int rc = q8_check(x, codes, scale, rows, width, dtype, "mgn_q8_rows")) return rc;
    if (rows == 0) return 0;
    const bool vec = q8_vec(x, codes, width, dtype);
    const hipStream_t st = (hipStream_t)stream;
    signed char* c = (signed char*)codes;
    if (dtype == MGN_F32) rows_dt<0>(vec, x, c, scale, rows, width, keep_nonzero, st);
    else if (dtype == MGN_BF16) rows_dt<1>(vec, x, c, scale, rows, width, keep_nonzero, st);
    else rows_dt<2>(vec, x, c, scale, rows, width, keep_nonzero, st);
    return check_launch("mgn_q8_rows");
}

extern "C" int mgn_q8_restore(const int8_t* codes, const float* scale, int64_t rows, int32_t width, int32_t dtype, void* x, void* stream) {
    if (const int rc = q8_check(x, codes, scale, rows, width, dtype, "mgn_q8_restore")) return rc;
    if (rows == 0) return 0;
    const bool vec = q8_vec(x, codes, width, dtype);
    const hipStream_t st = (hipStream_t)stream;
    const signed char* c = (const signed char*)codes;
    if (dtype == MGN_F32) restore_dt<0>(vec, c, scale, x, rows, width, st);
    else if (dtype == MGN_BF16) restore_dt<1>(vec, c, scale, x, rows, width, st);
    else restore_dt<2>(vec, c, scale, x, rows, width, st);
    return check_launch("mgn_q8_restore");
}
