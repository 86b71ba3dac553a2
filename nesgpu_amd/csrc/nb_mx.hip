// Microscaled rows: conversion from and to floating rows, and the RMS norm that writes them.
#include <algorithm>

#include "nb_mx.hpp"

namespace nb {

// ---- rows -> MX rows -------------------------------------------------------------------------------------------------
// A lane takes 8 consecutive elements (a "piece"), four lanes a block; pieces run over the padded row.  FLAT: rows of
// whole steps, so that input and output are one run of pieces without rows.
template <typename T, bool FP8, bool VEC, bool FLAT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                                                          const T *__restrict__ x, int64_t pieces, int64_t K,
                                                          int64_t row_pieces)
{
    NB_FLAT_LOOP(t, pieces)
    {
        if (t < pieces) {                      // pieces is a multiple of 16: blocks are whole here
            float v[8];
            if (FLAT) {
                mx_load8(v, x + 8 * t);
            } else {
                const int64_t r = t / row_pieces;
                mx_load_row8<VEC>(v, x + r * K, 8 * (t - r * row_pieces), K);
            }
            mx_emit8<FP8>(codes, scales, t, v);
        }
    }
}

template <typename T, bool FP8, bool VEC, bool FLAT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(T *__restrict__ out, const uint8_t *__restrict__ codes,
                                                            const uint8_t *__restrict__ scales, int64_t pieces, int64_t K,
                                                            int64_t row_pieces)
{
    NB_FLAT_LOOP(t, pieces)
    {
        if (t < pieces) {
            const uint32_t b = scales[t >> 2];
            float v[8];
            if (FP8) {
                const uint2 c = reinterpret_cast<const uint2 *>(codes)[t];
                mx_v2f d[4] = {__builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, false), __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, true),
                               __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, false), __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, true)};
#pragma unroll
                for (int i = 0; i < 4; i++) v[2 * i] = d[i][0], v[2 * i + 1] = d[i][1];
            } else {
                const uint32_t c = reinterpret_cast<const uint32_t *>(codes)[t];
                mx_v2f d[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1),
                               __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3)};
#pragma unroll
                for (int i = 0; i < 4; i++) v[2 * i] = d[i][0], v[2 * i + 1] = d[i][1];
            }
            // the scale as an exponent (exact down to the subnormals, whatever the byte); 255 stands for NaN
#pragma unroll
            for (int i = 0; i < 8; i++)
                v[i] = b == 255u ? __builtin_nanf("") : __builtin_ldexpf(v[i], (int)b - 127);
            if (FLAT) {
                mx_store8(out + 8 * t, v);
            } else {
                const int64_t r = t / row_pieces;
                mx_store_row8<VEC>(out + r * K, 8 * (t - r * row_pieces), K, v);
            }
        }
    }
}

// ---- RMS norm --------------------------------------------------------------------------------------------------------
// h = x + residual (fp32 sum, rounded to the residual's type: what is stored is what is normalised), y = h * r * w with
// r = 1 / sqrt(mean(h^2) + eps).  The sum of squares, r and the products are in 64 bits and y is rounded once to fp32:
// the codes have borders, and a y that is off by an fp32 rounding or two would fall on the other side of one every few
// hundred thousand elements.
struct RowWeight {
    const void *p;
    int type;
};
template <bool VEC>
__device__ __forceinline__ void mx_load_weight8(float (&w)[8], RowWeight weight, int64_t k0, int64_t K)
{
    if (weight.type == NB_TYPE_F32)
        mx_load_row8<VEC>(w, (const float *)weight.p, k0, K);
    else if (weight.type == NB_TYPE_F16)
        mx_load_row8<VEC>(w, (const _Float16 *)weight.p, k0, K);
    else
        mx_load_row8<VEC>(w, (const Bf16 *)weight.p, k0, K);
}

// Eight elements of a row as they lie in memory.  Loads leave them so, and the conversions come after: a row's loads are all
// under way together (converted one by one where they are loaded, the second of 8192 x 8192 rows in bf16 waits for the
// first), and 16-bit values keep to half the registers between the sum and the products.
template <typename T>
struct MxRaw {
    uint32_t w[sizeof(T) == 2 ? 4 : 8] = {};
    template <bool VEC>
    __device__ __forceinline__ void load(const T *row, int64_t k0, int64_t K)   // zeros past the row's end
    {
        if (VEC ? k0 < K : k0 + 8 <= K) {
            const auto *q = reinterpret_cast<const mx_words<VEC, T> *>(row + k0);
#pragma unroll
            for (int j = 0; j < (sizeof(T) == 2 ? 1 : 2); j++) {
                const auto a = q[j];
#pragma unroll
                for (int i = 0; i < 4; i++) w[4 * j + i] = a[i];
            }
        } else if (!VEC) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (k0 + i < K) {
                    if constexpr (sizeof(T) == 2)
                        w[i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, row[k0 + i]) << (16 * (i & 1));
                    else
                        w[i] = __builtin_bit_cast(uint32_t, row[k0 + i]);
                }
        }
    }
    __device__ __forceinline__ void set(int i, float v)                          // rounds; i upwards from a cleared start
    {
        if constexpr (__is_same(T, Bf16))
            w[i / 2] = i & 1 ? w[i / 2] | (uint32_t)mx_bf16(v) << 16 : mx_bf16(v);
        else if constexpr (__is_same(T, _Float16))
            w[i / 2] = i & 1 ? w[i / 2] | (uint32_t)mx_f16(v) << 16 : mx_f16(v);
        else
            w[i] = __builtin_bit_cast(uint32_t, v);
    }
    __device__ __forceinline__ float get(int i) const
    {
        if constexpr (sizeof(T) == 2)
            return mx_float(w[i / 2], i & 1, T{});
        else if constexpr (__is_same(T, int32_t))
            return (float)(int32_t)w[i];
        else
            return __builtin_bit_cast(float, w[i]);
    }
};
// what is normalised: the rows themselves or, with a residual, the sums rounded to its type
template <typename X, typename R>
struct MxHeldAs {
    typedef R type;
};
template <typename X>
struct MxHeldAs<X, NoType> {
    typedef X type;
};
template <bool VEC, int N, typename H, typename X, typename R>
__device__ __forceinline__ void norm_input(MxRaw<H> (&h)[N], const X *x, const R *residual, int64_t p, int64_t T, int64_t K)
{
    if constexpr (__is_same(R, NoType)) {
#pragma unroll
        for (int j = 0; j < N; j++) h[j].template load<VEC>(x, 8 * (p + T * j), K);
    } else {
        MxRaw<X> a[N];
#pragma unroll
        for (int j = 0; j < N; j++) {
            a[j].template load<VEC>(x, 8 * (p + T * j), K);
            h[j].template load<VEC>(residual, 8 * (p + T * j), K);
        }
#pragma unroll
        for (int j = 0; j < N; j++) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = a[j].get(i) + h[j].get(i);
#pragma unroll
            for (int i = 0; i < 8; i++) h[j].set(i, v[i]);
        }
    }
}
template <bool VEC, typename H>
__device__ __forceinline__ void norm_store(H *row, int64_t k0, int64_t K, const MxRaw<H> &h)
{
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = h.get(i);
    mx_store_row8<VEC>(row, k0, K, v);
}

template <int T>
__device__ __forceinline__ double row_sum(double s, double *part)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if (T > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
        __syncthreads();
        s = 0.0;
#pragma unroll
        for (int i = 0; i < T / 64; i++) s += part[i];
    }
    return s;
}

// T threads per row (a workgroup, or for T = 64 a wave of a workgroup of four rows).  N > 0: the row (at most 8 T N
// elements) stays in registers between the sum and the products; N = 0: rows of any length, read again for the products,
// out of the caches for the most part.
//
// Bound by memory: with a residual in bf16 7 + 1/32 bytes an element, 8192 x 8192 in 92 to 102 us (4.6 to 5.1 TB/s; a large
// copy 5.1).  The weights are loaded after the sum: taken before it they cost 16 registers per piece over the barrier and a
// third of the waves (151 us).  Without a residual the 64-bit products and their conversions show: 8192 x 8192 bf16, 3.0 bytes
// an element, 58 to 60 us (3.4 TB/s) over one set of rows, 70 over three in turn; fp32, 5.0 bytes, 79 us (4.3).  Int32 sums
// with an fp16 stream, 4096 x 1024: 8 us out of the caches, 10 to 11 over many sets (3.5 TB/s).
// A wave per row, without barriers, up to 1024 elements: 32768 x 1024 bf16 41 us, 15530 x 547 23 us; a workgroup of 256
// threads 52 and 34, of 128 43 and 24; four pieces a lane, up to 2048: 20000 x 1500 fp32 95 us, 79 with 256 threads.
// One piece per thread: 8 waves a SIMD (64 registers) 16384 x 4096 90 us, 95 with 68 registers; two pieces need their 92.  (int32
// with a 16-bit residual and 512 threads: two of the 64 spill.)
// Rows above 8192 are read twice: 4096 x 16384 bf16 105 us (held by 1024 threads of two pieces 107), 2000 x 32000 fp16
// 107 us (of four pieces 131), 3355 x 20001 fp32 215 us (219).
template <typename X, typename R, bool FP8, bool VEC, int T, int N>
__global__ __launch_bounds__(T == 64 ? 256 : T, N == 1 ? 8 : 1) void rms_norm_mx_kernel(uint8_t *codes, uint8_t *scales, R *residual_out,
                                                                      const X *x, const R *residual, RowWeight weight,
                                                                      double eps, int64_t rows, int64_t K,
                                                                      int64_t row_pieces)
{
    typedef typename MxHeldAs<X, R>::type H;
    __shared__ double part[T / 64 + 1];
    constexpr int kRows = T == 64 ? 4 : 1;
    const int tid = T == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
    for (int64_t row = (int64_t)blockIdx.x * kRows + (T == 64 ? threadIdx.x >> 6 : 0); row < rows;
         row += (int64_t)gridDim.x * kRows) {
        const X *xr = x + row * K;
        const R *rr = residual;
        R *ro = residual_out;
        if constexpr (!__is_same(R, NoType)) rr += row * K, ro += row * K;
        const int64_t out0 = row * row_pieces;
        double s = 0.0;
        if constexpr (N > 0) {
            MxRaw<H> h[N];
            norm_input<VEC>(h, xr, rr, tid, T, K);
#pragma unroll
            for (int j = 0; j < N; j++) {
                if constexpr (!__is_same(R, NoType)) norm_store<VEC>(ro, 8 * (tid + (int64_t)T * j), K, h[j]);
#pragma unroll
                for (int i = 0; i < 8; i++) s = fma((double)h[j].get(i), (double)h[j].get(i), s);
            }
            s = row_sum<T>(s, part);
            const double r = 1.0 / sqrt(s / (double)K + eps);
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int64_t p = tid + (int64_t)T * j;
                float w[8], v[8];
                mx_load_weight8<VEC>(w, weight, 8 * p, K);
                if (p < row_pieces) {                    // whole blocks: row_pieces and T are multiples of 4
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = 8 * p < K ? (float)(((double)h[j].get(i) * r) * (double)w[i]) : 0.f;
                    mx_emit8<FP8>(codes, scales, out0 + p, v);
                }
            }
        } else {
            for (int64_t p = tid; 8 * p < K; p += 2 * T) {
                MxRaw<H> h[2];
                norm_input<VEC>(h, xr, rr, p, T, K);
#pragma unroll
                for (int i = 0; i < 16; i++) s = fma((double)h[i / 8].get(i % 8), (double)h[i / 8].get(i % 8), s);
            }
            s = row_sum<T>(s, part);
            const double r = 1.0 / sqrt(s / (double)K + eps);
            for (int64_t p = tid; p < row_pieces; p += T) {
                float v[8], w[8];
                MxRaw<H> h[1];
                norm_input<VEC>(h, xr, rr, p, 0, K);
                mx_load_weight8<VEC>(w, weight, 8 * p, K);
                if constexpr (!__is_same(R, NoType)) norm_store<VEC>(ro, 8 * p, K, h[0]);
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = 8 * p < K ? (float)(((double)h[0].get(i) * r) * (double)w[i]) : 0.f;
                mx_emit8<FP8>(codes, scales, out0 + p, v);
            }
        }
        if (T > 64) __syncthreads();   // part[] is free for the next row
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------
static int mx_shape_check(int64_t rows, int64_t K, int format, const char *who)
{
    NB_REQUIRE(rows >= 0 && K >= 0, "%s: negative shape", who);
    NB_REQUIRE(format == NB_MX_FP4 || format == NB_MX_FP8, "%s: format %d", who, format);
    NB_REQUIRE(K <= (1LL << 40) && rows <= (1LL << 40) && (K == 0 || rows <= (1LL << 46) / mx_padded(K)), "%s: too large", who);
    return NB_OK;
}

template <typename T, bool FP8>
static void quantize_launch(uint8_t *codes, uint8_t *scales, const void *x, int64_t rows, int64_t K, hipStream_t st)
{
    const int64_t rp = mx_padded(K) / 8, pieces = rows * rp;
    const dim3 grid(grid_for(pieces)), block(256);
    const bool vec = K % 8 == 0 && aligned(x, 16);
    if (vec && K % kMxStep == 0)
        mx_quantize_kernel<T, FP8, true, true><<<grid, block, 0, st>>>(codes, scales, (const T *)x, pieces, K, rp);
    else if (vec)
        mx_quantize_kernel<T, FP8, true, false><<<grid, block, 0, st>>>(codes, scales, (const T *)x, pieces, K, rp);
    else
        mx_quantize_kernel<T, FP8, false, false><<<grid, block, 0, st>>>(codes, scales, (const T *)x, pieces, K, rp);
}

template <typename T, bool FP8>
static void dequantize_launch(void *out, const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t K,
                              hipStream_t st)
{
    const int64_t rp = mx_padded(K) / 8, pieces = rows * rp;
    const dim3 grid(grid_for(pieces)), block(256);
    const bool vec = K % 8 == 0 && aligned(out, 16);
    if (vec && K % kMxStep == 0)
        mx_dequantize_kernel<T, FP8, true, true><<<grid, block, 0, st>>>((T *)out, codes, scales, pieces, K, rp);
    else if (vec)
        mx_dequantize_kernel<T, FP8, true, false><<<grid, block, 0, st>>>((T *)out, codes, scales, pieces, K, rp);
    else
        mx_dequantize_kernel<T, FP8, false, false><<<grid, block, 0, st>>>((T *)out, codes, scales, pieces, K, rp);
}

struct NormArgs {
    uint8_t *codes, *scales;
    void *residual_out;
    const void *x, *residual;
    RowWeight weight;
    double eps;
    int64_t rows, K;
    hipStream_t st;
};

template <typename X, typename R, bool FP8, bool VEC, int T, int N>
static void norm_launch_n(const NormArgs &a)
{
    const int64_t groups = T == 64 ? ceil_div(a.rows, 4) : a.rows;
    rms_norm_mx_kernel<X, R, FP8, VEC, T, N>
        <<<dim3((unsigned)std::min<int64_t>(groups, 1 << 20)), dim3(T == 64 ? 256 : T), 0, a.st>>>(
            a.codes, a.scales, (R *)a.residual_out, (const X *)a.x, (const R *)a.residual, a.weight, a.eps, a.rows, a.K,
            mx_padded(a.K) / 8);
}

template <typename X, typename R, bool FP8, bool VEC>
static void norm_launch_vec(const NormArgs &a)
{
    const int64_t Kp = mx_padded(a.K);
    if (Kp <= 64 * 8)
        norm_launch_n<X, R, FP8, VEC, 64, 1>(a);
    else if (Kp <= 64 * 16)
        norm_launch_n<X, R, FP8, VEC, 64, 2>(a);
    else if (Kp <= 256 * 8)
        norm_launch_n<X, R, FP8, VEC, 256, 1>(a);
    else if (Kp <= 512 * 8)
        norm_launch_n<X, R, FP8, VEC, 512, 1>(a);
    else if (Kp <= 512 * 16)
        norm_launch_n<X, R, FP8, VEC, 512, 2>(a);
    else
        norm_launch_n<X, R, FP8, VEC, 1024, 0>(a);
}

template <typename X, typename R>
static void norm_launch(const NormArgs &a, int format, bool vec)
{
    if (format == NB_MX_FP8)
        vec ? norm_launch_vec<X, R, true, true>(a) : norm_launch_vec<X, R, true, false>(a);
    else
        vec ? norm_launch_vec<X, R, false, true>(a) : norm_launch_vec<X, R, false, false>(a);
}

}  // namespace nb

extern "C" {
int nb_mx_quantize(uint8_t *codes, uint8_t *scales, const void *x, int type, int format, int64_t rows, int64_t K,
                   nb_stream_t stream)
{
    const char *who = "nb_mx_quantize";
    if (int rc = nb::mx_shape_check(rows, K, format, who)) return rc;
    NB_REQUIRE(type == NB_TYPE_F32 || type == NB_TYPE_F16 || type == NB_TYPE_BF16, "%s: type %d", who, type);
    if (rows * K == 0) return NB_OK;
    NB_REQUIRE_PTR(codes);
    NB_REQUIRE_PTR(scales);
    NB_REQUIRE_PTR(x);
    NB_REQUIRE_ALIGNED(codes, 16);
    NB_REQUIRE_ALIGNED(scales, 4);
    NB_REQUIRE_ALIGNED(x, type == NB_TYPE_F32 ? 4 : 2);
    const hipStream_t st = nb::as_stream(stream);
    const bool fp8 = format == NB_MX_FP8;
    if (type == NB_TYPE_F32)
        fp8 ? nb::quantize_launch<float, true>(codes, scales, x, rows, K, st)
            : nb::quantize_launch<float, false>(codes, scales, x, rows, K, st);
    else if (type == NB_TYPE_F16)
        fp8 ? nb::quantize_launch<_Float16, true>(codes, scales, x, rows, K, st)
            : nb::quantize_launch<_Float16, false>(codes, scales, x, rows, K, st);
    else
        fp8 ? nb::quantize_launch<nb::Bf16, true>(codes, scales, x, rows, K, st)
            : nb::quantize_launch<nb::Bf16, false>(codes, scales, x, rows, K, st);
    return nb::check_launch(who);
}

int nb_mx_dequantize(void *out, int type, const uint8_t *codes, const uint8_t *scales, int format, int64_t rows,
                     int64_t K, nb_stream_t stream)
{
    const char *who = "nb_mx_dequantize";
    if (int rc = nb::mx_shape_check(rows, K, format, who)) return rc;
    NB_REQUIRE(type == NB_TYPE_F32 || type == NB_TYPE_F16 || type == NB_TYPE_BF16, "%s: type %d", who, type);
    if (rows * K == 0) return NB_OK;
    NB_REQUIRE_PTR(out);
    NB_REQUIRE_PTR(codes);
    NB_REQUIRE_PTR(scales);
    NB_REQUIRE_ALIGNED(codes, 16);
    NB_REQUIRE_ALIGNED(scales, 4);
    NB_REQUIRE_ALIGNED(out, type == NB_TYPE_F32 ? 4 : 2);
    const hipStream_t st = nb::as_stream(stream);
    const bool fp8 = format == NB_MX_FP8;
    if (type == NB_TYPE_F32)
        fp8 ? nb::dequantize_launch<float, true>(out, codes, scales, rows, K, st)
            : nb::dequantize_launch<float, false>(out, codes, scales, rows, K, st);
    else if (type == NB_TYPE_F16)
        fp8 ? nb::dequantize_launch<_Float16, true>(out, codes, scales, rows, K, st)
            : nb::dequantize_launch<_Float16, false>(out, codes, scales, rows, K, st);
    else
        fp8 ? nb::dequantize_launch<nb::Bf16, true>(out, codes, scales, rows, K, st)
            : nb::dequantize_launch<nb::Bf16, false>(out, codes, scales, rows, K, st);
    return nb::check_launch(who);
}

int nb_rms_norm_mx(uint8_t *codes, uint8_t *scales, void *residual_out, const void *x, int x_type, const void *residual,
                   int residual_type, const void *weight, int weight_type, double eps, int format, int64_t rows,
                   int64_t K, nb_stream_t stream)
{
    const char *who = "nb_rms_norm_mx";
    if (int rc = nb::mx_shape_check(rows, K, format, who)) return rc;
    NB_REQUIRE(x_type >= NB_TYPE_F32 && x_type <= NB_TYPE_I32, "%s: type %d", who, x_type);
    NB_REQUIRE(weight_type >= NB_TYPE_F32 && weight_type <= NB_TYPE_BF16, "%s: weight type %d", who, weight_type);
    NB_REQUIRE(eps >= 0.0, "%s: eps must not be negative", who);
    const bool with = residual != nullptr || residual_out != nullptr;
    if (with)
        NB_REQUIRE(residual_type >= NB_TYPE_F32 && residual_type <= NB_TYPE_BF16 &&
                       (x_type == NB_TYPE_I32 || residual_type == x_type),
                   "%s: a residual of type %d with inputs of type %d", who, residual_type, x_type);
    if (rows * K == 0) return NB_OK;
    NB_REQUIRE_PTR(codes);
    NB_REQUIRE_PTR(scales);
    NB_REQUIRE_PTR(x);
    NB_REQUIRE_PTR(weight);
    NB_REQUIRE_ALIGNED(codes, 16);
    NB_REQUIRE_ALIGNED(scales, 4);
    const auto size = [](int t) { return t == NB_TYPE_F32 || t == NB_TYPE_I32 ? 4 : 2; };
    NB_REQUIRE_ALIGNED(x, size(x_type));
    NB_REQUIRE_ALIGNED(weight, size(weight_type));
    if (with) {
        NB_REQUIRE_PTR(residual);
        NB_REQUIRE_PTR(residual_out);
        NB_REQUIRE_ALIGNED(residual, size(residual_type));
        NB_REQUIRE_ALIGNED(residual_out, size(residual_type));
    }
    const bool vec = K % 8 == 0 && nb::aligned(x, 16) && nb::aligned(weight, 16) &&
                     (!with || (nb::aligned(residual, 16) && nb::aligned(residual_out, 16)));
    const nb::NormArgs a{codes, scales, residual_out, x, residual, {weight, weight_type}, eps, rows, K, nb::as_stream(stream)};
    if (x_type == NB_TYPE_F32)
        with ? nb::norm_launch<float, float>(a, format, vec) : nb::norm_launch<float, nb::NoType>(a, format, vec);
    else if (x_type == NB_TYPE_F16)
        with ? nb::norm_launch<_Float16, _Float16>(a, format, vec) : nb::norm_launch<_Float16, nb::NoType>(a, format, vec);
    else if (x_type == NB_TYPE_BF16)
        with ? nb::norm_launch<nb::Bf16, nb::Bf16>(a, format, vec) : nb::norm_launch<nb::Bf16, nb::NoType>(a, format, vec);
    else if (!with)
        nb::norm_launch<int32_t, nb::NoType>(a, format, vec);
    else if (residual_type == NB_TYPE_F32)
        nb::norm_launch<int32_t, float>(a, format, vec);
    else if (residual_type == NB_TYPE_F16)
        nb::norm_launch<int32_t, _Float16>(a, format, vec);
    else
        nb::norm_launch<int32_t, nb::Bf16>(a, format, vec);
    return nb::check_launch(who);
}
}  // extern "C"
