// Shared pieces of the microscaled (MX) rows: element formats, scale bytes, loads of the activation types.
//
// A block of 32 consecutive elements of a row shares a scale 2^(b - 127), b one byte (255: the block stands for NaN).
// Elements are E2M1 (4 bits: 0, .5, 1, 1.5, 2, 3, 4, 6 and a sign; low nibble first) or E4M3 (8 bits, up to 448).  Rows
// are padded to whole steps of 128 elements with zero codes and zero scale bytes.
#pragma once
#include "nb_common.hpp"

namespace nb {

typedef int mx_v4i __attribute__((ext_vector_type(4)));
typedef int mx_v8i __attribute__((ext_vector_type(8)));
typedef float mx_v4f __attribute__((ext_vector_type(4)));
typedef short mx_v2s __attribute__((ext_vector_type(2)));
typedef float mx_v2f __attribute__((ext_vector_type(2)));

constexpr int kMxBlock = 32;   // elements per scale
constexpr int kMxStep = 128;   // elements per matrix instruction, and what rows are padded to

struct NoType {};
struct Bf16 {
    uint16_t bits;
};

// 16 bytes at an address that is a multiple of ALIGN only.  The hardware reads and writes memory at any multiple of 2 or 4
// bytes; rows of odd length keep their wide accesses.
template <int ALIGN>
struct MxWords;
template <>
struct MxWords<16> {
    typedef uint32_t type __attribute__((ext_vector_type(4)));
};
template <>
struct MxWords<4> {
    typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct MxWords<2> {
    typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};
template <bool VEC, typename T>
using mx_words = typename MxWords<VEC ? 16 : (int)sizeof(T)>::type;

__device__ __forceinline__ float mx_float(uint32_t w, int half, _Float16)
{
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(half ? w >> 16 : w & 0xFFFFu));
}
__device__ __forceinline__ float mx_float(uint32_t w, int half, Bf16)
{
    return __builtin_bit_cast(float, half ? w & 0xFFFF0000u : w << 16);
}
// 8 consecutive elements at p as floats (VEC: 16-byte aligned); int32 is converted (exact up to 2^24)
template <bool VEC = true, typename T>
__device__ __forceinline__ void mx_load8(float (&v)[8], const T *p)
{
    const auto *q = reinterpret_cast<const mx_words<VEC, T> *>(p);
    if constexpr (sizeof(T) == 4) {
        const auto a = q[0], b = q[1];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (__is_same(T, int32_t))
                v[i] = (float)(int32_t)a[i], v[4 + i] = (float)(int32_t)b[i];
            else
                v[i] = __builtin_bit_cast(float, (uint32_t)a[i]), v[4 + i] = __builtin_bit_cast(float, (uint32_t)b[i]);
        }
    } else {
        const auto a = q[0];
#pragma unroll
        for (int i = 0; i < 4; i++) v[2 * i] = mx_float(a[i], 0, T{}), v[2 * i + 1] = mx_float(a[i], 1, T{});
    }
}
__device__ __forceinline__ float mx_load1(const float *p) { return *p; }
__device__ __forceinline__ float mx_load1(const int32_t *p) { return (float)*p; }
__device__ __forceinline__ float mx_load1(const _Float16 *p) { return (float)*p; }
__device__ __forceinline__ float mx_load1(const Bf16 *p) { return __builtin_bit_cast(float, (uint32_t)p->bits << 16); }
// elements k0 .. k0 + 7 of a row of K, zeros past its end; VEC: K is a multiple of 8 and the address aligned
template <bool VEC, typename T>
__device__ __forceinline__ void mx_load_row8(float (&v)[8], const T *row, int64_t k0, int64_t K)
{
    if (VEC ? k0 < K : k0 + 8 <= K) {
        mx_load8<VEC>(v, row + k0);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = !VEC && k0 + i < K ? mx_load1(row + k0 + i) : 0.f;
    }
}

// fp32 -> the stored types, to nearest, ties to even
__device__ __forceinline__ uint16_t mx_bf16(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
__device__ __forceinline__ uint16_t mx_f16(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
template <bool VEC = true, typename T>
__device__ __forceinline__ void mx_store8(T *p, const float (&v)[8])
{
    auto *q = reinterpret_cast<mx_words<VEC, T> *>(p);
    if constexpr (sizeof(T) == 4) {
        mx_words<VEC, T> a, b;
#pragma unroll
        for (int i = 0; i < 4; i++)
            a[i] = __builtin_bit_cast(uint32_t, v[i]), b[i] = __builtin_bit_cast(uint32_t, v[4 + i]);
        q[0] = a, q[1] = b;
    } else {
        mx_words<VEC, T> a;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (__is_same(T, Bf16))
                a[i] = mx_bf16(v[2 * i]) | ((uint32_t)mx_bf16(v[2 * i + 1]) << 16);
            else
                a[i] = mx_f16(v[2 * i]) | ((uint32_t)mx_f16(v[2 * i + 1]) << 16);
        }
        q[0] = a;
    }
}
__device__ __forceinline__ void mx_store1(float *p, float v) { *p = v; }
__device__ __forceinline__ void mx_store1(_Float16 *p, float v) { *p = (_Float16)v; }
__device__ __forceinline__ void mx_store1(Bf16 *p, float v) { p->bits = mx_bf16(v); }
template <bool VEC, typename T>
__device__ __forceinline__ void mx_store_row8(T *row, int64_t k0, int64_t K, const float (&v)[8])
{
    if (VEC ? k0 < K : k0 + 8 <= K) {
        mx_store8<VEC>(row + k0, v);
    } else if (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (k0 + i < K) mx_store1(row + k0 + i, v[i]);
    }
}

// The scale byte of a block from the largest magnitude's bits: floor(log2 amax) - emax + 127 = exponent field - emax,
// at least 0 (zeros, subnormal blocks), 255 where the block holds an infinity or NaN (their bits compare above every
// finite value's as integers).
template <bool FP8>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits)
{
    const int field = (int)(amax_bits >> 23);
    const int b = field - (FP8 ? 8 : 2);
    return field == 255 ? 255u : (uint32_t)(b < 0 ? 0 : b);
}

// 8 elements -> their codes under scale byte b: 8 nibbles (E2M1, in .x) or 8 bytes (E4M3).  The conversion
// instructions divide by the scale, round to nearest even and saturate at 6; E4M3 would overflow to NaN, so the values
// are clamped to 448 scales first (exact: 448 * 2^(b - 127) is a float for every b <= 246, the largest a finite block
// gives).  A NaN block (b = 255) gets zero codes: its scale says what it is.
template <bool FP8>
__device__ __forceinline__ uint2 mx_codes8(const float (&v)[8], uint32_t b)
{
    if (b == 255u) return make_uint2(0u, 0u);
    // the scale operand 2^(b - 127); for b = 0 that is the subnormal 2^-127
    const float s = __builtin_bit_cast(float, b ? b << 23 : 0x00400000u);
    if (FP8) {
        const float top = 448.0f * s;
        mx_v2s lo = {0, 0}, hi = {0, 0};
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; i++) c[i] = __builtin_amdgcn_fmed3f(v[i], -top, top);
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, c[0], c[1], s, false);
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, c[2], c[3], s, true);
        hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, c[4], c[5], s, false);
        hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, c[6], c[7], s, true);
        return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
    }
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
    return make_uint2(w, 0u);
}

// Block maximum over the four lanes that hold a block's 8 elements each (magnitudes as integers)
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t m)
{
    uint32_t o = dpp_mov<0xB1>(m);   // quad_perm [1,0,3,2]
    m = m > o ? m : o;
    o = dpp_mov<0x4E>(m);            // quad_perm [2,3,0,1]
    return m > o ? m : o;
}

template <bool FP8>
__device__ __forceinline__ void mx_emit8(uint8_t *codes, uint8_t *scales, int64_t piece, const float (&v)[8])
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t a = __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu;
        m = m > a ? m : a;
    }
    const uint32_t b = mx_scale_byte<FP8>(mx_quad_max(m));
    const uint2 c = mx_codes8<FP8>(v, b);
    if (FP8)
        reinterpret_cast<uint2 *>(codes)[piece] = c;
    else
        reinterpret_cast<uint32_t *>(codes)[piece] = c.x;
    if ((piece & 3) == 0) scales[piece >> 2] = (uint8_t)b;
}

inline int64_t mx_padded(int64_t K) { return ceil_div(K, kMxStep) * kMxStep; }

}  // namespace nb
