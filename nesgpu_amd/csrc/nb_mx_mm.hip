// Product of microscaled rows: C[m, n] = sum_k A[m, k] B[n, k], A in E2M1 or E4M3, B in E2M1, on the scaled matrix
// instructions (v_mfma_scale_f32_16x16x128_f8f6f4: 128 positions of 16 + 16 rows, a scale byte per row and 32 positions).
//
// Fragments (checked against a plain sum over random codes and scales): lane l supplies row l % 16 and scale byte
// g = l / 16 of the step; of E2M1 the 32 positions 32 g ..., 16 bytes; of E4M3 the positions 16 g ... and 64 + 16 g ...,
// 16 bytes each.  acc[r] is C[4 g + r][l % 16].
//
// Sums.  The instruction adds the products of 8 neighbouring positions at 14 bits below the largest of them before
// they reach the fp32 accumulator: exact for E2M1 x E2M1 (products are multiples of 1/4 up to 36) but not for E4M3, whose
// values span 18 binades: a product 2^-14 of its neighbour is lost (relative error of a sum of normal values 4e-6, with
// a few columns 20 times larger 2e-5, measured over K = 8192).  The E4M3 operand is therefore split in two whose
// products fit: values of magnitude 4 and more (multiples of 1/2 up to 448) and smaller ones (multiples of 2^-9); two
// instructions per step, every sum exact to fp32.
#include <algorithm>

#include "nb_mx.hpp"

namespace nb {

// Bytes of E4M3 codes with magnitude >= 4 (code 0x48) as a mask; NaN (0x7F) among them.
__device__ __forceinline__ uint32_t mx_large_mask(uint32_t a)
{
    const uint32_t h = ((a & 0x7F7F7F7Fu) + 0x38383838u) & 0x80808080u;   // no carry between bytes: 0x7F + 0x38 < 0x100
    return (h << 1) - (h >> 7);
}

template <bool FP8>
struct MxA;
template <>
struct MxA<false> {
    mx_v8i v;
    __device__ __forceinline__ void load(const uint8_t *row, int g)
    {
        const mx_v4i a = *reinterpret_cast<const mx_v4i *>(row + 16 * g);
        v = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
    }
};
template <>
struct MxA<true> {
    mx_v8i v;
    __device__ __forceinline__ void load(const uint8_t *row, int g)
    {
        const mx_v4i a = *reinterpret_cast<const mx_v4i *>(row + 16 * g);
        const mx_v4i b = *reinterpret_cast<const mx_v4i *>(row + 64 + 16 * g);
        v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

__device__ __forceinline__ mx_v8i mx_frag4(const uint8_t *p)
{
    const mx_v4i b = *reinterpret_cast<const mx_v4i *>(p);
    return __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
}

template <typename O>
__device__ __forceinline__ void mx_store_out(O *c, float v) { mx_store1(c, v); }

// A workgroup makes one tile of 16 MT x 16 NT outputs; its W waves take every W-th step of K, fragments straight
// from memory, and their sums meet in shared memory in a fixed order.
template <bool FP8, typename O, int MT, int NT, int W>
__global__ __launch_bounds__(64 * W) void mx_mm_rows_kernel(O *__restrict__ C, const uint8_t *__restrict__ A,
                                                            const uint32_t *__restrict__ As, const uint8_t *__restrict__ B,
                                                            const uint32_t *__restrict__ Bs, int64_t M, int64_t N,
                                                            int64_t steps, int64_t ntiles)
{
    constexpr int ABYTES = FP8 ? 128 : 64;
    __shared__ float part[W][MT * NT][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
    const int64_t mt = blockIdx.x / ntiles, nt = blockIdx.x - mt * ntiles;
    const uint8_t *a[MT], *b[NT];
    const uint32_t *as[MT], *bs[NT];
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int64_t m = std::min<int64_t>(16 * (mt * MT + i) + r16, M - 1);   // rows past the end: the last one again
        a[i] = A + m * steps * ABYTES;
        as[i] = As + m * steps;
    }
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int64_t n = std::min<int64_t>(16 * (nt * NT + j) + r16, N - 1);
        b[j] = B + n * steps * 64;
        bs[j] = Bs + n * steps;
    }
    mx_v4f acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = mx_v4f{0.f, 0.f, 0.f, 0.f};
    for (int64_t s = wave; s < steps; s += W) {
        mx_v8i fb[NT];
        int sb[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) {
            fb[j] = mx_frag4(b[j] + s * 64 + 16 * g);
            sb[j] = (int)(bs[j][s] >> (8 * g));
        }
#pragma unroll
        for (int i = 0; i < MT; i++) {
            MxA<FP8> fa;
            fa.load(a[i] + s * ABYTES, g);
            const int sa = (int)(as[i][s] >> (8 * g));
            if (FP8) {
                mx_v8i hi, lo;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t m = mx_large_mask((uint32_t)fa.v[e]);
                    hi[e] = (int)((uint32_t)fa.v[e] & m);
                    lo[e] = (int)((uint32_t)fa.v[e] & ~m);
                }
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(lo, fb[j], acc[i][j], 0, 4, 0, sa, 0, sb[j]);
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(hi, fb[j], acc[i][j], 0, 4, 0, sa, 0, sb[j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < NT; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fa.v, fb[j], acc[i][j], 4, 4, 0, sa, 0, sb[j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) part[wave][i * NT + j][(4 * g + r) * 16 + r16] = acc[i][j][r];
    __syncthreads();
    for (int t = threadIdx.x; t < MT * NT * 256; t += 64 * W) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) v += part[w][t >> 8][t & 255];
        const int64_t m = 16 * (mt * MT + (t >> 8) / NT) + ((t & 255) >> 4);
        const int64_t n = 16 * (nt * NT + (t >> 8) % NT) + (t & 15);
        if (m < M && n < N) mx_store_out(C + m * N + n, v);
    }
}

struct MmArgs {
    void *C;
    const uint8_t *A, *B;
    const uint32_t *As, *Bs;
    int64_t M, N, steps;
    hipStream_t st;
};

template <bool FP8, typename O>
static int mm_launch(const MmArgs &a, const char *who)
{
    constexpr int MT = 1, NT = 2, W = 4;
    const int64_t mt = ceil_div(a.M, 16 * MT), nt = ceil_div(a.N, 16 * NT);
    NB_REQUIRE(mt * nt < (1LL << 31) / (64 * W) * 2, "%s: too many tiles", who);
    mx_mm_rows_kernel<FP8, O, MT, NT, W><<<dim3((unsigned)(mt * nt)), dim3(64 * W), 0, a.st>>>(
        (O *)a.C, a.A, a.As, a.B, a.Bs, a.M, a.N, a.steps, nt);
    return check_launch(who);
}

}  // namespace nb

extern "C" {
int nb_mx_mm_nt(void *C, int type, const uint8_t *A, const uint8_t *A_scales, int A_format, const uint8_t *B,
                const uint8_t *B_scales, int64_t M, int64_t N, int64_t K, nb_stream_t stream)
{
    const char *who = "nb_mx_mm_nt";
    NB_REQUIRE(M >= 0 && N >= 0 && K >= 1, "%s: bad shape", who);
    NB_REQUIRE(type >= NB_TYPE_F32 && type <= NB_TYPE_BF16, "%s: type %d", who, type);
    NB_REQUIRE(A_format == NB_MX_FP4 || A_format == NB_MX_FP8, "%s: format %d", who, A_format);
    NB_REQUIRE(M < (1LL << 31) && N < (1LL << 31) && K < (1LL << 31), "%s: too large", who);
    if (M * N == 0) return NB_OK;
    NB_REQUIRE_PTR(C);
    NB_REQUIRE_PTR(A);
    NB_REQUIRE_PTR(A_scales);
    NB_REQUIRE_PTR(B);
    NB_REQUIRE_PTR(B_scales);
    NB_REQUIRE_ALIGNED(C, type == NB_TYPE_F32 ? 4 : 2);
    NB_REQUIRE_ALIGNED(A, 16);
    NB_REQUIRE_ALIGNED(B, 16);
    NB_REQUIRE_ALIGNED(A_scales, 4);
    NB_REQUIRE_ALIGNED(B_scales, 4);
    const nb::MmArgs a{C, A, B, reinterpret_cast<const uint32_t *>(A_scales), reinterpret_cast<const uint32_t *>(B_scales),
                       M, N, nb::mx_padded(K) / nb::kMxStep, nb::as_stream(stream)};
    const bool fp8 = A_format == NB_MX_FP8;
    if (type == NB_TYPE_F32) return fp8 ? nb::mm_launch<true, float>(a, who) : nb::mm_launch<false, float>(a, who);
    if (type == NB_TYPE_F16) return fp8 ? nb::mm_launch<true, _Float16>(a, who) : nb::mm_launch<false, _Float16>(a, who);
    return fp8 ? nb::mm_launch<true, nb::Bf16>(a, who) : nb::mm_launch<false, nb::Bf16>(a, who);
}
}  // extern "C"
