// One token per row of logits from a supplied word: temperature, top-k, top-p, min-p.
//
// Each of the three filters keeps a prefix of the row in descending order (equal entries by index), so what is kept is
// "above a key, or equal to it at an index up to a cut", without a sort: the key comes from digit-by-digit histograms.
// Weights are integers (a weight of 1 is 2^f), so sums are the same in any order and are accumulated with atomics.
#include <algorithm>

#include "nb_mx.hpp"

namespace nb {

constexpr int64_t kTokenMaxV = 1 << 20;
constexpr int kTokenSeg = 512;                       // entries a wave takes at a time, 8 consecutive ones per lane
constexpr int kTokenMaxSegs = kTokenMaxV / kTokenSeg;

// Order-preserving keys; 0: an entry that is never drawn (NaN, -inf; no int32 entry is).  -0 and +0 are one key.
__device__ __forceinline__ uint32_t token_key(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    const uint32_t k = u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
    return v > -__builtin_inff() ? k : 0u;
}
template <typename T>
struct TokenKey {
    static __device__ __forceinline__ uint32_t key(const T *p) { return token_key(mx_load1(p)); }
    static __device__ __forceinline__ bool drawable(uint32_t k) { return k != 0; }
    static __device__ __forceinline__ double value(uint32_t k)
    {
        return (double)__builtin_bit_cast(float, k ^ (k >> 31 ? 0x80000000u : 0xFFFFFFFFu));
    }
};
template <>
struct TokenKey<int32_t> {
    static __device__ __forceinline__ uint32_t key(const int32_t *p) { return (uint32_t)*p ^ 0x80000000u; }
    static __device__ __forceinline__ bool drawable(uint32_t) { return true; }
    static __device__ __forceinline__ double value(uint32_t k) { return (double)(int32_t)(k ^ 0x80000000u); }
};

struct TokenArgs {
    int32_t *out;
    const void *logits;
    const uint32_t *words;
    const float *temperature, *top_p, *min_p;
    const int32_t *top_k;
    double temperature_all, top_p_all, min_p_all;
    int64_t top_k_all, R;
    int V, frac_bits;
};

struct TokenRow {
    uint32_t kmax;
    double vmax, rate, one;      // exponents per unit of the logits; a weight of 1
};
template <typename T>
__device__ __forceinline__ uint64_t token_weight(const TokenRow &r, uint32_t k)
{
    if (k == r.kmax) return (uint64_t)r.one;             // also where both are +inf
    if (!TokenKey<T>::drawable(k)) return 0;
    return (uint64_t)rint(exp2((TokenKey<T>::value(k) - r.vmax) * r.rate) * r.one);
}

template <typename U>
__device__ __forceinline__ U wave_sum(U v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_tokens_kernel(TokenArgs a)
{
    constexpr int WAVES = THREADS / 64;
    __shared__ uint64_t hist_w[256], seg_w[kTokenMaxSegs];
    __shared__ uint32_t hist_c[256], seg_c[kTokenMaxSegs];
    __shared__ uint32_t sh_key, sh_count, sh_ties;
    __shared__ uint64_t sh_sum;
    __shared__ int sh_digit, sh_cut;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x;
    const int V = a.V, segs = (V + kTokenSeg - 1) / kTokenSeg;
    const T *x = (const T *)a.logits + row * V;
    const auto for_each = [&](auto &&f) {
        for (int s = wave; s < segs; s += WAVES) {
            const int i0 = s * kTokenSeg + lane * 8;
            for (int e = 0; e < 8; e++)
                if (i0 + e < V) f(TokenKey<T>::key(x + i0 + e), i0 + e, s);
        }
    };
    if (threadIdx.x == 0) sh_key = 0, sh_cut = V, sh_sum = 0;
    __syncthreads();
    uint32_t m = 0;
    for_each([&](uint32_t k, int, int) { m = k > m ? k : m; });
    atomicMax(&sh_key, m);
    __syncthreads();
    TokenRow r;
    r.kmax = sh_key;
    if (!TokenKey<T>::drawable(r.kmax)) {
        if (threadIdx.x == 0) a.out[row] = -1;
        return;
    }
    const double temperature = a.temperature ? (double)a.temperature[row] : a.temperature_all;
    if (!(temperature > 0.0)) {
        int first = V;
        for_each([&](uint32_t k, int i, int) { first = k == r.kmax && i < first ? i : first; });
        atomicMin(&sh_cut, first);
        __syncthreads();
        if (threadIdx.x == 0) a.out[row] = sh_cut;
        return;
    }
    r.vmax = TokenKey<T>::value(r.kmax);
    r.rate = std::max(1.4426950408889634 / temperature, 1e-300);   // not 0: -inf * 0 is no exponent
    r.one = (double)(1ull << a.frac_bits);
    const int64_t top_k = a.top_k ? a.top_k[row] : a.top_k_all;
    const double top_p = a.top_p ? (double)a.top_p[row] : a.top_p_all;
    const double min_p = a.min_p ? (double)a.min_p[row] : a.min_p_all;
    const double min_w = std::min(min_p, 1.0) * r.one;

    // what is kept: keys above `key`, and `ties` of those equal to it, the first ones
    uint32_t key = 0, ties = 0xFFFFFFFFu, equal = 0;
    uint64_t total = 0;
    bool cut = false;
    // the shortest prefix of at least k entries, or of a weight of at least target; false: the row does not reach it
    const auto select = [&](bool by_count, int64_t k, double target) {
        uint32_t prefix = 0;
        uint64_t above_w = 0;
        uint32_t above_c = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            for (int t = threadIdx.x; t < 256; t += THREADS) hist_w[t] = 0, hist_c[t] = 0;
            if (threadIdx.x == 0) sh_digit = -1;
            __syncthreads();
            for_each([&](uint32_t q, int, int) {
                if (TokenKey<T>::drawable(q) && (shift == 24 || q >> (shift + 8) == prefix)) {
                    atomicAdd(&hist_c[(q >> shift) & 255], 1u);
                    atomicAdd((unsigned long long *)&hist_w[(q >> shift) & 255], (unsigned long long)token_weight<T>(r, q));
                }
            });
            __syncthreads();
            if (threadIdx.x == 0) {
                for (int d = 255; d >= 0; d--) {
                    const uint32_t c = hist_c[d];
                    if (!c) continue;
                    if (by_count ? (int64_t)above_c + c >= k : (double)(above_w + hist_w[d]) >= target) {
                        sh_digit = d, sh_count = above_c, sh_sum = above_w, sh_ties = c;
                        break;
                    }
                    above_c += c, above_w += hist_w[d];
                }
            }
            __syncthreads();
            if (sh_digit < 0) return false;
            above_c = sh_count, above_w = sh_sum, equal = sh_ties;
            prefix = (prefix << 8) | (uint32_t)sh_digit;
        }
        key = prefix;
        const uint64_t w = token_weight<T>(r, key);
        if (by_count) {
            ties = (uint32_t)(k - above_c);
        } else {
            uint32_t lo = 1, hi = equal;            // the fewest that reach the target
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                if ((double)(above_w + mid * w) >= target) hi = mid;
                else lo = mid + 1;
            }
            ties = lo;
        }
        total = above_w + ties * w;
        cut = true;
        return true;
    };
    if (top_k > 0 && top_k < V) select(true, top_k, 0.0);
    if (top_p < 1.0) {
        if (!cut) {
            uint64_t s = 0;
            for_each([&](uint32_t k, int, int) { s += token_weight<T>(r, k); });
            s = wave_sum(s);
            __syncthreads();
            if (threadIdx.x == 0) sh_sum = 0;
            __syncthreads();
            if (lane == 0) atomicAdd((unsigned long long *)&sh_sum, (unsigned long long)s);
            __syncthreads();
            total = sh_sum;
        }
        select(false, 0, top_p * (double)total);
    }
    // the index of the last tie that is kept
    int last = V;
    if (cut && ties < equal) {
        __syncthreads();
        for (int s = wave; s < segs; s += WAVES) {
            uint32_t c = 0;
            for (int e = 0; e < 8; e++) {
                const int i = s * kTokenSeg + lane * 8 + e;
                c += i < V && TokenKey<T>::key(x + i) == key;
            }
            c = wave_sum(c);
            if (lane == 0) seg_c[s] = c;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t left = ties;
            int s = 0;
            while (left > seg_c[s]) left -= seg_c[s++];
            int i = s * kTokenSeg;
            for (;; i++)
                if (TokenKey<T>::key(x + i) == key && --left == 0) break;
            sh_cut = i;
        }
        __syncthreads();
        last = sh_cut;
    }
    const auto kept = [&](int i) -> uint64_t {
        if (i >= V) return 0;
        const uint32_t k = TokenKey<T>::key(x + i);
        if (k < key || (k == key && i > last)) return 0;
        const uint64_t w = token_weight<T>(r, k);
        return (double)w < min_w ? 0 : w;
    };
    __syncthreads();
    for (int s = wave; s < segs; s += WAVES) {
        uint64_t w = 0;
        for (int e = 0; e < 8; e++) w += kept(s * kTokenSeg + lane * 8 + e);
        w = wave_sum(w);
        if (lane == 0) seg_w[s] = w;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        uint64_t all = 0;
        for (int s = 0; s < segs; s++) all += seg_w[s];
        // sum > word * all / 2^32 for integers: sum > the quotient's whole part
        const uint64_t word = a.words[row];
        uint64_t left = word * (all >> 32) + ((word * (all & 0xFFFFFFFFu)) >> 32);
        int s = 0;
        while (left >= seg_w[s]) left -= seg_w[s++];
        int i = s * kTokenSeg;
        for (uint64_t w; (w = kept(i)) <= left; i++) left -= w;
        a.out[row] = i;
    }
}

template <typename T>
static void token_launch(const TokenArgs &a, hipStream_t st)
{
    const dim3 grid((unsigned)a.R);
    if (a.V <= 2048)
        sample_tokens_kernel<T, 64><<<grid, dim3(64), 0, st>>>(a);
    else
        sample_tokens_kernel<T, 1024><<<grid, dim3(1024), 0, st>>>(a);
}

}  // namespace nb

extern "C" {
int64_t nb_sample_tokens_workspace_bytes(int64_t, int64_t) { return 0; }

int nb_sample_tokens(int32_t *out, const void *logits, int type, const uint32_t *words, const float *temperature,
                     double temperature_all, const int32_t *top_k, int64_t top_k_all, const float *top_p,
                     double top_p_all, const float *min_p, double min_p_all, int64_t R, int64_t V, void *workspace,
                     int64_t workspace_bytes, nb_stream_t stream)
{
    const char *who = "nb_sample_tokens";
    NB_REQUIRE(R >= 0 && V >= 1, "%s: bad shape", who);
    NB_REQUIRE(V <= nb::kTokenMaxV, "%s: rows of %lld entries, at most %lld", who, (long long)V, (long long)nb::kTokenMaxV);
    NB_REQUIRE(R < (1LL << 22), "%s: too many rows", who);
    NB_REQUIRE(type >= NB_TYPE_F32 && type <= NB_TYPE_I32, "%s: type %d", who, type);
    NB_REQUIRE(temperature || temperature_all == temperature_all, "%s: temperature is NaN", who);
    NB_REQUIRE(top_p || top_p_all == top_p_all, "%s: top_p is NaN", who);
    NB_REQUIRE(min_p || min_p_all == min_p_all, "%s: min_p is NaN", who);
    if (R == 0) return NB_OK;
    NB_REQUIRE_PTR(out);
    NB_REQUIRE_PTR(logits);
    NB_REQUIRE_PTR(words);
    NB_REQUIRE_ALIGNED(out, 4);
    NB_REQUIRE_ALIGNED(words, 4);
    NB_REQUIRE_ALIGNED(logits, type == NB_TYPE_F32 || type == NB_TYPE_I32 ? 4 : 2);
    NB_REQUIRE_ALIGNED(temperature, 4);
    NB_REQUIRE_ALIGNED(top_k, 4);
    NB_REQUIRE_ALIGNED(top_p, 4);
    NB_REQUIRE_ALIGNED(min_p, 4);
    (void)workspace, (void)workspace_bytes;
    int log2v = 0;
    while ((1LL << log2v) < V) log2v++;
    const nb::TokenArgs a{out, logits, words, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all,
                          top_k_all, R, (int)V, std::min(52, 61 - log2v)};
    const hipStream_t st = nb::as_stream(stream);
    if (type == NB_TYPE_F32)
        nb::token_launch<float>(a, st);
    else if (type == NB_TYPE_F16)
        nb::token_launch<_Float16>(a, st);
    else if (type == NB_TYPE_BF16)
        nb::token_launch<nb::Bf16>(a, st);
    else
        nb::token_launch<int32_t>(a, st);
    return nb::check_launch(who);
}
}  // extern "C"
