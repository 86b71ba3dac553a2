// One token per row of logits from a supplied word: temperature, top-k, top-p, min-p.
//
// Each of the three filters keeps a prefix of the row in descending order (equal entries by index), so what is kept is
// "above a key, or equal to it at an index up to a cut", without a sort: a histogram over the logits' distance below the
// row's maximum names the bin the border lies in, and only that bin's entries are looked at digit by digit.  Weights are
// integers (a weight of 1 is 2^f): sums over a row are the same in any order, and are accumulated with atomics.
//
// Rows of at most 64 entries: a wave per row, ranks by comparing all pairs.  Up to 16384: a workgroup per row.  Longer
// ones: one kernel over chunks of 8192 entries (the exponentials, which bound the whole, are then spread over the card
// however few the rows), one workgroup per row to finish from the chunks' histograms.
// Measured (MI355X, logits N(0, 2.5^2)): see the table in the launch function.
#include <algorithm>

#include "nb_mx.hpp"

namespace nb {

constexpr int64_t kTokenMaxV = 1 << 20;
constexpr int kTokenLocalV = 16384;                  // rows that one workgroup handles from beginning to end
constexpr int kGroup = 8;                            // entries of a lane's load: aligned pieces of memory, whatever the row's start
constexpr int kSegGroups = 64;                       // a segment: the groups of one load of a wave
constexpr int kTokenMaxSegs = kTokenMaxV / (kGroup * kSegGroups) + 1;
constexpr int kChunkGroups = 1024;
constexpr int kTokenMaxChunks = kTokenMaxV / (kGroup * kChunkGroups) + 1;
constexpr int kSlots = 256;                          // bins of 1/8 of an octave of the weights below the maximum; the last
                                                     // one holds all that is further below
constexpr int kSlotsPerOctave = 8;
constexpr int kTokenList = 4096;                     // entries of a border bin that fit LDS

// Order-preserving keys; 0: an entry that is never drawn (NaN, -inf; no int32 entry is).  -0 and +0 are one key.
__device__ __forceinline__ uint32_t token_key(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return v > -__builtin_inff() ? k : 0u;
}
template <typename T>
struct TokenKey {
    static __device__ __forceinline__ bool drawable(uint32_t k) { return k != 0; }
    static __device__ __forceinline__ double value(uint32_t k)
    {
        return (double)__builtin_bit_cast(float, k ^ (k >> 31 ? 0x80000000u : 0xFFFFFFFFu));
    }
    static __device__ __forceinline__ uint32_t key1(const T *p) { return token_key(mx_load1(p)); }
    static __device__ __forceinline__ void key8(uint32_t (&k)[8], const T *p)
    {
        float v[8];
        mx_load8(v, p);
#pragma unroll
        for (int e = 0; e < 8; e++) k[e] = token_key(v[e]);
    }
    // a key not above (not below) those of all logits of at least (at most) v, a few units of fp32 off
    static __device__ __forceinline__ uint32_t below(double v)
    {
        if (!(v > -3e38)) return 0u;
        const uint32_t k = token_key((float)(v < 3e38 ? v : 3e38));
        return k > 8u ? k - 8u : 0u;
    }
    static __device__ __forceinline__ uint32_t above(double v)
    {
        if (!(v < 3e38)) return 0xFFFFFFFFu;
        return token_key((float)(v > -3e38 ? v : -3e38)) + 8u;
    }
};
template <>
struct TokenKey<int32_t> {
    static __device__ __forceinline__ bool drawable(uint32_t) { return true; }
    static __device__ __forceinline__ double value(uint32_t k) { return (double)(int32_t)(k ^ 0x80000000u); }
    static __device__ __forceinline__ uint32_t key1(const int32_t *p) { return (uint32_t)*p ^ 0x80000000u; }
    static __device__ __forceinline__ void key8(uint32_t (&k)[8], const int32_t *p)
    {
        const uint4 a = reinterpret_cast<const uint4 *>(p)[0], b = reinterpret_cast<const uint4 *>(p)[1];
        k[0] = a.x, k[1] = a.y, k[2] = a.z, k[3] = a.w, k[4] = b.x, k[5] = b.y, k[6] = b.z, k[7] = b.w;
#pragma unroll
        for (int e = 0; e < 8; e++) k[e] ^= 0x80000000u;
    }
    static __device__ __forceinline__ uint32_t below(double v)
    {
        if (!(v > -2147483640.0)) return 0u;
        return ((uint32_t)(int32_t)floor(v < 2147483640.0 ? v : 2147483640.0) ^ 0x80000000u) - 2u;
    }
    static __device__ __forceinline__ uint32_t above(double v)
    {
        if (!(v < 2147483640.0)) return 0xFFFFFFFFu;
        return ((uint32_t)(int32_t)floor(v > -2147483640.0 ? v : -2147483640.0) ^ 0x80000000u) + 2u;
    }
};

struct TokenArgs {
    int32_t *out;
    const void *logits;
    const uint32_t *words;
    const float *temperature, *top_p, *min_p;
    const int32_t *top_k;
    double temperature_all, top_p_all, min_p_all;
    int64_t top_k_all, R;
    int V, frac_bits, chunks;
    uint8_t *workspace;
};

// A row as groups of eight entries that start at multiples of 16 bytes: group j holds the entries 8 j - lead ...
template <typename T>
struct TokenLogits {
    const T *row;
    int V, lead, groups;
    __device__ __forceinline__ TokenLogits(const void *logits, int64_t r, int V_) : row((const T *)logits + r * V_), V(V_)
    {
        lead = (int)(((uintptr_t)row & 15) / sizeof(T));
        groups = (V + lead + kGroup - 1) / kGroup;
    }
    // keys of group j and which of its entries can be drawn
    __device__ __forceinline__ uint32_t load(uint32_t (&k)[8], int j) const
    {
        const int i0 = j * kGroup - lead;
        uint32_t have = 0;
        if (i0 >= 0 && i0 + kGroup <= V) {
            TokenKey<T>::key8(k, row + i0);
#pragma unroll
            for (int e = 0; e < 8; e++) have |= (uint32_t)TokenKey<T>::drawable(k[e]) << e;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool in = i0 + e >= 0 && i0 + e < V;
                k[e] = in ? TokenKey<T>::key1(row + i0 + e) : 0u;
                have |= (uint32_t)(in && TokenKey<T>::drawable(k[e])) << e;
            }
        }
        return have;
    }
};

// 2^t for t <= 0 as an integer multiple of 2^-frac, rounded: 2^t = 2^n 2^f with n the nearest integer, 2^f by its Taylor
// sum in f ln 2, |f ln 2| <= 0.347, to the 12th power (the rest is below 2e-16 of it), then a shift of the 53-bit
// significand.
__device__ __forceinline__ uint64_t token_exp2(double t, int frac)
{
    if (!(t > -64.0)) return 0;
    constexpr double ln2 = 0.69314718055994530942;
    const double n = rint(t), f = (t - n) * ln2;
    constexpr double c[13] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320,
                              1.0 / 362880, 1.0 / 3628800, 1.0 / 39916800, 1.0 / 479001600};
    double p = c[12];
#pragma unroll
    for (int i = 11; i >= 0; i--) p = fma(p, f, c[i]);
    const uint64_t bits = __builtin_bit_cast(uint64_t, p);
    const int shift = 1075 - frac - (int)(bits >> 52) - (int)n;      // p = significand * 2^(exponent - 1075)
    if (shift >= 64) return 0;
    const uint64_t m = (bits & 0xFFFFFFFFFFFFFull) | 0x10000000000000ull;
    return shift ? (m + (1ull << (shift - 1))) >> shift : m;
}

// How a row's logits become weights, relative to a maximum (the row's, or a chunk's)
template <typename T>
struct TokenScale {
    uint32_t kmax;
    double vmax, rate;      // octaves of the weight per unit of the logits
    int frac;
    __device__ __forceinline__ TokenScale(uint32_t kmax_, double rate_, int frac_)
        : kmax(kmax_), vmax(TokenKey<T>::value(kmax_)), rate(rate_), frac(frac_) {}
    __device__ __forceinline__ uint64_t weight(uint32_t k) const
    {
        if (k == kmax) return 1ull << frac;                          // also where both are +inf
        return token_exp2((TokenKey<T>::value(k) - vmax) * rate, frac);
    }
    // Bins lie on one grid for all chunks of a row; they are the same for equal logits and rise with them.
    static __device__ __forceinline__ double bin(uint32_t k, double rate)
    {
        return floor(TokenKey<T>::value(k) * (rate * kSlotsPerOctave));
    }
    // bins below the maximum's; the infinity's own bin is 0
    __device__ __forceinline__ int slot(uint32_t k, double top) const
    {
        if (k == kmax) return 0;
        const double d = top - bin(k, rate);
        return d < kSlots - 1 ? (int)d : kSlots - 1;
    }
};

struct TokenSettings {
    double rate, top_p, min_p;
    int64_t top_k;
    bool greedy;
    __device__ __forceinline__ TokenSettings(const TokenArgs &a, int64_t row)
    {
        const double temperature = a.temperature ? (double)a.temperature[row] : a.temperature_all;
        greedy = !(temperature > 0.0);
        rate = std::max(1.4426950408889634 / temperature, 1e-300);   // not 0: -inf * 0 is no exponent
        top_k = a.top_k ? a.top_k[row] : a.top_k_all;
        if (top_k <= 0 || top_k >= a.V) top_k = 0;
        top_p = a.top_p ? (double)a.top_p[row] : a.top_p_all;
        min_p = a.min_p ? (double)a.min_p[row] : a.min_p_all;
    }
    __device__ __forceinline__ bool cut() const { return top_k > 0 || top_p < 1.0; }
};

template <typename U>
__device__ __forceinline__ U wave_sum(U v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
template <typename U>
__device__ __forceinline__ U wave_max(U v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const U w = __shfl_xor(v, o);
        v = v > w ? v : w;
    }
    return v;
}
// sum over the lanes up to and including this one
template <typename U>
__device__ __forceinline__ U wave_scan(U v, int lane)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const U w = __shfl_up(v, o);
        if (lane >= o) v += w;
    }
    return v;
}
// floor(word * all / 2^32): a sum of integers is above word / 2^32 of all exactly where it is above this
__device__ __forceinline__ uint64_t token_bar(uint32_t word, uint64_t all)
{
    return (uint64_t)word * (all >> 32) + (((uint64_t)word * (all & 0xFFFFFFFFu)) >> 32);
}

// ---- rows of at most 64 entries: a wave per row ------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void sample_short_kernel(TokenArgs a)
{
    const int lane = threadIdx.x & 63, V = a.V;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.R) return;                              // whole waves; no barrier follows
    const TokenSettings set(a, row);
    const T *x = (const T *)a.logits + row * V;
    const uint32_t key = lane < V ? TokenKey<T>::key1(x + lane) : 0u;
    const bool have = lane < V && TokenKey<T>::drawable(key);
    if (!__ballot(have)) {
        if (lane == 0) a.out[row] = -1;
        return;
    }
    const uint32_t kmax = wave_max(have ? key : 0u);
    if (set.greedy) {
        const uint64_t at = __ballot(have && key == kmax);
        if (lane == 0) a.out[row] = __builtin_ctzll(at);
        return;
    }
    const TokenScale<T> scale(kmax, set.rate, a.frac_bits);
    uint64_t w = have ? scale.weight(key) : 0;
    bool keep = have;
    if (set.cut()) {
        int rank = 0;                                    // entries before this one, and their weight
        uint64_t before = 0;
        for (int j = 0; j < V; j++) {
            const uint32_t k = __builtin_amdgcn_readlane(key, j);
            const uint64_t wj = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(w >> 32), j) << 32) |
                                (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)w, j);
            const bool first = __builtin_amdgcn_readlane(have, j) && (k > key || (k == key && j < lane));
            rank += first;
            before += first ? wj : 0;
        }
        if (set.top_k) keep = keep && rank < set.top_k;
        if (set.top_p < 1.0) {
            const uint64_t all = wave_sum(keep ? w : 0);
            keep = keep && (rank == 0 || (double)before < set.top_p * (double)all);
        }
    }
    keep = keep && !((double)w < std::min(set.min_p, 1.0) * (double)(1ull << a.frac_bits));
    w = keep ? w : 0;
    const uint64_t sum = wave_scan(w, lane), all = __shfl(sum, 63);
    const uint64_t at = __ballot(sum > token_bar(a.words[row], all));
    if (lane == 0) a.out[row] = __builtin_ctzll(at);
}

// ---- long rows, first kernel: a chunk's maximum, its weights' sum and, where the row is cut, their histogram ------------
struct TokenChunk {
    uint64_t sum;                  // of the weights relative to the chunk's maximum
    uint32_t kmax, have;           // have: whether the chunk holds anything that can be drawn
    uint64_t weight[kSlots];       // by bins below the chunk's maximum
    uint32_t count[kSlots];
};
static_assert(sizeof(TokenChunk) % 16 == 0, "records of the workspace");

template <typename T>
__global__ __launch_bounds__(512) void token_chunk_kernel(TokenArgs a)
{
    __shared__ uint64_t hist_w[kSlots], sh_sum;
    __shared__ uint32_t hist_c[kSlots], sh_max[8], sh_have[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / a.chunks;
    const int chunk = (int)(blockIdx.x - row * a.chunks);
    const TokenSettings set(a, row);
    const TokenLogits<T> x(a.logits, row, a.V);
    TokenChunk *out = reinterpret_cast<TokenChunk *>(a.workspace) + blockIdx.x;
    uint32_t k[2][8], have[2], m = 0;
#pragma unroll
    for (int q = 0; q < 2; q++) {
        const int j = chunk * kChunkGroups + q * 512 + tid;
        have[q] = 0;
        if (j < x.groups) have[q] = x.load(k[q], j);
    }
#pragma unroll
    for (int q = 0; q < 2; q++)
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (have[q] >> e & 1) m = k[q][e] > m ? k[q][e] : m;
    const uint64_t any = __ballot(have[0] | have[1]);
    m = wave_max(m);
    if (lane == 0) sh_max[wave] = m, sh_have[wave] = any != 0;
    for (int t = tid; t < kSlots; t += 512) hist_w[t] = 0, hist_c[t] = 0;
    if (tid == 0) sh_sum = 0;
    __syncthreads();
    uint32_t h = 0;
#pragma unroll
    for (int w = 0; w < 8; w++) m = sh_max[w] > m ? sh_max[w] : m, h |= sh_have[w];
    if (h && !set.greedy) {
        const TokenScale<T> scale(m, set.rate, a.frac_bits);
        const double top = TokenScale<T>::bin(m, set.rate);
        const bool cut = set.cut(), counted = set.top_k > 0;
        uint64_t sum = 0;
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (have[q] >> e & 1) {
                    const uint64_t w = scale.weight(k[q][e]);
                    sum += w;
                    if (cut) {
                        const int s = scale.slot(k[q][e], top);
                        atomicAdd((unsigned long long *)&hist_w[s], (unsigned long long)w);
                        if (counted) atomicAdd(&hist_c[s], 1u);
                    }
                }
        sum = wave_sum(sum);
        if (lane == 0) atomicAdd((unsigned long long *)&sh_sum, (unsigned long long)sum);
        __syncthreads();
        if (cut)
            for (int t = tid; t < kSlots; t += 512) out->weight[t] = hist_w[t], out->count[t] = hist_c[t];
    }
    if (tid == 0) out->sum = sh_sum, out->kmax = m, out->have = h;
}

// ---- a workgroup per row ----------------------------------------------------------------------------------------------
// LOCAL: from the logits alone; else from the chunks' records.
template <typename T, int THREADS, bool LOCAL>
__global__ __launch_bounds__(THREADS) void sample_row_kernel(TokenArgs a)
{
    constexpr int WAVES = THREADS / 64;
    constexpr int SEGS = LOCAL ? kTokenLocalV / (kGroup * kSegGroups) + 1 : kTokenMaxSegs;
    __shared__ uint64_t seg_w[SEGS];
    __shared__ uint32_t seg_c[SEGS];
    __shared__ double slot_w[kSlots];
    __shared__ uint64_t hist_w[kSlots];                  // LOCAL: by slot; in select(): by digit
    __shared__ uint32_t hist_c[kSlots], slot_c[kSlots];
    __shared__ uint32_t list[kTokenList];
    __shared__ double chunk_f[LOCAL ? 1 : kTokenMaxChunks];
    __shared__ int chunk_off[LOCAL ? 1 : kTokenMaxChunks];
    __shared__ uint32_t sh_key[WAVES], sh_have[WAVES], sh_n, sh_count, sh_ties;
    __shared__ uint64_t sh_sum;
    __shared__ double sh_before;
    __shared__ int sh_at;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const TokenSettings set(a, row);
    const TokenLogits<T> x(a.logits, row, a.V);
    const int segs = (x.groups + kSegGroups - 1) / kSegGroups;
    const TokenChunk *chunk = reinterpret_cast<const TokenChunk *>(a.workspace) + row * a.chunks;
    // f(keys, which can be drawn, first entry's index, segment): every wave takes whole segments
    const auto for_groups = [&](auto &&f) {
        for (int s = wave; s < segs; s += WAVES) {
            uint32_t k[8], have = 0;
            const int j = s * kSegGroups + lane;
            if (j < x.groups) have = x.load(k, j);
            f(k, have, j * kGroup - x.lead, s);
        }
    };
    // the row's maximum
    uint32_t m = 0, any = 0;
    if (LOCAL) {
        for_groups([&](const uint32_t (&k)[8], uint32_t have, int, int) {
            any |= have;
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (have >> e & 1) m = k[e] > m ? k[e] : m;
        });
    } else {
        for (int c = tid; c < a.chunks; c += THREADS)
            if (chunk[c].have) any = 1, m = chunk[c].kmax > m ? chunk[c].kmax : m;
    }
    m = wave_max(m);
    any = __ballot(any) != 0;
    if (lane == 0) sh_key[wave] = m, sh_have[wave] = any;
    if (tid == 0) sh_at = a.V;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) m = sh_key[w] > m ? sh_key[w] : m, any |= sh_have[w];
    if (!any) {
        if (tid == 0) a.out[row] = -1;
        return;
    }
    const TokenScale<T> scale(m, set.rate, a.frac_bits);
    const double top = TokenScale<T>::bin(m, set.rate);
    const double one = (double)(1ull << a.frac_bits);
    if (set.greedy) {
        for_groups([&](const uint32_t (&k)[8], uint32_t have, int i0, int) {
            for (int e = 0; e < 8; e++)
                if ((have >> e & 1) && k[e] == m) {
                    atomicMin(&sh_at, i0 + e);
                    break;
                }
        });
        __syncthreads();
        if (tid == 0) a.out[row] = sh_at;
        return;
    }

    if constexpr (!LOCAL) {
        for (int c = tid; c < a.chunks; c += THREADS) {
            const uint32_t cm = chunk[c].kmax;
            const double d = cm == m ? 0.0 : top - TokenScale<T>::bin(cm, set.rate);
            chunk_off[c] = !chunk[c].have ? kSlots : d < kSlots - 1 ? (int)d : kSlots - 1;
            chunk_f[c] = !chunk[c].have ? 0.0 : cm == m ? 1.0 : exp2((TokenKey<T>::value(cm) - scale.vmax) * set.rate);
        }
        __syncthreads();
    }
    // what is kept: keys above `key`, and `ties` of those equal to it, the first ones
    uint32_t key = 0, ties = 0xFFFFFFFFu, equal = 0;
    if (set.cut()) {
        // ---- the row's histogram -------------------------------------------------------------------------------------
        if (LOCAL) {
            for (int t = tid; t < kSlots; t += THREADS) hist_w[t] = 0, hist_c[t] = 0;
            __syncthreads();
            for_groups([&](const uint32_t (&k)[8], uint32_t have, int, int) {
                for (int e = 0; e < 8; e++)
                    if (have >> e & 1) {
                        const int s = scale.slot(k[e], top);
                        atomicAdd((unsigned long long *)&hist_w[s], (unsigned long long)scale.weight(k[e]));
                        if (set.top_k) atomicAdd(&hist_c[s], 1u);
                    }
            });
            __syncthreads();
            for (int t = tid; t < kSlots; t += THREADS) slot_w[t] = (double)hist_w[t], slot_c[t] = hist_c[t];
        } else {
            // a chunk's bin s lies chunk_off bins lower in the row, its weights are chunk_f of the row's; chunk after chunk, so
            // the sums have one order.  The last slot also takes all that lies below it (a wave of its own).
            if (tid < kSlots - 1) {
                double w = 0.0;
                uint32_t n = 0;
#pragma unroll 8
                for (int c = 0; c < a.chunks; c++) {
                    const int s = tid - chunk_off[c];
                    if (s >= 0) w += chunk_f[c] * (double)chunk[c].weight[s], n += chunk[c].count[s];
                }
                slot_w[tid] = w, slot_c[tid] = n;
            } else if (wave == kSlots / 64) {
                double w = 0.0;
                uint32_t n = 0;
                for (int c = 0; c < a.chunks; c++) {
                    if (chunk_off[c] >= kSlots) continue;
                    for (int s = kSlots - 1 - chunk_off[c] + lane; s < kSlots; s += 64)
                        w += chunk_f[c] * (double)chunk[c].weight[s], n += chunk[c].count[s];
                }
                w = wave_sum(w), n = wave_sum(n);
                if (lane == 0) slot_w[kSlots - 1] = w, slot_c[kSlots - 1] = n;
            }
        }
        __syncthreads();
        // ---- borders ---------------------------------------------------------------------------------------------------
        double total = 0.0;                              // what top_p is a part of
        bool have_total = false;
        // Digit by digit among the entries that `each` hands out and f accepts: the shortest prefix of at least k
        // entries, or of a weight of at least target, `before` entries or weight lying above all of them.  The row has to
        // reach it among them.
        const auto digits = [&](auto &&each, bool by_count, int64_t k, double target, uint32_t before_c, double before_w) {
            uint32_t prefix = 0;
            for (int shift = 24; shift >= 0; shift -= 8) {
                __syncthreads();
                for (int t = tid; t < kSlots; t += THREADS) hist_w[t] = 0, hist_c[t] = 0;
                __syncthreads();
                each([&](uint32_t q) {
                    if (shift == 24 || q >> (shift + 8) == prefix) {
                        atomicAdd(&hist_c[(q >> shift) & 255], 1u);
                        atomicAdd((unsigned long long *)&hist_w[(q >> shift) & 255], (unsigned long long)scale.weight(q));
                    }
                });
                __syncthreads();
                if (wave == 0) {                         // lane l: the digits 255 - 4 l down to 252 - 4 l
                    uint32_t c[4], cs = 0;
                    uint64_t w[4], ws = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        c[e] = hist_c[255 - 4 * lane - e], w[e] = hist_w[255 - 4 * lane - e];
                        cs += c[e], ws += w[e];
                    }
                    uint32_t ca = wave_scan(cs, lane) - cs;
                    uint64_t wa = wave_scan(ws, lane) - ws;
                    int found = -1;
                    uint32_t fc = 0, fn = 0;
                    uint64_t fw = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool here = c[e] && (by_count ? (int64_t)before_c + ca + c[e] >= k
                                                            : before_w + (double)(wa + w[e]) >= target);
                        if (found < 0 && here) found = 255 - 4 * lane - e, fc = ca, fw = wa, fn = c[e];
                        ca += c[e], wa += w[e];
                    }
                    // the last digit that holds anything, should rounding put the target above all
                    const uint64_t hit = __ballot(found >= 0), some = __ballot(cs != 0);
                    if (hit) {
                        if (lane == __builtin_ctzll(hit)) sh_at = found, sh_count = fc, sh_sum = fw, sh_ties = fn;
                    } else if (some && lane == 63 - __builtin_clzll(some)) {
                        uint32_t cb = ca - cs;
                        uint64_t wb = wa - ws;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if (c[e]) sh_at = 255 - 4 * lane - e, sh_ties = c[e], sh_count = cb, sh_sum = wb;
                            cb += c[e], wb += w[e];
                        }
                    }
                }
                __syncthreads();
                before_c += sh_count;
                before_w += (double)sh_sum;
                equal = sh_ties;
                prefix = (prefix << 8) | (uint32_t)sh_at;
            }
            key = prefix;
            const uint64_t w = scale.weight(key);
            if (by_count) {
                const int64_t left = k - before_c;
                ties = left < (int64_t)equal ? (uint32_t)left : equal;
            } else {
                uint32_t lo = 1, hi = equal;             // the fewest that reach the target
                while (lo < hi) {
                    const uint32_t mid = (lo + hi) / 2;
                    if (before_w + (double)(mid * w) >= target) hi = mid;
                    else lo = mid + 1;
                }
                ties = lo;
            }
            total = before_w + (double)(ties * w);
        };
        const auto select = [&](bool by_count, int64_t k, double target) {
            __syncthreads();
            // the slot that the border lies in: lane l has the slots 4 l ... 4 l + 3
            if (wave == 0) {
                uint32_t c[4], cs = 0;
                double w[4], ws = 0.0;
#pragma unroll
                for (int e = 0; e < 4; e++) c[e] = slot_c[4 * lane + e], w[e] = slot_w[4 * lane + e], cs += c[e], ws += w[e];
                double wa = wave_scan(ws, lane) - ws;
                uint32_t ca = wave_scan(cs, lane) - cs;
                int found = -1;
                uint32_t fc = 0;
                double fw = 0.0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool here = by_count ? c[e] && (int64_t)ca + c[e] >= k : w[e] > 0.0 && wa + w[e] >= target;
                    if (found < 0 && here) found = 4 * lane + e, fc = ca, fw = wa;
                    ca += c[e], wa += w[e];
                }
                const uint64_t hit = __ballot(found >= 0);
                if (!hit) {
                    if (lane == 0) sh_at = -1;
                } else if (lane == __builtin_ctzll(hit)) {
                    sh_at = found, sh_count = fc, sh_before = fw;
                }
                if (lane == 0) sh_n = 0;
            }
            __syncthreads();
            const int slot = sh_at;
            const uint32_t before_c = sh_count;
            const double before_w = sh_before;
            __syncthreads();
            if (slot < 0) return;                        // the row has no more than that: nothing is cut
            // keys that can lie in the slot, a little more than those that do
            const double per = set.rate * kSlotsPerOctave;
            const uint32_t lowest = slot == kSlots - 1 ? 0u : TokenKey<T>::below((top - slot) / per);
            const uint32_t span = (slot == 0 ? 0xFFFFFFFFu : TokenKey<T>::above((top - slot + 1.0) / per)) - lowest;
            const auto in_slot = [&](uint32_t q) { return q - lowest <= span && scale.slot(q, top) == slot; };
            for_groups([&](const uint32_t (&q)[8], uint32_t have, int, int) {
                for (int e = 0; e < 8; e++)
                    if ((have >> e & 1) && in_slot(q[e])) {
                        const uint32_t at = atomicAdd(&sh_n, 1u);
                        if (at < kTokenList) list[at] = q[e];
                    }
            });
            __syncthreads();
            const uint32_t n = sh_n;
            if (n <= kTokenList) {
                digits([&](auto &&f) { for (uint32_t i = tid; i < n; i += THREADS) f(list[i]); }, by_count, k, target,
                       before_c, before_w);
            } else {                                     // a slot of very many: from memory again for every digit
                digits([&](auto &&f) {
                    for_groups([&](const uint32_t (&q)[8], uint32_t have, int, int) {
                        for (int e = 0; e < 8; e++)
                            if ((have >> e & 1) && in_slot(q[e])) f(q[e]);
                    });
                }, by_count, k, target, before_c, before_w);
            }
            have_total = true;
        };
        if (set.top_k) select(true, set.top_k, 0.0);
        if (set.top_p < 1.0) {
            if (!have_total) {
                double w = 0.0;
#pragma unroll
                for (int e = 0; e < 4; e++) w += slot_w[4 * lane + e];
                total = wave_sum(w);
            }
            select(false, 0, set.top_p * total);
        }
    }
    // ---- the index of the last tie that is kept ----------------------------------------------------------------------------
    int last = a.V;
    if (ties < equal) {
        __syncthreads();
        for_groups([&](const uint32_t (&k)[8], uint32_t have, int, int s) {
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) c += (have >> e & 1) && k[e] == key;
            c = wave_sum(c);
            if (lane == 0) seg_c[s] = c;
        });
        __syncthreads();
        if (wave == 0) {
            uint32_t left = ties;                        // among the segments from base on
            int base = 0;
            for (;; base += 64) {
                const uint32_t c = base + lane < segs ? seg_c[base + lane] : 0;
                const uint32_t run = wave_scan(c, lane);
                const uint64_t hit = __ballot(run >= left);
                if (hit || base + 64 >= segs) {
                    const int l = hit ? __builtin_ctzll(hit) : 63;
                    left -= __shfl(run, l) - __shfl(c, l);
                    base += l;
                    break;
                }
                left -= __shfl(run, 63);
            }
            uint32_t k[8], have = 0, c = 0;
            const int j = base * kSegGroups + lane;
            if (j < x.groups) have = x.load(k, j);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                have = (have >> e & 1) && k[e] != key ? have & ~(1u << e) : have;
                c += have >> e & 1;
            }
            const uint32_t run = wave_scan(c, lane);
            const uint64_t hit = __ballot(run >= left);
            if (hit && lane == __builtin_ctzll(hit)) {
                left -= run - c;
                for (int e = 0; e < 8; e++)
                    if ((have >> e & 1) && --left == 0) sh_at = j * kGroup - x.lead + e;
            }
        }
        __syncthreads();
        last = sh_at;
    }
    // ---- the draw ----------------------------------------------------------------------------------------------------------
    const double min_w = std::min(set.min_p, 1.0) * one;
    // no entry below this reaches min_p (a little lower than it need be; the weights decide)
    uint32_t lowest = set.min_p > 0.0 ? TokenKey<T>::below(scale.vmax + log2(std::min(set.min_p, 1.0)) / set.rate) : 0u;
    lowest = lowest > key ? lowest : key;
    const auto draw = [&](const TokenScale<T> &sc, int seg0, int seg1, auto &&bar_of) {
        const auto kept = [&](uint32_t k, int i) -> uint64_t {
            if (k < lowest || (k == key && i > last)) return 0;
            const uint64_t w = sc.weight(k);
            return (double)w < min_w ? 0 : w;
        };
        __syncthreads();
        for (int s = seg0 + wave; s < seg1; s += WAVES) {
            uint32_t k[8], have = 0;
            const int j = s * kSegGroups + lane;
            if (j < x.groups) have = x.load(k, j);
            uint64_t w = 0;
            for (int e = 0; e < 8; e++)
                if (have >> e & 1) w += kept(k[e], j * kGroup - x.lead + e);
            w = wave_sum(w);
            if (lane == 0) seg_w[s] = w;
        }
        __syncthreads();
        if (wave != 0) return;
        uint64_t all = 0;
        for (int s = seg0 + lane; s < seg1; s += 64) all += seg_w[s];
        all = wave_sum(all);
        uint64_t bar = bar_of(all);                      // below all: some segment reaches over it
        int base = seg0;
        for (;; base += 64) {
            const uint64_t c = base + lane < seg1 ? seg_w[base + lane] : 0;
            const uint64_t run = wave_scan(c, lane);
            const uint64_t hit = __ballot(run > bar);
            if (hit || base + 64 >= seg1) {
                const int l = hit ? __builtin_ctzll(hit) : 63;
                bar -= __shfl(run, l) - __shfl(c, l);
                base += l;
                break;
            }
            bar -= __shfl(run, 63);
        }
        uint32_t k[8], have = 0;
        uint64_t w[8], sum = 0;
        const int j = base * kSegGroups + lane;
        if (j < x.groups) have = x.load(k, j);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            w[e] = have >> e & 1 ? kept(k[e], j * kGroup - x.lead + e) : 0;
            sum += w[e];
        }
        const uint64_t run = wave_scan(sum, lane);
        const uint64_t hit = __ballot(run > bar);
        if (hit && lane == __builtin_ctzll(hit)) {
            uint64_t acc = run - sum;
            int i = -1;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                acc += w[e];
                if (i < 0 && acc > bar) i = j * kGroup - x.lead + e;
            }
            a.out[row] = i;
        }
    };
    const uint32_t word = a.words[row];
    if constexpr (!LOCAL) {
        if (!set.cut() && !(set.min_p > 0.0)) {
            // nothing is cut off: the chunk from the chunks' sums, then that chunk's entries alone
            if (wave == 0) {
                double all = 0.0, before = 0.0;
                for (int c0 = 0; c0 < a.chunks; c0 += 64)
                    all += wave_sum(c0 + lane < a.chunks ? chunk_f[c0 + lane] * (double)chunk[c0 + lane].sum : 0.0);
                const double bar = (double)word * 0x1p-32 * all;
                int at = -1, seen = -1;                  // the chunk that reaches over the bar; the last with any weight
                double from = 0.0;
                for (int c0 = 0; c0 < a.chunks && at < 0; c0 += 64) {
                    const double v = c0 + lane < a.chunks ? chunk_f[c0 + lane] * (double)chunk[c0 + lane].sum : 0.0;
                    const double run = wave_scan(v, lane);
                    const uint64_t hit = __ballot(v > 0.0 && before + run > bar), some = __ballot(v > 0.0);
                    const int l = hit ? __builtin_ctzll(hit) : some ? 63 - __builtin_clzll(some) : -1;
                    if (l >= 0) {
                        seen = c0 + l;
                        from = before + __shfl(run - v, l);
                        if (hit) at = c0 + l;
                    }
                    before += __shfl(run, 63);
                }
                at = at < 0 ? seen : at;
                if (lane == 0) sh_at = at, sh_before = (bar - from) / chunk_f[at];
            }
            __syncthreads();
            const int at = sh_at;
            const double left = sh_before;
            constexpr int kSegsPerChunk = kChunkGroups / kSegGroups;
            const int seg1 = (at + 1) * kSegsPerChunk < segs ? (at + 1) * kSegsPerChunk : segs;
            draw(TokenScale<T>(chunk[at].kmax, set.rate, a.frac_bits), at * kSegsPerChunk, seg1, [&](uint64_t all) {
                const uint64_t b = left > 0.0 ? (uint64_t)left : 0;
                return b < all ? b : all - 1;
            });
            return;
        }
    }
    draw(scale, 0, segs, [&](uint64_t all) { return token_bar(word, all); });
}

static int token_chunks(int64_t V) { return (int)ceil_div(V + kGroup - 1, kChunkGroups * kGroup); }

template <typename T>
static int token_launch(const TokenArgs &a, hipStream_t st, const char *who)
{
    if (a.V <= 64)
        sample_short_kernel<T><<<dim3((unsigned)ceil_div(a.R, 4)), dim3(256), 0, st>>>(a);
    else if (a.V <= 2048)
        sample_row_kernel<T, 256, true><<<dim3((unsigned)a.R), dim3(256), 0, st>>>(a);
    else if (a.V <= kTokenLocalV)
        sample_row_kernel<T, 1024, true><<<dim3((unsigned)a.R), dim3(1024), 0, st>>>(a);
    else {
        token_chunk_kernel<T><<<dim3((unsigned)(a.R * a.chunks)), dim3(512), 0, st>>>(a);
        if (const int rc = check_launch(who)) return rc;
        sample_row_kernel<T, 1024, false><<<dim3((unsigned)a.R), dim3(1024), 0, st>>>(a);
    }
    return check_launch(who);
}

}  // namespace nb

extern "C" {
int64_t nb_sample_tokens_workspace_bytes(int64_t R, int64_t V)
{
    if (R <= 0 || V <= nb::kTokenLocalV || V > nb::kTokenMaxV || R >= (1LL << 22)) return 0;
    return R * nb::token_chunks(V) * (int64_t)sizeof(nb::TokenChunk);
}

int nb_sample_tokens(int32_t *out, const void *logits, int type, const uint32_t *words, const float *temperature,
                     double temperature_all, const int32_t *top_k, int64_t top_k_all, const float *top_p,
                     double top_p_all, const float *min_p, double min_p_all, int64_t R, int64_t V, void *workspace,
                     int64_t workspace_bytes, nb_stream_t stream)
{
    const char *who = "nb_sample_tokens";
    NB_REQUIRE(R >= 0 && V >= 1, "%s: bad shape", who);
    NB_REQUIRE(V <= nb::kTokenMaxV, "%s: rows of %lld entries, at most %lld", who, (long long)V, (long long)nb::kTokenMaxV);
    NB_REQUIRE(R < (1LL << 22) && R * V < (1LL << 34), "%s: too many rows", who);
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
    const int64_t need = nb_sample_tokens_workspace_bytes(R, V);
    NB_REQUIRE(workspace_bytes >= need, "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
               (long long)need);
    if (need) {
        NB_REQUIRE_PTR(workspace);
        NB_REQUIRE_ALIGNED(workspace, 16);
    }
    int log2v = 0;
    while ((1LL << log2v) < V) log2v++;
    const nb::TokenArgs a{out, logits, words, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all,
                          top_k_all, R, (int)V, std::min(52, 61 - log2v), nb::token_chunks(V), (uint8_t *)workspace};
    const hipStream_t st = nb::as_stream(stream);
    if (type == NB_TYPE_F32) return nb::token_launch<float>(a, st, who);
    if (type == NB_TYPE_F16) return nb::token_launch<_Float16>(a, st, who);
    if (type == NB_TYPE_BF16) return nb::token_launch<nb::Bf16>(a, st, who);
    return nb::token_launch<int32_t>(a, st, who);
}
}  // extern "C"
