// One token per row of logits from a supplied word: temperature, top-k, top-p, min-p.
//
// Each of the three filters keeps a prefix of the row in descending order (equal entries by index), so what is kept is
// "above a key, or equal to it at an index up to a cut", without a sort: a histogram over the logits' distance below the
// row's maximum names the bin the border lies in, and only that bin's entries are looked at digit by digit.  Weights are
// integers (a weight of 1 is 2^f): sums over a row are the same in any order, and are accumulated with atomics.
//
// Rows of at most 64 entries: a wave per row, ranks by comparing all pairs.  Up to 16376: a workgroup per row.  Longer
// ones: one kernel over chunks of 8192 entries (the exponentials, which bound the whole, are then spread over the card
// however few the rows), one workgroup per row to finish from the chunks' histograms.
//
// What bounds it: few rows, the latency of about ten phases that follow each other (a phase 1 to 4 us, most of it waiting for
// one workgroup's instructions and for memory).  Rows of 65 to 16376 entries that outnumber what the card holds, instructions:
// 4000 x 8000 bf16 without a cut 69 us, with top_p 165, where the bytes would take 13; an entry's weight is made once for the
// histogram and once for the draw, its bin by a chain of its own, and registers spill: to 128 (four waves a SIMD) 38 to 43
// vector registers of the forms with four groups a thread (156 to 176 bytes a lane), 7 to 10 of those with two, 7 and 17 to 18
// of the long rows' kernel with 512 and 1024 threads; none with one group.  256 x 131072 bf16 with a cut, 93 us: 48 us the
// exponentials' kernel (37 instructions an entry, two thirds of the cycles), 45 us the rows' kernel, 10 of them the second look
// at every logit at what the last cache gives to all CUs (7 TB/s).  A border's bin of more entries than the list holds costs a
// pass over the row per digit: 4 x 131072 equal logits 518 us, of N(0, 0.001^2) 298 us.
#include <algorithm>
#include <type_traits>

#include "nb_mx.hpp"

namespace nb {

constexpr int64_t kTokenMaxV = 1 << 20;
constexpr int kTokenLocalV = 16376;                  // rows that one workgroup handles from beginning to end
constexpr int kGroup = 8;                            // entries of a lane's load: aligned pieces of memory, whatever the row's start
constexpr int kSegGroups = 64;                       // a segment: the groups of one load of a wave
constexpr int kTokenMaxSegs = kTokenMaxV / (kGroup * kSegGroups) + 1;
constexpr int kChunkGroups = 1024;
constexpr int kTokenMaxChunks = kTokenMaxV / (kGroup * kChunkGroups) + 1;
constexpr int kSlots = 256;                          // bins of 1/8 of an octave of the weights below the maximum; the last
                                                     // one holds all that is further below
constexpr int kSlotsPerOctave = 8;

// Order-preserving keys; 0: an entry that is never drawn (NaN, -inf; no int32 entry is).  -0 and +0 are one key.
__device__ __forceinline__ uint32_t token_key(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return v > -__builtin_inff() ? k : 0u;
}
template <typename T>
struct TokenKey {
    // bits at a key's end that are clear in positive logits' keys and set in negative ones'
    static constexpr int kFree = __is_same(T, Bf16) ? 16 : __is_same(T, _Float16) ? 13 : 0;
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
    typedef float Value;                                 // holds every logit, and -inf
    static __device__ __forceinline__ void value8(float (&d)[8], const T *p) { mx_load8(d, p); }
    static __device__ __forceinline__ uint32_t key_of(double v) { return token_key((float)v); }
    // Near: a window of keys as the cheapest test on logits as they lie in memory, at most a little wider: two operations an
    // entry.  Differences are monotonic in v, so their roundings are too.
    struct Near {
        float middle, reach;
        __device__ __forceinline__ Near(uint32_t from, uint32_t to)              // 0, and what is above +inf's key: no end
        {
            const float lo = from < 0x00800000u ? -3.402823466e38f : (float)value(from);
            const float hi = to > 0xFF800000u ? __builtin_inff() : to < 0x00800000u ? -3.402823466e38f : (float)value(to);
            const bool all = !(hi - lo < __builtin_inff());
            middle = all ? 0.f : 0.5f * lo + 0.5f * hi;
            reach = all ? __builtin_inff() : fmaxf(hi - middle, middle - lo);
        }
        __device__ __forceinline__ bool any(const T *p) const                    // of a group's entries; NaNs are not
        {
            float v[8], least = __builtin_inff();
            mx_load8(v, p);
#pragma unroll
            for (int e = 0; e < 8; e += 2) least = fminf(fminf(least, fabsf(v[e] - middle)), fabsf(v[e + 1] - middle));
            return least <= reach;
        }
    };
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
    static constexpr int kFree = 0;
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
    typedef double Value;
    static __device__ __forceinline__ void value8(double (&d)[8], const int32_t *p)
    {
        const int4 a = reinterpret_cast<const int4 *>(p)[0], b = reinterpret_cast<const int4 *>(p)[1];
        d[0] = a.x, d[1] = a.y, d[2] = a.z, d[3] = a.w, d[4] = b.x, d[5] = b.y, d[6] = b.z, d[7] = b.w;
    }
    static __device__ __forceinline__ uint32_t key_of(double v) { return (uint32_t)(int32_t)v ^ 0x80000000u; }
    struct Near {
        uint32_t from, span;
        __device__ __forceinline__ Near(uint32_t from_, uint32_t to) : from(from_), span(to - from_) {}
        __device__ __forceinline__ bool any(const int32_t *p) const
        {
            uint32_t k[8], least = 0xFFFFFFFFu;
            key8(k, p);
#pragma unroll
            for (int e = 0; e < 8; e++) least = k[e] - from < least ? k[e] - from : least;
            return least <= span;
        }
    };
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

// A row as groups of eight entries that start at multiples of 16 bytes: group j holds the entries 8 j - lead ...  The
// first and the last group may reach past the row's ends: their keys are put into LDS once, entry by entry.
struct TokenEdges {
    uint32_t key[2][kGroup], have[2];
};
template <typename T>
struct TokenLogits {
    const T *row;
    int V, lead, groups;
    const TokenEdges *edges;
    __device__ __forceinline__ TokenLogits(const void *logits, int64_t r, int V_, const TokenEdges *e = nullptr)
        : row((const T *)logits + r * V_), V(V_), edges(e)
    {
        lead = (int)(((uintptr_t)row & 15) / sizeof(T));
        groups = (V + lead + kGroup - 1) / kGroup;
    }
    // by the first wave; the edges are there behind the caller's next barrier
    __device__ __forceinline__ void find_edges(TokenEdges *e) const
    {
        if (threadIdx.x >= 64) return;
        const int lane = threadIdx.x, i = (lane < 8 ? 0 : groups - 1) * kGroup - lead + (lane & 7);
        const bool in = lane < 16 && i >= 0 && i < V;    // lanes 0-7: the first group, 8-15: the last
        const uint32_t k = in ? TokenKey<T>::key1(row + i) : 0u;
        const uint64_t have = __ballot(in && TokenKey<T>::drawable(k));
        if (lane < 16) e->key[lane >> 3][lane & 7] = k;
        if (lane == 0) e->have[0] = (uint32_t)have & 255u, e->have[1] = (uint32_t)(have >> 8) & 255u;
    }
    __device__ __forceinline__ bool whole(int j) const
    {
        const int i0 = j * kGroup - lead;
        return i0 >= 0 && i0 + kGroup <= V;
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
            const int which = j ? 1 : 0;
            have = edges->have[which];
#pragma unroll
            for (int e = 0; e < 8; e++) k[e] = edges->key[which][e];
        }
        return have;
    }
    // an edge group's logits, -inf for those that are not there or cannot be drawn
    static __device__ __forceinline__ void edge_values(typename TokenKey<T>::Value (&d)[8], int j, const TokenEdges *edges)
    {
        const int which = j ? 1 : 0;
#pragma unroll
        for (int e = 0; e < 8; e++)
            d[e] = (typename TokenKey<T>::Value)(edges->have[which] >> e & 1 ? TokenKey<T>::value(edges->key[which][e])
                                                                             : -__builtin_inf());
    }
};

// Weights.  With u = 256 times the octaves of a weight: u = 256 n + j + r, |r| <= 1/2 and 0 <= j < 256, and 2^(u / 256) is 2^n by
// the exponent, 2^(j / 256) from a table, which also holds the weight of 1, 2^frac (frac <= 51), and 2^(r / 256) by its
// Taylor sum to the fourth power, whose rest is below 4e-17.  Adding 1.5 * 2^52 rounds u to an integer that then is the low
// word; adding 2^52 does the same for the weight, whose bits below the exponent are the integer.
constexpr int kExpTable = 256;
struct TokenExp {
    double power[kExpTable];                             // 2^(j / 256), j = 0 ... 255
};
constexpr TokenExp token_powers()
{
    TokenExp t{};
    for (int j = 0; j < kExpTable; j++) {
        const double x = 0.69314718055994530942 * j / kExpTable;
        double sum = 0.0, term = 1.0;
        for (int i = 1; i < 32; i++) sum += term, term = term * x / i;
        t.power[j] = sum;
    }
    return t;
}
__device__ const TokenExp kTokenPowers = token_powers();
// the table into LDS, by the whole workgroup; the caller's next barrier makes it visible
__device__ __forceinline__ void token_exp_table(TokenExp *t, int frac)
{
    const double one = (double)(1ull << frac);
    for (int j = threadIdx.x; j < kExpTable; j += blockDim.x) t->power[j] = kTokenPowers.power[j] * one;
}
constexpr double kExpHalf = 6755399441055744.0;          // 1.5 * 2^52
constexpr double kExpZero = -20000.0;                    // u from here on: 2^-78, 0 for every frac
__device__ __forceinline__ int token_low(double y) { return (int)(uint32_t)__builtin_bit_cast(uint64_t, y); }
struct TokenTaylor {
    double c[5];
    // of 2^((r - at) / 256)
    __device__ __forceinline__ explicit TokenTaylor(double at = 0.0)
    {
        constexpr double a = 0.69314718055994530942 / kExpTable;
        constexpr double k[5] = {1.0, a, a * a / 2, a * a * a / 6, a * a * a * a / 24};
        const double f = fma(fma(fma(fma(k[4], -at, k[3]), -at, k[2]), -at, k[1]), -at, 1.0);
#pragma unroll
        for (int i = 0; i < 5; i++) c[i] = f * k[i];
    }
    // the weight of i + r, i = 256 n + j
    __device__ __forceinline__ uint64_t weight(int i, double r, const TokenExp *t) const
    {
        const double p = fma(fma(fma(fma(c[4], r, c[3]), r, c[2]), r, c[1]), r, c[0]) * t->power[i & (kExpTable - 1)];
        const uint64_t bits = __builtin_bit_cast(uint64_t, p);           // never near a subnormal: n >= -79
        const uint32_t high = (uint32_t)(bits >> 32) + ((uint32_t)(i & ~(kExpTable - 1)) << 12);
        const double v = __builtin_bit_cast(double, (uint64_t)high << 32 | (uint32_t)bits) + 4503599627370496.0;
        return __builtin_bit_cast(uint64_t, v) & 0xFFFFFFFFFFFFFull;
    }
};
__device__ __forceinline__ uint64_t token_exp2(double u, const TokenExp *t)
{
    u = fmax(u, kExpZero);
    const double y = u + kExpHalf;
    return TokenTaylor().weight(token_low(y), u - (y - kExpHalf), t);
}

// Bins.  A logit v lies at step rint(256 v * octaves per unit) of one grid for all chunks of a row, 32 steps to a bin: the same
// for equal logits and rising with them.  Only the low words of steps are used: below the maximum by less than 20000
// steps, or taken to lie there.  A maximum beyond 2^50 steps is alone: another fp32 value is 2^26 steps off, another int32 2^19,
// and has no weight.
constexpr int kStepsPerBin = kExpTable / kSlotsPerOctave;
__device__ __forceinline__ bool token_alone(double vmax, double rate256) { return !(fabs(vmax) * rate256 < 0x1p50); }

// How a row's logits become weights, relative to a maximum (the row's, or a chunk's)
template <typename T>
struct TokenScale {
    uint32_t kmax;
    double vmax, rate256;   // 256 times the octaves of the weight per unit of the logits
    double low;             // what lies further below has no weight
    int frac, last;         // last: the last step of the maximum's bin
    bool alone;
    const TokenExp *table;
    __device__ __forceinline__ TokenScale(uint32_t kmax_, double rate, int frac_, const TokenExp *t)
        : kmax(kmax_), vmax(TokenKey<T>::value(kmax_)), rate256(rate * kExpTable), low(vmax + kExpZero / rate256), frac(frac_),
          last(token_low(fma(vmax, rate256, kExpHalf)) | (kStepsPerBin - 1)), alone(token_alone(vmax, rate256)), table(t) {}
    __device__ __forceinline__ uint64_t weight(uint32_t k) const
    {
        const uint64_t w = token_exp2((TokenKey<T>::value(k) - vmax) * rate256, table);
        return k == kmax ? 1ull << frac : w;             // also where both are +inf
    }
    // bins below the maximum's
    __device__ __forceinline__ int slot(uint32_t k) const
    {
        if (k == kmax) return 0;
        const uint32_t step = (uint32_t)token_low(fma(fmax(TokenKey<T>::value(k), low), rate256, kExpHalf));
        const uint32_t d = ((uint32_t)last - step) / kStepsPerBin;
        return alone || d >= kSlots ? kSlots - 1 : (int)d;
    }
    // keys that can lie in a slot, a little more than those that do: from ... to; of the last one those that have a weight
    __device__ __forceinline__ void window(int s, uint32_t &from, uint32_t &to) const
    {
        from = kmax, to = kmax;                          // alone: no other has a weight
        if (alone) return;
        const double end = (fma(vmax, rate256, kExpHalf) - kExpHalf) + (double)(last & (kStepsPerBin - 1)) -
                           (double)(token_low(fma(vmax, rate256, kExpHalf)) & (kStepsPerBin - 1)) - (double)(s * kStepsPerBin);
        from = TokenKey<T>::below(s < kSlots - 1 ? (end - kStepsPerBin + 0.5) / rate256 : vmax - (frac + 1) * (double)kExpTable / rate256);
        const uint32_t above = s ? TokenKey<T>::above((end + 0.5) / rate256) : kmax;
        to = above < kmax ? above : kmax;
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
    // whether anything is cut off a row, and whether by a count or a sum
    __device__ __forceinline__ bool cut() const { return top_k > 0 || top_p < 1.0 || min_p > 0.0; }
    __device__ __forceinline__ bool ranked() const { return top_k > 0 || top_p < 1.0; }
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
    __shared__ TokenExp table;
    token_exp_table(&table, a.frac_bits);
    __syncthreads();
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
    const TokenScale<T> scale(kmax, set.rate, a.frac_bits, &table);
    uint64_t w = have ? scale.weight(key) : 0;
    bool keep = have;
    if (set.ranked()) {
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

// A workgroup takes chunk after chunk, the next one's loads under way while it works on one (a workgroup per chunk spent
// most of its life waiting for them).  256 x 131072 bf16: 40 us, with the histogram 48, for the maximum alone 17.
// Two workgroups a CU; three with 80 registers and spills 46 to 63, four 57 to 73.
constexpr int kChunkGrid = 512;
template <typename T>
__global__ __launch_bounds__(512, 4) void token_chunk_kernel(TokenArgs a)
{
    typedef typename TokenKey<T>::Value Value;
    constexpr int WORDS = sizeof(T) / 2;                 // 16-byte words of a group
    __shared__ TokenExp table;
    __shared__ TokenEdges edges;
    __shared__ uint64_t hist_w[kSlots], sh_sum;
    __shared__ uint32_t hist_c[kSlots];
    __shared__ Value sh_max[2][8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t items = (uint32_t)(a.R * a.chunks);
    uint4 next[2][WORDS];
    bool next_whole[2] = {false, false};
    const auto request = [&](uint32_t item) {
        if (item >= items) return;
        const uint32_t row = item / (uint32_t)a.chunks;
        const TokenLogits<T> x(a.logits, row, a.V);
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const int j = (int)(item - row * a.chunks) * kChunkGroups + q * 512 + tid;
            next_whole[q] = x.whole(j);
            if (next_whole[q]) {
#pragma unroll
                for (int w = 0; w < WORDS; w++) next[q][w] = reinterpret_cast<const uint4 *>(x.row + (j * kGroup - x.lead))[w];
            }
        }
    };
    request(blockIdx.x);
    for (int t = tid; t < kSlots; t += 512) hist_w[t] = 0, hist_c[t] = 0;
    token_exp_table(&table, a.frac_bits);
    if (tid == 0) sh_sum = 0;
    int turn = 0;
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x, turn ^= 1) {
        const int64_t row = item / (uint32_t)a.chunks;
        const int chunk = (int)(item - (uint32_t)row * a.chunks);
        const TokenLogits<T> x(a.logits, row, a.V);
        const TokenSettings set(a, row);
        TokenChunk *out = reinterpret_cast<TokenChunk *>(a.workspace) + item;
        Value d[2][8];
        bool whole[2];
#pragma unroll
        for (int q = 0; q < 2; q++) {
            whole[q] = next_whole[q];
            TokenKey<T>::value8(d[q], reinterpret_cast<const T *>(next[q]));
        }
        request(item + gridDim.x);
        const int j0 = chunk * kChunkGroups + tid;
        if (chunk == 0 || chunk * kChunkGroups + kChunkGroups >= x.groups) {     // chunks with an edge of the row
            __syncthreads();
            x.find_edges(&edges);
            __syncthreads();
        }
#pragma unroll
        for (int q = 0; q < 2; q++)
            if (!whole[q]) {
#pragma unroll
                for (int e = 0; e < 8; e++) d[q][e] = -(Value)__builtin_inf();
                if (j0 + q * 512 < x.groups) x.edge_values(d[q], j0 + q * 512, &edges);
            }
        Value m = -(Value)__builtin_inf();
#pragma unroll
        for (int e = 0; e < 8; e++) m = fmax(m, fmax(d[0][e], d[1][e]));         // without NaNs
        m = wave_max(m);
        if (lane == 0) sh_max[turn][wave] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++) m = fmax(m, sh_max[turn][w]);
        const bool any = m > -(Value)__builtin_inf();
        if (any && !set.greedy) {
            double rate256 = set.rate * kExpTable, from = m;
            if (token_alone(m, rate256)) {               // the maximum's likes share the weight, all others have none
#pragma unroll
                for (int q = 0; q < 2; q++)
#pragma unroll
                    for (int e = 0; e < 8; e++) d[q][e] = d[q][e] == m ? (Value)0 : -(Value)__builtin_inf();
                from = 0.0, rate256 = 1.0;
            }
            const double low = from + kExpZero / rate256, y0 = fma(from, rate256, kExpHalf);
            const int first = token_low(y0);
            const uint32_t last = (uint32_t)first | (kStepsPerBin - 1);
            const TokenTaylor taylor(fma(from, rate256, kExpHalf - y0));
            const bool cut = set.cut(), counted = set.top_k > 0;
            uint64_t sum = 0;
            // eight at a time: their chains of dependent operations run side by side
            const auto take = [&](const Value (&v)[8]) {
                int step[8];
                uint64_t w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const double x = fmax((double)v[e], low), y = fma(x, rate256, kExpHalf);     // NaN: low
                    step[e] = token_low(y);
                    w[e] = taylor.weight((int)((uint32_t)step[e] - (uint32_t)first), fma(x, rate256, kExpHalf - y), &table);
                }
#pragma unroll
                for (int e = 0; e < 8; e++) sum += w[e];
                if (cut) {
                    uint32_t at[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        at[e] = (last - (uint32_t)step[e]) / kStepsPerBin;
                        at[e] = at[e] < kSlots ? at[e] : kSlots - 1;
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (w[e]) atomicAdd((unsigned long long *)&hist_w[at[e]], (unsigned long long)w[e]);
                    if (counted) {
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            if (v[e] > -(Value)__builtin_inf()) atomicAdd(&hist_c[at[e]], 1u);
                    }
                }
            };
            take(d[0]);
            take(d[1]);
            sum = wave_sum(sum);
            if (lane == 0) atomicAdd((unsigned long long *)&sh_sum, (unsigned long long)sum);
            __syncthreads();
            if (cut)
                for (int t = tid; t < kSlots; t += 512) {
                    out->weight[t] = hist_w[t], out->count[t] = hist_c[t];
                    hist_w[t] = 0, hist_c[t] = 0;        // for the next chunk, behind its first barrier
                }
        }
        if (tid == 0) {
            out->sum = sh_sum, out->kmax = any ? TokenKey<T>::key_of(m) : 0u, out->have = any;
            sh_sum = 0;
        }
    }
}

// ---- a workgroup per row ----------------------------------------------------------------------------------------------
// HELD > 0: rows of at most HELD groups per thread, kept in registers; HELD = 0: longer ones, from the chunks' records, read
// again where entries matter.  The passes over the row are few and their code is kept short:
// with every step inlined where it is used (145 KB) fetching instructions took longer than all else.
struct TokenEntry {
    uint32_t key;
    int index;
};

template <typename T, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS, 4) void sample_row_kernel(TokenArgs a)
{
    constexpr bool LOCAL = HELD > 0;
    constexpr int WAVES = THREADS / 64;
    constexpr int SEGS = LOCAL ? kTokenLocalV / (kGroup * kSegGroups) + 1 : kTokenMaxSegs;
    constexpr int CHUNKS = LOCAL ? 1 : kTokenMaxChunks;
    constexpr uint32_t kList = LOCAL && THREADS > 128 ? 1024 : 8 * THREADS;   // entries of a border's bin that fit LDS
    __shared__ TokenExp table;
    __shared__ TokenEdges edges;
    // what is kept of a segment, tie counts before; of long rows the groups that have an entry in the border's bin, and the
    // indexes of those that tie, before either
    __shared__ uint64_t seg_w[LOCAL || SEGS > (int)kList / 2 ? SEGS : kList / 2];
    uint32_t *const found = reinterpret_cast<uint32_t *>(seg_w);
    __shared__ double slot_w[kSlots];
    __shared__ uint64_t hist_w[kSlots];                  // LOCAL: by slot; later by digit
    __shared__ uint32_t hist_c[kSlots], slot_c[kSlots];
    __shared__ TokenEntry list[kList];                   // the entries of the border's slot
    __shared__ double chunk_f[CHUNKS];
    __shared__ int chunk_off[CHUNKS];
    __shared__ uint64_t chunk_w[CHUNKS];                 // what is kept of a chunk
    __shared__ uint32_t chunk_k[CHUNKS];                 // their largest keys
    constexpr int PARTS = LOCAL ? 1 : THREADS / kSlots;
    __shared__ double part_w[PARTS][kSlots];             // a row's histogram from every PARTS-th chunk
    __shared__ uint32_t part_c[PARTS][kSlots];
    __shared__ uint32_t sh_key[WAVES], sh_have[WAVES], low_c[WAVES], sh_n, sh_count, sh_ties;
    __shared__ uint64_t sh_sum;
    __shared__ double low_w[WAVES], sh_before;
    __shared__ int sh_at;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    // the chunks' heads, a thread each, under way from the start
    static_assert(LOCAL || kTokenMaxChunks <= THREADS, "a thread per chunk");
    const TokenChunk *chunk = reinterpret_cast<const TokenChunk *>(a.workspace) + row * a.chunks;
    uint32_t head_max = 0, head_have = 0;
    uint64_t head_sum = 0;
    if (!LOCAL && tid < a.chunks) head_max = chunk[tid].kmax, head_have = chunk[tid].have, head_sum = chunk[tid].sum;
    token_exp_table(&table, a.frac_bits);
    if (tid == 0) sh_at = a.V;
    if (LOCAL)
        for (int t = tid; t < kSlots; t += THREADS) hist_w[t] = 0, hist_c[t] = 0;
    const TokenLogits<T> x(a.logits, row, a.V, &edges);
    x.find_edges(&edges);
    __syncthreads();
    const TokenSettings set(a, row);
    const int segs = (x.groups + kSegGroups - 1) / kSegGroups;
    uint32_t held[LOCAL ? HELD : 1][8], held_have[LOCAL ? HELD : 1];
    if constexpr (LOCAL) {
#pragma unroll
        for (int q = 0; q < HELD; q++) {
            const int j = q * THREADS + tid;
            held_have[q] = 0;
            if (j < x.groups) held_have[q] = x.load(held[q], j);
#pragma unroll
            for (int e = 0; e < 8; e++) held[q][e] = held_have[q] >> e & 1 ? held[q][e] : 0u;
        }
    }
    // f(keys, which of them there are, the first one's index, segment) for the segments seg0 ... seg1 - 1: every wave takes
    // whole segments; from memory, AHEAD of them are under way at once
    const auto for_groups = [&](auto ahead, int seg0, int seg1, auto &&f) {
        if constexpr (LOCAL) {
#pragma unroll
            for (int q = 0; q < HELD; q++)
                if (q * WAVES + wave < segs) f(held[q], held_have[q], (q * THREADS + tid) * kGroup - x.lead, q * WAVES + wave);
        } else {
            constexpr int AHEAD = decltype(ahead)::value;
#pragma unroll 1
            for (int s = seg0 + wave; s < seg1; s += AHEAD * WAVES) {
                uint32_t k[AHEAD][8], have[AHEAD];
#pragma unroll
                for (int q = 0; q < AHEAD; q++) {
                    const int j = (s + q * WAVES) * kSegGroups + lane;
                    have[q] = 0;
                    if (s + q * WAVES < seg1 && j < x.groups) have[q] = x.load(k[q], j);
                }
#pragma unroll
                for (int q = 0; q < AHEAD; q++)
                    if (s + q * WAVES < seg1)
                        f(k[q], have[q], ((s + q * WAVES) * kSegGroups + lane) * kGroup - x.lead, s + q * WAVES);
            }
        }
    };
    const std::integral_constant<int, 1> one_ahead{};
    // the row's maximum
    uint32_t m = 0, any = 0;
    if (LOCAL) {
        for_groups(one_ahead, 0, segs, [&](const uint32_t (&k)[8], uint32_t have, int, int) {
            any |= have;
#pragma unroll
            for (int e = 0; e < 8; e++) m = k[e] > m ? k[e] : m;
        });
    } else {
        any = head_have, m = head_have ? head_max : 0u;
    }
    m = wave_max(m);
    any = __ballot(any) != 0;
    if (lane == 0) sh_key[wave] = m, sh_have[wave] = any;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) m = sh_key[w] > m ? sh_key[w] : m, any |= sh_have[w];
    if (!any) {
        if (tid == 0) a.out[row] = -1;
        return;
    }
    if (set.greedy) {
        int seg0 = 0, seg1 = segs;
        if constexpr (!LOCAL) {                          // the first chunk with that maximum
            if (head_have && head_max == m) atomicMin(&sh_at, tid);
            __syncthreads();
            seg0 = sh_at * (kChunkGroups / kSegGroups);
            seg1 = seg0 + kChunkGroups / kSegGroups < segs ? seg0 + kChunkGroups / kSegGroups : segs;
            __syncthreads();
            if (tid == 0) sh_at = a.V;
            __syncthreads();
        }
        for_groups(one_ahead, seg0, seg1, [&](const uint32_t (&k)[8], uint32_t have, int i0, int) {
            int first = a.V;
#pragma unroll
            for (int e = 7; e >= 0; e--) first = (have >> e & 1) && k[e] == m ? i0 + e : first;
            if (first < a.V) atomicMin(&sh_at, first);
        });
        __syncthreads();
        if (tid == 0) a.out[row] = sh_at;
        return;
    }
    const TokenScale<T> scale(m, set.rate, a.frac_bits, &table);
    // The smallest key that reaches min_p (weights rise with keys): 64 keys at a time, six bits of it per turn.
    uint32_t min_key = 0;
    if (set.min_p > 0.0) {
        const double min_w = std::min(set.min_p, 1.0) * (double)(1ull << a.frac_bits);
#pragma unroll 1
        for (int shift = 26;; shift = shift > 2 ? shift - 6 : 0) {
            const uint64_t k = (uint64_t)min_key + ((uint64_t)lane << shift);    // none below min_key reaches it
            const uint64_t hit = __ballot(k >= m || (double)scale.weight((uint32_t)k) >= min_w);
            if (hit & 1) break;
            min_key += ((hit ? (uint32_t)__builtin_ctzll(hit) : 64u) - 1) << shift;
            min_key += 1;
        }
    }
    if constexpr (!LOCAL) {
        if (tid < a.chunks) {
            chunk_k[tid] = head_max;
            chunk_off[tid] = head_have ? scale.slot(head_max) : kSlots;
            chunk_f[tid] = !head_have ? 0.0 : head_max == m ? 1.0 : exp2((TokenKey<T>::value(head_max) - scale.vmax) * set.rate);
            chunk_w[tid] = head_have ? head_sum : 0;
        }
        __syncthreads();
    }
    // what is kept: keys above `key`, and `ties` of those equal to it, the first ones
    uint32_t key = 0, ties = 0xFFFFFFFFu, equal = 0;
    int border = kSlots;                                 // the slot it lies in; kSlots: all are kept
    bool listed = false;                                 // whether `list` holds all of that slot,
    uint32_t list_n = 0;                                 // and how many it has
    if (set.ranked() || (!LOCAL && set.cut())) {
        // ---- the row's histogram -------------------------------------------------------------------------------------
        if (LOCAL) {
            for_groups(one_ahead, 0, segs, [&](const uint32_t (&k)[8], uint32_t have, int, int) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint64_t w = scale.weight(k[e]);
                    const int s = scale.slot(k[e]);
                    if ((have >> e & 1) && w) atomicAdd((unsigned long long *)&hist_w[s], (unsigned long long)w);
                    if ((have >> e & 1) && set.top_k) atomicAdd(&hist_c[s], 1u);
                }
            });
            __syncthreads();
            for (int t = tid; t < kSlots; t += THREADS) slot_w[t] = (double)hist_w[t], slot_c[t] = hist_c[t];
        } else {
            // a chunk's bin s lies chunk_off bins lower in the row, its weights are chunk_f of the row's; every PARTS-th chunk
            // after the other, then the parts, so the sums have one order.  The last bin also takes all that lies below it.
            const int part = tid / kSlots, mine = tid % kSlots;
            double w = 0.0, low = 0.0;
            uint32_t n = 0, low_n = 0;
#pragma unroll 5
            for (int c = part; c < a.chunks; c += PARTS) {
                const int off = chunk_off[c], s = mine - off;
                const bool below = off < kSlots && mine + off >= kSlots - 1;
                uint64_t here_w = 0, below_w = 0;
                uint32_t here_n = 0, below_n = 0;
                if (s >= 0) here_w = chunk[c].weight[s], here_n = chunk[c].count[s];
                if (below) below_w = chunk[c].weight[mine], below_n = chunk[c].count[mine];
                w += chunk_f[c] * (double)here_w, n += here_n;
                low += chunk_f[c] * (double)below_w, low_n += below_n;
            }
            part_w[part][mine] = w, part_c[part][mine] = n;
            low = wave_sum(low), low_n = wave_sum(low_n);
            if (lane == 0) low_w[wave] = low, low_c[wave] = low_n;
            __syncthreads();
            if (tid < kSlots - 1) {
                w = part_w[0][tid], n = part_c[0][tid];
#pragma unroll
                for (int q = 1; q < PARTS; q++) w += part_w[q][tid], n += part_c[q][tid];
                slot_w[tid] = w, slot_c[tid] = n;
            } else if (tid == kSlots - 1) {
                w = 0.0, n = 0;
#pragma unroll
                for (int v = 0; v < WAVES; v++) w += low_w[v], n += low_c[v];
                slot_w[tid] = w, slot_c[tid] = n;
            }
        }
        __syncthreads();
        // ---- the borders, one after the other: top_k, top_p, min_p -----------------------------------------------------
        uint32_t from = 0, to = 0;                       // the window of keys around the last border's slot
        double total = 0.0;                              // what top_p is a part of
        bool have_total = false;
#pragma unroll 1
        for (int which = 0; which < 3; which++) {
            const bool by_count = which == 0;
            if (which == 0 ? !set.top_k : which == 1 ? !(set.top_p < 1.0) : LOCAL || !(set.min_p > 0.0)) continue;
            if (which == 1 && !have_total) {
                double w = 0.0;
#pragma unroll
                for (int e = 0; e < 4; e++) w += slot_w[4 * lane + e];
                total = wave_sum(w);
            }
            const int64_t count = set.top_k;
            const double target = set.top_p * total;
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
                    const bool here = by_count ? c[e] && (int64_t)ca + c[e] >= count : w[e] > 0.0 && wa + w[e] >= target;
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
            int slot = sh_at;
            uint32_t before_c = sh_count;
            double before_w = sh_before;
            if (which == 2) slot = scale.slot(min_key);
            if (slot < 0 || slot > border) continue;     // the row has no more than that: nothing is cut
            if (slot != border || !listed) {             // else the list of the border before is the one
                // keys that can lie there, a little more than those that do
                scale.window(slot, from, to);
                // the entries of a group that lie in the slot, into the list
                const auto put = [&](const uint32_t (&keys)[8], uint32_t have, int i0) {
                    uint32_t near = 0;
#pragma unroll
                    for (int e = 0; e < 8; e++) near |= (uint32_t)(keys[e] >= from && keys[e] <= to) << e;
#pragma unroll 1
                    for (near &= have; near; near &= near - 1) {
                        const int e = __builtin_ctz(near);
                        uint32_t k = keys[0];
#pragma unroll
                        for (int d = 1; d < 8; d++) k = d == e ? keys[d] : k;
                        if (scale.slot(k) != slot) continue;
                        const uint32_t at = atomicAdd(&sh_n, 1u);
                        if (at < kList) list[at] = TokenEntry{k, i0 + e};
                    }
                };
                if constexpr (LOCAL) {
#pragma unroll
                    for (int q = 0; q < HELD; q++) put(held[q], held_have[q], (q * THREADS + tid) * kGroup - x.lead);
                } else {
                    // One workgroup looks at the whole row, which its instructions bound: first for the groups that have such an
                    // entry, then, a thread each, for the entries.  (Entry by entry at once, a wave goes through all of that
                    // for the few of its lanes that have one: 17 us more for 131072 entries.)
                    constexpr int WORDS = sizeof(T) / 2, AHEAD = 8 / WORDS;      // 16-byte words of a group
                    const typename TokenKey<T>::Near near(from, to);
#pragma unroll 1
                    for (int s = wave; s < segs; s += AHEAD * WAVES) {
                        uint4 raw[AHEAD][WORDS];
#pragma unroll
                        for (int q = 0; q < AHEAD; q++) {
                            const int j = (s + q * WAVES) * kSegGroups + lane;
                            if (x.whole(j)) {
#pragma unroll
                                for (int w = 0; w < WORDS; w++)
                                    raw[q][w] = reinterpret_cast<const uint4 *>(x.row + (j * kGroup - x.lead))[w];
                            }
                        }
#pragma unroll
                        for (int q = 0; q < AHEAD; q++) {
                            const int j = (s + q * WAVES) * kSegGroups + lane;
                            if (j < x.groups && (!x.whole(j) || near.any(reinterpret_cast<const T *>(raw[q])))) {
                                const uint32_t at = atomicAdd(&sh_n, 1u);
                                if (at < kList) found[at] = j;
                            }
                        }
                    }
                    __syncthreads();
                    const uint32_t n = sh_n;
                    __syncthreads();
                    if (n <= kList) {                    // else it stays: too many for the list
                        if (tid == 0) sh_n = 0;
                        __syncthreads();
#pragma unroll 1
                        for (uint32_t i = tid; i < n; i += THREADS) {
                            uint32_t k[8];
                            const int j = (int)found[i];
                            const uint32_t have = x.load(k, j);
                            put(k, have, j * kGroup - x.lead);
                        }
                    }
                }
                __syncthreads();
                list_n = sh_n;
                listed = list_n <= kList;
                border = slot;
            }
            if (which == 2) continue;                    // the entries below min_key stay out by their keys
            if (list_n == 0) continue;                   // nothing with a weight below the slots before: nothing is cut
            if (list_n <= 64) {
                // few enough for a lane each: what lies above an entry, by comparing all pairs (every wave does the same)
                const uint32_t q = (uint32_t)lane < list_n ? list[lane].key : 0u;
                const uint64_t w = (uint32_t)lane < list_n ? scale.weight(q) : 0;
                uint32_t above_c = 0, same = 0;
                uint64_t above_w = 0;
#pragma unroll 1
                for (uint32_t j = 0; j < list_n; j++) {
                    const uint32_t kj = __builtin_amdgcn_readlane(q, j);
                    const uint64_t wj = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(w >> 32), j) << 32) |
                                        (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)w, j);
                    above_c += kj > q, above_w += kj > q ? wj : 0, same += kj == q;
                }
                // the border's key: the largest with which the prefix is long enough; should rounding have put the target
                // above all of them, the smallest
                const bool here = (uint32_t)lane < list_n && (by_count ? (int64_t)before_c + above_c + same >= count
                                                                      : before_w + (double)(above_w + same * w) >= target);
                const uint64_t hit = __ballot(here);
                const uint32_t big = wave_max(here ? q : 0u), small = ~wave_max((uint32_t)lane < list_n ? ~q : 0u);
                key = hit ? big : small;
                const int l = __builtin_ctzll(__ballot((uint32_t)lane < list_n && q == key));
                equal = __shfl(same, l);
                before_c += __shfl(above_c, l);
                before_w += (double)__shfl(above_w, l);
            } else {
                // Digit by digit among the slot's keys, from the list or, where it has too many, from the row every time; only
                // the bits in which the list's keys differ (logits of 16 bits have few) or the window's.
                int top_bit = from ^ to ? 32 - __builtin_clz(from ^ to) : 1, low_bit = TokenKey<T>::kFree;
                if (top_bit <= low_bit) top_bit = low_bit + 1;
                uint32_t prefix = top_bit < 32 ? from >> top_bit : 0;
                if (listed) {
                    uint32_t both = 0xFFFFFFFFu, one = 0;
                    for (uint32_t i = tid; i < list_n; i += THREADS) both &= list[i].key, one |= list[i].key;
#pragma unroll
                    for (int o = 32; o; o >>= 1) both &= __shfl_xor(both, o), one |= __shfl_xor(one, o);
                    if (lane == 0) sh_key[wave] = both, sh_have[wave] = one;
                    __syncthreads();
#pragma unroll
                    for (int w = 0; w < WAVES; w++) both &= sh_key[w], one |= sh_have[w];
                    const uint32_t differ = both ^ one;
                    top_bit = differ ? 32 - __builtin_clz(differ) : 1;
                    low_bit = differ ? __builtin_ctz(differ) : 0;
                    prefix = top_bit < 32 ? both >> top_bit : 0;
                }
#pragma unroll 1
                for (int shift = top_bit; shift > low_bit;) {
                    const int width = shift - low_bit < 8 ? shift - low_bit : 8;
                    shift -= width;
                    __syncthreads();
                    for (int t = tid; t < kSlots; t += THREADS) hist_w[t] = 0, hist_c[t] = 0;
                    __syncthreads();
                    const auto add = [&](uint32_t q) {
                        if (shift + width == 32 || q >> (shift + width) == prefix) {
                            const uint32_t d = (q >> shift) & ((1u << width) - 1u);
                            atomicAdd(&hist_c[d], 1u);
                            atomicAdd((unsigned long long *)&hist_w[d], (unsigned long long)scale.weight(q));
                        }
                    };
                    if (listed) {
                        for (uint32_t i = tid; i < list_n; i += THREADS) add(list[i].key);
                    } else {
                        for_groups(one_ahead, 0, segs, [&](const uint32_t (&keys)[8], uint32_t have, int, int) {
                            uint32_t near = 0;
#pragma unroll
                            for (int e = 0; e < 8; e++) near |= (uint32_t)(keys[e] >= from && keys[e] <= to) << e;
#pragma unroll 1
                            for (near &= have; near; near &= near - 1) {
                                const int e = __builtin_ctz(near);
                                uint32_t k = keys[0];
#pragma unroll
                                for (int d = 1; d < 8; d++) k = d == e ? keys[d] : k;
                                if (scale.slot(k) == slot) add(k);
                            }
                        });
                    }
                    __syncthreads();
                    if (wave == 0) {                     // lane l: the digits 255 - 4 l down to 252 - 4 l
                        uint32_t c[4], cs = 0;
                        uint64_t w[4], ws = 0;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            c[e] = hist_c[255 - 4 * lane - e], w[e] = hist_w[255 - 4 * lane - e];
                            cs += c[e], ws += w[e];
                        }
                        uint32_t ca = wave_scan(cs, lane) - cs;
                        uint64_t wa = wave_scan(ws, lane) - ws;
                        int found = -1, seen = -1;       // seen: the last digit that holds anything
                        uint32_t fc = 0, fn = 0;
                        uint64_t fw = 0;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const bool here = c[e] && (by_count ? (int64_t)before_c + ca + c[e] >= count
                                                                : before_w + (double)(wa + w[e]) >= target);
                            if (found < 0 && (here || c[e])) {
                                fc = ca, fw = wa, fn = c[e];
                                seen = 255 - 4 * lane - e;
                                if (here) found = seen;
                            }
                            ca += c[e], wa += w[e];
                        }
                        // should rounding have put the target above all of them: the last one
                        const uint64_t hit = __ballot(found >= 0), some = __ballot(seen >= 0);
                        const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
                        if (lane == l) sh_at = seen, sh_count = fc, sh_sum = fw, sh_ties = fn;
                    }
                    __syncthreads();
                    before_c += sh_count;
                    before_w += (double)sh_sum;
                    equal = sh_ties;
                    prefix = (prefix << width) | (uint32_t)sh_at;
                }
                // bits below low_bit are the same in all keys, or, of 16-bit types, go with the sign
                const uint32_t rest = (1u << low_bit) - 1u;
                key = (prefix << low_bit) | (rest & (listed ? list[0].key : prefix >> (31 - low_bit) & 1 ? 0u : ~0u));
            }
            // the ties of `key` that are kept, before_c entries or before_w of weight lying above them
            const uint64_t w = scale.weight(key);
            if (by_count) {
                const int64_t left = count - before_c;
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
            have_total = true;
        }
    }
    const uint32_t lowest = key > min_key ? key : min_key;
    // ---- the index of the last tie that is kept ----------------------------------------------------------------------------
    int last = a.V;
    if (!LOCAL && listed && ties < equal && key >= lowest) {
        // all entries equal to `key` are in the list: the one with ties - 1 of them before it
        __syncthreads();
        if (tid == 0) sh_n = 0;
        __syncthreads();
        for (uint32_t i = tid; i < list_n; i += THREADS)
            if (list[i].key == key) found[atomicAdd(&sh_n, 1u)] = (uint32_t)list[i].index;
        __syncthreads();
        const uint32_t n = sh_n;
        for (uint32_t i = tid; i < n; i += THREADS) {
            const uint32_t mine = found[i];
            uint32_t before = 0;
#pragma unroll 8
            for (uint32_t j = 0; j < n; j++) before += found[j] < mine;
            if (before == ties - 1) sh_at = (int)mine;
        }
        __syncthreads();
        last = sh_at;
    } else if (ties < equal && key >= lowest) {
        __syncthreads();
        for_groups(one_ahead, 0, segs, [&](const uint32_t (&k)[8], uint32_t have, int, int s) {
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) c += (have >> e & 1) && k[e] == key;
            c = wave_sum(c);
            if (lane == 0) seg_w[s] = c;
        });
        __syncthreads();
        if (wave == 0) {
            uint32_t left = ties;                        // among the segments from base on
            int base = 0;
            for (;; base += 64) {
                const uint32_t c = base + lane < segs ? (uint32_t)seg_w[base + lane] : 0;
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
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if ((have >> e & 1) && --left == 0) sh_at = j * kGroup - x.lead + e;
            }
        }
        __syncthreads();
        last = sh_at;
    }
    // ---- the draw ----------------------------------------------------------------------------------------------------------
    const auto passes = [&](uint32_t k, int i) { return k >= lowest && (k != key || i <= last); };
    const uint32_t word = a.words[row];
    int seg0 = 0, seg1 = segs;                           // where the token lies
    uint32_t drawn_max = m;                              // what the weights are relative to there
    bool by_chunks = false;
    if constexpr (!LOCAL) {
        // The chunk first.  What is kept of every one: of the slots above the border's all, which its histogram holds, of the
        // border's slot the entries of the list.
        by_chunks = border == kSlots || listed;
        if (by_chunks && border < kSlots) {
            for (int c = wave; c < a.chunks; c += WAVES) {
                uint64_t w = 0;
                const int below = border - chunk_off[c];             // the chunk's slots above the row's border
#pragma unroll
                for (int q = 0; q < kSlots / 64; q++)
                    if (q * 64 + lane < below) w += chunk[c].weight[q * 64 + lane];
                w = wave_sum(w);
                if (lane == 0) chunk_w[c] = w;
            }
            __syncthreads();
            for (uint32_t i = tid; i < list_n; i += THREADS) {
                const TokenEntry q = list[i];
                if (!passes(q.key, q.index)) continue;
                const int c = (q.index + x.lead) / (kGroup * kChunkGroups);
                const TokenScale<T> sc(chunk_k[c], set.rate, a.frac_bits, &table);
                atomicAdd((unsigned long long *)&chunk_w[c], (unsigned long long)sc.weight(q.key));
            }
        }
        if (by_chunks) {
            __syncthreads();
            if (wave == 0) {
                double all = 0.0, before = 0.0;
                for (int c0 = 0; c0 < a.chunks; c0 += 64)
                    all += wave_sum(c0 + lane < a.chunks ? chunk_f[c0 + lane] * (double)chunk_w[c0 + lane] : 0.0);
                const double bar = (double)word * 0x1p-32 * all;
                int at = -1, seen = -1;                  // the chunk that reaches over the bar; the last with any weight
                double from = 0.0;
                for (int c0 = 0; c0 < a.chunks && at < 0; c0 += 64) {
                    const double v = c0 + lane < a.chunks ? chunk_f[c0 + lane] * (double)chunk_w[c0 + lane] : 0.0;
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
            constexpr int kSegsPerChunk = kChunkGroups / kSegGroups;
            seg0 = sh_at * kSegsPerChunk;
            seg1 = seg0 + kSegsPerChunk < segs ? seg0 + kSegsPerChunk : segs;
            drawn_max = chunk_k[sh_at];
        }
    }
    const TokenScale<T> drawn(drawn_max, set.rate, a.frac_bits, &table);
    const auto kept = [&](uint32_t k, int i, bool have) -> uint64_t {
        return have && passes(k, i) ? drawn.weight(k) : 0;
    };
    __syncthreads();
    for_groups(one_ahead, seg0, seg1, [&](const uint32_t (&k)[8], uint32_t have, int i0, int s) {
        uint64_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) w += kept(k[e], i0 + e, have >> e & 1);
        w = wave_sum(w);
        if (lane == 0) seg_w[s] = w;
    });
    __syncthreads();
    if (wave != 0) return;
    uint64_t all = 0;
    for (int s = seg0 + lane; s < seg1; s += 64) all += seg_w[s];
    all = wave_sum(all);
    uint64_t bar = token_bar(word, all);                 // below all: some segment reaches over it
    if (by_chunks) {
        const double left = sh_before;
        bar = left > 0.0 ? (uint64_t)left : 0;
        bar = bar < all ? bar : all - 1;
    }
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
        w[e] = kept(k[e], j * kGroup - x.lead + e, have >> e & 1);
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
}

static int token_chunks(int64_t V) { return (int)ceil_div(V + kGroup - 1, kChunkGroups * kGroup); }
// Rows of one launch, more of them in launches that follow each other: a grid's threads are counted in 32 bits, and the
// chunks' records of a launch are kept below 6.5 GB (the next launch takes the same memory).
static int64_t token_rows(int64_t V)
{
    return V <= 64 ? 1LL << 24 : V <= kTokenLocalV ? 1LL << 21 : (1LL << 21) / token_chunks(V);
}

template <typename T>
static int token_launch(const TokenArgs &a, hipStream_t st, const char *who)
{
    // Borders, in microseconds without a cut / with top_p = 0.9, logits N(0, 2.5^2), this kernel / the one on the other side:
    //   4096 x 64 fp32        9 /  15      15 /  25 (64 threads)
    //   5818 x 500 fp32       - /  29       - /  66 (256 threads), 10 x 500 12, 12
    //   5338 x 741 bf16       - /  43       - /  68 (256 threads), 10 x 1000 14, 14
    //   1024 x 2000 bf16     10 /  21      26 /  65 (1024 threads)
    //    200 x 8000 bf16     10 /  25       9 /  27 (1024 threads of one group)
    //    256 x 16000 bf16    13 /  28      18 /  37 (by chunks)
    // A CU holds 1024 threads of these; where rows outnumber what all of them hold, half the threads a row (with
    // top_p, a row's threads as they are / half of them):
    //   8, 1024, 4000 x 2000 bf16      15, 21,  67 /  19, 22,  54
    //   8,  512, 4000 x 4000 bf16      17, 23, 148 /  20, 24, 101
    //   8,  512, 4000 x 8000 bf16      24, 34, 219 /  31, 36, 165
    //  10,      1024 x 16000 fp32      29,     115 /  31,      83
    // fp32 and int32 have the same borders: at one the form for few rows takes as long as the other or up to 4 us less, a row above
    // it up to 10 us more (with top_p 512 rows of 8000 fp32 34 / 36, 513 46 / 40; 256 of 16000 int32 37 / 39, 257 55 / 45).
    // By chunks: 64 x 32768 bf16 17 / 31, 5 x 50001 fp16 17 / 32, 256 x 131072 bf16 51 / 93, the largest entry alone 20.  512
    // threads a row, 1024 for the longest: 1024 x 32768 bf16 113, 160; 400 x 131072 161, 155; 1 x 131072 fp32 43, 37.
    const auto launch = [&](auto *kernel, int threads) { kernel<<<dim3((unsigned)a.R), dim3(threads), 0, st>>>(a); };
    if (a.V <= 64) {
        sample_short_kernel<T><<<dim3((unsigned)ceil_div(a.R, 4)), dim3(256), 0, st>>>(a);
    } else if (a.V <= 64 * kGroup - 8) {                 // a row that starts inside a group reaches into one more
        launch(sample_row_kernel<T, 64, 1>, 64);
    } else if (a.V <= 128 * kGroup - 8) {
        launch(sample_row_kernel<T, 128, 1>, 128);
    } else if (a.V <= 256 * kGroup - 8) {
        a.R <= 1024 ? launch(sample_row_kernel<T, 256, 1>, 256) : launch(sample_row_kernel<T, 128, 2>, 128);
    } else if (a.V <= 512 * kGroup - 8) {
        a.R <= 512 ? launch(sample_row_kernel<T, 512, 1>, 512) : launch(sample_row_kernel<T, 256, 2>, 256);
    } else if (a.V <= 1024 * kGroup - 8) {
        a.R <= 512 ? launch(sample_row_kernel<T, 512, 2>, 512) : launch(sample_row_kernel<T, 256, 4>, 256);
    } else if (a.V <= kTokenLocalV) {
        a.R <= 256 ? launch(sample_row_kernel<T, 1024, 2>, 1024) : launch(sample_row_kernel<T, 512, 4>, 512);
    } else {
        token_chunk_kernel<T><<<dim3((unsigned)std::min<int64_t>(a.R * a.chunks, kChunkGrid)), dim3(512), 0, st>>>(a);
        if (const int rc = check_launch(who)) return rc;
        a.V <= 65536 ? launch(sample_row_kernel<T, 512, 0>, 512) : launch(sample_row_kernel<T, 1024, 0>, 1024);
    }
    return check_launch(who);
}

}  // namespace nb

extern "C" {
int64_t nb_sample_tokens_workspace_bytes(int64_t R, int64_t V)
{
    if (R <= 0 || V <= nb::kTokenLocalV || V > nb::kTokenMaxV) return 0;
    return std::min(R, nb::token_rows(V)) * nb::token_chunks(V) * (int64_t)sizeof(nb::TokenChunk);
}

int nb_sample_tokens(int32_t *out, const void *logits, int type, const uint32_t *words, const float *temperature,
                     double temperature_all, const int32_t *top_k, int64_t top_k_all, const float *top_p,
                     double top_p_all, const float *min_p, double min_p_all, int64_t R, int64_t V, void *workspace,
                     int64_t workspace_bytes, nb_stream_t stream)
{
    const char *who = "nb_sample_tokens";
    NB_REQUIRE(R >= 0 && V >= 1, "%s: bad shape", who);
    NB_REQUIRE(V <= nb::kTokenMaxV, "%s: rows of %lld entries, at most %lld", who, (long long)V, (long long)nb::kTokenMaxV);
    NB_REQUIRE(R <= (1LL << 40), "%s: too many rows", who);
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
    const int64_t most = nb::token_rows(V), size = type == NB_TYPE_F32 || type == NB_TYPE_I32 ? 4 : 2;
    const hipStream_t st = nb::as_stream(stream);
    for (int64_t r0 = 0; r0 < R; r0 += most) {
        const auto from = [&](auto *settings) { return settings ? settings + r0 : nullptr; };
        const nb::TokenArgs a{out + r0, (const uint8_t *)logits + r0 * V * size, words + r0, from(temperature), from(top_p),
                              from(min_p), from(top_k), temperature_all, top_p_all, min_p_all, top_k_all,
                              std::min(most, R - r0), (int)V, std::min(51, 61 - log2v), nb::token_chunks(V),
                              (uint8_t *)workspace};
        const int rc = type == NB_TYPE_F32   ? nb::token_launch<float>(a, st, who)
                       : type == NB_TYPE_F16 ? nb::token_launch<_Float16>(a, st, who)
                       : type == NB_TYPE_BF16 ? nb::token_launch<nb::Bf16>(a, st, who)
                                              : nb::token_launch<int32_t>(a, st, who);
        if (rc) return rc;
    }
    return NB_OK;
}
}  // extern "C"
