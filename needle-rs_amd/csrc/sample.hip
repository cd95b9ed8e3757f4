// A token drawn from each row of logits under a temperature, min-p, top-k and
// top-p, by a random number that is given.
//
// All rules cut the row's order (logits descending, equal ones by their number)
// behind some token, and the draw is a token of that order too: the first whose
// weights, added up, reach a target.  So no row is sorted:
//   a short top-k: the row's tokens are counted in bins that follow the order, those
//     up to the bin of the k-th are listed, and the list is put in order;
//   else: weights (with a top-k tokens too) are added up in the bins, the bin of a target
//     is found, its tokens' in finer ones, and the few of that are looked at one by one;
//   anything unusual (too many equal logits, infinite ones): the row is searched in
//     finer and finer bins, by the digits of the order.
// Weights are whole numbers, exp((l - M) / T) in units of 2^-s, worked out in fp64: a
// pick next to a border is the border's and not the rounding's, and sums of whole
// numbers are the same in any order.  s is 49, or less (37 or more) where a bound on the
// weights of all of a long row's tokens, before top-k and top-p, asks for it: their sum
// stays below 2^62.
//
// A block a row of up to kSlice logits, which stay in its registers.  Longer rows: a
// block a slice looks for its largest logit and lists its own short top-k; where
// there is none, the slices' bins are added up in a second launch, and the tokens of
// the bins that matter listed in a third; a block a row ends.
//
// What bounds it (MI355X; kernels):
//   one row of 8192, every rule: 5.6 us, one block's phases one after another.
//   1024 rows of 8192, top-p 0.9: 22.8 us (34 MB, 7 at a large copy's rate).  Vector
//     instructions, 70 a token: 30 for its weight and bin, the rest for the row's range,
//     the two searches and the scans.  (80 registers leave three blocks a CU; held to 64,
//     which spills, four blocks took no less.)
//   320 rows of 8191, the whole distribution: 14 us, two blocks on some of the CUs.
//   200 rows of 100003 (80 MB, 17 at a large copy's rate; a call): top-k 50 in all 34 us,
//     no top-k 85 (slices 20, bins 36, gather 22, draw 12), top-k 1000 87.  The bins: fp64
//     weights, five blocks a row with up to three slices one after another.
#include "nd_internal.h"
#include "nd_lanes.h"

#include <algorithm>

namespace {

constexpr int kSlice = 8192;
constexpr int kBins = 1024;
constexpr int kList = 512;       // tokens that are put in order, a thread each
constexpr int kShort = 448;      // the longest top-k that is listed whole
constexpr int kFew = 64;         // tokens of a bin that are looked at one by one
constexpr int kMostScale = 49;
constexpr uint32_t kNoBin = 0xffff;
constexpr int kMarked = -2;      // a row that is left to the search

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));  // rows may start anywhere

// A slice's largest and lowest logit (of tokens), a bound on its weights beside the
// largest, and the tokens listed, -1 for too many; a greedy row's: its first maximum.
struct Part {
    float top, low, sum;
    int listed;
};

struct Sample {
    const float *x, *temperature, *min_p, *top_p, *u;
    const int32_t *top_k;
    size_t x_stride;
    int n;
    int32_t *next;
    float *prob;
    int slices;       // of a row; more than one:
    int blocks;       // a row's, that share the slices in the second and third launch
    Part *part;       // [rows][slices]
    uint64_t *bins;   // [rows][kBins]
    uint64_t *list;   // [rows][slices][kList]
    uint32_t *count;  // [rows][kBins]
    int *scale;       // [rows], of rows by their bins
};

// The order of the floats as that of whole numbers, the largest first (-0 as 0).
__device__ inline uint32_t place_of(float l)
{
    const uint32_t u = __float_as_uint(l + 0.0f);
    return ~(u ^ (u >> 31 ? 0xffffffffu : 0x80000000u));
}

// w * u for 0 <= u <= 1, as the whole number below or above.
__device__ inline uint64_t part_of(uint64_t w, float u, bool up)
{
    const uint32_t b = __float_as_uint(u);
    const int e = int(b >> 23);
    const uint64_t m = e ? (b & 0x7fffffu) | 0x800000u : b & 0x7fffffu;
    const int sh = 150 - (e ? e : 1);  // u = m 2^-sh, sh 23 .. 149
    uint64_t hi = __umul64hi(w, m), lo = w * m, rest;
    if (sh >= 128) {
        rest = hi | lo;
        lo = 0;
    } else if (sh >= 64) {
        rest = lo | (sh > 64 ? hi << (128 - sh) : 0);
        lo = hi >> (sh - 64);
    } else {
        rest = lo << (64 - sh);
        lo = lo >> sh | hi << (64 - sh);
    }
    return lo + (up && rest ? 1 : 0);
}

// A row's rules.
struct Row {
    float top;          // its largest logit
    double by, low;     // log2(e) / T; tokens are those at top + low and above
    float bins;         // bins a unit of l
    int scale;
    float T, u, p;
    int k;
    bool greedy;
};

__device__ inline Row rules_of(const Sample &s, size_t row)
{
    Row r{};
    r.T = s.temperature ? s.temperature[row] : 1.0f;
    const float mp = s.min_p ? s.min_p[row] : 0.0f, u = s.u[row];
    r.k = s.top_k ? s.top_k[row] : 0;
    if (r.k >= s.n) r.k = 0;
    r.p = s.top_p ? s.top_p[row] : 1.0f;
    r.u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    r.greedy = !(r.T > 0.0f) || mp > 1.0f;
    r.by = r.greedy ? 1.0 : 1.4426950408889634 / double(r.T);
    // (weights below 2^-64 are no whole unit)
    r.low = fmax(-64.0 / r.by, -1e300);
    // (of an infinite temperature every weight is 1, which a min_p up to 1 lets stay)
    if (mp > 0.0f && r.T < INFINITY) r.low = fmax(r.low, mp < 1.0f ? double(r.T) * log(double(mp)) : 0.0);
    if (r.greedy) r.low = 0.0;
    return r;
}

// With the row's largest and lowest logit: 16 bins an octave of weights, or as many as
// the row's logits need.
__device__ inline void range_of(Row &r, float top, float low)
{
    r.top = top;
    if (top == INFINITY) r.low = 0.0;
    r.bins = fminf(fmaxf(16.0f * float(r.by), float(kBins - 1) / (top - low)), 1e30f);
}

// The logit's distance from the largest, exactly; a token's is r.low or more (that of
// -inf and of NaN is not; where the largest is infinite, so is no other finite one's).
__device__ inline double behind(const Row &r, float l) { return l == r.top ? 0.0 : double(l) - double(r.top); }
__device__ inline bool token(const Row &r, float l) { return behind(r, l) >= r.low; }

// 2^(d by) in units of 2^-scale (scale <= 50), to the nearest, for a d <= 0.  2^f, |f|
// <= 1/2, by the polynomial of degree 11 through its values at Chebyshev's nodes (2e-17
// of it off).  What 2^52 is added to keeps its whole part in the low 52 bits.  (f is
// written as the one operation that it is, lest one caller's is and another's is not:
// a token's weight is the same number wherever it is worked out.)
__device__ inline uint64_t units_of(double d, double by, int scale)
{
    // d by + scale as a whole number in the low bits of `at`, and the rest of it
    const double whole = 0x1.8p52 + double(scale), at = __builtin_fma(d, by, whole), f = __builtin_fma(d, by, whole - at);
    constexpr double c[] = {1.0,
                            0.6931471805599453,
                            0.24022650695910158,
                            0.055504108664821625,
                            0.009618129107587256,
                            0.001333355814640647,
                            0.00015403530463724353,
                            1.5252733841556773e-05,
                            1.3215432535912375e-06,
                            1.0178057087733941e-07,
                            7.074194297288521e-09,
                            4.4558179083360645e-10};
    double p = c[11];
#pragma unroll
    for (int i = 10; i >= 0; --i) p = __builtin_fma(p, f, c[i]);
    // (the exponent moves by at - 2^52 3/2: -64 .. 50)
    const int64_t q = __double_as_longlong(p) + int64_t(uint64_t(uint32_t(__double_as_longlong(at))) << 52);
    return uint64_t(__double_as_longlong(__longlong_as_double(q) + 0x1p52)) & 0xfffffffffffffull;
}

// The weight of a logit in units; 0: no token.
__device__ inline uint64_t weight_of(const Row &r, float l)
{
    const double d = behind(r, l);
    return d >= r.low ? units_of(d, r.by, r.scale) : 0;
}

// A little more than the weight; 0: no token.  (The argument is worked out in fp64, whose
// range holds any two logits' distance and any 1 / T, and rounded by 2^-24 of its size, of
// 64 at most.)
__device__ inline float bound_of(const Row &r, float l)
{
    const double d = behind(r, l);
    return d >= r.low ? __builtin_amdgcn_exp2f(float(d * r.by)) * 1.0001f : 0.0f;
}

// The scale for weights that come to `sum` or less: below 2^62 units.
__device__ inline int scale_of(float sum) { return min(62 - __builtin_amdgcn_frexp_expf(sum * 1.001f), kMostScale); }

__device__ inline int bin_of(const Row &r, float l)
{
    return l == r.top ? 0 : int(fminf((r.top - l) * r.bins, float(kBins - 1)));
}

// The same where the largest logit is finite.
__device__ inline uint32_t bin_below(const Row &r, float l) { return uint32_t(fminf((r.top - l) * r.bins, float(kBins - 1))); }

struct Shared {
    uint64_t weight[kBins], list[kList], sums[kList];
    uint64_t room[3][16], best[3];
    uint32_t count[kBins], listed, finer, bin;  // finer: what cut_in lists the second time
};

// Where a target lies: the token, the weights up to it and its own.
struct Cut {
    uint64_t place, upto, weight;
};

// The whole numbers of the threads before this one added up, and of all (a barrier;
// `room` is not used again before another).
template <int NT>
__device__ inline uint64_t block_scan(uint64_t v, uint64_t &before, uint64_t *room)
{
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const uint64_t up = ndl::wave_scan(v);
    if (lane == 63) room[w] = up;
    __syncthreads();
    // the waves' (16 at most) in the first lanes
    const uint64_t x = ndl::row_scan(room[lane & (NT / 64 - 1)]);
    before = up - v + (w ? ndl::of_lane(x, w - 1) : 0);
    return ndl::of_lane(x, NT / 64 - 1);
}

__device__ inline uint64_t order_of(float l, int i) { return uint64_t(place_of(l)) << 24 | uint32_t(i); }

// The logit of a place in the order (+0 for both zeros).
__device__ inline float logit_of(uint64_t place)
{
    const uint32_t u = ~uint32_t(place >> 24);
    return __uint_as_float(u ^ (u >> 31 ? 0x80000000u : 0xffffffffu));
}

__device__ inline void done(const Sample &s, size_t row, int next, double chance)
{
    if (threadIdx.x == 0) {
        s.next[row] = next;
        if (s.prob) s.prob[row] = float(chance);
    }
}

// top and low over the block; every thread gets both (a barrier, as block_scan).
template <int NT>
__device__ inline void meet(float &top, float &low, uint64_t *room)
{
    top = ndl::wave_max64(top);
    low = -ndl::wave_max64(-low);
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = uint64_t(__float_as_uint(low)) << 32 | __float_as_uint(top);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        const uint64_t x = room[i];
        top = fmaxf(top, __uint_as_float(uint32_t(x)));
        low = fminf(low, __uint_as_float(uint32_t(x >> 32)));
    }
}

template <int NT>
__device__ inline float sum_over(float v, uint64_t *room)
{
    v = ndl::wave_sum64(v);
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = __float_as_uint(v);
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) v += __uint_as_float(uint32_t(room[i]));
    return v;
}

// ---- a row by finer and finer bins --------------------------------------------

// Any row, whatever its logits and rules, from memory: a block.
template <int NT>
__device__ __forceinline__ void search(const Sample &s, size_t row, Row r, Shared &h)
{
    const int t = threadIdx.x;
    const float *x = s.x + row * s.x_stride;
    constexpr int B = kBins / NT;
    auto clear = [&]() {
        __syncthreads();
        for (int b = t; b < kBins; b += NT) h.count[b] = 0, h.weight[b] = 0;
        __syncthreads();
    };
    auto add = [&](int b, uint64_t w) {
        atomicAdd(&h.count[b], 1u);
        atomicAdd(reinterpret_cast<unsigned long long *>(&h.weight[b]), w);
    };
    uint64_t tokens = 0, all = 0;
    auto scan = [&]() {  // to sums up to each bin
        __syncthreads();
        uint64_t c[B], w[B], cs = 0, ws = 0, cb, wb;
#pragma unroll
        for (int e = 0; e < B; ++e) cs += c[e] = h.count[B * t + e], ws += w[e] = h.weight[B * t + e];
        tokens = block_scan<NT>(cs, cb, h.room[0]);
        all = block_scan<NT>(ws, wb, h.room[1]);
#pragma unroll
        for (int e = 0; e < B; ++e) {
            h.count[B * t + e] = uint32_t(cb += c[e]);
            h.weight[B * t + e] = wb += w[e];
        }
        __syncthreads();
    };
    auto each = [&](auto f) {
#pragma unroll 1
        for (int i = t; i < s.n; i += NT) {
            const float l = x[i];
            const uint64_t w = weight_of(r, l);
            if (w) f(l, i, w);
        }
    };
    // the unit
    float bound = 0.0f;
#pragma unroll 1
    for (int i = t; i < s.n; i += NT) bound += bound_of(r, x[i]);
    bound = sum_over<NT>(bound, h.room[2]);
    r.scale = scale_of(bound);
    // The cuts one after another: behind the k-th token, where the weights come to
    // top_p, and the draw: each the first token at which the tokens or the weights reach
    // `target`, 1 .. all of them.
    bool whole = false;  // the row's own bins stand in h
    uint64_t sum = 0, target = 0;
    for (int stage = 0; stage < 3; ++stage) {
        if (!whole) {
            clear();
            each([&](float l, int, uint64_t w) { add(bin_of(r, l), w); });
            scan();
            whole = true;
            if (stage == 0) sum = all;
        }
        const bool by_count = stage == 0;
        if (stage == 0) {
            if (!(r.k > 0 && uint64_t(r.k) < tokens)) continue;
            target = uint64_t(r.k);
        } else if (stage == 1) {
            if (!(r.p < 1.0f)) continue;
            target = part_of(sum, fmaxf(r.p, 0.0f), true);
            target = target ? target : 1;
        } else {
            target = part_of(sum, r.u, false) + 1;
            target = target < sum ? target : sum;
        }
        uint64_t before = 0, beforew = 0, prefix = 0;
        int bin = -1;
        // finer and finer: the row's bins, then digits of the order, ten bits each (of 56:
        // the first digit has six)
        for (int shift = 60;; shift -= 10) {
            // the bin in which the target lies
            for (int b = t; b < kBins; b += NT) {
                const uint64_t now = before + (by_count ? h.count[b] : h.weight[b]);
                const uint64_t was = before + (b == 0 ? 0 : by_count ? h.count[b - 1] : h.weight[b - 1]);
                if (was < target && now >= target) h.bin = uint32_t(b);
            }
            if (t == 0) h.listed = 0;
            __syncthreads();
            const int b = int(h.bin);
            const uint32_t many = h.count[b] - (b ? h.count[b - 1] : 0);
            before += b ? (by_count ? h.count[b - 1] : h.weight[b - 1]) : 0;
            beforew += b ? h.weight[b - 1] : 0;
            if (bin < 0)
                bin = b;
            else
                prefix = prefix << 10 | uint32_t(b);
            __syncthreads();
            auto in = [&](float l, int i) { return bin_of(r, l) == bin && order_of(l, i) >> shift == prefix; };
            if (many <= uint32_t(kList)) {
                each([&](float l, int i, uint64_t) {
                    if (in(l, i)) h.list[atomicAdd(&h.listed, 1u)] = order_of(l, i);
                });
                __syncthreads();
                uint64_t mine = 0, w = 0;
                if (uint32_t(t) < many) {
                    mine = h.list[t];
                    w = weight_of(r, logit_of(mine));
                    h.sums[t] = w;
                }
                __syncthreads();
                if (uint32_t(t) < many) {
                    uint64_t upto = 0, rank = 0;
#pragma unroll 1
                    for (uint32_t j = 0; j < many; ++j)
                        if (h.list[j] <= mine) upto += h.sums[j], ++rank;
                    const uint64_t now = before + (by_count ? rank : upto);
                    if (now >= target && now - (by_count ? 1 : w) < target) {
                        h.best[0] = mine;
                        h.best[1] = beforew + upto;
                        h.best[2] = w;
                    }
                }
                __syncthreads();
                break;
            }
            // too many: their next ten bits
            whole = false;
            clear();
            each([&](float l, int i, uint64_t w) {
                if (in(l, i)) add(int(order_of(l, i) >> (shift - 10) & 1023), w);
            });
            scan();
        }
        if (stage < 2)
            sum = h.best[1];
        else
            done(s, row, int(h.best[0] & 0xffffff), double(h.best[2]) / double(sum));
        __syncthreads();
    }
}

// ---- the common ways ------------------------------------------------------------

// A slice's logits in registers (what is no token, NaN too, is -inf), and their bins,
// two a word.
template <int NT>
struct Held {
    static constexpr int kPer = kSlice / NT;
    float v[kPer];
    uint32_t b[kPer / 2];
    int t0;
    __device__ inline int at(int j) const { return t0 + (j >> 2) * 4 * NT + 4 * int(threadIdx.x) + (j & 3); }
    __device__ inline void load(const float *x, int from, int n)
    {
        t0 = from;
#pragma unroll
        for (int c = 0; c < kPer / 4; ++c) {
            const int k = at(4 * c);
            if (k + 4 <= n) {
                const float4u l = *reinterpret_cast<const float4u *>(x + k);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * c + e] = l[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * c + e] = k + e < n ? x[k + e] : -INFINITY;
            }
        }
    }
    __device__ inline void clean()
    {
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[j] = v[j] > -INFINITY ? v[j] : -INFINITY;
    }
    // (cleaned) the largest and the lowest token's
    __device__ inline void range(float &top, float &low)
    {
        top = -INFINITY, low = INFINITY;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const bool is = v[j] > -INFINITY;
            low = fminf(low, is ? v[j] : INFINITY);
            v[j] = is ? v[j] : -INFINITY;
            top = fmaxf(top, v[j]);
        }
    }
    // the tokens' bins, and in those their weights (of a finite top)
    template <bool WEIGHTS, bool COUNT>
    __device__ inline void lay(const Row &r, Shared &h)
    {
        const double top = double(r.top);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const double d = double(v[j]) - top;
            uint32_t bin = kNoBin;
            if (d >= r.low) {
                bin = bin_below(r, v[j]);
                if constexpr (COUNT) atomicAdd(&h.count[bin], 1u);
                if constexpr (WEIGHTS)
                    atomicAdd(reinterpret_cast<unsigned long long *>(&h.weight[bin]), units_of(d, r.by, r.scale));
            }
            b[j / 2] = j & 1 ? b[j / 2] | bin << 16 : bin;
        }
    }
    // f of the tokens of bins from .. to and of one more
    template <typename F>
    __device__ inline void each(const Row &, uint32_t from, uint32_t to, F f) const
    {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const uint32_t bin = j & 1 ? b[j / 2] >> 16 : b[j / 2] & 0xffff;
            if (bin - from <= to - from) {
                float l = v[j];
                asm volatile("" : "+v"(l));  // (the order of all of them is not worked out ahead, and kept)
                f(l, order_of(l, at(j)));
            }
        }
    }
    // the number of the first logit that is `top`, over the block
    __device__ inline int first(float top, uint64_t *room) const
    {
        int i = 0x7fffffff;
#pragma unroll
        for (int j = kPer - 1; j >= 0; --j) i = v[j] == top ? at(j) : i;
#pragma unroll
        for (int d = 32; d; d /= 2) i = min(i, __shfl_xor(i, d));
        if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = uint64_t(i);
        __syncthreads();
        for (int k = 0; k < NT / 64; ++k) i = min(i, int(room[k]));
        return i;
    }
};

// What the slices have listed, a wave a slice.  The first of a wave are asked for ahead of
// the row's rules.
template <int NT>
struct Lists {
    const uint64_t *list;
    const Part *part;
    int slices, many0;
    uint64_t o0;
    __device__ inline Lists(const Sample &s, size_t row)
        : list(s.list + row * s.slices * kList), part(s.part + row * s.slices), slices(s.slices), many0(0), o0(0)
    {
        const int i = int(threadIdx.x >> 6);
        if (i < slices) {
            many0 = part[i].listed;
            o0 = list[size_t(i) * kList + (threadIdx.x & 63)];
        }
    }
    template <typename F>
    __device__ inline void all(const Row &r, F f) const
    {
        const int lane = int(threadIdx.x & 63), first = int(threadIdx.x >> 6);
        auto take = [&](uint64_t o) {
            const float l = logit_of(o);
            if (token(r, l)) f(l, o);
        };
        if (lane < many0) take(o0);
        for (int j = lane + 64; j < many0; j += 64) take(list[size_t(first) * kList + j]);
        for (int i = first + NT / 64; i < slices; i += NT / 64) {
            const int many = part[i].listed;
            for (int j = lane; j < many; j += 64) take(list[size_t(i) * kList + j]);
        }
    }
    template <bool WEIGHTS, bool COUNT>
    __device__ inline void lay(const Row &r, Shared &h) const
    {
        all(r, [&](float l, uint64_t) { atomicAdd(&h.count[bin_of(r, l)], 1u); });
    }
    template <typename F>
    __device__ inline void each(const Row &r, uint32_t from, uint32_t to, F f) const
    {
        all(r, [&](float l, uint64_t o) {
            if (uint32_t(bin_of(r, l)) - from <= to - from) f(l, o);
        });
    }
};

__device__ inline void enlist(Shared &h, uint64_t o, uint32_t &listed)
{
    const uint32_t at = atomicAdd(&listed, 1u);  // (what is beyond the list's room is counted alone)
    if (at < uint32_t(kList)) h.list[at] = o;
}

// A thread's bins' tokens (or weights) and those before them.
template <int NT, typename T>
struct Bins {
    static constexpr int B = kBins / NT;
    uint64_t v[B], before, all;
    __device__ inline void read(const T *from, uint64_t *room)
    {
        uint64_t sum = 0;
#pragma unroll
        for (int e = 0; e < B; ++e) sum += v[e] = from[B * int(threadIdx.x) + e];
        all = block_scan<NT>(sum, before, room);
    }
    // f of the bin in which they reach `target`, and of what comes before it
    template <typename F>
    __device__ inline void with(uint64_t target, F f) const
    {
        uint64_t was = before;
#pragma unroll
        for (int e = 0; e < B; ++e) {
            if (was < target && was + v[e] >= target) f(uint32_t(B * int(threadIdx.x) + e), was, v[e]);
            was += v[e];
        }
    }
    // f of what comes before bin b, and of the bin
    template <typename F>
    __device__ inline void at(uint32_t b, F f) const
    {
        uint64_t was = before;
#pragma unroll
        for (int e = 0; e < B; ++e) {
            if (uint32_t(B * int(threadIdx.x) + e) == b) f(was, v[e]);
            was += v[e];
        }
    }
};

// Lists the tokens up to the bin of the `want`-th and says how many, -1: more than a
// list holds; `want` becomes the tokens' number, if that is less.  h.count and
// h.listed are 0.
template <int NT, typename Src>
__device__ inline int list_first(const Row &r, int &want, Shared &h, Src &src)
{
    src.template lay<false, true>(r, h);
    __syncthreads();
    Bins<NT, uint32_t> c;
    c.read(h.count, h.room[1]);
    want = min(want, int(c.all));
    c.with(uint64_t(want), [&](uint32_t bin, uint64_t was, uint64_t v) {
        h.bin = bin;
        h.best[0] = was + v;
    });
    __syncthreads();
    const int many = int(h.best[0]);
    if (many > kList) return -1;
    src.each(r, 0, h.bin, [&](float, uint64_t o) { enlist(h, o, h.listed); });
    __syncthreads();
    return many;
}

// f of the places of the list's first `many` and their number in it, four at a time: what
// is behind them counts as the last of all (a barrier).
template <typename F>
__device__ inline void listed_all(Shared &h, int many, F f)
{
    const int t = threadIdx.x, all = (many + 3) & ~3;
    if (t >= many && t < all) h.list[t] = ~uint64_t(0);
    __syncthreads();
    if ((t & ~63) >= many) return;  // (a wave without a place in it)
    for (int j = 0; j < all; j += 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f(h.list[j + e], j + e);
    }
}

// Draws from the first `want` of the `many` tokens listed.
template <int NT>
__device__ inline void draw_listed(const Sample &s, size_t row, Row r, int want, int many, Shared &h)
{
    const int t = threadIdx.x;
    r.scale = kMostScale;
    const uint64_t own = t < many ? h.list[t] : 0;
    int rank = 0;
    listed_all(h, many, [&](uint64_t o, int) { rank += o < own; });
    if (t < many) h.sums[rank] = own;
    __syncthreads();
    const uint64_t mine = t < want ? h.sums[t] : 0, w = t < want ? weight_of(r, logit_of(mine)) : 0;
    uint64_t before;
    uint64_t sum = block_scan<NT>(w, before, h.room[2]);
    if (r.p < 1.0f) {
        uint64_t need = part_of(sum, fmaxf(r.p, 0.0f), true);
        need = need ? need : 1;
        if (before < need && before + w >= need) h.best[1] = before + w;
        __syncthreads();
        sum = h.best[1];
    }
    uint64_t target = part_of(sum, r.u, false) + 1;
    target = target < sum ? target : sum;
    if (before < target && before + w >= target) {
        s.next[row] = int32_t(mine & 0xffffff);
        if (s.prob) s.prob[row] = float(double(w) / double(sum));
    }
}

// A token's place in its bin, 0 .. kBins - 1 in the order.
__device__ inline int part_of_bin(const Row &r, float l, uint32_t bin)
{
    const float x = l == r.top ? 0.0f : __builtin_fmaf(r.top - l, r.bins, -float(bin));
    return int(fminf(fmaxf(x * float(kBins), 0.0f), float(kBins - 1)));
}

// The token of a bin of `src` at which the tokens (COUNT) or the weights reach `target`;
// `skip` of them, and weights `skipw`, lie before the bin.  The bin's tokens are
// listed, a thread each, and, where they are more than a few, sorted into finer
// ones (gone through once more for that, if they are more than a list holds).  false:
// too many all the same.
template <int NT, bool COUNT, typename Src>
__device__ inline bool cut_in(uint64_t target, uint32_t bin, uint64_t skip, uint64_t skipw, const Row &r,
                              Shared &h, const Src &src, Cut &cut)
{
    const int t = threadIdx.x;
    constexpr int B = kBins / NT;
    // (the two lists' lengths are cleared here, both: between the barrier that ends the first
    // list and a wave's reading of its length nothing may write that)
    if (t == 0) h.listed = h.finer = 0;
    __syncthreads();
    src.each(r, bin, bin, [&](float, uint64_t o) { enlist(h, o, h.listed); });
#pragma unroll
    for (int e = 0; e < B; ++e) h.weight[B * t + e] = 0, h.count[B * t + e] = 0;
    __syncthreads();
    int many = int(h.listed);
    const bool all = many <= kList;  // are listed
    uint64_t mine = 0, w = 0;
    bool in = all && t < many;
    if (in) {
        mine = h.list[t];
        w = weight_of(r, logit_of(mine));
    }
    if (many > kFew) {
        auto lay = [&](int b, uint64_t v) {
            atomicAdd(reinterpret_cast<unsigned long long *>(&h.weight[b]), v);
            if constexpr (COUNT) atomicAdd(&h.count[b], 1u);
        };
        const int part = in ? part_of_bin(r, logit_of(mine), bin) : -1;
        if (in) lay(part, w);
        if (!all) src.each(r, bin, bin, [&](float l, uint64_t) { lay(part_of_bin(r, l, bin), weight_of(r, l)); });
        __syncthreads();
        Bins<NT, uint64_t> bw;
        bw.read(h.weight, h.room[1]);
        if constexpr (COUNT) {
            Bins<NT, uint32_t> bc;
            bc.read(h.count, h.room[2]);
            bc.with(target - skip, [&](uint32_t b, uint64_t was, uint64_t) {
                h.bin = b;
                h.best[0] = skip + was;
            });
            __syncthreads();
            bw.at(h.bin, [&](uint64_t was, uint64_t) { h.best[1] = skipw + was; });
        } else {
            bw.with(target - skip, [&](uint32_t b, uint64_t was, uint64_t) {
                h.bin = b;
                h.best[0] = h.best[1] = skip + was;
            });
        }
        __syncthreads();
        skip = h.best[0], skipw = h.best[1];
        const int fine = int(h.bin);
        if (in && part == fine) enlist(h, mine, h.finer);
        if (!all)
            src.each(r, bin, bin, [&](float l, uint64_t o) {
                if (part_of_bin(r, l, bin) == fine) enlist(h, o, h.finer);
            });
        __syncthreads();
        many = int(h.finer);
        in = t < many;
        if (in && many <= kList) {
            mine = h.list[t];
            w = weight_of(r, logit_of(mine));
        }
    }
    if (many > kList) return false;
    if (in) h.sums[t] = w;
    uint64_t upto = 0;
    uint32_t rank = 0;
    listed_all(h, many, [&](uint64_t o, int j) {
        const bool is = o <= mine;
        upto += is ? h.sums[j] : 0;
        rank += is;
    });
    if (in) {
        const uint64_t now = skip + (COUNT ? rank : upto);
        if (now >= target && now - (COUNT ? 1 : w) < target) {
            h.best[0] = mine;
            h.best[1] = skipw + upto;
            h.best[2] = w;
        }
    }
    __syncthreads();
    cut = Cut{h.best[0], h.best[1], h.best[2]};
    __syncthreads();
    return true;
}

// Draws from all tokens by their bins' weights in h.weight (and, with a top-k, their
// number in h.count); false: too many in a bin.
template <int NT, typename Src>
__device__ inline bool draw_binned(const Sample &s, size_t row, const Row &r, Shared &h, const Src &src)
{
    Bins<NT, uint64_t> w;
    w.read(h.weight, h.room[1]);
    uint64_t sum = w.all;
    Cut cut{};
    auto find = [&](uint64_t target) {
        w.with(target, [&](uint32_t b, uint64_t was, uint64_t) {
            h.bin = b;
            h.best[0] = was;
        });
        __syncthreads();
        const uint32_t bin = h.bin;
        const uint64_t skip = h.best[0];
        return cut_in<NT, false>(target, bin, skip, skip, r, h, src, cut);
    };
    if (r.k > 0) {
        Bins<NT, uint32_t> c;
        c.read(h.count, h.room[2]);
        if (uint64_t(r.k) < c.all) {
            c.with(uint64_t(r.k), [&](uint32_t b, uint64_t was, uint64_t) {
                h.bin = b;
                h.best[0] = was;
            });
            __syncthreads();
            const uint32_t bin = h.bin;
            const uint64_t skip = h.best[0];
            w.at(bin, [&](uint64_t was, uint64_t) { h.best[1] = was; });
            __syncthreads();
            const uint64_t skipw = h.best[1];
            if (!cut_in<NT, true>(uint64_t(r.k), bin, skip, skipw, r, h, src, cut)) return false;
            sum = cut.upto;
        }
    }
    if (r.p < 1.0f) {
        const uint64_t need = part_of(sum, fmaxf(r.p, 0.0f), true);
        if (!find(need ? need : 1)) return false;
        sum = cut.upto;
    }
    const uint64_t target = part_of(sum, r.u, false) + 1;
    if (!find(target < sum ? target : sum)) return false;
    done(s, row, int(cut.place & 0xffffff), double(cut.weight) / double(sum));
    return true;
}

constexpr int kThreads = 512;  // of a row's block, or a slice's

// Rows of one slice: a block a row.  SEARCH: what is unusual is searched here, at the
// price of registers; else the row is marked for a launch after this one.  Rows of 8192,
// top-p 0.9, with and without (us, a launch more of half a microsecond not counted): 320
// 12.8, 13.5; 512 14.6, 14.9; 1024 23.8, 22.4; 3000 59, 51.  (Of 1024 threads, with: 1 row
// 8.1 against 7.8, 320 17.2, 1024 34.)
template <bool SEARCH>
__global__ __launch_bounds__(kThreads) void sample_kernel(Sample s, size_t first)
{
    constexpr int NT = kThreads;
    __shared__ Shared h;
    const size_t row = first + blockIdx.x;
    const int t = threadIdx.x;
    Held<NT> v;
    v.load(s.x + row * s.x_stride, 0, s.n);
    Row r = rules_of(s, row);
    for (int b = t; b < kBins; b += NT) h.weight[b] = 0, h.count[b] = 0;
    if (t == 0) h.listed = 0;
    float top, low;
    v.range(top, low);
    meet<NT>(top, low, h.room[0]);
    if (top == -INFINITY) return done(s, row, -1, 0.0);
    range_of(r, top, low);
    if (r.greedy) return done(s, row, v.first(top, h.room[1]), 1.0);
    if (top < INFINITY) {
        if (r.k > 0 && r.k <= kShort) {
            int want = r.k;
            const int many = list_first<NT>(r, want, h, v);
            if (many >= 0) return draw_listed<NT>(s, row, r, want, many, h);
        } else {
            r.scale = kMostScale;
            if (r.k > 0)
                v.template lay<true, true>(r, h);
            else
                v.template lay<true, false>(r, h);
            __syncthreads();
            if (draw_binned<NT>(s, row, r, h, v)) return;
        }
    }
    if constexpr (SEARCH) {
        __syncthreads();
        search<NT>(s, row, r, h);
    } else if (t == 0) {
        s.next[row] = kMarked;
    }
}

// The rows marked.
__global__ __launch_bounds__(kThreads) void search_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x;
    if (s.next[row] != kMarked) return;
    const float *x = s.x + row * s.x_stride;
    Row r = rules_of(s, row);
    float top = -INFINITY, low = INFINITY;
    for (int i = threadIdx.x; i < s.n; i += kThreads) {
        const float l = x[i];
        top = l > top ? l : top;
        low = l > -INFINITY ? fminf(low, l) : low;
    }
    meet<kThreads>(top, low, h.room[0]);
    range_of(r, top, low);
    search<kThreads>(s, row, r, h);
}

// ---- rows of several slices -------------------------------------------------------

constexpr int kDraw = 1024;    // of a row's

enum Way { kSearch, kListed, kBinned };
__device__ inline Way way_of(const Row &r)
{
    return r.top == INFINITY ? kSearch : r.k > 0 && r.k <= kShort ? kListed : kBinned;
}

// A row's largest and lowest logit from its parts (a barrier).
template <int NT>
__device__ inline void join_parts(const Sample &s, size_t row, Row &r, uint64_t *room)
{
    const Part *part = s.part + row * s.slices;
    float top = -INFINITY, low = INFINITY;
    for (int i = threadIdx.x; i < s.slices; i += NT) {
        top = fmaxf(top, part[i].top);
        low = fminf(low, part[i].low);
    }
    meet<NT>(top, low, room);
    range_of(r, top, low);
}

// And the unit, by the bound on its weights (a barrier).  Only the bins' launch works it
// out, and leaves it for the draw: in another order of the sum it may be another.
__device__ inline void join_scale(const Sample &s, size_t row, Row &r, uint64_t *room)
{
    const Part *part = s.part + row * s.slices;
    float b = 0.0f;
    for (int i = threadIdx.x; i < s.slices; i += kThreads)
        if (part[i].top > -INFINITY) b += part[i].sum * bound_of(r, part[i].top);
    r.scale = scale_of(sum_over<kThreads>(b, room));
}

// A slice's part and its own short top-k.
__global__ __launch_bounds__(kThreads) void slice_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x / unsigned(s.slices);
    const int slice = int(blockIdx.x % unsigned(s.slices)), t = threadIdx.x;
    Held<kThreads> v;
    v.load(s.x + row * s.x_stride, slice * kSlice, s.n);
    Row r = rules_of(s, row);
    for (int b = t; b < kBins; b += kThreads) {
        h.count[b] = 0;
        if (slice == 0) s.bins[row * kBins + b] = 0, s.count[row * kBins + b] = 0;
    }
    if (t == 0) h.listed = 0;
    float top, low;
    v.range(top, low);
    meet<kThreads>(top, low, h.room[0]);
    range_of(r, top, low);
    Part p{top, low, 0.0f, 0};
    if (top > -INFINITY) {
        if (r.greedy) {
            p.listed = v.first(top, h.room[1]);
        } else if (way_of(r) == kListed) {
            int want = r.k;
            p.listed = list_first<kThreads>(r, want, h, v);
            if (t < p.listed) s.list[(row * s.slices + slice) * kList + t] = h.list[t];
        } else if (way_of(r) == kBinned) {
            float b = 0.0f;
#pragma unroll
            for (int j = 0; j < v.kPer; ++j) b += bound_of(r, v.v[j]);
            p.sum = sum_over<kThreads>(b, h.room[1]);
        }
    }
    if (t == 0) s.part[row * s.slices + slice] = p;
}

// Of rows without a short top-k: the weights, and with a long one the tokens' number, in
// their rows' bins.
__global__ __launch_bounds__(kThreads) void bins_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x / unsigned(s.blocks);
    const int block = int(blockIdx.x % unsigned(s.blocks)), t = threadIdx.x;
    Row r = rules_of(s, row);
    if (r.greedy || (r.k > 0 && r.k <= kShort)) return;
    Held<kThreads> v;
    v.load(s.x + row * s.x_stride, block * kSlice, s.n);
    for (int b = t; b < kBins; b += kThreads) {
        h.weight[b] = 0;
        if (r.k > 0) h.count[b] = 0;
    }
    join_parts<kThreads>(s, row, r, h.room[0]);
    if (r.top == -INFINITY || way_of(r) != kBinned) return;
    join_scale(s, row, r, h.room[1]);
    if (block == 0 && t == 0) s.scale[row] = r.scale;
    for (int slice = block;;) {
        v.clean();
        if (r.k > 0)
            v.template lay<true, true>(r, h);
        else
            v.template lay<true, false>(r, h);
        slice += s.blocks;
        if (slice >= s.slices) break;
        v.load(s.x + row * s.x_stride, slice * kSlice, s.n);
    }
    __syncthreads();
    for (int b = t; b < kBins; b += kThreads) {
        if (const uint64_t w = h.weight[b])
            atomicAdd(reinterpret_cast<unsigned long long *>(&s.bins[row * kBins + b]), w);
        if (r.k > 0)
            if (const uint32_t c = h.count[b]) atomicAdd(&s.count[row * kBins + b], c);
    }
}

// Which bins of a row matter: that of the k-th token (`cut`), those where the weights may
// come to top_p, whatever token the first k end at, and those where the draw may be.
struct Range {
    uint32_t from, to;
    __device__ inline bool has(uint32_t bin) const { return bin - from <= to - from; }
};

struct Matter {
    uint32_t cut;
    Range nucleus, draw;
    __device__ inline bool has(uint32_t bin) const { return bin == cut || nucleus.has(bin) || draw.has(bin); }
};

__device__ inline uint32_t scalar(uint32_t x) { return uint32_t(__builtin_amdgcn_readfirstlane(int(x))); }

template <int NT>
__device__ inline Matter matter_of(const Sample &s, size_t row, const Row &r, Shared &h)
{
    Bins<NT, uint64_t> w;
    w.read(s.bins + row * kBins, h.room[2]);
    Matter m{kNoBin, Range{kNoBin, kNoBin}, Range{}};
    uint64_t least = w.all, most = w.all;  // that stay
    if (r.k > 0) {
        Bins<NT, uint32_t> c;
        c.read(s.count + row * kBins, h.room[1]);
        if (uint64_t(r.k) < c.all) {
            c.with(uint64_t(r.k), [&](uint32_t b, uint64_t, uint64_t) { h.bin = b; });
            __syncthreads();
            m.cut = scalar(h.bin);
            w.at(m.cut, [&](uint64_t was, uint64_t v) {
                h.best[0] = was;
                h.best[1] = was + v;
            });
            __syncthreads();
            // (its last token may weigh less than half a unit)
            least = h.best[0] ? h.best[0] : 1;
            most = h.best[1];
        }
    }
    // the bins of the tokens at which the weights reach a .. z, and what those come to
    auto reach = [&](uint64_t a, uint64_t z) {
        w.with(a, [&](uint32_t b, uint64_t, uint64_t) { h.sums[0] = b; });
        w.with(z, [&](uint32_t b, uint64_t was, uint64_t v) {
            h.sums[1] = b;
            h.sums[2] = was + v;
        });
        __syncthreads();
        return Range{scalar(uint32_t(h.sums[0])), scalar(uint32_t(h.sums[1]))};
    };
    if (r.p < 1.0f) {
        const uint64_t a = part_of(least, fmaxf(r.p, 0.0f), true), z = part_of(most, fmaxf(r.p, 0.0f), true);
        least = a ? a : 1;
        m.nucleus = reach(least, z ? z : 1);
        most = h.sums[2] < most ? h.sums[2] : most;
        __syncthreads();
    }
    const uint64_t a = part_of(least, r.u, false) + 1, z = part_of(most, r.u, false) + 1;
    m.draw = reach(a < least ? a : least, z < most ? z : most);
    return m;
}

// The tokens of those bins, slice by slice.
__global__ __launch_bounds__(kThreads) void gather_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x / unsigned(s.blocks);
    const int block = int(blockIdx.x % unsigned(s.blocks)), t = threadIdx.x;
    Row r = rules_of(s, row);
    if (r.greedy || (r.k > 0 && r.k <= kShort)) return;
    Held<kThreads> v;
    v.load(s.x + row * s.x_stride, block * kSlice, s.n);
    join_parts<kThreads>(s, row, r, h.room[0]);
    if (r.top == -INFINITY || way_of(r) != kBinned) return;
    const Matter m = matter_of<kThreads>(s, row, r, h);
    for (int slice = block;;) {
        if (t == 0) h.listed = 0;
        __syncthreads();
        v.clean();
#pragma unroll
        for (int j = 0; j < v.kPer; ++j) {
            const uint32_t bin = bin_below(r, v.v[j]);
            if (m.has(bin) && token(r, v.v[j])) enlist(h, order_of(v.v[j], v.at(j)), h.listed);
        }
        __syncthreads();
        const int many = int(h.listed);
        if (t < many && many <= kList) s.list[(row * s.slices + slice) * kList + t] = h.list[t];
        if (t == 0) s.part[row * s.slices + slice].listed = many <= kList ? many : -1;
        slice += s.blocks;
        if (slice >= s.slices) break;
        v.load(s.x + row * s.x_stride, slice * kSlice, s.n);
        __syncthreads();
    }
}

__global__ __launch_bounds__(kDraw) void draw_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x;
    const int t = threadIdx.x;
    const Lists<kDraw> lists(s, row);
    Row r = rules_of(s, row);
    h.count[t] = 0;
    if (t == 0) h.listed = 0;
    join_parts<kDraw>(s, row, r, h.room[0]);
    if (r.top == -INFINITY) return done(s, row, -1, 0.0);
    const Part *part = s.part + row * s.slices;
    if (r.greedy) {
        if (t == 0) {
            int i = 0;
            while (part[i].top != r.top) ++i;
            done(s, row, part[i].listed, 1.0);
        }
        return;
    }
    int few = 1;
    for (int i = t; i < s.slices; i += kDraw) few &= part[i].listed >= 0;
    if (__syncthreads_and(few)) {
        if (way_of(r) == kListed) {
            int want = r.k;
            const int many = list_first<kDraw>(r, want, h, lists);
            if (many >= 0) return draw_listed<kDraw>(s, row, r, want, many, h);
        } else if (way_of(r) == kBinned) {
            r.scale = s.scale[row];
            h.weight[t] = s.bins[row * kBins + t];
            h.count[t] = s.count[row * kBins + t];
            __syncthreads();
            if (draw_binned<kDraw>(s, row, r, h, lists)) return;
        }
    }
    __syncthreads();
    search<kDraw>(s, row, r, h);
}

size_t slices_of(size_t n) { return (n + kSlice - 1) / kSlice; }

size_t row_bytes(size_t slices) { return slices > 1 ? kBins * 12 + slices * (kList * 8 + sizeof(Part)) + 4 : 0; }

}  // namespace

extern "C" {

size_t nd_sample_rows_work(nd_ctx *, size_t count, size_t n) { return count * row_bytes(slices_of(n)); }

int nd_sample_rows(nd_ctx *ctx, const float *x, size_t x_stride, size_t count, size_t n,
                   const nd_sampling *sampling, const float *u, int32_t *next, float *prob,
                   void *work, size_t work_bytes)
{
    ND_ENTER(ctx);
    ND_REQUIRE(n > 0 && n <= (size_t(1) << 24), "n %zu must be in 1..2^24", n);
    ND_REQUIRE(count <= 0x7fffffff, "count %zu above 2^31 - 1", count);
    if (count == 0) return ND_OK;
    ND_REQUIRE(x && u && next, "null buffer");
    ND_REQUIRE(count == 1 || x_stride >= n, "row stride %zu below n %zu", x_stride, n);
    const nd_sampling none{}, &r = sampling ? *sampling : none;
    const size_t slices = slices_of(n);
    Sample s{x, r.temperature, r.min_p, r.top_p, u, r.top_k, x_stride, int(n), next, prob, int(slices), 0, nullptr, nullptr, nullptr, nullptr, nullptr};
    // (a row's blocks, of about four a CU; each finds out what matters for itself)
    s.blocks = int(std::min(slices, std::max<size_t>(1, 1024 / count)));
    if (slices > 1) {
        void *ws = nullptr;
        if (int rc = nd::call_workspace(ctx, count * row_bytes(slices), work, work_bytes, &ws)) return rc;
        s.bins = static_cast<uint64_t *>(ws);
        s.list = s.bins + count * kBins;
        s.count = reinterpret_cast<uint32_t *>(s.list + count * slices * kList);
        s.part = reinterpret_cast<Part *>(s.count + count * kBins);
        s.scale = reinterpret_cast<int *>(s.part + count * slices);
    }
    // HIP counts a launch's threads in 32 bits: rows beyond that go in further launches
    const size_t most = 0xffffffff / kDraw / slices;
    // two blocks a CU are what its registers hold
    const bool few = count <= 2 * size_t(ctx->num_cus > 0 ? ctx->num_cus : 256);
    for (size_t first = 0; first < count; first += most) {
        const unsigned rows = unsigned(std::min(most, count - first)), blocks = rows * unsigned(slices);
        if (slices == 1) {
            if (few) {
                hipLaunchKernelGGL(sample_kernel<true>, dim3(rows), dim3(kThreads), 0, ctx->stream, s, first);
                if (int rc = nd::check_launch("sample_rows")) return rc;
            } else {
                hipLaunchKernelGGL(sample_kernel<false>, dim3(rows), dim3(kThreads), 0, ctx->stream, s, first);
                if (int rc = nd::check_launch("sample_rows")) return rc;
                hipLaunchKernelGGL(search_kernel, dim3(rows), dim3(kThreads), 0, ctx->stream, s, first);
                if (int rc = nd::check_launch("sample_search")) return rc;
            }
            continue;
        }
        hipLaunchKernelGGL(slice_kernel, dim3(blocks), dim3(kThreads), 0, ctx->stream, s, first);
        if (int rc = nd::check_launch("sample_slices")) return rc;
        // (only rows without a short top-k have anything to do here, which the host does not see)
        hipLaunchKernelGGL(bins_kernel, dim3(rows * unsigned(s.blocks)), dim3(kThreads), 0, ctx->stream, s, first);
        if (int rc = nd::check_launch("sample_bins")) return rc;
        hipLaunchKernelGGL(gather_kernel, dim3(rows * unsigned(s.blocks)), dim3(kThreads), 0, ctx->stream, s, first);
        if (int rc = nd::check_launch("sample_gather")) return rc;
        hipLaunchKernelGGL(draw_kernel, dim3(rows), dim3(kDraw), 0, ctx->stream, s, first);
        if (int rc = nd::check_launch("sample_draw")) return rc;
    }
    return ND_OK;
}

}  // extern "C"
