// A token drawn from each row of logits under a temperature, min-p, top-k and
// top-p, by a random number that is given.
//
// All rules cut the row's order (logits descending, equal ones by their number)
// behind some token, and the draw is a token of that order too: the first whose
// weights, added up, reach a target.  So no row is sorted:
//   a short top-k: the row's tokens are counted in bins that follow the order, those
//     up to the bin of the k-th are listed, and the list is put in order;
//   else: weights are added up in the bins, the bin of a target is found, and its
//     tokens alone are listed;
//   anything unusual (more tokens in a bin than a list holds, infinite logits): the
//     row is searched in finer and finer bins, by the digits of the order.
// Weights are whole numbers, exp((l - M) / T) in units of 2^-s, worked out in fp64: a
// pick next to a border is the border's and not the rounding's, and sums of whole
// numbers are the same in any order.  s is 49, or less where a bound on a long row's
// sum asks for it: the sum stays below 2^62 and has 2^49 units at least.
//
// A block a row of up to kSlice logits, which stay in its registers.  Longer rows: a
// block a slice looks for its largest logit and lists its own short top-k; where
// there is none, the slices' bins are added up in a second launch, and the tokens of
// the bins that matter listed in a third; a block a row ends.
#include "nd_internal.h"
#include "nd_lanes.h"

#include <algorithm>

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kPer = 8, kSlice = kPer * kThreads;
constexpr int kBins = kThreads;  // one a thread
constexpr int kList = 512;       // tokens that are put in order, a thread each
constexpr int kShort = 448;      // the longest top-k that is listed
constexpr int kMostScale = 49;
constexpr uint32_t kNoBin = 0xffff;

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
    Part *part;       // [rows][slices]
    uint64_t *bins;   // [rows][kBins]
    uint64_t *list;   // [rows][slices][kList]
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
    if (mp > 0.0f) r.low = fmax(r.low, double(r.T) * log(double(mp)));
    if (r.greedy || mp >= 1.0f) r.low = 0.0;
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

// 2^z in units of 2^-scale (scale <= 50), to the nearest, for a z <= 0.  2^f, |f| <=
// 1/2, by the polynomial of degree 11 through its values at Chebyshev's nodes (2e-17
// of it off).  What 2^52 is added to keeps its whole part in the low 52 bits.
__device__ inline uint64_t units_of(double z, int scale)
{
    const double n = __builtin_rint(z), f = z - n;
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
    const double q = __builtin_ldexp(p, int(n) + scale) + 0x1p52;
    return uint64_t(__double_as_longlong(q)) & 0xfffffffffffffull;
}

// The weight of a logit in units; 0: no token.
__device__ inline uint64_t weight_of(const Row &r, float l)
{
    const double d = behind(r, l);
    return d >= r.low ? units_of(d * r.by, r.scale) : 0;
}

// A little more than the weight (and 1 for some that are no tokens).
__device__ inline float bound_of(const Row &r, float l)
{
    // (the argument is off by 2^-22 of its size, of 64 at most where it counts; a factor
    // of 0 would make no number of -inf)
    const float d = l == r.top ? 0.0f : l - r.top;
    return l > -INFINITY ? __builtin_amdgcn_exp2f(d * fmaxf(float(r.by), 0x1p-149f)) * 1.0001f : 0.0f;
}

// The scale for weights that come to `sum` or less: below 2^62 units.
__device__ inline int scale_of(float sum) { return min(62 - __builtin_amdgcn_frexp_expf(sum * 1.001f), kMostScale); }

__device__ inline int bin_of(const Row &r, float l)
{
    return l == r.top ? 0 : int(fminf((r.top - l) * r.bins, float(kBins - 1)));
}

struct Shared {
    uint64_t weight[kBins], list[kList], sums[kList];
    uint64_t room[kWaves], range[kWaves], best[3];
    uint32_t count[kBins], listed, bin, in[3];
};

// Where a target lies: the token, the weights up to it and its own.
struct Cut {
    uint64_t place, upto, weight;
};

// The whole numbers of the threads before this one added up, and of all.
__device__ inline uint64_t block_scan(uint64_t v, uint64_t &before, uint64_t *room)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t up = ndl::wave_scan(v);
    if (lane == 63) room[w] = up;
    __syncthreads();
    uint64_t all = 0, mine = up - v;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const uint64_t x = room[i];
        mine += i < w ? x : 0;
        all += x;
    }
    __syncthreads();
    before = mine;
    return all;
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

// ---- a row by finer and finer bins --------------------------------------------

// Any row, whatever its logits and rules, from memory: a block.
__device__ __forceinline__ void search(const Sample &s, size_t row, Row r, Shared &h)
{
    const int t = threadIdx.x, lane = t & 63;
    const float *x = s.x + row * s.x_stride;
    auto clear = [&]() {
        __syncthreads();
        h.count[t] = 0, h.weight[t] = 0;
        __syncthreads();
    };
    auto add = [&](int b, uint64_t w) {
        atomicAdd(&h.count[b], 1u);
        atomicAdd(reinterpret_cast<unsigned long long *>(&h.weight[b]), w);
    };
    uint64_t tokens = 0, all = 0;
    auto scan = [&]() {  // to sums up to each bin
        __syncthreads();
        uint64_t c = h.count[t], w = h.weight[t], before;
        tokens = block_scan(c, before, h.room);
        h.count[t] = uint32_t(before + c);
        all = block_scan(w, before, h.room);
        h.weight[t] = before + w;
        __syncthreads();
    };
    auto each = [&](auto f) {
#pragma unroll 1
        for (int i = t; i < s.n; i += kThreads) {
            const float l = x[i];
            const uint64_t w = weight_of(r, l);
            if (w) f(l, i, w);
        }
    };
    // the unit
    float bound = 0.0f;
#pragma unroll 1
    for (int i = t; i < s.n; i += kThreads) bound += bound_of(r, x[i]);
    bound = ndl::wave_sum64(bound);
    __syncthreads();
    if (lane == 0) h.room[t >> 6] = __float_as_uint(bound);
    __syncthreads();
    bound = 0.0f;
    for (int i = 0; i < kWaves; ++i) bound += __uint_as_float(uint32_t(h.room[i]));
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
            {
                const uint64_t now = before + (by_count ? h.count[t] : h.weight[t]);
                const uint64_t was = before + (t == 0 ? 0 : by_count ? h.count[t - 1] : h.weight[t - 1]);
                if (was < target && now >= target) h.bin = uint32_t(t);
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

// top and low over the block; every thread gets both (a barrier).
__device__ inline void meet(float &top, float &low, Shared &h)
{
    top = ndl::wave_max64(top);
    low = -ndl::wave_max64(-low);
    if ((threadIdx.x & 63) == 0) h.range[threadIdx.x >> 6] = uint64_t(__float_as_uint(low)) << 32 | __float_as_uint(top);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const uint64_t x = h.range[i];
        top = fmaxf(top, __uint_as_float(uint32_t(x)));
        low = fminf(low, __uint_as_float(uint32_t(x >> 32)));
    }
}

__device__ inline float sum_over(float v, uint64_t *room)
{
    v = ndl::wave_sum64(v);
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = __float_as_uint(v);
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) v += __uint_as_float(uint32_t(room[i]));
    __syncthreads();
    return v;
}

// A slice's logits in registers (what is no token, NaN too, is -inf), and their bins,
// two a word.
struct Held {
    float v[kPer];
    uint32_t b[kPer / 2];
    int t0;
    __device__ inline int at(int j) const { return t0 + (j >> 2) * 4 * kThreads + 4 * int(threadIdx.x) + (j & 3); }
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
    // the largest and the lowest token's
    __device__ inline void range(float &top, float &low)
    {
        top = -INFINITY, low = INFINITY;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            v[j] = v[j] > -INFINITY ? v[j] : -INFINITY;
            top = fmaxf(top, v[j]);
            low = fminf(low, v[j] > -INFINITY ? v[j] : INFINITY);
        }
    }
    // the tokens' bins, and, in h.weight, their number or weights
    template <bool WEIGHTS>
    __device__ inline void lay(const Row &r, Shared &h)
    {
        const double top = double(r.top);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const double d = double(v[j]) - top;  // (a finite top)
            uint32_t bin = kNoBin;
            if (d >= r.low) {
                bin = uint32_t(bin_of(r, v[j]));
                if constexpr (WEIGHTS)
                    atomicAdd(reinterpret_cast<unsigned long long *>(&h.weight[bin]), units_of(d * r.by, r.scale));
                else
                    atomicAdd(reinterpret_cast<uint32_t *>(&h.weight[bin]), 1u);
            }
            b[j / 2] = j & 1 ? b[j / 2] | bin << 16 : bin;
        }
    }
    template <typename F>
    __device__ inline void each(F f) const
    {
#pragma unroll
        for (int j = 0; j < kPer; ++j) f(v[j], at(j), j & 1 ? b[j / 2] >> 16 : b[j / 2] & 0xffff);
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
        for (int k = 0; k < kWaves; ++k) i = min(i, int(room[k]));
        return i;
    }
};

// What the slices have listed, a wave a slice.
struct Lists {
    const uint64_t *list;
    const Part *part;
    int slices;
    template <typename F>
    __device__ inline void all(F f) const
    {
        for (int i = int(threadIdx.x >> 6); i < slices; i += kWaves)
            for (int j = int(threadIdx.x & 63); j < part[i].listed; j += 64) f(list[size_t(i) * kList + j]);
    }
    // (their bins are worked out twice)
    template <bool WEIGHTS>
    __device__ inline void lay(const Row &r, Shared &h) const
    {
        all([&](uint64_t o) {
            const float l = logit_of(o);
            if (token(r, l)) atomicAdd(reinterpret_cast<uint32_t *>(&h.weight[bin_of(r, l)]), 1u);
        });
    }
};

// The tokens of bins from .. to of `src`, added to the list; what is beyond its room is
// counted alone.
__device__ inline void collect(const Held &src, const Row &, uint32_t from, uint32_t to, Shared &h)
{
    src.each([&](float l, int i, uint32_t bin) {
        if (bin - from <= to - from) {
            const uint32_t at = atomicAdd(&h.listed, 1u);
            if (at < uint32_t(kList)) h.list[at] = order_of(l, i);
        }
    });
}

__device__ inline void collect(const Lists &src, const Row &r, uint32_t from, uint32_t to, Shared &h)
{
    src.all([&](uint64_t o) {
        const float l = logit_of(o);
        if (token(r, l) && uint32_t(bin_of(r, l)) - from <= to - from) {
            const uint32_t at = atomicAdd(&h.listed, 1u);
            if (at < uint32_t(kList)) h.list[at] = o;
        }
    });
}

// Lists the tokens up to the bin of the `want`-th and says how many, -1: more than a
// list holds; `want` becomes the tokens' number, if that is less.  h.weight and
// h.listed are 0.
template <typename Src>
__device__ inline int list_first(const Row &r, int &want, Shared &h, Src &src)
{
    const int t = threadIdx.x;
    src.template lay<false>(r, h);
    __syncthreads();
    const uint64_t mine = uint32_t(h.weight[t]);
    uint64_t before;
    const int all = int(block_scan(mine, before, h.room));
    want = min(want, all);
    if (int(before) < want && int(before + mine) >= want) {
        h.bin = uint32_t(t);
        h.best[0] = before + mine;
    }
    __syncthreads();
    const int last = int(h.bin), many = int(h.best[0]);
    if (many > kList) return -1;
    collect(src, r, 0, uint32_t(last), h);
    __syncthreads();
    return many;
}

// Draws from the first `want` of the `many` tokens listed.
__device__ inline void draw_listed(const Sample &s, size_t row, Row r, int want, int many, Shared &h)
{
    const int t = threadIdx.x;
    r.scale = kMostScale;
    if (t < many) {
        const uint64_t mine = h.list[t];
        int rank = 0;
        for (int j = 0; j < many; ++j) rank += h.list[j] < mine;
        h.sums[rank] = mine;
    }
    __syncthreads();
    const uint64_t mine = t < want ? h.sums[t] : 0, w = t < want ? weight_of(r, logit_of(mine)) : 0;
    uint64_t before;
    uint64_t sum = block_scan(w, before, h.room);
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

// The bin in which the weights up to it reach `target` and those before it, from the
// weight of each thread's bin (a barrier).
__device__ inline uint32_t bin_with(uint64_t target, uint64_t before, uint64_t mine, uint64_t &skip, Shared &h, int place)
{
    if (before < target && before + mine >= target) {
        h.best[place] = before;
        h.in[place] = threadIdx.x;
    }
    __syncthreads();
    skip = h.best[place];
    return h.in[place];
}

// Of the tokens listed (`many`, of bins one after another, `skip` being the weights of
// the bins before them) the one at which the weights reach `target` (barriers).
__device__ inline Cut cut_at(uint64_t target, uint64_t skip, int many, const Row &r, Shared &h)
{
    const int t = threadIdx.x;
    uint64_t mine = 0, w = 0;
    if (t < many) {
        mine = h.list[t];
        w = weight_of(r, logit_of(mine));
        h.sums[t] = w;
    }
    __syncthreads();
    if (t < many) {
        uint64_t upto = skip;
        for (int j = 0; j < many; ++j) upto += h.list[j] <= mine ? h.sums[j] : 0;
        if (upto >= target && upto - w < target) {
            h.best[0] = mine;
            h.best[1] = upto;
            h.best[2] = w;
        }
    }
    __syncthreads();
    const Cut cut{h.best[0], h.best[1], h.best[2]};
    __syncthreads();
    return cut;
}

// Draws from all tokens by their bins' weights in h.weight; false: a bin that matters
// has more tokens than a list holds.
__device__ inline bool draw_binned(const Sample &s, size_t row, const Row &r, Shared &h, const Held &src)
{
    const int t = threadIdx.x;
    const uint64_t mine = h.weight[t];
    uint64_t before, skip;
    uint64_t sum = block_scan(mine, before, h.room);
    uint32_t listed = kNoBin;
    int many = 0;
    Cut cut{};
    auto find = [&](uint64_t target) {
        const uint32_t bin = bin_with(target, before, mine, skip, h, 0);
        if (bin != listed) {
            __syncthreads();
            if (t == 0) h.listed = 0;
            __syncthreads();
            collect(src, r, bin, bin, h);
            __syncthreads();
            listed = bin;
            many = int(h.listed);
        }
        if (many > kList) return false;
        cut = cut_at(target, skip, many, r, h);
        return true;
    };
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

// Rows of one slice: a block a row.
__global__ __launch_bounds__(kThreads) void sample_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x;
    const int t = threadIdx.x;
    Held v;
    v.load(s.x + row * s.x_stride, 0, s.n);
    Row r = rules_of(s, row);
    h.weight[t] = 0;
    if (t == 0) h.listed = 0;
    float top, low;
    v.range(top, low);
    meet(top, low, h);
    if (top == -INFINITY) return done(s, row, -1, 0.0);
    range_of(r, top, low);
    if (r.greedy) return done(s, row, v.first(top, h.room), 1.0);
    if (r.k > 0 && r.k <= kShort && top < INFINITY) {
        int want = r.k;
        const int many = list_first(r, want, h, v);
        if (many >= 0) return draw_listed(s, row, r, want, many, h);
    } else if (r.k <= 0 && top < INFINITY) {
        r.scale = kMostScale;
        v.lay<true>(r, h);
        __syncthreads();
        if (draw_binned(s, row, r, h, v)) return;
    }
    search(s, row, r, h);
}

// ---- rows of several slices -------------------------------------------------------

enum Way { kSearch, kListed, kBinned };
__device__ inline Way way_of(const Row &r)
{
    return r.top == INFINITY ? kSearch : r.k <= 0 ? kBinned : r.k <= kShort ? kListed : kSearch;
}

// A row's largest and lowest logit and the bound on its weights, from its parts.
__device__ inline float join_parts(const Sample &s, size_t row, Row &r, Shared &h)
{
    const Part *part = s.part + row * s.slices;
    float top = -INFINITY, low = INFINITY;
    for (int i = threadIdx.x; i < s.slices; i += kThreads) {
        top = fmaxf(top, part[i].top);
        low = fminf(low, part[i].low);
    }
    meet(top, low, h);
    range_of(r, top, low);
    if (top == -INFINITY || top == INFINITY) return 1.0f;
    float b = 0.0f;
    for (int i = threadIdx.x; i < s.slices; i += kThreads)
        if (part[i].top > -INFINITY) b += part[i].sum * bound_of(r, part[i].top);
    return sum_over(b, h.room);
}

// A slice's part and its own short top-k.
__global__ __launch_bounds__(kThreads) void slice_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x / unsigned(s.slices);
    const int slice = int(blockIdx.x % unsigned(s.slices)), t = threadIdx.x;
    Held v;
    v.load(s.x + row * s.x_stride, slice * kSlice, s.n);
    Row r = rules_of(s, row);
    h.weight[t] = 0;
    if (t == 0) h.listed = 0;
    float top, low;
    v.range(top, low);
    meet(top, low, h);
    range_of(r, top, low);
    if (slice == 0) s.bins[row * kBins + t] = 0;
    Part p{top, low, 0.0f, 0};
    if (top > -INFINITY) {
        if (r.greedy) {
            p.listed = v.first(top, h.room);
        } else if (way_of(r) == kListed) {
            int want = r.k;
            p.listed = list_first(r, want, h, v);
            if (t < p.listed) s.list[(row * s.slices + slice) * kList + t] = h.list[t];
        } else if (way_of(r) == kBinned) {
            float b = 0.0f;
#pragma unroll
            for (int j = 0; j < kPer; ++j) b += bound_of(r, v.v[j]);
            p.sum = sum_over(b, h.room);
        }
    }
    if (t == 0) s.part[row * s.slices + slice] = p;
}

// The weights of the slices of rows without a top-k in their rows' bins.
__global__ __launch_bounds__(kThreads) void bins_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x / unsigned(s.slices);
    const int slice = int(blockIdx.x % unsigned(s.slices)), t = threadIdx.x;
    Row r = rules_of(s, row);
    if (r.greedy || r.k > 0) return;
    Held v;
    v.load(s.x + row * s.x_stride, slice * kSlice, s.n);
    h.weight[t] = 0;
    float top, low;
    v.range(top, low);
    const float bound = join_parts(s, row, r, h);
    if (r.top == -INFINITY || way_of(r) != kBinned) return;
    r.scale = scale_of(bound);
    v.lay<true>(r, h);
    __syncthreads();
    if (const uint64_t w = h.weight[t])
        atomicAdd(reinterpret_cast<unsigned long long *>(&s.bins[row * kBins + t]), w);
}

// Which bins of a row matter: the one where the weights come to top_p (`last`), and
// those where the draw may be, whatever token of `last` the run ends at (from .. to).
struct Bins {
    uint32_t from, to, last;
    uint64_t skip, skip_last, sum;  // weights before `from`, before `last`, of all
};

__device__ inline Bins bins_of(const Sample &s, size_t row, const Row &r, Shared &h)
{
    const uint64_t mine = s.bins[row * kBins + threadIdx.x];
    Bins b{};
    uint64_t before, most, least, no;
    b.sum = block_scan(mine, before, h.room);
    most = least = b.sum;
    b.last = kBins;
    if (r.p < 1.0f) {
        const uint64_t need = part_of(b.sum, fmaxf(r.p, 0.0f), true);
        b.last = bin_with(need ? need : 1, before, mine, b.skip_last, h, 0);
        if (threadIdx.x == b.last) h.sums[0] = before + mine;
        __syncthreads();
        least = b.skip_last + 1;
        most = h.sums[0];
    }
    const uint64_t a = part_of(least, r.u, false) + 1, z = part_of(most, r.u, false) + 1;
    b.from = bin_with(a < least ? a : least, before, mine, b.skip, h, 1);
    b.to = bin_with(z < most ? z : most, before, mine, no, h, 2);
    __syncthreads();
    return b;
}

// The tokens of those bins.
__global__ __launch_bounds__(kThreads) void gather_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x / unsigned(s.slices);
    const int slice = int(blockIdx.x % unsigned(s.slices)), t = threadIdx.x;
    Row r = rules_of(s, row);
    if (r.greedy || r.k > 0) return;
    Held v;
    v.load(s.x + row * s.x_stride, slice * kSlice, s.n);
    if (t == 0) h.listed = 0;
    float top, low;
    v.range(top, low);
    join_parts(s, row, r, h);
    if (r.top == -INFINITY || way_of(r) != kBinned) return;
    const Bins b = bins_of(s, row, r, h);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const uint32_t bin = token(r, v.v[j]) ? uint32_t(bin_of(r, v.v[j])) : kNoBin;
        if (bin == b.last || bin - b.from <= b.to - b.from) {
            const uint32_t at = atomicAdd(&h.listed, 1u);
            if (at < uint32_t(kList)) h.list[at] = order_of(v.v[j], v.at(j));
        }
    }
    __syncthreads();
    const int many = int(h.listed);
    if (t < many && many <= kList) s.list[(row * s.slices + slice) * kList + t] = h.list[t];
    if (t == 0) s.part[row * s.slices + slice].listed = many <= kList ? many : -1;
}

__global__ __launch_bounds__(kThreads) void draw_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x;
    const int t = threadIdx.x;
    Row r = rules_of(s, row);
    h.weight[t] = 0;
    if (t == 0) h.listed = 0;
    const float bound = join_parts(s, row, r, h);
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
    Lists lists{s.list + row * s.slices * kList, part, s.slices};
    int few = 1;
    for (int i = t; i < s.slices; i += kThreads) few &= part[i].listed >= 0;
    if (__syncthreads_and(few)) {
        if (way_of(r) == kListed) {
            int want = r.k;
            const int many = list_first(r, want, h, lists);
            if (many >= 0) return draw_listed(s, row, r, want, many, h);
        } else if (way_of(r) == kBinned) {
            r.scale = scale_of(bound);
            const Bins b = bins_of(s, row, r, h);
            // the tokens of one run of bins, then of the other
            auto find = [&](uint64_t target, uint32_t from, uint32_t to, uint64_t skip, Cut &cut) {
                if (t == 0) h.listed = 0;
                __syncthreads();
                collect(lists, r, from, to, h);
                __syncthreads();
                const int many = int(h.listed);
                if (many > kList) return false;
                cut = cut_at(target, skip, many, r, h);
                return true;
            };
            Cut cut{};
            uint64_t sum = b.sum;
            bool good = true;
            if (r.p < 1.0f) {
                const uint64_t need = part_of(sum, fmaxf(r.p, 0.0f), true);
                good = find(need ? need : 1, b.last, b.last, b.skip_last, cut);
                sum = cut.upto;
            }
            const uint64_t target = part_of(sum, r.u, false) + 1;
            if (good && find(target < sum ? target : sum, b.from, b.to, b.skip, cut))
                return done(s, row, int(cut.place & 0xffffff), double(cut.weight) / double(sum));
        }
    }
    search(s, row, r, h);
}

size_t slices_of(size_t n) { return (n + kSlice - 1) / kSlice; }

size_t row_bytes(size_t slices) { return slices > 1 ? kBins * 8 + slices * (kList * 8 + sizeof(Part)) : 0; }

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
    Sample s{x, r.temperature, r.min_p, r.top_p, u, r.top_k, x_stride, int(n), next, prob, int(slices)};
    if (slices > 1) {
        void *ws = nullptr;
        if (int rc = nd::call_workspace(ctx, count * row_bytes(slices), work, work_bytes, &ws)) return rc;
        s.bins = static_cast<uint64_t *>(ws);
        s.list = s.bins + count * kBins;
        s.part = reinterpret_cast<Part *>(s.list + count * slices * kList);
    }
    // HIP counts a launch's threads in 32 bits: rows beyond that go in further launches
    const size_t most = 0xffffffff / kThreads / slices;
    for (size_t first = 0; first < count; first += most) {
        const unsigned rows = unsigned(std::min(most, count - first)), blocks = rows * unsigned(slices);
        if (slices == 1) {
            hipLaunchKernelGGL(sample_kernel, dim3(rows), dim3(kThreads), 0, ctx->stream, s, first);
            if (int rc = nd::check_launch("sample_rows")) return rc;
            continue;
        }
        hipLaunchKernelGGL(slice_kernel, dim3(blocks), dim3(kThreads), 0, ctx->stream, s, first);
        if (int rc = nd::check_launch("sample_slices")) return rc;
        // (only rows without a top-k have anything to do here, which the host does not see)
        hipLaunchKernelGGL(bins_kernel, dim3(blocks), dim3(kThreads), 0, ctx->stream, s, first);
        if (int rc = nd::check_launch("sample_bins")) return rc;
        hipLaunchKernelGGL(gather_kernel, dim3(blocks), dim3(kThreads), 0, ctx->stream, s, first);
        if (int rc = nd::check_launch("sample_gather")) return rc;
        hipLaunchKernelGGL(draw_kernel, dim3(rows), dim3(kThreads), 0, ctx->stream, s, first);
        if (int rc = nd::check_launch("sample_draw")) return rc;
    }
    return ND_OK;
}

}  // extern "C"
