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
// numbers are the same in any order.  s is 53 for a list, and else chosen by a bound
// on the row's sum, so that the sum has 2^60 .. 2^62 units whatever the row's shape.
//
// A block a row of up to kSlice logits, which stay in its registers.  Longer rows: a
// block a slice looks for its largest logit and lists its own short top-k; where
// there is none the slices' bins are added up in a second launch; a block a row ends.
#include "nd_internal.h"
#include "nd_lanes.h"

#include <algorithm>

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kPer = 16, kSlice = kPer * kThreads;
constexpr int kBins = 1024;                // two a thread
constexpr int kList = kThreads;            // tokens that are put in order, one a thread
constexpr int kShort = kList - 64;         // the longest top-k that is listed

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
    // (weights below 2^-64 are no whole unit; where none is asked for, of any logit)
    r.low = -64.0 / r.by;
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

__device__ inline bool token(const Row &r, float l)
{
    // (not the difference of two infinities)
    return l == r.top || (l > -INFINITY && double(l) - double(r.top) >= r.low);
}

// 2^z in whole units of 2^-scale, to the nearest; -65 <= z <= 0.  2^f for |f| <= 1/2 by
// the series of e^(f ln 2) to the 13th power, whose next term is below 2^-57.
__device__ inline uint64_t units_of(double z, int scale)
{
    const double n = __builtin_rint(z), f = z - n;
    constexpr double c[] = {1.0,
                            0.693147180559945309417,
                            0.240226506959100712333,
                            0.0555041086648215799531,
                            0.00961812910762847716198,
                            0.00133335581464284434234,
                            0.000154035303933816099544,
                            1.52527338040598402800e-5,
                            1.32154867901443094884e-6,
                            1.01780860092396997275e-7,
                            7.05491162080112332988e-9,
                            4.44553827187081149760e-10,
                            2.56784359934882051420e-11,
                            1.36914888539041288810e-12};
    double p = c[13];
#pragma unroll
    for (int i = 12; i >= 0; --i) p = __builtin_fma(p, f, c[i]);
    // p = m 2^(e - 52), m of 53 bits
    const uint64_t b = uint64_t(__double_as_longlong(p)), m = (b & 0xfffffffffffffull) | 0x10000000000000ull;
    const int sh = int(b >> 52) - 1023 + int(n) + scale - 52;
    if (sh >= 0) return m << sh;
    return sh < -53 ? 0 : ((m >> (-sh - 1)) + 1) >> 1;
}

// The weight of a logit in units; 0: no token.
__device__ inline uint64_t weight_of(const Row &r, float l)
{
    if (!token(r, l)) return 0;
    return l == r.top ? uint64_t(1) << r.scale : units_of((double(l) - double(r.top)) * r.by, r.scale);
}

// A little more than the weight.
__device__ inline float bound_of(const Row &r, float l)
{
    if (!token(r, l)) return 0.0f;
    // (the argument is off by 2^-22 of its size, which is 64 at most)
    return l == r.top ? 1.0f : __builtin_amdgcn_exp2f(float((double(l) - double(r.top)) * r.by)) * 1.0001f;
}

// The scale for weights that come to `sum` or less: below 2^62 units.
__device__ inline int scale_of(float sum) { return 62 - __builtin_amdgcn_frexp_expf(sum * 1.001f); }

__device__ inline int bin_of(const Row &r, float l)
{
    return l == r.top ? 0 : int(fminf((r.top - l) * r.bins, float(kBins - 1)));
}

struct Shared {
    uint32_t count[kBins];
    uint64_t weight[kBins], list[kList], sums[kList];
    uint64_t room[kWaves], best[3];
    uint32_t listed, bin;
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
        for (int b = t; b < kBins; b += kThreads) h.count[b] = 0, h.weight[b] = 0;
        __syncthreads();
    };
    auto add = [&](int b, uint64_t w) {
        atomicAdd(&h.count[b], 1u);
        atomicAdd(reinterpret_cast<unsigned long long *>(&h.weight[b]), w);
    };
    uint64_t tokens = 0, all = 0;
    auto scan = [&]() {  // to sums up to each bin
        __syncthreads();
        const uint32_t c0 = h.count[2 * t], c1 = h.count[2 * t + 1];
        const uint64_t w0 = h.weight[2 * t], w1 = h.weight[2 * t + 1];
        uint64_t c, w;
        tokens = block_scan(uint64_t(c0) + c1, c, h.room);
        all = block_scan(w0 + w1, w, h.room);
        h.count[2 * t] = uint32_t(c) + c0;
        h.count[2 * t + 1] = uint32_t(c) + c0 + c1;
        h.weight[2 * t] = w + w0;
        h.weight[2 * t + 1] = w + w0 + w1;
        __syncthreads();
    };
    auto each = [&](auto f) {
        for (int i = t; i < s.n; i += kThreads) {
            const float l = x[i];
            const uint64_t w = weight_of(r, l);
            if (w) f(l, i, w);
        }
    };
    // the unit
    float bound = 0.0f;
    for (int i = t; i < s.n; i += kThreads) bound += bound_of(r, x[i]);
    bound = ndl::wave_sum64(bound);
    __syncthreads();
    if (lane == 0) h.room[t >> 6] = __float_as_uint(bound);
    __syncthreads();
    bound = 0.0f;
    for (int i = 0; i < kWaves; ++i) bound += __uint_as_float(uint32_t(h.room[i]));
    r.scale = scale_of(bound);
    auto count_row = [&]() {
        clear();
        each([&](float l, int, uint64_t w) { add(bin_of(r, l), w); });
        scan();
    };
    bool whole = false;  // the row's own bins stand in h
    // The first token at which the tokens (by_count) or the weights reach `target`,
    // 1 .. all of them.
    auto find = [&](uint64_t target, bool by_count) {
        if (!whole) count_row();
        whole = true;
        uint64_t before = 0, beforew = 0, prefix = 0;
        int level = -1, bin = -1;  // finer: digits of the order, ten bits each
        for (;;) {
            // the bin in which the target lies
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int b = 2 * t + e;
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
            if (level < 0)
                bin = b;
            else
                prefix = prefix << 10 | uint32_t(b);
            const int shift = 60 - 10 * (level + 1);  // (56 bits of order: the first digit has six)
            __syncthreads();
            if (many <= uint32_t(kList)) {
                each([&](float l, int i, uint64_t) {
                    if (bin_of(r, l) == bin && (level < 0 || order_of(l, i) >> shift == prefix))
                        h.list[atomicAdd(&h.listed, 1u)] = order_of(l, i);
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
                const Cut cut{h.best[0], h.best[1], h.best[2]};
                __syncthreads();
                return cut;
            }
            // too many: their next ten bits
            ++level;
            whole = false;
            clear();
            const int down = 60 - 10 * (level + 1);
            each([&](float l, int i, uint64_t w) {
                if (bin_of(r, l) != bin) return;
                const uint64_t o = order_of(l, i);
                if (level == 0 || o >> (down + 10) == prefix) add(int(o >> down & 1023), w);
            });
            scan();
        }
    };
    count_row();
    whole = true;
    uint64_t sum = all;
    if (r.k > 0 && uint64_t(r.k) < tokens) sum = find(uint64_t(r.k), true).upto;
    if (r.p < 1.0f) {
        const uint64_t need = part_of(sum, fmaxf(r.p, 0.0f), true);
        sum = find(need ? need : 1, false).upto;
    }
    const uint64_t target = part_of(sum, r.u, false) + 1;
    const Cut drawn = find(target < sum ? target : sum, false);
    done(s, row, int(drawn.place & 0xffffff), double(drawn.weight) / double(sum));
}

// ---- the common ways ------------------------------------------------------------

// top and low over the block (kWaves places of room); every thread gets both.
__device__ inline void meet(float &top, float &low, uint64_t *room)
{
    top = ndl::wave_max64(top);
    low = -ndl::wave_max64(-low);
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = uint64_t(__float_as_uint(low)) << 32 | __float_as_uint(top);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        top = fmaxf(top, __uint_as_float(uint32_t(room[i])));
        low = fminf(low, __uint_as_float(uint32_t(room[i] >> 32)));
    }
    __syncthreads();
}

// The tokens listed: those up to the bin of the `want`-th, counted by `each`.  -1: more
// than a list holds.  Leaves `want` as the tokens there are, if those are fewer.
template <typename Each>
__device__ inline int list_first(const Row &r, int &want, Shared &h, Each each)
{
    const int t = threadIdx.x;
    h.count[2 * t] = h.count[2 * t + 1] = 0;
    if (t == 0) h.listed = 0;
    __syncthreads();
    each([&](float l, int) {
        if (token(r, l)) atomicAdd(&h.count[bin_of(r, l)], 1u);
    });
    __syncthreads();
    const uint32_t c0 = h.count[2 * t], c1 = h.count[2 * t + 1];
    uint64_t before;
    const int all = int(block_scan(uint64_t(c0) + c1, before, h.room));
    want = min(want, all);
    const int was = int(before), mid = was + int(c0), now = mid + int(c1);
    if (was < want && now >= want) {
        h.bin = uint32_t(2 * t + (mid < want));
        h.best[0] = uint64_t(mid < want ? now : mid);
    }
    __syncthreads();
    const int last = int(h.bin), many = int(h.best[0]);
    if (many > kList) return -1;
    each([&](float l, int i) {
        if (token(r, l) && bin_of(r, l) <= last) h.list[atomicAdd(&h.listed, 1u)] = order_of(l, i);
    });
    __syncthreads();
    return many;
}

// Draws from the first `want` of the `many` tokens listed.
__device__ inline void draw_listed(const Sample &s, size_t row, Row r, int want, int many, Shared &h)
{
    const int t = threadIdx.x;
    r.scale = 53;
    uint64_t mine = 0;
    if (t < many) {
        mine = h.list[t];
        int rank = 0;
        for (int j = 0; j < many; ++j) rank += h.list[j] < mine;
        h.sums[rank] = mine;
    }
    __syncthreads();
    mine = t < want ? h.sums[t] : 0;
    const uint64_t w = t < want ? weight_of(r, logit_of(mine)) : 0;
    uint64_t before;
    uint64_t sum = block_scan(w, before, h.room);
    if (r.p < 1.0f) {
        uint64_t need = part_of(sum, fmaxf(r.p, 0.0f), true);
        need = need ? need : 1;
        if (before < need && before + w >= need) h.best[0] = before + w;
        __syncthreads();
        sum = h.best[0];
    }
    uint64_t target = part_of(sum, r.u, false) + 1;
    target = target < sum ? target : sum;
    if (before < target && before + w >= target) {
        s.next[row] = int32_t(mine & 0xffffff);
        if (s.prob) s.prob[row] = float(double(w) / double(sum));
    }
}

// Draws from all tokens by their bins' weights, which stand in h.weight (r.scale is
// set); false: a bin that matters has more tokens than a list holds.
template <typename Each>
__device__ inline bool draw_binned(const Sample &s, size_t row, const Row &r, Shared &h, Each each)
{
    const int t = threadIdx.x;
    const uint64_t w0 = h.weight[2 * t], w1 = h.weight[2 * t + 1];
    uint64_t before;
    uint64_t sum = block_scan(w0 + w1, before, h.room);
    int listed = -1;  // the bin that is listed
    uint64_t skip = 0;
    // the token at which the weights reach `target`
    auto find = [&](uint64_t target, Cut &cut) {
        if (before < target && before + w0 + w1 >= target) {
            const bool second = before + w0 < target;
            h.bin = uint32_t(2 * t + second);
            h.best[0] = second ? before + w0 : before;
        }
        if (t == 0) h.listed = 0;
        __syncthreads();
        const int bin = int(h.bin);
        skip = h.best[0];
        if (bin != listed) {
            each([&](float l, int i) {
                if (token(r, l) && bin_of(r, l) == bin) {
                    const uint32_t at = atomicAdd(&h.listed, 1u);
                    if (at < uint32_t(kList)) h.list[at] = order_of(l, i);
                }
            });
            listed = bin;
            __syncthreads();
            if (t == 0) h.best[1] = h.listed;
        }
        __syncthreads();
        const int many = int(h.best[1]);
        if (many > kList) return false;
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
                h.room[0] = mine;
                h.room[1] = upto;
                h.room[2] = w;
            }
        }
        __syncthreads();
        cut = Cut{h.room[0], h.room[1], h.room[2]};
        __syncthreads();
        return true;
    };
    Cut cut{};
    if (r.p < 1.0f) {
        const uint64_t need = part_of(sum, fmaxf(r.p, 0.0f), true);
        if (!find(need ? need : 1, cut)) return false;
        sum = cut.upto;
    }
    const uint64_t target = part_of(sum, r.u, false) + 1;
    if (!find(target < sum ? target : sum, cut)) return false;
    done(s, row, int(cut.place & 0xffffff), double(cut.weight) / double(sum));
    return true;
}

// A slice's logits in registers; what is no token (NaN too) is -inf.
struct Held {
    float v[kPer];
    int t0;
    __device__ inline void load(const float *x, int from, int n)
    {
        t0 = from;
        const int cnt = min(kSlice, n - from);
#pragma unroll
        for (int c = 0; c < kPer / 4; ++c) {
            const int k = c * 4 * kThreads + 4 * int(threadIdx.x);
            if (k + 4 <= cnt) {
                const float4u l = *reinterpret_cast<const float4u *>(x + from + k);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * c + e] = l[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * c + e] = k + e < cnt ? x[from + k + e] : -INFINITY;
            }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[j] = v[j] > -INFINITY ? v[j] : -INFINITY;
    }
    __device__ inline int at(int j) const { return t0 + (j >> 2) * 4 * kThreads + 4 * int(threadIdx.x) + (j & 3); }
    __device__ inline void range(float &top, float &low) const
    {
        top = -INFINITY, low = INFINITY;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            top = fmaxf(top, v[j]);
            low = v[j] > -INFINITY ? fminf(low, v[j]) : low;
        }
    }
    template <typename F>
    __device__ inline void each(F f) const
    {
#pragma unroll
        for (int j = 0; j < kPer; ++j) f(v[j], at(j));
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

// The weights of `each` in the bins, in units of r.scale.
template <typename Each>
__device__ inline void add_weights(const Row &r, Shared &h, Each each)
{
    const int t = threadIdx.x;
    h.weight[2 * t] = h.weight[2 * t + 1] = 0;
    __syncthreads();
    each([&](float l, int) {
        const uint64_t w = weight_of(r, l);
        if (w) atomicAdd(reinterpret_cast<unsigned long long *>(&h.weight[bin_of(r, l)]), w);
    });
    __syncthreads();
}

__device__ inline float sum_bounds(const Row &r, const Held &v, uint64_t *room)
{
    float b = 0.0f;
    v.each([&](float l, int) { b += bound_of(r, l); });
    b = ndl::wave_sum64(b);
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = __float_as_uint(b);
    __syncthreads();
    b = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) b += __uint_as_float(uint32_t(room[i]));
    __syncthreads();
    return b;
}

// Rows of one slice: a block a row.
__global__ __launch_bounds__(kThreads) void sample_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x;
    Held v;
    v.load(s.x + row * s.x_stride, 0, s.n);
    Row r = rules_of(s, row);
    float top, low;
    v.range(top, low);
    meet(top, low, h.room);
    if (top == -INFINITY) return done(s, row, -1, 0.0);
    range_of(r, top, low);
    if (r.greedy) return done(s, row, v.first(top, h.room), 1.0);
    auto each = [&](auto f) { v.each(f); };
    if (r.k > 0 && r.k <= kShort && top < INFINITY) {
        int want = r.k;
        const int many = list_first(r, want, h, each);
        if (many >= 0) return draw_listed(s, row, r, want, many, h);
    } else if (r.k <= 0 && top < INFINITY) {
        r.scale = scale_of(sum_bounds(r, v, h.room));
        add_weights(r, h, each);
        if (draw_binned(s, row, r, h, each)) return;
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
__device__ inline float join_parts(const Sample &s, size_t row, Row &r, uint64_t *room)
{
    const Part *part = s.part + row * s.slices;
    float top = -INFINITY, low = INFINITY;
    for (int i = threadIdx.x; i < s.slices; i += kThreads) {
        top = fmaxf(top, part[i].top);
        low = fminf(low, part[i].low);
    }
    meet(top, low, room);
    range_of(r, top, low);
    if (top == -INFINITY || top == INFINITY) return 1.0f;
    float b = 0.0f;
    for (int i = threadIdx.x; i < s.slices; i += kThreads)
        if (part[i].top > -INFINITY) b += part[i].sum * bound_of(r, part[i].top);
    b = ndl::wave_sum64(b);
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = __float_as_uint(b);
    __syncthreads();
    b = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) b += __uint_as_float(uint32_t(room[i]));
    __syncthreads();
    return b;
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
    float top, low;
    v.range(top, low);
    meet(top, low, h.room);
    range_of(r, top, low);
    if (slice == 0) s.bins[row * kBins + 2 * t] = s.bins[row * kBins + 2 * t + 1] = 0;
    Part p{top, low, 0.0f, 0};
    if (top > -INFINITY) {
        if (r.greedy) {
            p.listed = v.first(top, h.room);
        } else if (way_of(r) == kListed) {
            int want = r.k;
            p.listed = list_first(r, want, h, [&](auto f) { v.each(f); });
            if (t < p.listed) s.list[(row * s.slices + slice) * kList + t] = h.list[t];
        } else if (way_of(r) == kBinned) {
            p.sum = sum_bounds(r, v, h.room);
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
    const float bound = join_parts(s, row, r, h.room);
    if (r.top == -INFINITY || way_of(r) != kBinned) return;
    r.scale = scale_of(bound);
    add_weights(r, h, [&](auto f) { v.each(f); });
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (const uint64_t w = h.weight[2 * t + e])
            atomicAdd(reinterpret_cast<unsigned long long *>(&s.bins[row * kBins + 2 * t + e]), w);
}

__global__ __launch_bounds__(kThreads) void draw_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const size_t row = first + blockIdx.x;
    const int t = threadIdx.x;
    Row r = rules_of(s, row);
    const float bound = join_parts(s, row, r, h.room);
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
    if (way_of(r) == kListed) {
        int most = 0;
        for (int i = t; i < s.slices; i += kThreads) most |= part[i].listed;
        if (!__syncthreads_or(most < 0)) {
            // a wave a slice's list
            const uint64_t *list = s.list + row * s.slices * kList;
            int want = r.k;
            const int many = list_first(r, want, h, [&](auto f) {
                for (int i = t >> 6; i < s.slices; i += kWaves)
                    for (int j = t & 63; j < part[i].listed; j += 64) {
                        const uint64_t o = list[size_t(i) * kList + j];
                        f(logit_of(o), int(o & 0xffffff));
                    }
            });
            if (many >= 0) return draw_listed(s, row, r, want, many, h);
        }
    } else if (way_of(r) == kBinned) {
        r.scale = scale_of(bound);
        h.weight[2 * t] = s.bins[row * kBins + 2 * t];
        h.weight[2 * t + 1] = s.bins[row * kBins + 2 * t + 1];
        const float *x = s.x + row * s.x_stride;
        const bool drawn = draw_binned(s, row, r, h, [&](auto f) {
            for (int i0 = 0; i0 < s.n; i0 += kSlice) {
                Held v;
                v.load(x, i0, s.n);
                v.each(f);
            }
        });
        if (drawn) return;
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
        hipLaunchKernelGGL(draw_kernel, dim3(rows), dim3(kThreads), 0, ctx->stream, s, first);
        if (int rc = nd::check_launch("sample_draw")) return rc;
    }
    return ND_OK;
}

}  // extern "C"
