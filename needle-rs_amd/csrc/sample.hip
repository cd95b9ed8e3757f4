// A token drawn from each row of logits under a temperature, min-p, top-k and
// top-p, by a random number that is given.
//
// All three rules cut the row's order (logits descending, equal ones by their
// number) behind some token, and the draw is a token of that order too: the first
// whose weights, added up, reach a target.  So nothing is sorted: the row's tokens
// are counted and their weights added up in bins that follow the order, the bin of
// a target is found, and only its tokens are looked at one by one (in finer bins
// first, where there are many).
// Weights are whole numbers, exp((l - M) / T) in units of 2^-s: worked out in fp64,
// so that a pick next to a border is the border's and not the rounding's, and sums
// of whole numbers are the same in any order.  s is chosen by a bound on the row's
// sum, so that the sum has 2^60 .. 2^62 units whatever the row's shape.
#include "nd_internal.h"
#include "nd_lanes.h"

#include <algorithm>

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kBins = 1024;    // two a thread
constexpr int kList = kThreads;  // tokens that are looked at one by one

struct Sample {
    const float *x, *temperature, *min_p, *top_p, *u;
    const int32_t *top_k;
    size_t x_stride;
    int n;
    int32_t *next;
    float *prob;
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

struct Row {
    float top;        // its largest logit
    double by, low;   // 1 / T; logits above top + low and at it are tokens
    float bins;       // bins a unit of l
    int scale;
};

// 2^s exp((l - top) / T); 0: no token.
__device__ inline uint64_t weight_of(const Row &r, float l)
{
    if (!(l > -INFINITY)) return 0;
    if (l == r.top) return uint64_t(1) << r.scale;
    const double d = double(l) - double(r.top);
    if (!(d >= r.low)) return 0;
    return uint64_t(__double2ll_rn(ldexp(exp(d * r.by), r.scale)));
}

// More than 2^32 exp((l - top) / T), and not much.
__device__ inline uint64_t bound_of(const Row &r, float l)
{
    if (!(l > -INFINITY)) return 0;
    if (l == r.top) return uint64_t(1) << 32;
    const double d = double(l) - double(r.top);
    if (!(d >= r.low)) return 0;
    // (the argument is off by 2^-23 of its size, of 150 at most where it counts)
    return uint64_t(__builtin_amdgcn_exp2f(float(d * r.by) * 1.4426950f) * 0x1.0002p32f) + 2;
}

__device__ inline int bin_of(const Row &r, float l)
{
    return l == r.top ? 0 : int(fminf((r.top - l) * r.bins, float(kBins - 1)));
}

struct Shared {
    uint32_t count[kBins];
    uint64_t weight[kBins], list[kList], sums[kList];
    uint64_t room[kWaves], best[2];
    uint32_t roomc[kWaves], listed, bin, low;
};

// Where a target lies: the token, the weights up to it and its own.
struct Cut {
    uint64_t place, upto, weight;
};

template <typename T>
__device__ inline T block_scan(T v, T &before, T *room)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    T up = v;
    for (int d = 1; d < 64; d *= 2) {
        const T o = __shfl_up(up, d);
        if (lane >= d) up += o;
    }
    if (lane == 63) room[w] = up;
    __syncthreads();
    T all = 0, mine = 0;
    for (int i = 0; i < kWaves; ++i) {
        mine += i < w ? room[i] : 0;
        all += room[i];
    }
    __syncthreads();
    before = mine + up - v;
    return all;
}

// A block a row.
__global__ __launch_bounds__(kThreads) void sample_kernel(Sample s, size_t first)
{
    __shared__ Shared h;
    const int t = threadIdx.x, lane = t & 63;
    const size_t row = first + blockIdx.x;
    const float *x = s.x + row * s.x_stride;
    float top = -INFINITY, low = INFINITY;
    for (int i = t; i < s.n; i += kThreads) {
        const float l = x[i];
        top = fmaxf(top, l);
        if (l > -INFINITY) low = fminf(low, l);
    }
    top = ndl::wave_max64(top);
    low = -ndl::wave_max64(-low);
    if (lane == 0) h.sums[t >> 6] = uint64_t(__float_as_uint(low)) << 32 | __float_as_uint(top);
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) {
        top = fmaxf(top, __uint_as_float(uint32_t(h.sums[i])));
        low = fminf(low, __uint_as_float(uint32_t(h.sums[i] >> 32)));
    }
    const float T = s.temperature ? s.temperature[row] : 1.0f;
    if (top == -INFINITY) {
        if (t == 0) {
            s.next[row] = -1;
            if (s.prob) s.prob[row] = 0.0f;
        }
        return;
    }
    const float mp = s.min_p ? s.min_p[row] : 0.0f;
    const int k = s.top_k ? s.top_k[row] : 0;
    const float p = s.top_p ? s.top_p[row] : 1.0f;
    float u = s.u[row];
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    Row r;
    r.top = top;
    const bool greedy = !(T > 0.0f) || mp > 1.0f;
    r.by = greedy ? 1.0 : 1.0 / double(T);
    r.low = mp > 0.0f ? double(T) * log(double(mp)) : -INFINITY;
    if (greedy || mp >= 1.0f || top == INFINITY) r.low = 0.0;
    // 16 bins an octave of weights, or as many as the row's logits need
    r.bins = fminf(fmaxf(16.0f * 1.4426950f * float(r.by), float(kBins - 1) / (top - low)), 1e30f);

    // ---- the unit: weights to 2^-32, each a little too large, come to little more
    // than the sum (the largest alone is 1, what 2^24 are too large 2^-6) ----
    uint64_t most = 0;
    for (int i = t; i < s.n; i += kThreads) most += bound_of(r, x[i]);
    for (int d = 32; d; d /= 2) most += __shfl_xor(most, d);
    __syncthreads();
    if (lane == 0) h.sums[t >> 6] = most;
    __syncthreads();
    most = 0;
    for (int i = 0; i < kWaves; ++i) most += h.sums[i];
    r.scale = 62 + 32 - (64 - __clzll(most));  // most < 2^bits, the sum below 2^(bits - 32)

    // ---- the row's bins: their tokens and weights, then those up to each ----
    auto clear = [&]() {
        for (int b = t; b < kBins; b += kThreads) h.count[b] = 0, h.weight[b] = 0;
        __syncthreads();
    };
    auto add = [&](int b, uint64_t w) {
        atomicAdd(&h.count[b], 1u);
        atomicAdd(reinterpret_cast<unsigned long long *>(&h.weight[b]), w);
    };
    struct Sum {
        uint32_t count;
        uint64_t weight;
    };
    auto scan = [&]() {
        __syncthreads();
        const uint32_t c0 = h.count[2 * t], c1 = h.count[2 * t + 1];
        const uint64_t w0 = h.weight[2 * t], w1 = h.weight[2 * t + 1];
        uint32_t c;
        uint64_t w;
        Sum all;
        all.count = block_scan(c0 + c1, c, h.roomc);
        all.weight = block_scan(w0 + w1, w, h.room);
        h.count[2 * t] = c + c0;
        h.count[2 * t + 1] = c + c0 + c1;
        h.weight[2 * t] = w + w0;
        h.weight[2 * t + 1] = w + w0 + w1;
        __syncthreads();
        return all;
    };
    auto each = [&](auto f) {
        for (int i = t; i < s.n; i += kThreads) {
            const float l = x[i];
            const uint64_t w = weight_of(r, l);
            if (w) f(l, i, w);
        }
    };
    auto order_of = [&](float l, int i) { return uint64_t(place_of(l)) << 24 | uint32_t(i); };
    Sum all{};
    auto count_row = [&]() {
        clear();
        each([&](float l, int, uint64_t w) { add(bin_of(r, l), w); });
        all = scan();
    };
    bool whole = false;  // the row's own bins stand in h
    // The first token at which the tokens (by_count) or the weights reach `target`,
    // 1 .. all of them.
    auto find = [&](uint64_t target, bool by_count) {
        if (!whole) count_row();
        whole = true;
        uint64_t before = 0, beforew = 0;
        int level = -1, bin = -1;  // finer: digits of the order, ten bits each
        uint64_t prefix = 0;
        Cut cut{};
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
            const uint64_t skip = b ? (by_count ? h.count[b - 1] : h.weight[b - 1]) : 0;
            beforew += b ? h.weight[b - 1] : 0;
            before += skip;
            if (level < 0) bin = b;
            else prefix = prefix << 10 | uint32_t(b);
            const int shift = 60 - 10 * (level + 1);  // order >> shift == prefix so far (56 bits: digits from 60 down)
            auto in = [&](float l, int i) {
                return bin_of(r, l) == bin && (level < 0 || order_of(l, i) >> shift == prefix);
            };
            __syncthreads();
            if (many <= uint32_t(kList)) {
                each([&](float l, int i, uint64_t) {
                    if (in(l, i)) h.list[atomicAdd(&h.listed, 1u)] = order_of(l, i);
                });
                __syncthreads();
                uint64_t mine = ~uint64_t(0), w = 0;
                if (uint32_t(t) < many) {
                    mine = h.list[t];
                    w = weight_of(r, x[mine & 0xffffff]);
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
                    }
                }
                __syncthreads();
                cut.place = h.best[0];
                cut.upto = h.best[1];
                cut.weight = weight_of(r, x[cut.place & 0xffffff]);
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
    Cut drawn{};
    uint64_t sum = 1;
    if (greedy) {
        drawn = find(1, true);
        drawn.weight = sum;
    } else {
        count_row();
        whole = true;
        sum = all.weight;
        if (k > 0 && uint32_t(k) < all.count) sum = find(uint64_t(k), true).upto;
        if (p < 1.0f) sum = find(max(part_of(sum, fmaxf(p, 0.0f), true), uint64_t(1)), false).upto;
        drawn = find(min(part_of(sum, u, false) + 1, sum), false);
    }
    if (t == 0) {
        s.next[row] = int32_t(drawn.place & 0xffffff);
        if (s.prob) s.prob[row] = float(double(drawn.weight) / double(sum));
    }
}

}  // namespace

extern "C" {

size_t nd_sample_rows_work(nd_ctx *, size_t, size_t) { return 0; }

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
    Sample s{x, r.temperature, r.min_p, r.top_p, u, r.top_k, x_stride, int(n), next, prob};
    // HIP counts a launch's threads in 32 bits: rows beyond that go in further launches
    const size_t most = 0xffffffff / kThreads;
    for (size_t first = 0; first < count; first += most) {
        const unsigned rows = unsigned(std::min(most, count - first));
        hipLaunchKernelGGL(sample_kernel, dim3(rows), dim3(kThreads), 0, ctx->stream, s, first);
        if (int rc = nd::check_launch("sample_rows")) return rc;
    }
    return ND_OK;
}

}  // extern "C"
