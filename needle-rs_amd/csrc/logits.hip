// Logits under a request's rules -- penalties for repeated tokens, biases,
// grammar masks -- and the greedy pick.
//
// A block takes a slice of kSlice tokens of one row, asks for its logits, counts
// the history's tokens that fall into the slice in LDS meanwhile (whole numbers:
// the order of the atomics changes nothing), and passes over the logits once.  A
// token with a bias is left to the thread that holds its entry of the list; where
// one is listed twice the list is gone through in order, as many entries at a time
// as do not meet (64 rows with lists of 300 14 us, of 2000 23; a thread that looks
// through the list for its token's other entries took 46 and 750).
// Bound by memory: 4 bytes in and 4 out a logit, the history a second time for
// every slice after the first (from L2).  Written past the caches: 1024 rows of
// 8192 17.9 -> 15.9 us (15.9 is what a copy of as many bytes takes), 200 of 100003
// 42.6 -> 38.7 (34.4), of which the history costs 2.5 and the join of a row's
// slices 3; read past them too it was slower (18.2, 43.3), and so were slices of
// 4096 (25.1, 48.9) and blocks of 256 (19.5, 49.0) or 1024 threads (22.3, 47.6).
//
// Every step is one fp32 rounding (the file is compiled without contraction),
// so results do not depend on slice, lane or the presence of other rules.
#include "nd_internal.h"
#include "nd_lanes.h"

#include <algorithm>

namespace {

constexpr int kThreads = 512;
constexpr int kSlice = 8192;  // 32 KiB of counts: four blocks a CU
constexpr int kChunk = 4 * kThreads, kChunks = kSlice / kChunk;

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));  // rows may start anywhere
typedef int int4u __attribute__((ext_vector_type(4), aligned(4)));
constexpr uint32_t kEver = 1u << 30, kBias = 1u << 31;  // beside the count of a token

struct Pick {
    float v;
    int i;
};

// The first of equal maxima; a NaN never wins.
__device__ inline void take(Pick &a, float v, int i)
{
    if (v > a.v || (v == a.v && i < a.i)) a = Pick{v, i};
}

__device__ inline int clamp_len(const int32_t *len, size_t row, size_t most)
{
    const int m = int(most);
    return len ? min(max(len[row], 0), m) : m;
}

template <int H>
__device__ inline void meet(Pick &a)
{
    const float v = ndl::wave_xor<H>(a.v);
    take(a, v, ndl::wave_xor_int<H>(a.i));
}

__device__ inline void meet_wave(Pick &a)
{
    meet<32>(a), meet<16>(a), meet<8>(a), meet<4>(a), meet<2>(a), meet<1>(a);
}

constexpr int kNone = 0x7fffffff;

__global__ __launch_bounds__(kThreads) void adjust_kernel(const float *x, size_t x_stride, size_t first, int n, int slices,
                                                          nd_logits_rules r, float *y, size_t y_stride,
                                                          int32_t *next, Pick *part)
{
    __shared__ __align__(16) uint32_t st[kSlice];
    __shared__ int twice, turn[kThreads];
    __shared__ Pick best[kThreads / 64];
    const size_t row = first + blockIdx.x / unsigned(slices);
    const int slice = int(blockIdx.x % unsigned(slices)), t0 = slice * kSlice, t = threadIdx.x;
    const int cnt = min(kSlice, n - t0);
    const float *xr = x + row * x_stride + t0;
    float *yr = y ? y + row * y_stride + t0 : nullptr;

    // ---- the slice's logits, on their way while the tokens are counted ----
    float v[kChunks][4];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int k = c * kChunk + 4 * t;
        if (k + 4 <= cnt) {
            const float4u l = *reinterpret_cast<const float4u *>(xr + k);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c][e] = l[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c][e] = k + e < cnt ? xr[k + e] : 0.0f;
        }
    }
    const uint32_t *mask = nullptr;
    if (r.mask) {
        const int m = r.mask_row ? r.mask_row[row] : int(row);
        if (m >= 0 && size_t(m) < r.mask_rows) mask = r.mask + size_t(m) * r.mask_stride + (t0 >> 5);
    }
    const int nh = r.hist ? clamp_len(r.hist_len, row, r.hist_stride) : 0;
    const int nb = r.bias ? clamp_len(r.bias_len, row, r.bias_stride) : 0;
    const bool marks = nh > 0 || nb > 0;
    const float rep = r.repeat ? r.repeat[row] : 1.0f;
    const float fr = r.frequency ? r.frequency[row] : 0.0f, pr = r.presence ? r.presence[row] : 0.0f;
    const int32_t *bi = r.bias_id + row * r.bias_stride;
    const float *bv = r.bias + row * r.bias_stride;
    if (marks) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
            *reinterpret_cast<uint4 *>(&st[c * kChunk + 4 * t]) = make_uint4(0, 0, 0, 0);
        if (t == 0) twice = 0;
        __syncthreads();
        const int32_t *h = r.hist + row * r.hist_stride;
        const int from = r.out_from ? r.out_from[row] : 0;
        auto count = [&](int tok, int i) {
            const uint32_t k = uint32_t(tok) - uint32_t(t0);
            if (k < uint32_t(cnt)) {
                atomicOr(&st[k], kEver);
                if (i >= from) atomicAdd(&st[k], 1u);
            }
        };
        for (int i = 4 * t; i < nh; i += kChunk) {
            if (i + 4 <= nh) {
                const int4u q = *reinterpret_cast<const int4u *>(h + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) count(q[e], i + e);
            } else {
                for (int e = i; e < nh; ++e) count(h[e], e);
            }
        }
        for (int i = t; i < nb; i += kThreads) {
            const uint32_t k = uint32_t(bi[i]) - uint32_t(t0);
            if (k < uint32_t(cnt) && (atomicOr(&st[k], kBias) & kBias)) twice = 1;
        }
        __syncthreads();
    }
    // the penalties of a token's marks
    auto penal = [&](float l, uint32_t s) {
        const uint32_t c = s & (kEver - 1);
        if ((s & kEver) && r.repeat) l = l > 0.0f ? l / rep : l * rep;
        if (c && r.frequency) l -= float(c) * fr;
        if (c && r.presence) l -= pr;
        return l;
    };
    const bool again = marks && twice;
    Pick b{-INFINITY, kNone};
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int k = c * kChunk + 4 * t;
        if (k >= cnt) continue;
        uint4 s = make_uint4(0, 0, 0, 0);
        if (marks) s = *reinterpret_cast<const uint4 *>(&st[k]);
        const uint32_t sv[4] = {s.x, s.y, s.z, s.w};
        const uint32_t allowed = mask ? mask[k >> 5] >> (k & 31) : 0xfu;
        const uint32_t any = s.x | s.y | s.z | s.w;
        if (any & ~kBias) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c][e] = penal(v[c][e], sv[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!(allowed >> e & 1)) v[c][e] = -INFINITY;
            if (k + e < cnt && !(sv[e] & kBias) && v[c][e] > b.v) b = Pick{v[c][e], t0 + k + e};
        }
        if (yr) {
            if (k + 4 <= cnt && !(any & kBias)) {
                __builtin_nontemporal_store(float4u{v[c][0], v[c][1], v[c][2], v[c][3]},
                                            reinterpret_cast<float4u *>(yr + k));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k + e < cnt && !(sv[e] & kBias)) yr[k + e] = v[c][e];
            }
        }
    }
    // ---- tokens with a bias: a thread an entry of the list ----
    if (!again) {
        for (int i = t; i < nb; i += kThreads) {
            const uint32_t k = uint32_t(bi[i]) - uint32_t(t0);
            if (k >= uint32_t(cnt)) continue;
            float l = penal(xr[k], st[k]) + bv[i];
            if (mask && !(mask[k >> 5] >> (k & 31) & 1)) l = -INFINITY;
            if (yr) yr[k] = l;
            if (l > -INFINITY) take(b, l, t0 + int(k));
        }
    } else {
        // Some token of the slice is listed twice.  The thread of a logit takes its
        // marks, in whose place comes the sum of its biases, to which the list's
        // entries are added in order: of those that meet (in a slot of `turn`) the
        // first goes, the others wait.
        turn[t] = kNone;
        uint32_t was[4 * kChunks];
#pragma unroll
        for (int i = 0; i < 4 * kChunks; ++i) {
            uint32_t &s = st[(i >> 2) * kChunk + 4 * t + (i & 3)];
            was[i] = s;
            s = 0x80000000u;  // -0
        }
        __syncthreads();
        for (int i = 0; i < nb; i += kThreads) {
            const uint32_t k = i + t < nb ? uint32_t(bi[i + t]) - uint32_t(t0) : ~0u;
            const float v = i + t < nb ? bv[i + t] : 0.0f;
            bool left = k < uint32_t(cnt);
            do {
                if (left) atomicMin(&turn[k % kThreads], t);
                __syncthreads();
                if (left && turn[k % kThreads] == t) {
                    st[k] = __float_as_uint(__uint_as_float(st[k]) + v);
                    turn[k % kThreads] = kNone;
                    left = false;
                }
            } while (__syncthreads_or(left));
        }
#pragma unroll
        for (int i = 0; i < 4 * kChunks; ++i) {
            if (!(was[i] & kBias)) continue;
            const int k = (i >> 2) * kChunk + 4 * t + (i & 3);
            float l = penal(xr[k], was[i]) + __uint_as_float(st[k]);
            if (mask && !(mask[k >> 5] >> (k & 31) & 1)) l = -INFINITY;
            if (yr) yr[k] = l;
            if (l > -INFINITY) take(b, l, t0 + k);
        }
    }
    if (!next) return;
    meet_wave(b);
    if ((t & 63) == 0) best[t >> 6] = b;
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < kThreads / 64; ++w) take(b, best[w].v, best[w].i);
        if (slices == 1)
            next[row] = b.i == kNone ? -1 : b.i;
        else
            part[row * slices + slice] = b;
    }
}

// A wave a row: the best of its slices.
__global__ __launch_bounds__(64) void join_kernel(const Pick *__restrict__ part, size_t first, int slices,
                                                  int32_t *__restrict__ next)
{
    const size_t row = first + blockIdx.x;
    Pick b{-INFINITY, kNone};
    for (int s = threadIdx.x; s < slices; s += 64) {
        const Pick p = part[row * slices + s];
        take(b, p.v, p.i);
    }
    meet_wave(b);
    if (threadIdx.x == 0) next[row] = b.i == kNone ? -1 : b.i;
}

size_t slices_of(size_t n) { return (n + kSlice - 1) / kSlice; }

}  // namespace

extern "C" {

size_t nd_logits_adjust_work(nd_ctx *, size_t count, size_t n)
{
    const size_t s = slices_of(n);
    return s > 1 ? count * s * sizeof(Pick) : 0;
}

int nd_logits_adjust(nd_ctx *ctx, const float *x, size_t x_stride, size_t count, size_t n,
                     const nd_logits_rules *rules, float *y, size_t y_stride, int32_t *next,
                     void *work, size_t work_bytes)
{
    ND_ENTER(ctx);
    ND_REQUIRE(rules, "null rules");
    ND_REQUIRE(n > 0 && n <= (size_t(1) << 24), "n %zu must be in 1..2^24", n);
    if (count == 0 || (!y && !next)) return ND_OK;
    ND_REQUIRE(x, "null buffer");
    ND_REQUIRE(count == 1 || (x_stride >= n && (!y || y_stride >= n)), "row strides below n %zu", n);
    const size_t slices = slices_of(n);
    ND_REQUIRE(count <= 0x7fffffff, "count %zu above 2^31 - 1", count);
    const nd_logits_rules &r = *rules;
    ND_REQUIRE(!r.hist || r.hist_stride < (size_t(1) << 30), "hist_stride too large");
    ND_REQUIRE(!r.bias == !r.bias_id, "bias and bias_id are given together or not at all");
    ND_REQUIRE(!r.bias || r.bias_stride < (size_t(1) << 30), "bias_stride too large");
    ND_REQUIRE(!r.mask || r.mask_stride >= (n + 31) / 32, "mask_stride %zu below %zu words", r.mask_stride,
               (n + 31) / 32);
    ND_REQUIRE(!r.mask || r.mask_row || r.mask_rows >= count, "%zu mask rows for %zu rows", r.mask_rows, count);
    if (y && y != x) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
        ND_REQUIRE(a + ((count - 1) * x_stride + n) * 4 <= b || b + ((count - 1) * y_stride + n) * 4 <= a,
                   "y overlaps x");
    }
    ND_REQUIRE(y != x || count == 1 || x_stride == y_stride, "y is x with another stride");
    Pick *part = nullptr;
    if (next && slices > 1) {
        void *p = nullptr;
        if (int rc = nd::call_workspace(ctx, count * slices * sizeof(Pick), work, work_bytes, &p)) return rc;
        part = static_cast<Pick *>(p);
    }
    // HIP counts a launch's threads in 32 bits: rows beyond that go in further launches
    const size_t most = size_t(0xffffffff / kThreads) / slices;
    for (size_t first = 0; first < count; first += most) {
        const unsigned rows = unsigned(std::min(most, count - first));
        hipLaunchKernelGGL(adjust_kernel, dim3(rows * unsigned(slices)), dim3(kThreads), 0, ctx->stream, x, x_stride,
                           first, int(n), int(slices), r, y, y_stride, next, part);
        if (int rc = nd::check_launch("logits_adjust")) return rc;
        if (part) {
            hipLaunchKernelGGL(join_kernel, dim3(rows), dim3(64), 0, ctx->stream, part, first, int(slices), next);
            if (int rc = nd::check_launch("logits_join")) return rc;
        }
    }
    return ND_OK;
}

}  // extern "C"
