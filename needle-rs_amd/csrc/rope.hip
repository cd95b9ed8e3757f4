// Rotary positions, alone and on the way into the int8 cache, and the cache
// read back.
//
// A turn is y = (u cos a - w sin a, u sin a + w cos a) for a pair (u, w) and
// the angle a = pos f.  Angle, sine, cosine and products are fp64: at position
// 10^6 an fp32 angle is off by 0.03, and where the result is quantised a code
// next to a border should not depend on how the products were rounded.  A block
// works out each (row, pair) once, in LDS, for all heads of the row.  A group of
// 16, 32 or 64 lanes takes a head vector, four elements a lane, so that a code's
// scale is a maximum over the group's registers.
// (Lane moves stay within a group, whose lanes are all there; other groups of a wave
// may be elsewhere.)
// All three calls are bound by memory, a value read and written once, results past
// the caches (kernel times): 6001 rows of 12 x 64 7.5 us = 4.9 TB/s; 8000 rows of 12
// q, 12 k and 12 v heads of 64 25.4 us = 4.4 TB/s, their read-back 12.5 us = 5.0;
// 16 windows of 8001 positions of 2 kv heads, 48 and 64 long, read in 23.9 us = 6.1.
#include "nd_internal.h"
#include "nd_kv_internal.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace ndkv;

constexpr int kThreads = 256;
constexpr int kMaxPairs = kMaxDim / 2;

// A rope as the kernels take it, for heads of 2 P elements or fewer: a launch
// copies its arguments, and most heads are short.
template <int P>
struct TurnOf {
    int layout, rot;
    double gain;
    double f[P];
};
using Turn = TurnOf<kMaxPairs>;

// What a rope or write launch works on: rows of nq q heads, and of a
// cache's k and v heads, any of them absent.
struct Rows {
    size_t rows, first, per_block;  // first: the launch's first row
    const int32_t *pos, *rot_pos;
    const float *q, *k, *v;
    float *q_out;
    size_t q_stride, q_out_stride, k_stride, v_stride, kv_stride;
    uint8_t *kv;
    int nq, dim;
};

// Sine and cosine of |a| < 2^42: a - n pi / 2 with pi / 2 in two parts (the first
// fma is exact but for the last bit of what is left, so the remainder is off by
// 2^-53 of at most pi / 4), then the two Taylor series, whose first terms left out
// are r^17 / 17! < 5e-17 and r^18 / 18! < 3e-18.
__device__ inline void sine_cosine(double a, double &sn, double &c)
{
    const double n = __builtin_rint(a * 0.63661977236758134);
    double r = __builtin_fma(-n, 0x1.921fb54442d18p+0, a);
    r = __builtin_fma(-n, 0x1.1a62633145c07p-54, r);
    const double x = r * r;
    double s = -1.0 / 1307674368000.0, t = 1.0 / 20922789888000.0;  // 1 / 15!, 1 / 16!
    s = __builtin_fma(s, x, 1.0 / 6227020800.0);
    t = __builtin_fma(t, x, -1.0 / 87178291200.0);
    s = __builtin_fma(s, x, -1.0 / 39916800.0);
    t = __builtin_fma(t, x, 1.0 / 479001600.0);
    s = __builtin_fma(s, x, 1.0 / 362880.0);
    t = __builtin_fma(t, x, -1.0 / 3628800.0);
    s = __builtin_fma(s, x, -1.0 / 5040.0);
    t = __builtin_fma(t, x, 1.0 / 40320.0);
    s = __builtin_fma(s, x, 1.0 / 120.0);
    t = __builtin_fma(t, x, -1.0 / 720.0);
    s = __builtin_fma(s, x, -1.0 / 6.0);
    t = __builtin_fma(t, x, 1.0 / 24.0);
    t = __builtin_fma(t, x, -0.5);
    s = __builtin_fma(s * x, r, r);
    t = __builtin_fma(t, x, 1.0);
    const int q = int(int64_t(n) & 3);
    const double u = q & 1 ? t : s, v = q & 1 ? s : t;
    sn = q & 2 ? -u : u;
    c = (q + 1) & 2 ? -v : v;
}

// Where a row lies in the cache, worked out once a block: its block and slot, and
// its position (-1: left out).
struct Place {
    size_t off;
    int slot, p;
};
constexpr int kMaxRows = 16;

__device__ inline Place place_of(const int32_t *pos, size_t i, size_t per_block, size_t kv_stride, int cap)
{
    const int p = pos[i];
    const size_t b = per_block == 1 ? i : (i | per_block) >> 32 ? i / per_block : uint32_t(i) / uint32_t(per_block);
    return Place{b * kv_stride, p < 0 ? 0 : p % cap, p};
}

typedef float float4a __attribute__((ext_vector_type(4)));
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));  // rows may start anywhere
typedef float float2u __attribute__((ext_vector_type(2), aligned(4)));

// G lanes a head vector, four elements a lane: element 4 l + e of the head.  FOUR:
// every head is a multiple of 4 long, and with halves rot / 2 is too, so that a
// lane's partners are four neighbours.  A group keeps its heads for all rows of
// the block: q heads, then k heads, then v heads.
template <int G, bool FOUR>
__global__ __launch_bounds__(kThreads) void turn_kernel(TurnOf<2 * G> tn, Rows r, Geom g, int rpb)
{
    extern __shared__ double2 cs[];  // [rpb][rot / 2]: gain cos, gain sin
    __shared__ Place at_row[kMaxRows];
    const int t = threadIdx.x, l = t % G, e0 = 4 * l, groups = blockDim.x / G;
    const int half = tn.rot / 2;
    const bool pairs = tn.layout == ND_ROPE_PAIRS;
    // where pair k of a row lies in LDS: what the lanes of a group read at once,
    // pairs 4 l + e or 2 l + e / 2, one after another
    const int q4 = half / 4, q2 = half / 2;
    auto place_in = [&](int k) { return !FOUR ? k : pairs ? (k & 1) * q2 + k / 2 : (k & 3) * q4 + k / 4; };

    // the lane's elements of a head, as they are
    auto load = [&](const float *x, int dim, float (&y)[4]) {
        if (FOUR ? e0 < dim : e0 + 4 <= dim) {
            const float4u q = *reinterpret_cast<const float4u *>(x + e0);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = q[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = !FOUR && e0 + e < dim ? x[e0 + e] : 0.0f;
        }
    };
    // and turned
    auto turn = [&](const float *x, int row, float (&y)[4]) {
        if (e0 >= tn.rot) return;
        const double2 *a = cs + row * half;
        if (pairs) {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                if (!FOUR && e0 + e >= tn.rot) continue;
                const double2 z = a[FOUR ? (e / 2) * q2 + l : (e0 + e) / 2];
                const double u = y[e], w = y[e + 1];
                y[e] = float(u * z.x - w * z.y);
                y[e + 1] = float(u * z.y + w * z.x);
            }
        } else if (FOUR) {
            const bool second = e0 >= half;
            const int j = second ? e0 - half : e0;
            const float4u o = *reinterpret_cast<const float4u *>(x + (second ? j : e0 + half));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double2 z = a[e * q4 + j / 4];
                y[e] = float(double(y[e]) * z.x + double(second ? o[e] : -o[e]) * z.y);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (e0 + e >= tn.rot) continue;
                const bool second = e0 + e >= half;
                const int j = second ? e0 + e - half : e0 + e;
                const float o = x[second ? j : j + half];
                y[e] = float(double(y[e]) * a[j].x + double(second ? o : -o) * a[j].y);
            }
        }
    };
    // quant_into (cache.rs:80-104) and the store of k or v head h; heads are
    // multiples of 16 long
    auto keep = [&](const Place &place, const float (&y)[4], int h, int dim, size_t part, size_t scales) {
        float m = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float av = y[e] < 0.0f ? -y[e] : y[e];
            if (av > m) m = av;
        }
        m = fmaxf(m, ndl::wave_xor<1>(m));
        m = fmaxf(m, ndl::wave_xor<2>(m));
        m = fmaxf(m, ndl::wave_xor<4>(m));
        m = fmaxf(m, ndl::wave_xor<8>(m));
        if (G >= 32) m = fmaxf(m, ndl::wave_xor<16>(m));
        if (G >= 64) m = fmaxf(m, ndl::wave_xor<32>(m));
        if (place.p < 0) return;
        const float scale = m > 0.0f ? m / 127.0f : 1.0f;
        const float inv = 1.0f / scale;
        uint32_t codes = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) codes |= (uint32_t(int32_t(int8_t(quant_code(y[e], inv)))) & 0xffu) << (8 * e);
        uint8_t *blk = r.kv + place.off;
        const size_t at = size_t(h) * g.cap + place.slot;
        if (e0 < dim) *reinterpret_cast<uint32_t *>(blk + part + at * dim + e0) = codes;
        if (l == 0) reinterpret_cast<float *>(blk + scales)[at] = scale;
    };

    const size_t i0 = r.first + size_t(blockIdx.x) * rpb;
    const int rows = int(min(size_t(rpb), r.rows - i0));
    if (t < rows) at_row[t] = place_of(r.pos, i0 + t, r.per_block, r.kv_stride, r.kv ? g.cap : 1);
    for (int j = t; j < rows * half; j += blockDim.x) {
        const int row = j / half, k = j - row * half;
        const int p = r.rot_pos ? r.rot_pos[i0 + row] : r.pos[i0 + row];
        double sn, c;
        sine_cosine(double(p) * tn.f[k], sn, c);
        cs[row * half + place_in(k)] = double2{tn.gain * c, tn.gain * sn};
    }
    __syncthreads();
    const int heads = r.nq + (r.kv ? 2 * g.KVH : 0);
    for (int h = t / G; h < heads; h += groups) {
        float y[4];
        if (h < r.nq) {
            const float *x = r.q + i0 * r.q_stride + size_t(h) * r.dim;
            float *out = r.q_out + i0 * r.q_out_stride + size_t(h) * r.dim;
            for (int row = 0; row < rows; ++row, x += r.q_stride, out += r.q_out_stride) {
                load(x, r.dim, y);
                turn(x, row, y);
                if (at_row[row].p < 0) continue;  // left out; what was read is memory all the same
                if (FOUR ? e0 < r.dim : e0 + 4 <= r.dim) {
                    __builtin_nontemporal_store(float4u{y[0], y[1], y[2], y[3]}, reinterpret_cast<float4u *>(out + e0));
                } else if (!FOUR) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e0 + e < r.dim) out[e0 + e] = y[e];
                }
            }
        } else if (h < r.nq + g.KVH) {
            const int hk = h - r.nq;
            const float *x = r.k + i0 * r.k_stride + size_t(hk) * g.QK;
            for (int row = 0; row < rows; ++row, x += r.k_stride) {
                load(x, g.QK, y);
                turn(x, row, y);
                keep(at_row[row], y, hk, g.QK, 0, g.ks_off);
            }
        } else {
            const int hk = h - r.nq - g.KVH;
            const float *x = r.v + i0 * r.v_stride + size_t(hk) * g.VD;
            for (int row = 0; row < rows; ++row, x += r.v_stride) {
                load(x, g.VD, y);
                keep(at_row[row], y, hk, g.VD, g.v_off, g.vs_off);
            }
        }
    }
}

// Sixteen bytes of a result a lane: four codes of a head vector and its scale.
// Item j of a row is dword j of its K heads, then of its V heads.
__global__ __launch_bounds__(kThreads) void read_kernel(Geom g, const uint8_t *__restrict__ kv,
                                                        size_t kv_stride, size_t rows, size_t first,
                                                        size_t per_block, const int32_t *__restrict__ pos,
                                                        float *__restrict__ k, float *__restrict__ v, int rpb,
                                                        uint32_t by_qk, uint32_t by_vd)
{
    __shared__ Place at_row[kMaxRows];
    const int wk = k ? g.KVH * g.QK / 4 : 0, wv = v ? g.KVH * g.VD / 4 : 0, items = wk + wv;
    const size_t i0 = first + size_t(blockIdx.x) * rpb;
    const int n = int(min(size_t(rpb), rows - i0));
    if (int(threadIdx.x) < n) at_row[threadIdx.x] = place_of(pos, i0 + threadIdx.x, per_block, kv_stride, g.cap);
    __syncthreads();
    for (int row = 0, j = threadIdx.x;; j += kThreads) {
        while (j >= items) j -= items, ++row;
        if (row >= n) break;
        const size_t i = i0 + row;
        const bool isv = j >= wk;
        // dword d of the heads: d / (dim / 4) by 2^32 / (dim / 4) rounded up, d below 2^16 64
        const int d = isv ? j - wk : j, dim = isv ? g.VD : g.QK, e = 4 * d;
        const int h = int(__umulhi(uint32_t(d), isv ? by_vd : by_qk));
        const Place &place = at_row[row];
        const uint8_t *blk = kv + place.off;
        const size_t at = size_t(h) * g.cap + place.slot;
        const uint32_t c = *reinterpret_cast<const uint32_t *>(blk + (isv ? g.v_off : 0) + at * dim + (e - h * dim));
        const float s = reinterpret_cast<const float *>(blk + (isv ? g.vs_off : g.ks_off))[at];
        float4a o;
#pragma unroll
        for (int b = 0; b < 4; ++b) o[b] = place.p < 0 ? 0.0f : float(int32_t(c << (24 - 8 * b)) >> 24) * s;
        float *out = (isv ? v : k) + i * size_t(g.KVH) * dim + e;
        __builtin_nontemporal_store(float4u(o), reinterpret_cast<float4u *>(out));
    }
}

void freqs(const nd_rope *r, double *f)
{
    for (int j = 0; j < r->rot_dim / 2; ++j) {
        f[j] = std::pow(r->theta, -2.0 * j / r->rot_dim);
        if (r->scaling == ND_ROPE_LINEAR) {
            f[j] /= r->factor;
        } else if (r->scaling == ND_ROPE_PARTS) {
            const double turns = r->trained * f[j] / 6.283185307179586;
            const double g = std::fmin(std::fmax((turns - r->turns_lo) / (r->turns_hi - r->turns_lo), 0.0), 1.0);
            f[j] *= g + (1.0 - g) / r->factor;
        }
    }
}

// Checks a rope and fills the kernels' form of it.
int make_turn(const nd_rope *r, Turn &t)
{
    ND_REQUIRE(r, "null rope");
    ND_REQUIRE(r->layout == ND_ROPE_HALVES || r->layout == ND_ROPE_PAIRS, "rope layout %d unknown", r->layout);
    ND_REQUIRE(r->scaling >= ND_ROPE_PLAIN && r->scaling <= ND_ROPE_PARTS, "rope scaling %d unknown", r->scaling);
    ND_REQUIRE(r->rot_dim >= 2 && r->rot_dim % 2 == 0 && r->rot_dim <= kMaxDim,
               "rot_dim %d must be even and in 2..%d", r->rot_dim, kMaxDim);
    ND_REQUIRE(std::isfinite(r->theta) && r->theta > 0, "theta must be positive");
    ND_REQUIRE(std::isfinite(r->gain), "gain must be finite");
    if (r->scaling != ND_ROPE_PLAIN)
        ND_REQUIRE(std::isfinite(r->factor) && r->factor > 0, "factor must be positive");
    if (r->scaling == ND_ROPE_PARTS) {
        ND_REQUIRE(std::isfinite(r->trained) && r->trained > 0, "trained must be positive");
        ND_REQUIRE(r->turns_lo >= 0 && std::isfinite(r->turns_hi) && r->turns_hi > r->turns_lo,
                   "0 <= turns_lo < turns_hi is required");
    }
    t.layout = r->layout;
    t.rot = r->rot_dim;
    t.gain = r->gain;
    freqs(r, t.f);
    // (the angles' reduction: 2^31 positions of 2^10 are below 2^42)
    for (int j = 0; j < t.rot / 2; ++j)
        ND_REQUIRE(t.f[j] <= 1024.0, "frequency %d, %g a position, is above 1024", j, t.f[j]);
    return ND_OK;
}

// Whether writing row i at y + i*ys (w elements) can touch a row of x, other
// than the row itself where both are one buffer of rows.
bool clash(const float *x, size_t xs, const float *y, size_t ys, size_t wx, size_t wy, size_t rows)
{
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
    const uintptr_t ae = a + ((rows - 1) * xs + wx) * 4, be = b + ((rows - 1) * ys + wy) * 4;
    if (ae <= b || be <= a) return false;
    if (rows > 1 && xs != ys) return true;
    // rows side by side in rows of one buffer
    const uintptr_t d = a < b ? b - a : a - b, first = (a < b ? wx : wy) * 4, second = (a < b ? wy : wx) * 4;
    return !(d >= first && (rows == 1 || d + second <= xs * 4));
}

// Rows a block, so that there are `want` blocks or more of it, at most `most`.
size_t rows_a_block(size_t rows, size_t want, size_t most) { return std::min(std::max<size_t>(rows / want, 1), most); }

// Launches of at most 2^23 blocks of rpb rows (HIP counts a launch's threads in 32
// bits): f(first row, blocks) for each.
template <typename F>
void launches(size_t rows, size_t rpb, F f)
{
    const size_t most = (size_t(1) << 23) * rpb;
    for (size_t i = 0; i < rows; i += most) f(i, dim3(unsigned((std::min(most, rows - i) + rpb - 1) / rpb)));
}

template <int G>
void launch_heads(nd_ctx *ctx, const Turn &turn, Rows a, const Geom &g, bool four)
{
    // four rows a block give each lane a few heads and leave blocks for all CUs (us,
    // 8000 rows of 12 + 24 heads with their read-back: 2 / 4 / 8 rows 43.6 / 41.5 /
    // 46.9; 6001 rows of 12 heads 9.5 / 8.8 / 8.9)
    const size_t rpb = rows_a_block(a.rows, 1024, 4);
    // as many groups as give each the same number of heads (36 heads: 12 groups)
    const int most = kThreads / G, heads = a.nq + (a.kv ? 2 * g.KVH : 0), turns = (heads + most - 1) / most;
    const int threads = ((heads + turns - 1) / turns * G + 63) / 64 * 64;
    TurnOf<2 * G> t;
    t.layout = turn.layout;
    t.rot = turn.rot;
    t.gain = turn.gain;
    std::copy(turn.f, turn.f + turn.rot / 2, t.f);
    auto *fn = four ? turn_kernel<G, true> : turn_kernel<G, false>;
    launches(a.rows, rpb, [&](size_t first, dim3 grid) {
        a.first = first;
        hipLaunchKernelGGL(fn, grid, dim3(threads), rpb * (turn.rot / 2) * sizeof(double2), ctx->stream, t, a, g,
                           int(rpb));
    });
}

int launch_turn(nd_ctx *ctx, const Turn &turn, const Rows &a, const Geom &g, const char *what)
{
    const int longest = a.kv ? std::max(g.QK, g.VD) : a.dim;
    const bool four = a.dim % 4 == 0 && (turn.layout == ND_ROPE_PAIRS ? turn.rot % 4 == 0 : turn.rot % 8 == 0);
    if (longest <= 64)
        launch_heads<16>(ctx, turn, a, g, four);
    else if (longest <= 128)
        launch_heads<32>(ctx, turn, a, g, four);
    else
        launch_heads<64>(ctx, turn, a, g, four);
    return nd::check_launch(what);
}

}  // namespace

extern "C" {

int nd_rope_freqs(const nd_rope *r, double *freq)
{
    nd::clear_error();
    Turn t;
    if (int rc = make_turn(r, t)) return rc;
    ND_REQUIRE(freq, "null buffer");
    std::copy(t.f, t.f + t.rot / 2, freq);
    return ND_OK;
}

int nd_rope_rows(nd_ctx *ctx, const nd_rope *r, size_t rows, const int32_t *pos, size_t heads,
                 size_t dim, const float *x, size_t x_stride, float *y, size_t y_stride)
{
    ND_ENTER(ctx);
    Turn turn;
    if (int rc = make_turn(r, turn)) return rc;
    ND_REQUIRE(heads > 0 && heads <= 65536, "heads %zu must be in 1..65536", heads);
    ND_REQUIRE(dim >= size_t(r->rot_dim) && dim <= kMaxDim, "dim %zu must be in rot_dim %d..%d", dim,
               r->rot_dim, kMaxDim);
    if (rows == 0) return ND_OK;
    ND_REQUIRE(x && y && pos, "null buffer");
    ND_REQUIRE(rows <= 0x7fffffff, "too many rows");
    const size_t w = heads * dim;
    ND_REQUIRE(rows == 1 || (x_stride >= w && y_stride >= w), "row strides %zu, %zu below a row's %zu elements",
               x_stride, y_stride, w);
    ND_REQUIRE((x == y && (rows == 1 || x_stride == y_stride)) || !clash(x, x_stride, y, y_stride, w, w, rows),
               "y overlaps x");
    Rows a{};
    a.rows = rows;
    a.per_block = 1;
    a.pos = pos;
    a.q = x;
    a.q_out = y;
    a.q_stride = x_stride;
    a.q_out_stride = y_stride;
    a.nq = int(heads);
    a.dim = int(dim);
    return launch_turn(ctx, turn, a, Geom{}, "rope_rows");
}

int nd_kv_write_rope(nd_ctx *ctx, const nd_kv_geom *g, const nd_rope *r, void *kv, size_t kv_stride,
                     size_t count, size_t per_block, const int32_t *pos, const int32_t *rot_pos,
                     const float *q, size_t q_stride, float *q_out, size_t q_out_stride,
                     const float *k, size_t k_stride, const float *v, size_t v_stride)
{
    ND_ENTER(ctx);
    if (int rc = check_geom(g)) return rc;
    Turn turn;
    if (int rc = make_turn(r, turn)) return rc;
    ND_REQUIRE(r->rot_dim <= g->qk_head_dim, "rot_dim %d above qk_head_dim %d", r->rot_dim, g->qk_head_dim);
    ND_REQUIRE(per_block > 0, "per_block must be positive");
    ND_REQUIRE(g->num_heads <= 65536, "num_heads %d above 65536", g->num_heads);
    if (count == 0) return ND_OK;
    ND_REQUIRE(kv && pos && k && v, "null buffer");
    ND_REQUIRE(!q == !q_out, "q and q_out are given together or not at all");
    ND_REQUIRE(count <= 0x7fffffff, "count too large");
    ND_REQUIRE((reinterpret_cast<uintptr_t>(kv) & 255) == 0 && kv_stride % 256 == 0,
               "kv blocks must be 256-byte aligned");
    const size_t wq = size_t(g->num_heads) * g->qk_head_dim, wk = size_t(g->num_kv_heads) * g->qk_head_dim,
                 wv = size_t(g->num_kv_heads) * g->v_head_dim;
    ND_REQUIRE(count == 1 || (k_stride >= wk && v_stride >= wv && (!q || (q_stride >= wq && q_out_stride >= wq))),
               "row strides below a row's elements");
    if (q) {
        ND_REQUIRE((q == q_out && (count == 1 || q_stride == q_out_stride)) ||
                       !clash(q, q_stride, q_out, q_out_stride, wq, wq, count),
                   "q_out overlaps q");
        ND_REQUIRE(!clash(k, k_stride, q_out, q_out_stride, wk, wq, count) &&
                       !clash(v, v_stride, q_out, q_out_stride, wv, wq, count),
                   "q_out overlaps k or v");
    }
    Rows a{};
    a.rows = count;
    a.per_block = per_block;
    a.pos = pos;
    a.rot_pos = rot_pos;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.q_stride = q_stride;
    a.q_out_stride = q_out_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.kv_stride = kv_stride;
    a.kv = static_cast<uint8_t *>(kv);
    a.nq = q ? g->num_heads : 0;
    a.dim = g->qk_head_dim;
    return launch_turn(ctx, turn, a, make_geom(g), "kv_write_rope");
}

int nd_kv_read(nd_ctx *ctx, const nd_kv_geom *g, const void *kv, size_t kv_stride, size_t count,
               size_t per_block, const int32_t *pos, float *k, float *v)
{
    ND_ENTER(ctx);
    if (int rc = check_geom(g)) return rc;
    ND_REQUIRE(per_block > 0, "per_block must be positive");
    ND_REQUIRE(g->num_kv_heads <= 65536, "num_kv_heads %d above 65536", g->num_kv_heads);
    if (count == 0 || (!k && !v)) return ND_OK;
    ND_REQUIRE(kv && pos, "null buffer");
    ND_REQUIRE(count <= 0x7fffffff, "count too large");
    ND_REQUIRE((reinterpret_cast<uintptr_t>(kv) & 255) == 0 && kv_stride % 256 == 0,
               "kv blocks must be 256-byte aligned");
    const size_t rpb = rows_a_block(count, 2048, kMaxRows);
    auto up = [](int d) { return uint32_t(((uint64_t(1) << 32) + d - 1) / d); };
    const Geom kg = make_geom(g);
    launches(count, rpb, [&](size_t first, dim3 grid) {
        hipLaunchKernelGGL(read_kernel, grid, dim3(kThreads), 0, ctx->stream, kg, static_cast<const uint8_t *>(kv),
                           kv_stride, count, first, per_block, pos, k, v, int(rpb), up(g->qk_head_dim / 4),
                           up(g->v_head_dim / 4));
    });
    return nd::check_launch("kv_read");
}

}  // extern "C"
