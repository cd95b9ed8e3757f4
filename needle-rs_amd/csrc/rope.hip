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
// All three calls are bound by memory: a value is read and written once.
#include "nd_internal.h"
#include "nd_kv_internal.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace ndkv;

constexpr int kThreads = 256;
constexpr int kMaxPairs = kMaxDim / 2;

struct Turn {
    int layout, rot;
    double gain;
    double f[kMaxPairs];
};

// What a rope or write launch works on: rows of q heads (nq), k heads (nk)
// and v heads (nk), any of them absent.
struct Rows {
    size_t rows, per_block;
    const int32_t *pos, *rot_pos;
    const float *q, *k, *v;
    float *q_out;
    size_t q_stride, q_out_stride, k_stride, v_stride, kv_stride;
    uint8_t *kv;
    int nq, dim;
};

typedef float float4a __attribute__((ext_vector_type(4)));
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));  // rows may start anywhere
typedef float float2u __attribute__((ext_vector_type(2), aligned(4)));

// G lanes a head vector, four elements a lane: element 4 l + e of the head.  FOUR:
// every head is a multiple of 4 long, and with halves rot / 2 is too, so that a
// lane's partners are four neighbours.
template <int G, bool FOUR>
__global__ __launch_bounds__(kThreads) void turn_kernel(Turn tn, Rows r, Geom g, int rpb)
{
    extern __shared__ double2 cs[];  // [rpb][rot / 2]: gain cos, gain sin
    constexpr int GROUPS = kThreads / G;
    const int t = threadIdx.x, l = t % G;
    const int half = tn.rot / 2;
    const bool pairs = tn.layout == ND_ROPE_PAIRS;
    const int heads = r.nq + (r.kv ? 2 * g.KVH : 0);
    auto head = [&](size_t i0, int row, int h) {
        const size_t i = i0 + row;
        const int p = r.pos[i];
        const bool isq = h < r.nq, isv = h >= r.nq + g.KVH;
        const int hk = h - r.nq - (isv ? g.KVH : 0);
        const int dim = isq ? r.dim : isv ? g.VD : g.QK;
        const float *x = isq ? r.q + i * r.q_stride + size_t(h) * dim
                         : isv ? r.v + i * r.v_stride + size_t(hk) * dim
                               : r.k + i * r.k_stride + size_t(hk) * dim;
        const int e0 = 4 * l;
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (FOUR ? e0 < dim : e0 + 4 <= dim) {
            const float4u q = *reinterpret_cast<const float4u *>(x + e0);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = q[e];
        } else if (!FOUR) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = e0 + e < dim ? x[e0 + e] : 0.0f;
        }
        if (!isv && e0 < tn.rot) {
            const double2 *a = cs + row * half;
            if (pairs) {
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    if (e0 + e >= tn.rot) continue;
                    const double2 z = a[(e0 + e) / 2];
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
                    const double2 z = a[j + e];
                    y[e] = float(double(y[e]) * z.x + double(o[e]) * (second ? z.y : -z.y));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (e0 + e >= tn.rot) continue;
                    const bool second = e0 + e >= half;
                    const int j = second ? e0 + e - half : e0 + e;
                    const double2 z = a[j];
                    y[e] = float(double(y[e]) * z.x + double(x[second ? j : j + half]) * (second ? z.y : -z.y));
                }
            }
        }
        if (p < 0) return;  // left out; what was read is memory all the same
        if (isq) {
            float *out = r.q_out + i * r.q_out_stride + size_t(h) * dim;
            if (FOUR ? e0 < dim : e0 + 4 <= dim) {
                *reinterpret_cast<float4u *>(out + e0) = float4u{y[0], y[1], y[2], y[3]};
            } else if (!FOUR) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e0 + e < dim) out[e0 + e] = y[e];
            }
        } else {
            // quant_into (cache.rs:80-104): heads are multiples of 16 long
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
            const float scale = m > 0.0f ? m / 127.0f : 1.0f;
            const float inv = 1.0f / scale;
            uint32_t codes = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                codes |= (uint32_t(int32_t(int8_t(quant_code(y[e], inv)))) & 0xffu) << (8 * e);
            uint8_t *blk = r.kv + (i / r.per_block) * r.kv_stride;
            const size_t at = size_t(hk) * g.cap + p % g.cap;
            if (e0 < dim)
                *reinterpret_cast<uint32_t *>(blk + (isv ? g.v_off : 0) + at * dim + e0) = codes;
            if (l == 0) reinterpret_cast<float *>(blk + (isv ? g.vs_off : g.ks_off))[at] = scale;
        }
    };
    for (size_t i0 = size_t(blockIdx.x) * rpb; i0 < r.rows; i0 += size_t(gridDim.x) * rpb) {
        const int rows = int(min(size_t(rpb), r.rows - i0));
        if (i0 >= size_t(gridDim.x) * rpb) __syncthreads();
        for (int j = t; j < rows * half; j += kThreads) {
            const int row = j / half;
            const int p = r.rot_pos ? r.rot_pos[i0 + row] : r.pos[i0 + row];
            double sn, c;
            sincos(double(p) * tn.f[j - row * half], &sn, &c);
            cs[j] = double2{tn.gain * c, tn.gain * sn};
        }
        __syncthreads();
        int row = 0, h = t / G;
        while (h >= heads && row < rows) h -= heads, ++row;
        while (row < rows) {
            head(i0, row, h);
            h += GROUPS;
            while (h >= heads && row < rows) h -= heads, ++row;
        }
    }
}

// Sixteen bytes of a result a lane: four codes of a head vector and its scale.
// Item j of a row is dword j of its K heads, then of its V heads.
__global__ __launch_bounds__(kThreads) void read_kernel(Geom g, const uint8_t *__restrict__ kv,
                                                        size_t kv_stride, size_t rows, size_t per_block,
                                                        const int32_t *__restrict__ pos,
                                                        float *__restrict__ k, float *__restrict__ v, int rpb)
{
    const int wk = k ? g.KVH * g.QK / 4 : 0, wv = v ? g.KVH * g.VD / 4 : 0, items = wk + wv;
    for (size_t i0 = size_t(blockIdx.x) * rpb; i0 < rows; i0 += size_t(gridDim.x) * rpb) {
        const int n = int(min(size_t(rpb), rows - i0));
        for (int row = 0, j = threadIdx.x;; j += kThreads) {
            while (j >= items) j -= items, ++row;
            if (row >= n) break;
            const size_t i = i0 + row;
            const bool isv = j >= wk;
            const int dim = isv ? g.VD : g.QK, e = 4 * (isv ? j - wk : j), h = e / dim;
            const int p = pos[i];
            const uint8_t *blk = kv + (i / per_block) * kv_stride;
            const size_t at = size_t(h) * g.cap + (p < 0 ? 0 : p % g.cap);
            const uint32_t c = *reinterpret_cast<const uint32_t *>(blk + (isv ? g.v_off : 0) + at * dim + (e - h * dim));
            const float s = reinterpret_cast<const float *>(blk + (isv ? g.vs_off : g.ks_off))[at];
            float4a o;
#pragma unroll
            for (int b = 0; b < 4; ++b) o[b] = p < 0 ? 0.0f : float(int32_t(c << (24 - 8 * b)) >> 24) * s;
            float *out = (isv ? v : k) + i * size_t(g.KVH) * dim + e;
            *reinterpret_cast<float4u *>(out) = o;
        }
    }
}

int check_rope(const nd_rope *r)
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
    return ND_OK;
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

Turn make_turn(const nd_rope *r)
{
    Turn t{};
    t.layout = r->layout;
    t.rot = r->rot_dim;
    t.gain = r->gain;
    freqs(r, t.f);
    return t;
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

// Blocks of them: the kernels go round where there are more than a launch holds
// (HIP counts its threads in 32 bits).
dim3 row_blocks(size_t rows, size_t rpb) { return dim3(unsigned(std::min<size_t>((rows + rpb - 1) / rpb, size_t(1) << 23))); }

int launch_turn(nd_ctx *ctx, const nd_rope *r, const Rows &a, const Geom &g, const char *what)
{
    const int longest = a.kv ? std::max(g.QK, g.VD) : a.dim, half = r->rot_dim / 2;
    const bool four = a.dim % 4 == 0 && (r->layout == ND_ROPE_PAIRS ? r->rot_dim % 4 == 0 : half % 4 == 0);
    const size_t rpb = rows_a_block(a.rows, 2048, 8);
    const size_t lds = rpb * half * sizeof(double2);
    auto *fn = longest <= 64    ? (four ? turn_kernel<16, true> : turn_kernel<16, false>)
               : longest <= 128 ? (four ? turn_kernel<32, true> : turn_kernel<32, false>)
                                : (four ? turn_kernel<64, true> : turn_kernel<64, false>);
    hipLaunchKernelGGL(fn, row_blocks(a.rows, rpb), dim3(kThreads), lds, ctx->stream, make_turn(r), a, g, int(rpb));
    return nd::check_launch(what);
}

}  // namespace

extern "C" {

int nd_rope_freqs(const nd_rope *r, double *freq)
{
    nd::clear_error();
    if (int rc = check_rope(r)) return rc;
    ND_REQUIRE(freq, "null buffer");
    freqs(r, freq);
    return ND_OK;
}

int nd_rope_rows(nd_ctx *ctx, const nd_rope *r, size_t rows, const int32_t *pos, size_t heads,
                 size_t dim, const float *x, size_t x_stride, float *y, size_t y_stride)
{
    ND_ENTER(ctx);
    if (int rc = check_rope(r)) return rc;
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
    return launch_turn(ctx, r, a, Geom{}, "rope_rows");
}

int nd_kv_write_rope(nd_ctx *ctx, const nd_kv_geom *g, const nd_rope *r, void *kv, size_t kv_stride,
                     size_t count, size_t per_block, const int32_t *pos, const int32_t *rot_pos,
                     const float *q, size_t q_stride, float *q_out, size_t q_out_stride,
                     const float *k, size_t k_stride, const float *v, size_t v_stride)
{
    ND_ENTER(ctx);
    if (int rc = check_geom(g)) return rc;
    if (int rc = check_rope(r)) return rc;
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
    return launch_turn(ctx, r, a, make_geom(g), "kv_write_rope");
}

int nd_kv_read(nd_ctx *ctx, const nd_kv_geom *g, const void *kv, size_t kv_stride, size_t count,
               size_t per_block, const int32_t *pos, float *k, float *v)
{
    ND_ENTER(ctx);
    if (int rc = check_geom(g)) return rc;
    ND_REQUIRE(per_block > 0, "per_block must be positive");
    if (count == 0 || (!k && !v)) return ND_OK;
    ND_REQUIRE(kv && pos, "null buffer");
    ND_REQUIRE(count <= 0x7fffffff, "count too large");
    ND_REQUIRE((reinterpret_cast<uintptr_t>(kv) & 255) == 0 && kv_stride % 256 == 0,
               "kv blocks must be 256-byte aligned");
    const size_t rpb = rows_a_block(count, 2048, 16);
    hipLaunchKernelGGL(read_kernel, row_blocks(count, rpb), dim3(kThreads), 0, ctx->stream,
                       make_geom(g), static_cast<const uint8_t *>(kv), kv_stride, count, per_block, pos, k, v,
                       int(rpb));
    return nd::check_launch("kv_read");
}

}  // extern "C"
