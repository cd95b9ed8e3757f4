// Rotary positions, alone and on the way into the int8 cache, and the cache
// read back.
//
// A turn is y = (u cos a - w sin a, u sin a + w cos a) for a pair (u, w) and
// the angle a = pos f.  Angle, sine, cosine and products are fp64: at position
// 10^6 an fp32 angle is off by 0.03, and where the result is quantised a code
// next to a border should not depend on how the products were rounded.  Each
// (row, pair) is worked out once a block, in LDS, for all heads of the row.
// All three calls are bound by memory: a value is read and written once.
#include "nd_internal.h"
#include "nd_kv_internal.h"

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

// A block per row, a wave per head vector in turn.
__global__ __launch_bounds__(kThreads) void turn_kernel(Turn tn, Rows r, Geom g)
{
    __shared__ double cs[kMaxPairs], sn[kMaxPairs];
    __shared__ float buf[kThreads / 64][kMaxDim];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int half = tn.rot / 2;
    const int heads = r.nq + (r.kv ? 2 * g.KVH : 0);
    for (size_t i = blockIdx.x; i < r.rows; i += gridDim.x) {
        const int p = r.pos[i];
        if (p < 0) continue;  // the same for the whole block
        const double at = r.rot_pos ? double(r.rot_pos[i]) : double(p);
        __syncthreads();
        for (int j = threadIdx.x; j < half; j += kThreads) {
            double s, c;
            sincos(at * tn.f[j], &s, &c);
            cs[j] = tn.gain * c;
            sn[j] = tn.gain * s;
        }
        __syncthreads();
        for (int h = w; h < heads; h += kThreads / 64) {
            const bool isq = h < r.nq, isv = h >= r.nq + g.KVH;
            const int hk = h - r.nq - (isv ? g.KVH : 0);
            const int dim = isq ? r.dim : isv ? g.VD : g.QK;
            const float *x = isq ? r.q + i * r.q_stride + size_t(h) * dim
                             : isv ? r.v + i * r.v_stride + size_t(hk) * dim
                                   : r.k + i * r.k_stride + size_t(hk) * dim;
            for (int e = lane; e < dim; e += 64) {
                float y = x[e];
                if (!isv && e < tn.rot) {
                    const bool second = tn.layout == ND_ROPE_PAIRS ? e & 1 : e >= half;
                    const int j = tn.layout == ND_ROPE_PAIRS ? e / 2 : second ? e - half : e;
                    const int other = tn.layout == ND_ROPE_PAIRS ? e ^ 1 : second ? e - half : e + half;
                    const double u = y, o = x[other];
                    y = float(second ? o * sn[j] + u * cs[j] : u * cs[j] - o * sn[j]);
                }
                buf[w][e] = y;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (isq) {
                float *y = r.q_out + i * r.q_out_stride + size_t(h) * dim;
                for (int e = lane; e < dim; e += 64) y[e] = buf[w][e];
            } else {
                uint8_t *blk = r.kv + (i / r.per_block) * r.kv_stride;
                const size_t at_slot = size_t(hk) * g.cap + p % g.cap;
                int8_t *dst = reinterpret_cast<int8_t *>(blk + (isv ? g.v_off : 0)) + at_slot * dim;
                float scale, inv;
                quant_scale_wave(buf[w], dim, scale, inv);
                for (int e = lane; e < dim; e += 64) dst[e] = int8_t(quant_code(buf[w][e], inv));
                if (lane == 0) reinterpret_cast<float *>(blk + (isv ? g.vs_off : g.ks_off))[at_slot] = scale;
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// A wave per (row, head) of k or v.
__global__ __launch_bounds__(kThreads) void read_kernel(Geom g, const uint8_t *__restrict__ kv,
                                                        size_t kv_stride, size_t rows, size_t per_block,
                                                        const int32_t *__restrict__ pos,
                                                        float *__restrict__ k, float *__restrict__ v)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const size_t units = rows * size_t(g.KVH) * 2;
    for (size_t u = size_t(blockIdx.x) * (kThreads / 64) + w; u < units; u += size_t(gridDim.x) * (kThreads / 64)) {
        const bool isv = u & 1;
        const size_t i = u / 2 / g.KVH;
        const int h = int(u / 2 % g.KVH), dim = isv ? g.VD : g.QK;
        float *out = isv ? v : k;
        if (!out) continue;
        out += (i * g.KVH + h) * dim;
        const int p = pos[i];
        const uint8_t *blk = kv + (i / per_block) * kv_stride;
        const size_t at = size_t(h) * g.cap + (p < 0 ? 0 : p % g.cap);
        const int8_t *src = reinterpret_cast<const int8_t *>(blk + (isv ? g.v_off : 0)) + at * dim;
        const float s = reinterpret_cast<const float *>(blk + (isv ? g.vs_off : g.ks_off))[at];
        for (int e = lane; e < dim; e += 64) out[e] = p < 0 ? 0.0f : float(src[e]) * s;
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

unsigned row_blocks(size_t rows) { return unsigned(rows < (size_t(1) << 20) ? rows : size_t(1) << 20); }

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
    hipLaunchKernelGGL(turn_kernel, dim3(row_blocks(rows)), dim3(kThreads), 0, ctx->stream, make_turn(r), a, Geom{});
    return nd::check_launch("rope_rows");
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
    hipLaunchKernelGGL(turn_kernel, dim3(row_blocks(count)), dim3(kThreads), 0, ctx->stream, make_turn(r), a,
                       make_geom(g));
    return nd::check_launch("kv_write_rope");
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
    hipLaunchKernelGGL(read_kernel, dim3(row_blocks(count * g->num_kv_heads)), dim3(kThreads), 0, ctx->stream,
                       make_geom(g), static_cast<const uint8_t *>(kv), kv_stride, count, per_block, pos, k, v);
    return nd::check_launch("kv_read");
}

}  // extern "C"
