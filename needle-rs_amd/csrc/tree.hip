// Attention of drafted trees over the int8 cache: every node of a session's
// tree attends to a window of the committed positions and to the nodes its
// mask names, whose keys and values lie in the same ring behind them.
//
// A block a (node, query head): each thread walks its own positions with a
// running maximum and sum (scores in bits: e^s = 2^(s log2 e)), and the
// threads' sums meet at the end.
#include "nd_internal.h"
#include "nd_kv_internal.h"

namespace {

using namespace ndkv;

constexpr int kThreads = 256;
constexpr int kMaxNodes = 256;

struct Tree {
    const uint8_t *kv;
    size_t kv_stride;
    const int32_t *base, *length, *lo;
    const uint32_t *mask;
    const float *q;
    float *out;
    int nodes, words;
    float scale2;  // scale log2(e)
};

template <int QK, bool QQ>
__global__ __launch_bounds__(kThreads) void tree_kernel(Geom g, Tree tr)
{
    constexpr int VD = 64, NW = kThreads / 64;
    __shared__ float qs[QK];
    __shared__ float mo[NW][VD], mm[NW], ml[NW];
    const int head = blockIdx.x % g.H, node = blockIdx.x / g.H;
    const size_t ses = blockIdx.y;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int len = tr.length ? tr.length[ses] : tr.nodes;
    float *out = tr.out + ((ses * tr.nodes + node) * g.H + head) * VD;
    const size_t row = ses * tr.nodes + node;
    const int base = tr.base[ses], lo = tr.lo[row];
    const bool wrong = len < 0 || len > tr.nodes;
    if (!wrong && node >= len) return;
    const int first = min(lo, base);
    if (wrong || base < 0 || lo < 0 || base > 0x7fffffff - kMaxNodes || base - first + len > g.cap) {
        if (t < VD) out[t] = NAN;
        return;
    }
    const int kvh = head / (g.H / g.KVH);
    const uint8_t *blk = tr.kv + ses * tr.kv_stride;
    const int8_t *kb = reinterpret_cast<const int8_t *>(blk) + size_t(kvh) * g.cap * QK;
    const int8_t *vb = reinterpret_cast<const int8_t *>(blk + g.v_off) + size_t(kvh) * g.cap * VD;
    const float *ksb = reinterpret_cast<const float *>(blk + g.ks_off) + size_t(kvh) * g.cap;
    const float *vsb = reinterpret_cast<const float *>(blk + g.vs_off) + size_t(kvh) * g.cap;
    const float *q = tr.q + (row * g.H + head) * QK;
    for (int e = t; e < QK; e += kThreads) qs[e] = q[e];
    __syncthreads();
    if (QQ) {
        if (w == 0) {
            float sc, inv;
            quant_scale_wave(qs, QK, sc, inv);
            for (int e = lane; e < QK; e += 64) qs[e] = quant_code(qs[e], inv) * sc;
        }
        __syncthreads();
    }
    const uint32_t *bits = tr.mask + row * tr.words;
    float m = -INFINITY, l = 0.0f, acc[VD];
#pragma unroll
    for (int e = 0; e < VD; ++e) acc[e] = 0.0f;
    const int before = base - first;
    for (int i = t; i < before + len; i += kThreads) {
        const int j = i - before;
        if (j >= 0 && !(bits[j >> 5] >> (j & 31) & 1)) continue;
        const int slot = int((uint32_t(first) + uint32_t(i)) % uint32_t(g.cap));
        float s = 0.0f;
        const int8_t *k = kb + size_t(slot) * QK, *v = vb + size_t(slot) * VD;
        for (int e = 0; e < QK; ++e) s += qs[e] * float(k[e]);
        s = s * ksb[slot] * tr.scale2;
        const float mn = fmaxf(m, s);
        const float al = m == mn ? 1.0f : exp2f(m - mn), p = exp2f(s - mn), wt = p * vsb[slot];
        l = l * al + p;
#pragma unroll
        for (int e = 0; e < VD; ++e) acc[e] = acc[e] * al + wt * float(v[e]);
        m = mn;
    }
    const float M = wave_max(m);
    const float f = m == -INFINITY ? (l != l ? NAN : 0.0f) : exp2f(m - M);
    l = wave_sum(l * f);
#pragma unroll
    for (int e = 0; e < VD; ++e) {
        const float o = wave_sum(m == -INFINITY ? 0.0f : acc[e] * f);
        if (lane == 0) mo[w][e] = o;
    }
    if (lane == 0) mm[w] = M, ml[w] = l;
    __syncthreads();
    if (t < VD) {
        float MM = -INFINITY, O = 0.0f, L = 0.0f;
        for (int i = 0; i < NW; ++i) MM = fmaxf(MM, mm[i]);
        for (int i = 0; i < NW; ++i) {
            const float fi = mm[i] == -INFINITY ? 0.0f : exp2f(mm[i] - MM);
            O += mo[i][t] * fi;
            L += ml[i] * (ml[i] != ml[i] ? 1.0f : fi);
        }
        out[t] = L == 0.0f ? 0.0f : O / L;
    }
}

}  // namespace

extern "C" {

size_t nd_attend_tree_i8_work(nd_ctx *, const nd_kv_geom *, size_t, size_t) { return 0; }

int nd_attend_tree_i8(nd_ctx *ctx, const nd_kv_geom *g, const void *kv, size_t kv_stride,
                      size_t count, size_t nodes, const int32_t *base, const int32_t *length,
                      const int32_t *lo, const uint32_t *mask, const float *q, float scale,
                      int quant_query, float *out, void *work, size_t work_bytes)
{
    ND_ENTER(ctx);
    if (int rc = check_geom(g)) return rc;
    ND_REQUIRE((g->qk_head_dim == 48 || g->qk_head_dim == 64) && g->v_head_dim == 64,
               "no tree attention for qk %d, v %d", g->qk_head_dim, g->v_head_dim);
    ND_REQUIRE(nodes >= 1 && nodes <= kMaxNodes, "nodes %zu must be in 1..%d", nodes, kMaxNodes);
    if (count == 0) return ND_OK;
    ND_REQUIRE(kv && base && lo && mask && q && out, "null buffer");
    ND_REQUIRE(count <= 65535, "count %zu above 65535", count);
    ND_REQUIRE(g->num_heads <= 4096, "num_heads %d above 4096", g->num_heads);
    ND_REQUIRE((reinterpret_cast<uintptr_t>(kv) & 255) == 0 && kv_stride % 256 == 0,
               "kv blocks must be 256-byte aligned");
    Tree t{};
    t.kv = static_cast<const uint8_t *>(kv);
    t.kv_stride = kv_stride;
    t.base = base;
    t.length = length;
    t.lo = lo;
    t.mask = mask;
    t.q = q;
    t.out = out;
    t.nodes = int(nodes);
    t.words = int((nodes + 31) / 32);
    t.scale2 = float(double(scale) * 1.4426950408889634);
    const dim3 grid(unsigned(nodes * g->num_heads), unsigned(count));
    const bool q48 = g->qk_head_dim == 48;
    auto *fn = q48 ? (quant_query ? tree_kernel<48, true> : tree_kernel<48, false>)
                   : (quant_query ? tree_kernel<64, true> : tree_kernel<64, false>);
    hipLaunchKernelGGL(fn, grid, dim3(kThreads), 0, ctx->stream, make_geom(g), t);
    return nd::check_launch("attend_tree_i8");
}

}  // extern "C"
