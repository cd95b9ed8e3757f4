// Attention of drafted trees over the int8 cache: every node of a session's
// tree attends to a window of the committed positions and to the nodes its
// mask names, whose keys and values lie in the same ring behind them.
//
// On the matrix cores.  The columns of a (session, kv head) are its (node,
// query head) pairs: a wave owns 16 of them and walks chunks of 32
// positions with an online softmax; the waves of a block own the same columns
// and take the chunks in turn, and meet in LDS at the end.  The committed
// positions and the tree are chunked apart, so that a chunk of the tree is a
// word of the mask.
//   scores  S[pos][col] = K Q^T, v_mfma 16x16, A = 16 positions' int8 rows.
//           With quant_query both sides are codes and the dot is an exact
//           integer; else the fp32 query is two f16 pieces of a head scaled by
//           a power of two (error 2^-23 of an element at most, either way, less
//           than fp32's own steps leave a sum of products).
//   softmax scores stay without the column's factor cf (scale, query scale):
//           the maximum m is kept before it and e = 2^(fma(t, cf, -m cf)).
//   values  O^T[v][col] = V^T P^T: a score tile's result layout is the layout
//           of the weights the product needs.  MFMA c takes V columns 4 n + c,
//           a dword a position.  The weights e vs are two f16 pieces, off by
//           2^-23 of the weight or of the column's largest so far (a maximum on
//           values next to zero is no measure of the rest: the sums then go on
//           against a lower one); V's codes are exact in f16.  A chunk with a V
//           scale 2^-9 or less of the largest met takes the fp32 matrix product
//           instead, all 24 bits at any size: the values of one position may be
//           far smaller than its neighbours' and yet decide the output.
// Sums and statistics are fp32.
//
// What bounds it: where the cache streams (one query head a kv head) HBM, 64
// sessions x 13 nodes x 12 heads x 64 at 2048 positions 39.3 us = 5.0 TB/s; with
// grouped heads the VALU, about 146 operations a chunk (the exponentials 32, V's
// conversion 40), 64 x 16 nodes x 12 heads over 2 at 2000 21.5 us; small trees the
// 7 us from launch to merge.  One column tile a wave at four waves a SIMD: two
// tiles, which share V's conversion but leave three waves, gain at 100 million
// scores (128 sessions x 4000 65.9 -> 57.4) and lose below (64 x 2000 23.9 -> 26.7,
// 12 kv heads 32.1 -> 44.0).
#include "nd_attn_pieces.h"
#include "nd_internal.h"
#include "nd_kv_internal.h"

#include <algorithm>
#include <type_traits>

namespace {

using namespace ndkv;
using namespace ndap;

constexpr int kMaxNodes = 256;
constexpr int VD = 64, kCols = 16;

struct Tree {
    const uint8_t *kv;
    size_t kv_stride;
    const int32_t *base, *length, *lo;
    const uint32_t *mask;
    const float *q;
    float *out, *part_o, *part_ml;
    int nodes, words, splits, rep;
    uint32_t units;
    Divisor by_splits, by_kvh;
    float scale2;  // |scale| log2(e); below 0 where scale is no number
    int negative;  // scale < 0
};

template <int QK, bool QQ, int NW>
__global__ __launch_bounds__(NW * 64, 4) void tree_kernel(Geom g, Tree tr)
{
    constexpr int SL = QK / 4, KD = SL / 4;  // a lane's slice of a K row; its dwords (3 or 4)
    constexpr int LD = VD + 4;
    __shared__ __align__(16) float sc_s[NW][64];
    __shared__ __align__(16) float mo[NW][kCols][LD];
    __shared__ floatx4_t ms[NW][kCols];  // maximum, more, weight

    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n = lane & 15, qd = lane >> 4;
    // blocks 8 apart share an XCD's L2: there a unit's column tiles follow each other
    const uint32_t unit = blockIdx.z * 8 + blockIdx.x, tile = blockIdx.y;
    if (unit >= tr.units) return;
    const uint32_t group = tr.by_splits.quotient(unit), split = unit - group * tr.splits;
    const uint32_t ses = tr.by_kvh.quotient(group), kvh = group - ses * uint32_t(g.KVH);
    const int R = tr.rep;

    // ---- the wave's columns: window and query operand, asked for before the
    // session's numbers are there (rows behind the tree's end are memory too).
    // f / R of a column f < 2^11: (f + 1/2) / R is 1/16 or more away from an
    // integer (R <= 8) ----
    const float inv_r = 1.0f / float(R);
    auto node_of = [&](int f) { return int((float(f) + 0.5f) * inv_r); };
    const int f = min(int(tile) * kCols + n, tr.nodes * R - 1);
    const int node = node_of(f), head = int(kvh) * R + f - node * R;
    const size_t row = size_t(ses) * tr.nodes + node;
    float v[SL];
    {
        const float *qh = tr.q + (row * g.H + head) * QK + qd * SL;
#pragma unroll
        for (int e = 0; e < SL; ++e) v[e] = qh[e];
    }
    const int l0 = tr.lo[row];
    const int base = tr.base[ses], len0 = tr.length ? tr.length[ses] : tr.nodes;
    const bool there = len0 >= 0 && len0 <= tr.nodes;
    const bool wrong = !there || base < 0 || base > 0x7fffffff - kMaxNodes;
    const int len = there ? len0 : tr.nodes;
    const int ncols = len * R;
    if (int(tile) * kCols >= ncols) return;
    const uint8_t *blk = tr.kv + size_t(ses) * tr.kv_stride;
    const rows_t kb = rows_at(blk + size_t(kvh) * g.cap * QK, uint32_t(g.cap) * QK);
    const rows_t vb = rows_at(blk + g.v_off + size_t(kvh) * g.cap * VD, uint32_t(g.cap) * VD);
    // K scales, and vs_off - ks_off bytes on (KVH cap 4, below 2^32) the V scales
    const uint32_t to_vs = uint32_t(g.vs_off - g.ks_off);
    const rows_t sb = rows_at(blk + g.ks_off + size_t(kvh) * g.cap * 4, to_vs + uint32_t(g.cap) * 4);
    const uint32_t cap = uint32_t(g.cap);

    const bool bad = wrong || l0 < 0 || base - min(l0, base) + len > g.cap;
    // these and columns past the end walk along whatever the others read
    const bool along = bad || int(tile) * kCols + n >= ncols;
    const uint32_t lo = along ? 0u : uint32_t(l0);  // first committed position
    // the first position that some column reads, and the first that all do
    uint32_t ulo = along ? uint32_t(base) : min(uint32_t(base), lo), tlo = lo;
    auto both = [&](auto distance) {
        constexpr int D = decltype(distance)::value;
        ulo = min(ulo, uint32_t(ndl::wave_xor_int<D>(int(ulo))));
        tlo = max(tlo, uint32_t(ndl::wave_xor_int<D>(int(tlo))));
    };
    both(std::integral_constant<int, 1>{});
    both(std::integral_constant<int, 2>{});
    both(std::integral_constant<int, 4>{});
    both(std::integral_constant<int, 8>{});
    ulo = __builtin_amdgcn_readfirstlane(ulo);
    tlo = __builtin_amdgcn_readfirstlane(tlo);

    // ---- the walk: committed positions up to the ring's end, from its start,
    // then the tree's nodes likewise, each in chunks of 32 (the last ones of a
    // part shorter).  A walk is no longer than the ring, so it wraps once ----
    const uint32_t before = uint32_t(base) - ulo, slo = ulo % cap;
    const uint32_t n0 = min(before, cap - slo), n1 = before - n0;
    const uint32_t s2 = slo + before >= cap ? slo + before - cap : slo + before;
    const uint32_t n2 = min(uint32_t(len), cap - s2), n3 = uint32_t(len) - n2;
    const int e0 = int((n0 + 31) / 32), e1 = e0 + int((n1 + 31) / 32), e2 = e1 + int((n2 + 31) / 32);
    // (a column past the end may be no bad one where all others are; its walk is empty)
    const int nch = any_of(!bad) ? e2 + int((n3 + 31) / 32) : 0;
    const int step = tr.splits * NW;
    int ch = int(split) * NW + w;
    uint32_t s0 = 0;   // the chunk's first slot,
    uint32_t p0 = 0;   // position or node,
    int left = 0;      // positions from there to the part's end; 0 behind the last chunk
    int stop = 0;      // the part's last chunk, and one
    bool tail = false;
    auto place = [=, &s0, &p0, &left, &stop, &tail](int i) {
        const uint32_t off = 32u * uint32_t(i >= e2 ? i - e2 : i >= e1 ? i - e1 : i >= e0 ? i - e0 : i);
        const uint32_t cnt = i >= e2 ? n3 : i >= e1 ? n2 : i >= e0 ? n1 : n0;
        tail = i >= e1;
        s0 = i >= nch ? 0u : (i >= e2 ? 0u : i >= e1 ? s2 : i >= e0 ? 0u : slo) + off;
        p0 = (i >= e2 ? n2 : i >= e1 ? 0u : i >= e0 ? ulo + n0 : ulo) + off;
        left = i >= nch ? 0 : int(cnt - off);
        stop = i >= e2 ? nch : i >= e1 ? e2 : i >= e0 ? e1 : e0;
    };
    uint32_t kr[2][KD], vr[8], word = 0;
    float scr = 0.0f;
    const uint32_t kl = uint32_t(n * QK + qd * SL), vl = uint32_t(4 * qd * VD + 4 * n);
    const uint32_t scl = (lane & 31) * 4 + (lane < 32 ? 0u : to_vs);
    // loads of K and V are never conditional: past the last chunk they read some slot
    auto load_k = [&]() {
        if (tail && left > 0) {
            // bits p0 .. p0 + 31 of the node's mask
            const int at = node_of(min(int(tile) * kCols + n, ncols - 1));
            const uint32_t *m = tr.mask + (size_t(ses) * tr.nodes + at) * tr.words + (p0 >> 5);
            word = m[0] >> (p0 & 31u);
            if ((p0 & 31u) && int(p0 >> 5) + 1 < tr.words) word |= m[1] << (32u - (p0 & 31u));
        }
        const uint32_t o = here(kl + s0 * QK);
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            if constexpr (KD == 3) {
                const auto r = __builtin_amdgcn_raw_buffer_load_b96(kb, o + 16 * a * QK, 0, 0);
#pragma unroll
                for (int d = 0; d < KD; ++d) kr[a][d] = r[d];
            } else {
                const auto r = __builtin_amdgcn_raw_buffer_load_b128(kb, o + 16 * a * QK, 0, 0);
#pragma unroll
                for (int d = 0; d < KD; ++d) kr[a][d] = r[d];
            }
        }
        scr = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(sb, scl + s0 * 4, 0, 0));
    };
    auto load_v = [&]() {
        const uint32_t o = here(vl + s0 * VD);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            vr[j] = __builtin_amdgcn_raw_buffer_load_b32(vb, o + (16 * (j >> 2) + (j & 3)) * VD, 0, 0);
    };
    place(ch);
    load_k();
    load_v();

    // ---- the query operand, while the first chunk is on its way ----
    float cf0;                        // factor of a score, in bits, is |cf0| 2^(kexp - sh)
    int sh;
    intx4_t qi;                       // QQ: codes
    uint32_t qp[2][KD == 3 ? 6 : 8];  // else: f16 pieces
    {
        if (tr.negative) {
            asm volatile("");  // (a branch)
#pragma unroll
            for (int e = 0; e < SL; ++e) v[e] = -v[e];
        }
        float a = 0.0f;
#pragma unroll
        for (int e = 0; e < SL; e += 2) a = max3(a, __builtin_fabsf(v[e]), __builtin_fabsf(v[e + 1]));
        a = fmaxf(a, ndl::wave_xor<16>(a));
        a = fmaxf(a, ndl::wave_xor<32>(a));
        float nan = 0.0f;
        if constexpr (QQ) {
            // quant_rows (model.rs:289-293): the codes and the head's scale
            const float qs = a > 0.0f ? a / 127.0f : 1.0f;
            const float inv = 1.0f / qs;
            uint32_t dw[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < SL; ++e) {
                // quant_code: half away from zero is truncation after adding
                // the float below a half, for every |y| < 2^22
                const float y = v[e] * inv;
                const float r = __builtin_amdgcn_fmed3f(y + copysignf(0.49999997f, y), -128.0f, 127.5f);
                nan = y != y ? y : nan;
                dw[e >> 2] |= (uint32_t(int32_t(r)) & 0xffu) << (8 * (e & 3));
            }
            qi = intx4_t{int(dw[0]), int(dw[1]), int(dw[2]), int(dw[3])};
            sh = -__builtin_amdgcn_frexp_expf(qs);
            cf0 = __builtin_amdgcn_ldexpf(qs, sh) * tr.scale2;
        } else {
            // the head in 2^14 .. 2^15, so that the second pieces are normal numbers
            sh = a > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(a) : 0;
#pragma unroll
            for (int e = 0; e < SL; ++e) {
                nan = v[e] - v[e] != 0.0f ? NAN : nan;
                v[e] = __builtin_amdgcn_ldexpf(v[e], sh);
            }
#pragma unroll
            for (int e = 0; e < SL; e += 2) split2(v[e], v[e + 1], qp[0][e / 2], qp[1][e / 2]);
            cf0 = tr.scale2;
        }
        // a query that has a NaN (or an infinity, which gives one) makes no number
        // of what its node sees, and zeros of nothing: cf0's sign says so until the
        // sum is known
        nan += ndl::wave_xor<16>(nan);
        nan += ndl::wave_xor<32>(nan);
        cf0 = nan != nan ? -__builtin_fabsf(cf0) : cf0;
    }
    // (a factor of 0 would make no number of a score of -inf)
    auto factor = [&](int k) {
        const float c = __builtin_amdgcn_ldexpf(__builtin_fabsf(cf0), k - sh);
        return c == 0.0f ? 0x1p-126f : c;
    };
    float cf = factor(0);

    // m_run: a score of the column that the sums are against (mu = m_run cf, in
    // bits).  Another is taken, and the sums scaled, where one gets more than kAhead
    // bits ahead of it (lim, in the scores' units), or all stay far behind
    constexpr float kAhead = 5.0f;
    float m_run = -INFINITY, lim = -INFINITY, mu = 0.0f, l_run = 0.0f;
    floatx4_t acc[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
    // K and V scales are taken in units of 2^kexp and 2^(vexp - 10), powers of
    // two that no finite one so far is above: scores before cf, and weights,
    // stay in range at any size of the cache's values
    int kexp = 0, vexp = 0;
    float top = 0.0f;                   // lanes below 32: 2^kexp, the others: 2^vexp
    int shift = lane < 32 ? 0 : 10;
    // Weights below 2^-2 lose bits of their second pieces.  Where a column has met a
    // larger one in a product of pieces, those bits are none of the result's, and it
    // meets one (an e of 1 and a V scale of 2 units or more) with each new m_run; not
    // where that lies in a chunk of small values, or where the unit of weights has
    // grown since, by more than 2^3.  From then on (watch: lim lets every chunk in)
    // a column goes on against the next chunk's own maximum, which may lie far below:
    // its sums are multiplied (up to 2^100)
    uint32_t watch = 0;
    int vmet = 0x10000;                 // vexp then, and 3

    for (; ch < nch; ch += step) {
        // ---- the positions each column sees ----
        const bool full = !tail && p0 >= tlo && left >= 32;
        uint32_t vis = 0xffffffffu;
        if (!full) {
            vis = left < 32 ? (1u << left) - 1u : 0xffffffffu;
            vis &= tail ? word : lo <= p0 ? 0xffffffffu : lo - p0 < 32u ? 0xffffffffu << (lo - p0) : 0u;
        }
        // ---- the chunk's scales, zero behind its end ----
        float sc = (lane & 31) < left ? scr : 0.0f;
        if (any_of(!(__builtin_fabsf(sc) <= top))) {
            // what no column sees may be anything: it sets no unit, and counts as one
            bool unseen = false;
            if (tail || p0 < tlo) {
                uint32_t seen = along ? 0u : vis;
                seen |= uint32_t(ndl::wave_xor_int<1>(int(seen)));
                seen |= uint32_t(ndl::wave_xor_int<2>(int(seen)));
                seen |= uint32_t(ndl::wave_xor_int<4>(int(seen)));
                seen |= uint32_t(ndl::wave_xor_int<8>(int(seen)));
                unseen = !(seen >> (lane & 31) & 1u);
                sc = unseen ? 0.0f : sc;
            }
            // a V scale that is no number makes no number of the columns that see
            // it, and only of those: a weight of 0 there would not stay 0
            const bool wild = lane >= 32 && !(__builtin_fabsf(sc) < INFINITY);
            const uint32_t wilds = uint32_t(__builtin_amdgcn_ballot_w64(wild) >> 32);
            if (wild) sc = 0.0f;
            if (vis & wilds) l_run = NAN;
            float h = __builtin_fabsf(sc) < INFINITY ? fmaxf(__builtin_fabsf(sc), top) : top;
            h = fmaxf(h, ndl::wave_xor<16>(h));
            h = fmaxf(h, ndl::wave_xor<8>(h));
            h = fmaxf(h, ndl::wave_xor<4>(h));
            h = fmaxf(h, ndl::wave_xor<2>(h));
            h = fmaxf(h, ndl::wave_xor<1>(h));
            const int was = lane < 32 ? kexp : vexp;
            const int now = h > top ? __builtin_amdgcn_frexp_expf(h) : was;
            top = h > top ? (now > 127 ? 0x1.fffffep127f : __builtin_amdgcn_ldexpf(1.0f, now)) : top;
            sc = unseen ? top : sc;
            shift += was - now;
            const int kn = __builtin_amdgcn_readlane(now, 0), vn = __builtin_amdgcn_readlane(now, 32);
            if (vn > vmet) {
                watch = 1;
                vmet = vn + 3;
            }
            m_run = __builtin_amdgcn_ldexpf(m_run, kexp - kn);
            cf = factor(kn);
            lim = watch || m_run == -INFINITY ? -INFINITY : m_run + kAhead * __builtin_amdgcn_rcpf(cf);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[c][i] = __builtin_amdgcn_ldexpf(acc[c][i], vexp - vn);
            kexp = kn;
            vexp = vn;
        }
        sc = __builtin_amdgcn_ldexpf(sc, shift);
        const uint32_t few = uint32_t(__builtin_amdgcn_ballot_w64(sc < 2.0f) >> 32);
        uint32_t small = left < 32 ? few & ((1u << left) - 1u) : few;
        sc_s[w][lane] = sc;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        floatx4_t ks[2], vs[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            ks[a] = *reinterpret_cast<const floatx4_t *>(&sc_s[w][16 * a + 4 * qd]);
            vs[a] = *reinterpret_cast<const floatx4_t *>(&sc_s[w][32 + 16 * a + 4 * qd]);
        }
        __builtin_amdgcn_wave_barrier();
        // ---- scores ----
        float s[8];
        if constexpr (QQ) {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const intx4_t kf{int(kr[a][0]), int(kr[a][1]), int(kr[a][2]), KD == 3 ? 0 : int(kr[a][KD - 1])};
                const intx4_t d = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, qi, intx4_t{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[4 * a + i] = float(d[i]) * ks[a][i];
            }
        } else {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                uint32_t kp[2 * KD];
#pragma unroll
                for (int d = 0; d < KD; ++d) {
                    const uint32_t u = kr[a][d] ^ 0x80808080u;
                    kp[2 * d] = f16_pair<0>(u);
                    kp[2 * d + 1] = f16_pair<1>(u);
                }
                floatx4_t d{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int pc = 1; pc >= 0; --pc) {  // the small pieces first
                    const uint32_t *qq = qp[pc];
                    // qk 48: a lane's last four codes, doubled to the 32-wide
                    // product's eight against four zeros of the query
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        vec4<f16x8_t>(kp[4], kp[5], kp[2 * KD - 2], kp[2 * KD - 1]),
                        KD == 3 ? vec4<f16x8_t>(qq[4], qq[5], 0u, 0u)
                                : vec4<f16x8_t>(qq[4], qq[5], qq[2 * KD - 2], qq[2 * KD - 1]),
                        d, 0, 0, 0);
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(vec4<f16x8_t>(kp[0], kp[1], kp[2], kp[3]),
                                                               vec4<f16x8_t>(qq[0], qq[1], qq[2], qq[3]), d, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[4 * a + i] = d[i] * ks[a][i];
            }
        }
        // the next chunk: its K lands during the softmax and the values
        if (ch + step < stop) [[likely]] {
            s0 += 32u * uint32_t(step);
            p0 += 32u * uint32_t(step);
            left -= 32 * step;
        } else {
            asm volatile("");  // (a branch, not thirty selects in every chunk)
            place(ch + step);
        }
        load_k();
        // ---- softmax: each lane its column's eight positions ----
        if (!full) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!(vis >> (16 * (j >> 2) + 4 * qd + (j & 3)) & 1u)) s[j] = -INFINITY;
        }
        const float m8 = max3(max3(s[0], s[1], s[2]), max3(s[3], s[4], s[5]), max3(s[6], s[7], s[7]));
        if (any_of(m8 > lim)) {
            // a row of zeros has a scale of 1, which is no measure of its values
            small |= uint32_t(__builtin_amdgcn_ballot_w64(sc == __builtin_amdgcn_ldexpf(1.0f, shift)) >> 32);
            float m_new = max3(m8, m_run, ndl::wave_xor<16>(m8));
            m_new = fmaxf(m_new, ndl::wave_xor<32>(m_new));
            if (watch && !small) [[unlikely]] {
                float m = fmaxf(m8, ndl::wave_xor<16>(m8)), l = fmaxf(l_run, ndl::wave_xor<16>(l_run));
                m = fmaxf(m, ndl::wave_xor<32>(m));
                l = fmaxf(l, ndl::wave_xor<32>(l));
                const float behind = mu - m * cf;
                const bool down = (m > -INFINITY) & (behind + float(__builtin_amdgcn_frexp_expf(l)) < 100.0f);
                m_new = down ? m : m_new;
                watch = any32((m_new > -INFINITY) & !down);
            }
            watch |= small;
            vmet = min(vmet, vexp + 3);
            const float mu_new = m_new == -INFINITY ? 0.0f : m_new * cf;
            // nothing is summed yet where there was no maximum
            const float al = m_run == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mu - mu_new);
            m_run = m_new;
            lim = watch || m_new == -INFINITY ? -INFINITY : m_new + kAhead * __builtin_amdgcn_rcpf(cf);
            mu = mu_new;
            l_run *= al;
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] *= al;
        }
        // the weights e vs, and the sum of e
        float wt[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], cf, -mu));
            l_run += e;
            wt[j] = e * vs[j >> 2][j & 3];
        }
        // ---- values ----
        if (small) [[unlikely]] {
            // (then the product below adds nothing: two ways that each end in
            // sums cost copies of all of them)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(i8_at(vr[j], c) * 0x1p-9f, wt[j], acc[c], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 8; ++j) wt[j] = 0.0f;
        }
        {
            uint32_t ph[4], pl[4], u[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) split2(wt[2 * j], wt[2 * j + 1], ph[j], pl[j]);
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = vr[j] ^ 0x80808080u;
            auto column = [&](auto cc) {
                constexpr int c = decltype(cc)::value;
                const f16x8_t vf = vec4<f16x8_t>(f16_codes<c>(u[0], u[1]), f16_codes<c>(u[2], u[3]),
                                                 f16_codes<c>(u[4], u[5]), f16_codes<c>(u[6], u[7]));
                acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, vec4<f16x8_t>(pl[0], pl[1], pl[2], pl[3]), acc[c],
                                                                0, 0, 0);
                acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, vec4<f16x8_t>(ph[0], ph[1], ph[2], ph[3]), acc[c],
                                                                0, 0, 0);
            };
            column(std::integral_constant<int, 0>{});
            column(std::integral_constant<int, 1>{});
            column(std::integral_constant<int, 2>{});
            column(std::integral_constant<int, 3>{});
        }
        load_v();  // lands during the next scores
    }

    // ---- the block's waves meet: each leaves its sums, and sixteen threads a
    // column, four values each, put them together ----
    l_run += ndl::wave_xor<16>(l_run);
    l_run += ndl::wave_xor<32>(l_run);
    l_run = (bad | ((__float_as_int(cf0) < 0) & (l_run != 0.0f))) ? NAN : l_run;
    // the sums are left as 2^more of what has a weight of 1/2 to 1: of values near
    // fp32's end the sum may be beyond it, the mean is not
    const int more = __builtin_amdgcn_frexp_expf(l_run);
    // (from here on the maximum is in bits)
    if (qd == 0)
        ms[w][n] = floatx4_t{m_run == -INFINITY ? -INFINITY : mu, float(more), __builtin_amdgcn_ldexpf(l_run, -more), 0.0f};
    // lane (n, qd) holds V columns 16 qd + 4 i + c
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        floatx4_t o;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = __builtin_amdgcn_ldexpf(acc[c][i], vexp - 1 - more);
        *reinterpret_cast<floatx4_t *>(&mo[w][n][16 * qd + 4 * i]) = o;
    }
    __syncthreads();
    const int col = t >> 4, fo = int(tile) * kCols + col;
    if (col >= kCols || fo >= ncols) return;
    // Against a maximum 2^3 above the largest, so that no sum of eight leaves the
    // values' range.  -inf: sums are 0, or NaN where a score was.  (m + more may be
    // rounded, M with it; m - M is not.)
    float M = -INFINITY, L = 0.0f;
    floatx4_t O{0.0f, 0.0f, 0.0f, 0.0f}, z[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        z[i] = ms[i][col];
        M = fmaxf(M, z[i][0] + z[i][1]);
    }
    M += 3.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const float by = z[i][0] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(z[i][0] - M + z[i][1]);
        L += z[i][2] * by;
        O += *reinterpret_cast<const floatx4_t *>(&mo[i][col][4 * (t & 15)]) * by;
    }
    const int no = node_of(fo);
    const size_t oh = (size_t(ses) * tr.nodes + no) * g.H + int(kvh) * R + fo - no * R;
    if (tr.splits == 1) {
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        *reinterpret_cast<floatx4_u *>(tr.out + oh * VD + 4 * (t & 15)) = O * inv;
    } else {
        const size_t at = oh * tr.splits + split;
        *reinterpret_cast<floatx4_t *>(tr.part_o + at * VD + 4 * (t & 15)) = O;
        if ((t & 15) == 0) {
            tr.part_ml[2 * at] = M;
            tr.part_ml[2 * at + 1] = L;
        }
    }
}

// The splits of a (row, head) meet: a wave each, a lane a column.
__global__ __launch_bounds__(256) void tree_join_kernel(int H, Tree tr, size_t total)
{
    const size_t oh = size_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (oh >= total) return;
    const int lane = threadIdx.x & 63;
    const size_t row = oh / H, ses = row / tr.nodes;
    const int len = tr.length ? tr.length[ses] : tr.nodes;
    // rows behind the tree's end have no partials and are left as they are
    if (len >= 0 && len <= tr.nodes && int(row - ses * tr.nodes) >= len) return;
    // a lane a split, then a lane a column
    float m = -INFINITY, l = 0.0f;
    if (lane < tr.splits) {
        const size_t at = oh * tr.splits + lane;
        m = tr.part_ml[2 * at];
        l = tr.part_ml[2 * at + 1];
    }
    const float M = wave_max(m), f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - M), L = wave_sum(l * f);
    const float by = L == 0.0f ? 0.0f : f / L;
    float O = 0.0f;
    for (int s = 0; s < tr.splits; ++s)
        O += tr.part_o[(oh * tr.splits + s) * VD + lane] * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(by), s));
    tr.out[oh * VD + lane] = O;
}

constexpr int kMaxSplits = 64;  // a lane each in the join

struct Plan {
    int nw;
    size_t tiles, splits;
};

Plan plan_of(nd_ctx *ctx, const nd_kv_geom *g, size_t count, size_t nodes)
{
    const size_t cus = size_t(ctx && ctx->num_cus > 0 ? ctx->num_cus : 256);
    const size_t cols = nodes * size_t(g->num_heads / g->num_kv_heads);
    const size_t groups = count * size_t(g->num_kv_heads);
    const size_t chunks = (size_t(g->cap) + 31) / 32 + (nodes + 31) / 32;
    Plan p;
    p.tiles = (cols + kCols - 1) / kCols;
    const size_t blocks = groups * p.tiles;
    // Eight waves a block below one and a half blocks a CU, four above (us, 4 / 8:
    // 96 blocks 9.5 / 8.8, 576 17.9 / 18.0, 768 23.9 / 23.5, 768 longer ones 35.8 /
    // 37.5, 1024 20.1 / 23.2)
    p.nw = blocks * 2 < cus * 3 ? 8 : 4;
    // A chunk costs a wave 0.55 us, a split about 0.25 at the join, the join's
    // launch 3: as many splits as balance the first two, no more than give every
    // SIMD two waves, and none that do not pay for the launch (us, one session x
    // 8000 in 1 / 4 / 8 / 10 splits 26.4 / 15.0 / 13.3 / 14.4; one of 12 kv heads x
    // 4000 in 1 / 4 / 6 / 8 18.4 / 12.7 / 12.5 / 12.8; 4 sessions x 4000 in 1 / 2 / 4
    // 18.5 / 15.8 / 16.7; 16 x 1000 in 1 / 2 8.8 / 11.9)
    const size_t fill = cus * 8 / (blocks * p.nw);
    p.splits = 1;
    while (p.splits < fill && p.splits < kMaxSplits && (p.splits + 1) * (p.splits + 1) * p.nw <= 2 * chunks) ++p.splits;
    if (chunks * (p.splits - 1) < 6 * p.nw * p.splits) p.splits = 1;
    return p;
}

template <int QK, bool QQ>
auto kernel_of(const Plan &p)
{
    return p.nw == 4 ? tree_kernel<QK, QQ, 4> : tree_kernel<QK, QQ, 8>;
}

// What a call and its workspace's size are refused for.
int check_tree(const nd_kv_geom *g, size_t count, size_t nodes)
{
    if (int rc = check_geom(g)) return rc;
    ND_REQUIRE((g->qk_head_dim == 48 || g->qk_head_dim == 64) && g->v_head_dim == VD,
               "no tree attention for qk %d, v %d", g->qk_head_dim, g->v_head_dim);
    ND_REQUIRE(nodes >= 1 && nodes <= kMaxNodes, "nodes %zu must be in 1..%d", nodes, kMaxNodes);
    ND_REQUIRE(count <= 65535, "count %zu above 65535", count);
    ND_REQUIRE(g->num_heads <= 4096, "num_heads %d above 4096", g->num_heads);
    // a buffer of one head's scales reaches from its K scales to its V scales
    ND_REQUIRE(size_t(g->num_kv_heads) * g->cap <= size_t(1) << 29, "%d kv heads x cap %d above 2^29",
               g->num_kv_heads, g->cap);
    return ND_OK;
}

size_t partial_floats(const nd_kv_geom *g, size_t count, size_t nodes, size_t splits)
{
    return splits > 1 ? count * nodes * g->num_heads * splits * (VD + 2) : 0;
}

}  // namespace

extern "C" {

size_t nd_attend_tree_i8_work(nd_ctx *ctx, const nd_kv_geom *g, size_t count, size_t nodes)
{
    nd::clear_error();
    if (!ctx || check_tree(g, count, nodes) != ND_OK || !count) return 0;
    return partial_floats(g, count, nodes, plan_of(ctx, g, count, nodes).splits) * sizeof(float);
}

int nd_attend_tree_i8(nd_ctx *ctx, const nd_kv_geom *g, const void *kv, size_t kv_stride,
                      size_t count, size_t nodes, const int32_t *base, const int32_t *length,
                      const int32_t *lo, const uint32_t *mask, const float *q, float scale,
                      int quant_query, float *out, void *work, size_t work_bytes)
{
    ND_ENTER(ctx);
    if (int rc = check_tree(g, count, nodes)) return rc;
    if (count == 0) return ND_OK;
    ND_REQUIRE(kv && base && lo && mask && q && out, "null buffer");
    ND_REQUIRE((reinterpret_cast<uintptr_t>(kv) & 255) == 0 && kv_stride % 256 == 0,
               "kv blocks must be 256-byte aligned");
    const uintptr_t qa = reinterpret_cast<uintptr_t>(q), oa = reinterpret_cast<uintptr_t>(out);
    const size_t heads = count * nodes * g->num_heads * sizeof(float);
    ND_REQUIRE(qa + heads * g->qk_head_dim <= oa || oa + heads * VD <= qa, "out overlaps q");
    const Plan p = plan_of(ctx, g, count, nodes);
    Tree t{};
    t.kv_stride = kv_stride;
    t.nodes = int(nodes);
    t.words = int((nodes + 31) / 32);
    t.rep = g->num_heads / g->num_kv_heads;
    t.by_splits = Divisor::of(uint32_t(p.splits));
    t.by_kvh = Divisor::of(uint32_t(g->num_kv_heads));
    t.splits = int(p.splits);
    t.scale2 = scale == scale ? float(double(scale < 0 ? -scale : scale) * 1.4426950408889634) : -1.0f;
    t.negative = scale < 0;
    if (p.splits > 1) {
        void *ws = nullptr;
        const size_t bytes = partial_floats(g, count, nodes, p.splits) * sizeof(float);
        if (int rc = nd::call_workspace(ctx, bytes, work, work_bytes, &ws)) return rc;
        t.part_o = static_cast<float *>(ws);
        t.part_ml = t.part_o + count * nodes * g->num_heads * p.splits * VD;
    }
    const bool q48 = g->qk_head_dim == 48;
    auto *fn = q48 ? (quant_query ? kernel_of<48, true>(p) : kernel_of<48, false>(p))
                   : (quant_query ? kernel_of<64, true>(p) : kernel_of<64, false>(p));
    // HIP counts a launch's threads in 32 bits: sessions beyond that go in further
    // launches (never those of a split call, whose waves are two a SIMD at most)
    const size_t per = size_t(g->num_kv_heads) * p.splits * p.tiles, most = std::max<size_t>(1, (size_t(1) << 18) / per);
    const Geom kg = make_geom(g);
    for (size_t s = 0; s < count; s += most) {
        const size_t m = std::min(most, count - s), rows = s * nodes;
        t.kv = static_cast<const uint8_t *>(kv) + s * kv_stride;
        t.base = base + s;
        t.length = length ? length + s : nullptr;
        t.lo = lo + rows;
        t.mask = mask + rows * t.words;
        t.q = q + rows * g->num_heads * g->qk_head_dim;
        t.out = out + rows * g->num_heads * VD;
        t.units = uint32_t(m * g->num_kv_heads * p.splits);
        hipLaunchKernelGGL(fn, dim3(8, unsigned(p.tiles), unsigned((t.units + 7) / 8)), dim3(p.nw * 64), 0, ctx->stream, kg, t);
        if (int rc = nd::check_launch("attend_tree_i8")) return rc;
        if (t.part_o) {
            const size_t total = m * nodes * g->num_heads;
            hipLaunchKernelGGL(tree_join_kernel, dim3(unsigned((total + 3) / 4)), dim3(256), 0, ctx->stream,
                               g->num_heads, t, total);
            if (int rc = nd::check_launch("tree_join")) return rc;
        }
    }
    return ND_OK;
}

}  // extern "C"
