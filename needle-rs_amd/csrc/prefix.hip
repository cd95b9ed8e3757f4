// A batch that shares its prompts: the rows of a step laid out from the requests'
// lengths, and attention over prefixes that are held once and over the sessions'
// own blocks.
#include "nd_attn_pieces.h"
#include "nd_internal.h"
#include "nd_kv_internal.h"

#include <algorithm>

namespace {

using namespace ndkv;
using namespace ndap;

constexpr int VD = 64, kCols = 16;
constexpr size_t kMaxSessions = 65535, kMaxRows = 256, kMaxAll = size_t(1) << 20, kMaxPrefixes = 2048;

// ---- the plan ---------------------------------------------------------------
//
// Attention is done in units: a quad of column tiles (16 (row, head) pairs of a kv
// head each) of one source -- a prefix, for all rows of its group, or a session's
// own block -- and a run of chunks of 32 positions.  A unit's four waves take its
// tiles (`wide` of them: 4, 2 or 1) and, where there are fewer than four, the
// chunks in turn.  The units are as long as leaves about kBlocks blocks, whatever
// the requests' lengths are, and each leaves its sums in slots, one a tile.
constexpr int kPlanMagic = 0x6e645031;
constexpr uint32_t kBlocks = 1024;     // four a CU
constexpr uint32_t kLeast = 2;         // chunks a wave, at least

struct Head {
    int magic, count, rows, prefixes, heads, kv_heads, cap, prefix_cap;
    int units, slots, window, pad[5];
};

// there: the rows the session has, bad: no number comes of them; prefix -1: none;
// at: its first row's place in the prefix's group.
struct Session {
    int there, bad, prefix, at;
    int used, lo, span, quads;  // own positions lo .. lo + span - 1; first quad
};

struct Group {
    int first, rows, begin, span;  // places in the order; positions
    int end, quads, pad0, pad1;    // the prefix's length; first quad
};

struct Place {
    int row, from;
};

struct Quad {
    int slot, runs, wide, pad;  // first slot, runs of chunks; slot + run * wide + tile
};

struct Unit {
    int source, quad, wide, slot;      // prefix, or ~session; of the source; first slot
    int begin, end, rows, first;       // chunks; rows of the source and the first's place
    int from, span, used, pad[5];      // positions; own: positions before the step
};

struct Layout {
    size_t session, group, quad, place, unit, bytes;  // offsets
    uint32_t quads_prefix, quads_own;                 // at most: of all prefixes, of a session
    uint32_t units, slots;                            // at most
};

struct Sizes {
    uint32_t count, rows, prefixes;
    int H, KVH, cap, pcap;
};

uint32_t ceil_div(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }

Layout layout_of(const Sizes &z)
{
    const uint64_t R = uint64_t(z.H / z.KVH), own = ceil_div(z.rows * R, kCols);
    const uint64_t all = ceil_div(uint64_t(z.count) * z.rows * R, kCols);
    Layout l{};
    l.quads_prefix = z.prefixes ? uint32_t((all + 3) / 4) + z.prefixes : 0;
    l.quads_own = uint32_t((own + 3) / 4);
    // units: a quad's last run may be short, the full ones come to kBlocks / KVH
    const uint32_t runs = std::max<uint32_t>(1, kBlocks / uint32_t(z.KVH));
    const uint64_t quads = l.quads_prefix + uint64_t(z.count) * l.quads_own;
    l.units = uint32_t(quads + runs);
    // slots: a quad of three tiles has four
    l.slots = uint32_t((z.prefixes ? all + 2 * z.prefixes : 0) + z.count * (own + (own % 4 == 3)) + 4 * runs);
    l.session = sizeof(Head);
    l.group = l.session + z.count * sizeof(Session);
    l.quad = l.group + z.prefixes * sizeof(Group);
    l.place = l.quad + quads * sizeof(Quad);
    l.unit = nd::align_up(l.place + size_t(z.count) * z.rows * sizeof(Place), 64);
    l.bytes = l.unit + l.units * sizeof(Unit);
    return l;
}

struct PlanOf {
    uint8_t *p;
    Layout l;
    __host__ __device__ Head *head() const { return reinterpret_cast<Head *>(p); }
    __host__ __device__ Session *session() const { return reinterpret_cast<Session *>(p + l.session); }
    __host__ __device__ Group *group() const { return reinterpret_cast<Group *>(p + l.group); }
    __host__ __device__ Quad *quad() const { return reinterpret_cast<Quad *>(p + l.quad); }
    __host__ __device__ Place *place() const { return reinterpret_cast<Place *>(p + l.place); }
    __host__ __device__ Unit *unit() const { return reinterpret_cast<Unit *>(p + l.unit); }
};

struct Requests {
    const int32_t *prefix_of, *prefix_len, *used, *length;
    int window;
};

// One session's numbers.
struct Want {
    int there, bad, prefix, used, prefix_len, from, lo, span;
    __device__ int rows() const { return bad ? 0 : there; }
};

__device__ inline Want want_of(const Sizes &z, const Requests &r, uint32_t i)
{
    Want w{};
    const int p = r.prefix_of ? r.prefix_of[i] : z.prefixes ? 0 : -1;
    const int m = r.length ? r.length[i] : int(z.rows), u = r.used[i];
    const bool some = p >= 0 && p < int(z.prefixes);
    const int L = some ? r.prefix_len[p] : 0;
    const bool fits = m >= 0 && m <= int(z.rows);
    w.there = fits ? m : int(z.rows);
    w.prefix = some ? p : -1;
    w.used = u;
    w.prefix_len = L;
    bool bad = !fits || p >= int(z.prefixes) || u < 0 || L < 0 || int64_t(L) + u + m > int64_t(1) << 31;
    if (!bad) {
        // the first row's window; the others' begin later
        w.lo = r.window ? int(max(int64_t(u) + 1 - r.window, int64_t(0))) : 0;
        w.from = r.window ? int(min(max(int64_t(L) + u + 1 - r.window, int64_t(0)), int64_t(L))) : 0;
        const int64_t span = int64_t(u) + m - w.lo;
        w.span = int(min(span, int64_t(z.cap)));
        bad = m > 0 && (span > z.cap || L - w.from > z.pcap);
    }
    w.bad = bad;
    return w;
}

// Chunks of 32 positions of a walk from `from`: chunks end at the ring's end.
__host__ __device__ inline uint32_t chunks_of(uint32_t from, uint32_t span, uint32_t cap)
{
    const uint32_t n0 = min(span, cap - from % cap), n1 = span - n0;
    return (n0 + 31) / 32 + (n1 + 31) / 32;
}

// What `tiles` tiles over `chunks` chunks come to: waves' chunks (weight), and, a
// wave having `each`, units and slots.  A last quad of three tiles is one of four.
struct Shares {
    uint32_t units, slots;
};

__device__ inline uint32_t wide_of(uint32_t tiles, uint32_t quad)
{
    const uint32_t left = tiles - 4 * quad;
    return left >= 3 ? 4 : left;
}

__device__ inline uint32_t runs_of(uint32_t wide, uint32_t chunks, uint32_t each)
{
    const uint64_t most = uint64_t(each) * (4 / wide);
    return uint32_t((chunks + most - 1) / most);
}

__device__ inline uint64_t weight_of(uint32_t tiles, uint32_t chunks)
{
    const uint32_t full = tiles / 4, rest = tiles % 4;
    return uint64_t(full) * chunks + (rest ? runs_of(wide_of(rest, 0), chunks, 1) : 0);
}

__device__ inline Shares shares_of(uint32_t tiles, uint32_t chunks, uint32_t each)
{
    const uint32_t full = tiles / 4, rest = tiles % 4;
    const uint32_t a = runs_of(4, chunks, each), wide = rest ? wide_of(rest, 0) : 1;
    const uint32_t b = rest ? runs_of(wide, chunks, each) : 0;
    return Shares{full * a + b, 4 * full * a + wide * b};
}

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64, kPlanSessions = 256;

// The sum of v over the block, and over the threads before this one.
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
    for (int i = 0; i < kPlanWaves; ++i) {
        mine += i < w ? room[i] : 0;
        all += room[i];
    }
    __syncthreads();
    before = mine + up - v;
    return all;
}

// A block lays out kPlanSessions sessions, and every blocks-th prefix.  What it has
// to know of the rest -- the groups, and what the sessions before its own come to --
// it works out from the requests itself (65535 of them are 64 a thread), so that
// one launch does without a word between blocks.  Whole numbers: the same plan
// whatever the order of the atomics.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(Sizes z, Requests r, PlanOf plan, nd_prefix_maps maps)
{
    __shared__ uint32_t rows_s[kMaxPrefixes], from_s[kMaxPrefixes], before_s[kMaxPrefixes];
    __shared__ uint32_t first_s[kMaxPrefixes], units_s[kMaxPrefixes], slots_s[kMaxPrefixes];
    __shared__ uint64_t room[kPlanWaves], weight_s;
    __shared__ int which_s[kPlanSessions], mine_s[kPlanSessions], there_s[kPlanSessions], at_s[kPlanSessions];
    __shared__ int used_s[kPlanSessions], len_s[kPlanSessions];
    __shared__ uint32_t units_at, slots_at;
    const int t = threadIdx.x, lane = t & 63;
    const uint32_t R = uint32_t(z.H / z.KVH), P = z.prefixes, S = z.count;
    const uint32_t s0 = blockIdx.x * kPlanSessions, s1 = min(S, s0 + kPlanSessions);
    for (uint32_t p = t; p < P; p += kPlanThreads) rows_s[p] = before_s[p] = 0, from_s[p] = 0xffffffffu;
    if (t == 0) weight_s = 0, units_at = slots_at = 0;
    __syncthreads();

    // ---- the groups, and all own walks ----
    uint64_t weight = 0;
    for (uint32_t i = t; i < S; i += kPlanThreads) {
        const Want w = want_of(z, r, i);
        const uint32_t m = uint32_t(w.rows());
        if (!m) continue;
        weight += weight_of((m * R + kCols - 1) / kCols, chunks_of(uint32_t(w.lo), uint32_t(w.span), uint32_t(z.cap)));
        if (w.prefix < 0) continue;
        atomicAdd(&rows_s[w.prefix], m);
        atomicMin(&from_s[w.prefix], uint32_t(w.from));
        if (i < s0) atomicAdd(&before_s[w.prefix], m);
    }
    for (int d = 32; d; d /= 2) weight += __shfl_xor(weight, d);
    if (lane == 0) atomicAdd(reinterpret_cast<unsigned long long *>(&weight_s), weight);
    __syncthreads();
    auto tiles_of = [&](uint32_t rows) { return (rows * R + kCols - 1) / kCols; };
    auto group_chunks = [&](uint32_t p) -> uint32_t {  // of a group with rows
        return chunks_of(from_s[p], uint32_t(r.prefix_len[p]) - from_s[p], uint32_t(z.pcap));
    };
    weight = 0;
    for (uint32_t p = t; p < P; p += kPlanThreads)
        if (rows_s[p]) weight += weight_of(tiles_of(rows_s[p]), group_chunks(p));
    for (int d = 32; d; d /= 2) weight += __shfl_xor(weight, d);
    if (lane == 0 && weight) atomicAdd(reinterpret_cast<unsigned long long *>(&weight_s), weight);
    __syncthreads();
    const uint64_t runs = max(1u, kBlocks / uint32_t(z.KVH));
    const uint32_t each = uint32_t(min(max(uint64_t(kLeast), (weight_s + runs - 1) / runs), uint64_t(1) << 20));

    // ---- where each group's rows, quads, units and slots begin ----
    uint32_t rows_all = 0, quads_all = 0, units_all = 0, slots_all = 0;
    for (uint32_t p0 = 0; p0 < P; p0 += kPlanThreads) {
        const uint32_t p = p0 + t, rows = p < P ? rows_s[p] : 0, tiles = tiles_of(rows);
        const uint32_t chunks = rows ? group_chunks(p) : 0;
        const Shares sh = shares_of(tiles, chunks, each);
        // (rows and quads below 2^20 each, units and slots below 2^32)
        uint64_t a, b;
        const uint64_t all_a = block_scan(uint64_t(rows) << 32 | (tiles + 3) / 4, a, room);
        const uint64_t all_b = block_scan(uint64_t(sh.units) << 32 | sh.slots, b, room);
        if (p < P) {
            first_s[p] = rows_all + uint32_t(a >> 32);
            units_s[p] = units_all + uint32_t(b >> 32);
            slots_s[p] = slots_all + uint32_t(b);
            if (blockIdx.x == 0) {
                Group g{};
                g.first = int(first_s[p]);
                g.rows = int(rows);
                g.begin = rows ? int(from_s[p]) : 0;
                g.end = rows ? r.prefix_len[p] : 0;
                g.span = g.end - g.begin;
                g.quads = int(quads_all + uint32_t(a));
                plan.group()[p] = g;
                if (maps.first) maps.first[p] = g.first;
            }
            // each block its share of the groups
            if (p % gridDim.x == blockIdx.x) {
                uint32_t slot = slots_s[p];
                for (uint32_t q = 0; 4 * q < tiles; ++q) {
                    const uint32_t wide = wide_of(tiles, q), n = runs_of(wide, chunks, each);
                    plan.quad()[quads_all + uint32_t(a) + q] = Quad{int(slot), int(n), int(wide), 0};
                    slot += n * wide;
                }
            }
        }
        rows_all += uint32_t(all_a >> 32);
        quads_all += uint32_t(all_a);
        units_all += uint32_t(all_b >> 32);
        slots_all += uint32_t(all_b);
    }
    __syncthreads();
    if (blockIdx.x == 0 && t == 0 && maps.first) maps.first[P] = int(rows_all);

    // ---- the groups' units ----
    for (uint32_t p = blockIdx.x; p < P; p += gridDim.x) {
        const uint32_t rows = rows_s[p];
        if (!rows) continue;
        const uint32_t tiles = tiles_of(rows), full = tiles / 4, chunks = group_chunks(p);
        const uint32_t a = runs_of(4, chunks, each);
        const Shares sh = shares_of(tiles, chunks, each);
        for (uint32_t i = t; i < sh.units; i += kPlanThreads) {
            const uint32_t q = i < full * a ? i / a : full, k = i - q * a;
            const uint32_t wide = wide_of(tiles, q), n = each * (4 / wide);
            Unit u{};
            u.source = int(p);
            u.quad = int(q);
            u.wide = int(wide);
            u.slot = int(slots_s[p] + 4 * q * a + k * wide);
            u.begin = int(k * n);
            u.end = int(min(chunks, (k + 1) * n));
            u.rows = int(rows);
            u.first = int(first_s[p]);
            u.from = int(from_s[p]);
            u.span = r.prefix_len[p] - int(from_s[p]);
            plan.unit()[units_s[p] + i] = u;
        }
    }

    // ---- what the sessions before this block's come to, and all ----
    Shares before{0, 0}, all{0, 0};
    for (uint32_t i = t; i < S; i += kPlanThreads) {
        if (blockIdx.x && i >= s1) break;
        const Want w = want_of(z, r, i);
        const uint32_t m = uint32_t(w.rows());
        if (!m) continue;
        const Shares sh = shares_of(tiles_of(m), chunks_of(uint32_t(w.lo), uint32_t(w.span), uint32_t(z.cap)), each);
        all.units += sh.units, all.slots += sh.slots;
        if (i < s0) before.units += sh.units, before.slots += sh.slots;
    }
    for (int d = 32; d; d /= 2) {
        before.units += __shfl_xor(before.units, d), before.slots += __shfl_xor(before.slots, d);
        all.units += __shfl_xor(all.units, d), all.slots += __shfl_xor(all.slots, d);
    }
    if (lane == 0) {
        atomicAdd(&units_at, blockIdx.x ? before.units : all.units);
        atomicAdd(&slots_at, blockIdx.x ? before.slots : all.slots);
    }
    __syncthreads();
    const uint32_t units0 = units_all + (blockIdx.x ? units_at : 0), slots0 = slots_all + (blockIdx.x ? slots_at : 0);
    if (blockIdx.x == 0 && t == 0)
        *plan.head() = Head{kPlanMagic, int(z.count), int(z.rows), int(P), z.H, z.KVH, z.cap, z.pcap,
                            int(units_all + units_at), int(slots_all + slots_at), r.window, {}};

    // ---- this block's sessions ----
    const uint32_t i = s0 + uint32_t(t);
    const bool mine = t < kPlanSessions && i < s1;
    Want w{};
    if (mine) w = want_of(z, r, i);
    const uint32_t m = mine ? uint32_t(w.rows()) : 0;
    const uint32_t tiles = tiles_of(m), chunks = m ? chunks_of(uint32_t(w.lo), uint32_t(w.span), uint32_t(z.cap)) : 0;
    const Shares sh = shares_of(tiles, chunks, each);
    if (t < kPlanSessions) which_s[t] = m ? w.prefix : -1, mine_s[t] = int(m);
    uint64_t at64;
    block_scan(uint64_t(sh.units) << 32 | sh.slots, at64, room);
    if (mine) {
        uint32_t at = w.prefix >= 0 ? before_s[w.prefix] : 0;
        for (int j = 0; j < t; ++j) at += which_s[j] == w.prefix ? uint32_t(mine_s[j]) : 0u;
        Session s{};
        s.there = w.there;
        s.bad = w.bad;
        s.prefix = w.bad ? -1 : w.prefix;
        s.at = int(at);
        s.used = w.used;
        s.lo = w.lo;
        s.span = w.span;
        s.quads = int(plan.l.quads_prefix + i * plan.l.quads_own);
        plan.session()[i] = s;
        uint32_t unit = units0 + uint32_t(at64 >> 32), slot = slots0 + uint32_t(at64);
        for (uint32_t q = 0; 4 * q < tiles; ++q) {
            const uint32_t wide = wide_of(tiles, q), n = each * (4 / wide), k1 = runs_of(wide, chunks, each);
            plan.quad()[uint32_t(s.quads) + q] = Quad{int(slot), int(k1), int(wide), 0};
            for (uint32_t k = 0; k < k1; ++k) {
                Unit u{};
                u.source = ~int(i);
                u.quad = int(q);
                u.wide = int(wide);
                u.slot = int(slot);
                u.begin = int(k * n);
                u.end = int(min(chunks, (k + 1) * n));
                u.rows = int(m);
                u.from = w.lo;
                u.span = w.span;
                u.used = w.used;
                plan.unit()[unit++] = u;
                slot += wide;
            }
        }
        there_s[t] = w.bad ? 0 : w.there;
        at_s[t] = int(at);
        used_s[t] = w.used;
        len_s[t] = w.prefix_len;
    }
    __syncthreads();

    // ---- their rows, and what lies behind the last of the order ----
    const uint32_t N = z.rows, total = (s1 > s0 ? s1 - s0 : 0) * N;
    for (uint32_t k = t; k < total; k += kPlanThreads) {
        const uint32_t j = k / N, n = k - j * N;
        const int row = int(s0 * N + k);
        int pos = -1, rot = -1, from = -1, lo = -1;
        if (int(n) < there_s[j]) {
            const int64_t at = int64_t(len_s[j]) + used_s[j] + n, open = r.window ? max(at + 1 - r.window, int64_t(0)) : 0;
            pos = used_s[j] + int(n);
            rot = int(at);
            from = int(min(open, int64_t(len_s[j])));
            lo = int(max(open - len_s[j], int64_t(0)));
            if (which_s[j] >= 0) {
                const uint32_t to = first_s[which_s[j]] + uint32_t(at_s[j]) + n;
                plan.place()[to] = Place{row, from};
                if (maps.order) maps.order[to] = row;
            }
        }
        if (maps.pos) maps.pos[row] = pos;
        if (maps.rot) maps.rot[row] = rot;
        if (maps.from) maps.from[row] = from;
        if (maps.lo) maps.lo[row] = lo;
    }
    if (maps.order)
        for (uint32_t k = rows_all + blockIdx.x * kPlanThreads + t; k < S * N; k += gridDim.x * kPlanThreads)
            maps.order[k] = -1;
}

// ---- attention ----------------------------------------------------------------

struct Attend {
    PlanOf plan;
    Sizes z;
    const uint8_t *kv, *pkv;
    size_t kv_stride, pkv_stride;
    const float *q;
    float *out;
    float scale;
    int quant_query;
};

// A wave a (row, head): 64 positions at a time, a lane each, then a lane a column.
template <int QK>
__global__ __launch_bounds__(64) void attend_kernel(Geom g, Geom gp, Attend a)
{
    __shared__ float qs[QK], ws[64];
    const int lane = threadIdx.x;
    const uint32_t row = blockIdx.x, head = blockIdx.y, kvh = head / uint32_t(a.z.H / a.z.KVH);
    const uint32_t i = row / a.z.rows, n = row - i * a.z.rows;
    const Head hd = *a.plan.head();
    float *out = a.out + (size_t(row) * a.z.H + head) * VD + lane;
    const bool fits = hd.magic == kPlanMagic && hd.count == int(a.z.count) && hd.rows == int(a.z.rows) &&
                      hd.prefixes == int(a.z.prefixes) && hd.heads == a.z.H && hd.kv_heads == a.z.KVH &&
                      hd.cap == a.z.cap && hd.prefix_cap == a.z.pcap;
    if (!fits) {
        *out = NAN;
        return;
    }
    const Session s = a.plan.session()[i];
    if (int(n) >= s.there) return;
    if (s.bad) {
        *out = NAN;
        return;
    }
    const float *qh = a.q + (size_t(row) * a.z.H + head) * QK;
    if (lane < QK) qs[lane] = qh[lane];
    __syncthreads();
    if (a.quant_query) {
        float sc, inv;
        quant_scale_wave(qs, QK, sc, inv);
        if (lane < QK) qs[lane] = quant_code(qs[lane], inv) * sc;
        __syncthreads();
    }
    float m = -INFINITY, l = 0.0f;
    double o = 0.0;  // (of values near fp32's end the sum is beyond it, the mean is not)
    auto walk = [&](const Geom &gg, const uint8_t *blk, uint32_t lo, int span) {
        const int8_t *kb = reinterpret_cast<const int8_t *>(blk) + size_t(kvh) * gg.cap * QK;
        const int8_t *vb = reinterpret_cast<const int8_t *>(blk + gg.v_off) + size_t(kvh) * gg.cap * VD;
        const float *ks = reinterpret_cast<const float *>(blk + gg.ks_off) + size_t(kvh) * gg.cap;
        const float *vs = reinterpret_cast<const float *>(blk + gg.vs_off) + size_t(kvh) * gg.cap;
        for (int done = 0; done < span; done += 64) {
            const uint32_t p0 = lo + uint32_t(done), cap = uint32_t(gg.cap);
            const int cnt = min(64, span - done), slot = int((p0 + uint32_t(min(lane, cnt - 1))) % cap);
            float dot = 0.0f;
            for (int e = 0; e < QK; ++e) dot += qs[e] * float(kb[size_t(slot) * QK + e]);
            const float sc = lane < cnt ? dot * ks[slot] * a.scale : -INFINITY;
            float top = fmaxf(m, wave_max(sc));
            if (top == -INFINITY) top = 0.0f;
            const float e = lane < cnt ? expf(sc - top) : 0.0f, al = m == -INFINITY ? 0.0f : expf(m - top);
            m = top;
            l = l * al + wave_sum(e);
            o *= al;
            ws[lane] = lane < cnt ? e * vs[slot] : 0.0f;
            __syncthreads();
            for (int j = 0; j < cnt; ++j) o += double(ws[j]) * double(vb[size_t((p0 + uint32_t(j)) % cap) * VD + lane]);
            __syncthreads();
        }
    };
    if (s.prefix >= 0) {
        const Group gr = a.plan.group()[s.prefix];
        const Place at = a.plan.place()[uint32_t(gr.first + s.at) + n];
        walk(gp, a.pkv + size_t(s.prefix) * a.pkv_stride, uint32_t(at.from), gr.end - at.from);
    }
    const int64_t end = int64_t(s.used) + n + 1, lo = hd.window ? max(end - hd.window, int64_t(0)) : 0;
    walk(g, a.kv + size_t(i) * a.kv_stride, uint32_t(lo), int(end - lo));
    *out = float(o / l);
}

// ---- the host's side ------------------------------------------------------------

int check_sizes(const nd_kv_geom *g, size_t count, size_t rows, size_t prefixes)
{
    if (int rc = check_geom(g)) return rc;
    ND_REQUIRE(g->num_heads <= 4096, "num_heads %d above 4096", g->num_heads);
    ND_REQUIRE(rows >= 1 && rows <= kMaxRows, "rows %zu must be in 1..%zu", rows, kMaxRows);
    ND_REQUIRE(count <= kMaxSessions, "count %zu above %zu", count, kMaxSessions);
    ND_REQUIRE(count * rows <= kMaxAll, "%zu sessions x %zu rows above %zu", count, rows, kMaxAll);
    ND_REQUIRE(prefixes <= kMaxPrefixes, "prefixes %zu above %zu", prefixes, kMaxPrefixes);
    return ND_OK;
}

int check_prefix_cap(size_t prefix_cap, size_t prefixes)
{
    ND_REQUIRE(prefixes == 0 || (prefix_cap > 0 && prefix_cap <= size_t(1) << 24), "prefix_cap %zu out of range",
               prefix_cap);
    return ND_OK;
}

Sizes sizes_of(const nd_kv_geom *g, size_t prefix_cap, size_t count, size_t rows, size_t prefixes)
{
    return Sizes{uint32_t(count), uint32_t(rows), uint32_t(prefixes), g->num_heads, g->num_kv_heads, g->cap,
                 prefixes ? int(prefix_cap) : 1};
}

}  // namespace

extern "C" {

size_t nd_prefix_plan_bytes(const nd_kv_geom *g, size_t count, size_t rows, size_t prefixes)
{
    nd::clear_error();
    if (check_sizes(g, count, rows, prefixes) != ND_OK) return 0;
    return layout_of(sizes_of(g, 1, count, rows, prefixes)).bytes;
}

int nd_prefix_plan(nd_ctx *ctx, const nd_kv_geom *g, size_t prefix_cap, size_t count, size_t rows,
                   size_t prefixes, const int32_t *prefix_of, const int32_t *prefix_len,
                   const int32_t *used, const int32_t *length, int32_t window, void *plan,
                   size_t plan_bytes, const nd_prefix_maps *maps)
{
    ND_ENTER(ctx);
    if (int rc = check_sizes(g, count, rows, prefixes)) return rc;
    if (int rc = check_prefix_cap(prefix_cap, prefixes)) return rc;
    ND_REQUIRE(window >= 0, "window %d below 0", window);
    ND_REQUIRE(plan && (count == 0 || used) && (prefixes == 0 || prefix_len), "null buffer");
    ND_REQUIRE((reinterpret_cast<uintptr_t>(plan) & 15) == 0, "plan must be 16-byte aligned");
    const Sizes z = sizes_of(g, prefix_cap, count, rows, prefixes);
    const Layout l = layout_of(z);
    ND_REQUIRE(plan_bytes >= l.bytes, "plan holds %zu bytes, %zu needed", plan_bytes, l.bytes);
    const unsigned blocks = unsigned(std::max<size_t>(1, (count + kPlanSessions - 1) / kPlanSessions));
    hipLaunchKernelGGL(plan_kernel, dim3(blocks), dim3(kPlanThreads), 0, ctx->stream, z,
                       Requests{prefix_of, prefix_len, used, length, window},
                       PlanOf{static_cast<uint8_t *>(plan), l}, maps ? *maps : nd_prefix_maps{});
    return nd::check_launch("prefix_plan");
}

size_t nd_attend_prefix_i8_work(nd_ctx *ctx, const nd_kv_geom *g, size_t count, size_t rows,
                                size_t prefixes)
{
    nd::clear_error();
    if (!ctx || check_sizes(g, count, rows, prefixes) != ND_OK || !count) return 0;
    return 0;
}

int nd_attend_prefix_i8(nd_ctx *ctx, const nd_kv_geom *g, const void *kv, size_t kv_stride,
                        size_t count, size_t rows, const void *prefix_kv, size_t prefix_stride,
                        size_t prefix_cap, size_t prefixes, const void *plan, const float *q,
                        float scale, int quant_query, float *out, void *work, size_t work_bytes)
{
    ND_ENTER(ctx);
    if (int rc = check_sizes(g, count, rows, prefixes)) return rc;
    if (int rc = check_prefix_cap(prefix_cap, prefixes)) return rc;
    ND_REQUIRE((g->qk_head_dim == 48 || g->qk_head_dim == 64) && g->v_head_dim == VD,
               "no prefix attention for qk %d, v %d", g->qk_head_dim, g->v_head_dim);
    // a buffer of one head's scales reaches from its K scales to its V scales
    const size_t most = std::max(size_t(g->cap), prefixes ? prefix_cap : 0);
    ND_REQUIRE(size_t(g->num_kv_heads) * most <= size_t(1) << 29, "%d kv heads x cap %zu above 2^29",
               g->num_kv_heads, most);
    if (count == 0) return ND_OK;
    ND_REQUIRE(kv && plan && q && out && (prefix_kv || !prefixes), "null buffer");
    ND_REQUIRE((reinterpret_cast<uintptr_t>(kv) & 255) == 0 && kv_stride % 256 == 0 &&
                   (reinterpret_cast<uintptr_t>(prefix_kv) & 255) == 0 && prefix_stride % 256 == 0,
               "kv blocks must be 256-byte aligned");
    ND_REQUIRE((reinterpret_cast<uintptr_t>(plan) & 15) == 0, "plan must be 16-byte aligned");
    const uintptr_t qa = reinterpret_cast<uintptr_t>(q), oa = reinterpret_cast<uintptr_t>(out);
    const size_t heads = count * rows * g->num_heads * sizeof(float);
    ND_REQUIRE(qa + heads * g->qk_head_dim <= oa || oa + heads * VD <= qa, "out overlaps q");
    Attend a{};
    a.z = sizes_of(g, prefix_cap, count, rows, prefixes);
    a.plan = PlanOf{const_cast<uint8_t *>(static_cast<const uint8_t *>(plan)), layout_of(a.z)};
    a.kv = static_cast<const uint8_t *>(kv);
    a.pkv = static_cast<const uint8_t *>(prefix_kv);
    a.kv_stride = kv_stride;
    a.pkv_stride = prefix_stride;
    a.q = q;
    a.out = out;
    a.scale = scale;
    a.quant_query = quant_query;
    nd_kv_geom pg = *g;
    pg.cap = a.z.pcap;
    auto *fn = g->qk_head_dim == 48 ? attend_kernel<48> : attend_kernel<64>;
    hipLaunchKernelGGL(fn, dim3(unsigned(count * rows), unsigned(g->num_heads)), dim3(64), 0, ctx->stream, make_geom(g),
                       make_geom(&pg), a);
    return nd::check_launch("attend_prefix_i8");
}

}  // extern "C"
