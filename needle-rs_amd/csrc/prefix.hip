// A batch that shares its prompts: the rows of a step laid out from the requests'
// lengths, and attention over prefixes that are held once and over the sessions'
// own blocks.
#include "nd_attn_pieces.h"
#include "nd_internal.h"
#include "nd_kv_internal.h"

#include <algorithm>
#include <type_traits>

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
    float *out, *part_o, *part_ml;  // sums of (slot, kv head, column), and their maximum and weight
    Divisor by_rep;
    float scale2;  // |scale| log2(e); below 0 where scale is no number
    int negative;  // scale < 0
};

__device__ inline bool made_for(const Head &h, const Sizes &z)
{
    return h.magic == kPlanMagic && h.count == int(z.count) && h.rows == int(z.rows) && h.prefixes == int(z.prefixes) &&
           h.heads == z.H && h.kv_heads == z.KVH && h.cap == z.cap && h.prefix_cap == z.pcap;
}

template <int QK, bool QQ>
__global__ __launch_bounds__(256, 4) void prefix_kernel(Geom gown, Geom gp, Attend at)
{
    constexpr int SL = QK / 4, KD = SL / 4;  // a lane's slice of a K row; its dwords (3 or 4)
    constexpr int LD = VD + 4, NW = 4;
    __shared__ __align__(16) float sc_s[NW][64];
    __shared__ __align__(16) float mo[NW][kCols][LD];
    __shared__ floatx4_t ms[NW][kCols];  // maximum, more, weight

    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n = lane & 15, qd = lane >> 4;
    const Head hd = *at.plan.head();
    if (!made_for(hd, at.z) || int(blockIdx.x) >= hd.units) return;
    const Unit un = at.plan.unit()[blockIdx.x];
    const uint32_t kvh = blockIdx.y, R = uint32_t(gown.H / gown.KVH);
    const bool own = un.source < 0;
    const int wide = un.wide, mine = w & (wide - 1), stream = w / wide, step = NW / wide;
    const uint32_t ncols = uint32_t(un.rows) * R, tile = 4 * uint32_t(un.quad) + uint32_t(mine);
    if (tile * kCols >= ncols) return;  // (of a quad of three tiles, whose waves do not meet)

    // ---- the wave's columns: what they see, and the query operand.  A column past
    // the end is a copy of the last ----
    const uint32_t f = min(tile * kCols + uint32_t(n), ncols - 1), r = at.by_rep.quotient(f);
    uint32_t row, lo, hi;
    if (own) {
        const uint32_t end = uint32_t(un.used) + r;  // the row's own position, below 2^31
        row = uint32_t(~un.source) * at.z.rows + r;
        lo = hd.window && end + 1 > uint32_t(hd.window) ? end + 1 - uint32_t(hd.window) : 0;
        hi = end;
    } else {
        const Place pl = at.plan.place()[uint32_t(un.first) + r];
        row = uint32_t(pl.row);
        lo = uint32_t(pl.from);
        hi = 0x7fffffff;
    }
    const uint32_t head = kvh * R + f - r * R;
    float v[SL];
    {
        const float *qh = at.q + (size_t(row) * gown.H + head) * QK + qd * SL;
#pragma unroll
        for (int e = 0; e < SL; ++e) v[e] = qh[e];
    }
    const uint32_t cap = uint32_t(own ? gown.cap : gp.cap);
    const uint8_t *blk = own ? at.kv + size_t(~un.source) * at.kv_stride : at.pkv + size_t(un.source) * at.pkv_stride;
    const size_t v_off = own ? gown.v_off : gp.v_off, ks_off = own ? gown.ks_off : gp.ks_off;
    const rows_t kb = rows_at(blk + size_t(kvh) * cap * QK, cap * QK);
    const rows_t vb = rows_at(blk + v_off + size_t(kvh) * cap * VD, cap * VD);
    // K scales, and vs_off - ks_off bytes on (KVH cap 4, below 2^32) the V scales
    const uint32_t to_vs = uint32_t((own ? gown.vs_off : gp.vs_off) - ks_off);
    const rows_t sb = rows_at(blk + ks_off + size_t(kvh) * cap * 4, to_vs + cap * 4);
    // the first position that all columns see, and the last
    uint32_t tlo = lo, thi = hi;
    auto both = [&](auto distance) {
        constexpr int D = decltype(distance)::value;
        tlo = max(tlo, uint32_t(ndl::wave_xor_int<D>(int(tlo))));
        thi = min(thi, uint32_t(ndl::wave_xor_int<D>(int(thi))));
    };
    both(std::integral_constant<int, 1>{});
    both(std::integral_constant<int, 2>{});
    both(std::integral_constant<int, 4>{});
    both(std::integral_constant<int, 8>{});
    tlo = __builtin_amdgcn_readfirstlane(tlo);
    thi = __builtin_amdgcn_readfirstlane(thi);

    // ---- the walk: up to the ring's end, then from its start, in chunks of 32 (the
    // last of a part shorter).  It is no longer than the ring, so it wraps once ----
    const uint32_t span = uint32_t(un.span), begin = uint32_t(un.from), slo = begin % cap;
    const uint32_t n0 = min(span, cap - slo), n1 = span - n0;
    const int e0 = int((n0 + 31) / 32), nch = un.end;
    int ch = un.begin + stream;
    uint32_t s0 = 0;   // the chunk's first slot,
    uint32_t p0 = 0;   // its position,
    int left = 0;      // positions from there to the part's end; 0 behind the last chunk
    int stop = 0;      // the part's last chunk, and one
    auto place = [=, &s0, &p0, &left, &stop](int i) {
        const bool second = i >= e0;
        const uint32_t off = 32u * uint32_t(second ? i - e0 : i);
        s0 = i >= nch ? 0u : (second ? 0u : slo) + off;
        p0 = begin + (second ? n0 : 0u) + off;
        left = i >= nch ? 0 : int((second ? n1 : n0) - off);
        stop = second ? nch : min(e0, nch);
    };
    uint32_t kr[2][KD], vr[8];
    float scr = 0.0f;
    const uint32_t kl = uint32_t(n * QK + qd * SL), vl = uint32_t(4 * qd * VD + 4 * n);
    const uint32_t scl = (lane & 31) * 4 + (lane < 32 ? 0u : to_vs);
    // loads of K and V are never conditional: past the last chunk they read some slot
    auto load_k = [&]() {
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
        if (at.negative) {
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
            cf0 = __builtin_amdgcn_ldexpf(qs, sh) * at.scale2;
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
            cf0 = at.scale2;
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
        const bool full = p0 >= tlo && p0 + 31 <= thi && left >= 32;
        uint32_t vis = 0xffffffffu;
        if (!full) {
            vis = left < 32 ? (1u << left) - 1u : 0xffffffffu;
            vis &= lo <= p0 ? 0xffffffffu : lo - p0 < 32u ? 0xffffffffu << (lo - p0) : 0u;
            vis &= hi < p0 ? 0u : hi - p0 < 31u ? (2u << (hi - p0)) - 1u : 0xffffffffu;
        }
        // ---- the chunk's scales, zero behind its end ----
        float sc = (lane & 31) < left ? scr : 0.0f;
        if (any_of(!(__builtin_fabsf(sc) <= top))) {
            // what no column sees may be anything: it sets no unit, and counts as one
            bool unseen = false;
            if (!full) {
                uint32_t seen = vis;
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

    // ---- the sums: a wave's own, or, where waves have shared a tile's chunks, put
    // together by sixteen threads a column ----
    l_run += ndl::wave_xor<16>(l_run);
    l_run += ndl::wave_xor<32>(l_run);
    l_run = ((__float_as_int(cf0) < 0) & (l_run != 0.0f)) ? NAN : l_run;
    // the sums are left as 2^more of what has a weight of 1/2 to 1: of values near
    // fp32's end the sum may be beyond it, the mean is not
    const int more = __builtin_amdgcn_frexp_expf(l_run);
    // (from here on the maximum is in bits; -inf: sums are 0, or NaN where a score was)
    const float mb = m_run == -INFINITY ? -INFINITY : mu, lb = __builtin_amdgcn_ldexpf(l_run, -more);
    const size_t slot = (size_t(un.slot) + mine) * gown.KVH + kvh;
    if (step == 1) {
        // (m + more may be rounded, M with it; m - M is not)
        const float M = mb + float(more), by = mb == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mb - M + float(more));
        float *po = at.part_o + (slot * kCols + n) * VD + 16 * qd;
        // lane (n, qd) holds V columns 16 qd + 4 i + c
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            floatx4_t o;
#pragma unroll
            for (int c = 0; c < 4; ++c) o[c] = __builtin_amdgcn_ldexpf(acc[c][i], vexp - 1 - more) * by;
            *reinterpret_cast<floatx4_t *>(po + 4 * i) = o;
        }
        if (qd == 0) *reinterpret_cast<floatx2_t *>(at.part_ml + (slot * kCols + n) * 2) = floatx2_t{M, lb * by};
        return;
    }
    if (qd == 0) ms[w][n] = floatx4_t{mb, float(more), lb, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        floatx4_t o;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = __builtin_amdgcn_ldexpf(acc[c][i], vexp - 1 - more);
        *reinterpret_cast<floatx4_t *>(&mo[w][n][16 * qd + 4 * i]) = o;
    }
    __syncthreads();
    const int col = t >> 4;
    for (int j = 0; j < wide; ++j) {
        // against a maximum 2^3 above the largest, so that no sum of eight leaves the
        // values' range
        float M = -INFINITY, L = 0.0f;
        floatx4_t O{0.0f, 0.0f, 0.0f, 0.0f};
        for (int i = j; i < NW; i += wide) M = fmaxf(M, ms[i][col][0] + ms[i][col][1]);
        M += 3.0f;
        for (int i = j; i < NW; i += wide) {
            const floatx4_t z = ms[i][col];
            const float by = z[0] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(z[0] - M + z[1]);
            L += z[2] * by;
            O += *reinterpret_cast<const floatx4_t *>(&mo[i][col][4 * (t & 15)]) * by;
        }
        const size_t to = ((size_t(un.slot) + j) * gown.KVH + kvh) * kCols + col;
        *reinterpret_cast<floatx4_t *>(at.part_o + to * VD + 4 * (t & 15)) = O;
        if ((t & 15) == 0) *reinterpret_cast<floatx2_t *>(at.part_ml + to * 2) = floatx2_t{M, L};
    }
}

// The sums of a (row, head) meet: a wave each, a lane a run of chunks, then a lane a
// column.
__global__ __launch_bounds__(256) void prefix_join_kernel(Attend at, uint32_t first, uint32_t total)
{
    const uint32_t oh = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (oh >= total) return;
    const int lane = threadIdx.x & 63;
    const uint32_t H = uint32_t(at.z.H), R = H / uint32_t(at.z.KVH), down = oh / H;
    const uint32_t row = first + down, head = oh - down * H, kvh = head / R, r = head - kvh * R;
    const uint32_t i = row / at.z.rows, n = row - i * at.z.rows;
    float *out = at.out + (size_t(row) * H + head) * VD + lane;
    if (!made_for(*at.plan.head(), at.z)) {
        *out = NAN;
        return;
    }
    const Session s = at.plan.session()[i];
    if (int(n) >= s.there) return;
    if (s.bad) {
        *out = NAN;
        return;
    }
    const uint32_t fp = (uint32_t(s.at) + n) * R + r, fo = n * R + r;
    Quad qp{}, qo = at.plan.quad()[uint32_t(s.quads) + fo / (4 * kCols)];
    if (s.prefix >= 0) qp = at.plan.quad()[uint32_t(at.plan.group()[s.prefix].quads) + fp / (4 * kCols)];
    const int all = qp.runs + qo.runs;
    float M = -INFINITY, L = 0.0f, O = 0.0f;
    for (int j0 = 0; j0 < all; j0 += 64) {
        const int j = j0 + lane, many = min(64, all - j0);
        const bool old = j < qp.runs;
        const uint32_t f = old ? fp : fo;
        size_t to = 0;
        float m = -INFINITY, l = 0.0f;
        if (j < all) {
            const uint32_t slot = (old ? uint32_t(qp.slot + j * qp.wide) : uint32_t(qo.slot + (j - qp.runs) * qo.wide)) +
                                  f / kCols % 4;
            to = (size_t(slot) * at.z.KVH + kvh) * kCols + f % kCols;
            m = at.part_ml[2 * to];
            l = at.part_ml[2 * to + 1];
        }
        // (a NaN among the weights is one of L; M is a number or -inf)
        const float top = fmaxf(M, wave_max(m)), by = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top);
        const float was = M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - top);
        M = top;
        // as means of what is there, so that no sum leaves the values' range
        const float part = l * by, now = L * was, sum = now + wave_sum(part);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        O *= now * inv;
        for (int e = 0; e < many; ++e) {
            const uint32_t a0 = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(to)), e));
            const uint32_t a1 = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(to >> 32)), e));
            const float b = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(by * inv), e));
            O += at.part_o[(size_t(a1) << 32 | a0) * VD + lane] * b;
        }
        L = sum;
    }
    *out = L != L ? NAN : O;
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

size_t partial_floats(const Sizes &z) { return size_t(layout_of(z).slots) * z.KVH * kCols * (VD + 2); }

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
    return partial_floats(sizes_of(g, 1, count, rows, prefixes)) * sizeof(float);
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
    a.by_rep = Divisor::of(uint32_t(g->num_heads / g->num_kv_heads));
    a.scale2 = scale == scale ? float(double(scale < 0 ? -scale : scale) * 1.4426950408889634) : -1.0f;
    a.negative = scale < 0;
    void *ws = nullptr;
    if (int rc = nd::call_workspace(ctx, partial_floats(a.z) * sizeof(float), work, work_bytes, &ws)) return rc;
    a.part_o = static_cast<float *>(ws);
    a.part_ml = a.part_o + size_t(a.plan.l.slots) * a.z.KVH * kCols * VD;
    nd_kv_geom pg = *g;
    pg.cap = a.z.pcap;
    auto *fn = g->qk_head_dim == 48 ? (quant_query ? prefix_kernel<48, true> : prefix_kernel<48, false>)
                                    : (quant_query ? prefix_kernel<64, true> : prefix_kernel<64, false>);
    hipLaunchKernelGGL(fn, dim3(a.plan.l.units, unsigned(g->num_kv_heads)), dim3(256), 0, ctx->stream, make_geom(g),
                       make_geom(&pg), a);
    if (int rc = nd::check_launch("attend_prefix_i8")) return rc;
    // HIP counts a launch's threads in 32 bits: rows beyond that go in further launches
    const size_t step = (size_t(1) << 25) / size_t(g->num_heads);
    for (size_t first = 0; first < count * rows; first += step) {
        const uint32_t total = uint32_t(std::min(step, count * rows - first) * g->num_heads);
        hipLaunchKernelGGL(prefix_join_kernel, dim3((total + 3) / 4), dim3(256), 0, ctx->stream, a, uint32_t(first), total);
        if (int rc = nd::check_launch("prefix_join")) return rc;
    }
    return ND_OK;
}

}  // extern "C"
