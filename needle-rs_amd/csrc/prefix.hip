// A batch that shares its prompts: the rows of a step laid out from the requests'
// lengths, and attention over prefixes that are held once and over the sessions'
// own blocks.
//
// A (row, head)'s positions lie in two sources, its prefix's block and its session's:
//   out = sum_s 2^(x_s - M) V_s / sum_s 2^(x_s - M),  x_s = scale log2(e) q . K_s
// A sum over any part of them is three numbers' worth: its own M, the weights' sum and
// the 64 weighted sums of V, and parts meet by M = max M_i, each times 2^(M_i - M).  So
// the rows of all sessions behind a prefix are columns of one matrix product over it:
// its codes are read for 16 columns at a time (a tile), or for 64 (four tiles together),
// and only the sessions' own blocks are read row by row.
//
// What bounds it (MI355X; a call, both kernels):
//   512 rows of 12 heads over 2 behind 8000 positions, fp32 queries: 48 us.  Vector
//     instructions: about 100 for a chunk of 512 scores (8 exponentials, 16 to split the
//     weights, 20 to turn the wave's share of K and V, 24 for scores and weights), of
//     which 20 more cost 3 us; 14 matrix products of 16 cycles lie beside them.
//   200 sessions of 12 x 64 heads, 500 own positions each, seven prompts: 50 us, 168 MB
//     at 3.4 TB/s (at 3.7 in the first kernel's 45); a large copy would take 35.
//   64 sessions behind 2000 positions, query codes: 12.5 us, of which 8.7 are the first
//     kernel, one pass through memory and four chunks a wave, and 4 the join's.
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
// Attention is done in units, a wave each: a column tile (16 (row, head) pairs of a kv
// head) of one source -- a prefix, for all rows of its group, or a session's own block
// -- and a run of its chunks of 32 positions, as long as leaves about kWaves waves
// whatever the requests' lengths are.  A unit leaves its sums in a slot of its own
// number.  A prefix's units are numbered so that a block's four take four tiles over
// the same chunks: unit base + 4 q runs + k w + j is run k of tile 4 q + j, w the
// tiles of quad q.
constexpr int kPlanMagic = 0x6e645031;
// Kernel times: with half as many waves 512 rows behind 8000 positions 46 -> 54 us, with
// twice as many 24 x 33 rows 26 -> 28 and their join 7.5 -> 9.3; with 3600, a card not quite
// full, 200 rows of 12 x 64 45 -> 42 (the last 14 blocks of a full one begin when others end),
// but 512 rows 46 -> 49 and 24 x 33 rows 25 -> 26.5.  With runs of 2 chunks 64
// rows 10.4 -> 11.4 and their join 4.3 -> 5.8, of 8 128 rows in windows 15 -> 17.
constexpr uint32_t kWaves = 4096;  // four a SIMD
constexpr uint32_t kLeast = 4;     // chunks a wave, at least
constexpr uint32_t kExtra = 3;     // what a unit costs beside its chunks, in chunks

struct Head {
    int magic, count, rows, prefixes, heads, kv_heads, cap, prefix_cap;
    int units, window, pad[6];
};

struct Place {
    int row, from;
};

// Where the sums of a row's heads are: their source's first unit, its runs and its
// tiles, and the column of the row's first head.
struct Seat {
    int unit, runs, tiles, column;
};

struct Seats {
    Seat prefix, own;
    int is, pad[7];  // 0: there, 1: bad, -1: not there
};

struct Unit {
    int source, tile, rows, first;  // prefix, or ~session; its rows, the first one's place
    int run, runs, from, span;      // chunks run, run + runs, .. of the positions from .. from + span - 1
    int used, chunks, pad[6];       // own: positions before the step; chunks of the span
};

struct Layout {
    size_t seat, place, unit, bytes;  // offsets
    uint32_t units;                   // at most
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
    // a tile's last run may be short, the full ones come to kWaves / KVH
    l.units = uint32_t((z.prefixes ? all + 4 * z.prefixes : 0) + z.count * own + std::max<uint32_t>(1, kWaves / uint32_t(z.KVH)));
    l.units = (l.units + 3) & ~3u;
    const size_t rows = size_t(z.count) * z.rows;
    l.seat = sizeof(Head);
    l.place = l.seat + rows * sizeof(Seats);
    l.unit = nd::align_up(l.place + rows * sizeof(Place), 64);
    l.bytes = l.unit + l.units * sizeof(Unit);
    return l;
}

struct PlanOf {
    uint8_t *p;
    Layout l;
    __host__ __device__ Head *head() const { return reinterpret_cast<Head *>(p); }
    __host__ __device__ Seats *seat() const { return reinterpret_cast<Seats *>(p + l.seat); }
    __host__ __device__ Place *place() const { return reinterpret_cast<Place *>(p + l.place); }
    __host__ __device__ Unit *unit() const { return reinterpret_cast<Unit *>(p + l.unit); }
};

struct Requests {
    const int32_t *prefix_of, *prefix_len, *used, *length;
    int window;
};

// One session's numbers, as they are given and as they are meant.
struct Given {
    int prefix, used, length;
};

struct Want {
    int there, bad, prefix, used, prefix_len, from, lo, span;
    __device__ int rows() const { return bad ? 0 : there; }
};

__device__ inline Given given_of(const Sizes &z, const Requests &r, uint32_t i)
{
    return Given{r.prefix_of ? r.prefix_of[i] : z.prefixes ? 0 : -1, r.used[i], r.length ? r.length[i] : int(z.rows)};
}

__device__ inline Want want_of(const Sizes &z, uint32_t window, const Given &g, const uint32_t *prefix_len)
{
    Want w;
    const bool some = uint32_t(g.prefix) < z.prefixes, fits = uint32_t(g.length) <= z.rows;
    const uint32_t L = some ? prefix_len[g.prefix] : 0, u = uint32_t(g.used), m = fits ? uint32_t(g.length) : z.rows;
    // the first row's window; the others' begin later
    const uint32_t end = L + u + 1, open = window && end > window ? end - window : 0;
    w.there = int(m);
    w.prefix = some ? g.prefix : -1;
    w.used = int(u);
    w.prefix_len = int(L);
    w.from = int(min(open, L));
    w.lo = int(open - min(open, L));
    const uint32_t span = u + m - uint32_t(w.lo);
    w.span = int(span);
    // (L and u below 2^31 each: their sum, and m, do not wrap)
    w.bad = !fits | (g.prefix >= int(z.prefixes)) | (int(u | L) < 0) || L + u > 0x80000000u - m ||
            (m && (span > uint32_t(z.cap) || L - uint32_t(w.from) > uint32_t(z.pcap)));
    return w;
}

// Chunks of 32 positions of a walk from `from`: chunks end at the ring's end.
__host__ __device__ inline uint32_t chunks_of(uint32_t from, uint32_t span, uint32_t cap)
{
    const uint32_t n0 = min(span, cap - (from < cap ? from : from % cap)), n1 = span - n0;
    return (n0 + 31) / 32 + (n1 + 31) / 32;
}

// Runs of `each` (< 2^21) chunks.
__device__ inline uint32_t runs_of(uint32_t chunks, uint32_t each)
{
    return chunks <= each ? uint32_t(chunks > 0) : (chunks + each - 1) / each;
}

constexpr int kPlanSessions = 64;

// The sum of v over the block, and over the threads before this one.
template <int NT>
__device__ inline void block_scan(uint64_t v, uint64_t &before, uint64_t &all, uint64_t *room)
{
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const uint64_t up = ndl::wave_scan(v);
    if (lane == 63) room[w] = up;
    __syncthreads();
    // the waves' (16 at most) in the first lanes
    const uint64_t x = ndl::row_scan(room[lane & (NT / 64 - 1)]);
    before = up - v + (w ? ndl::of_lane(x, w - 1) : 0);
    all = ndl::of_lane(x, NT / 64 - 1);
}

// 4001 sessions of up to 5 rows behind 90 prompts: 12.3 us, 0.9 MB written; 5 sessions:
// 5.7.  Latency: the requests, three scans, and the units one after another.  Blocks of
// 256 threads where they hold every session and prefix (of 1024 there: 6.4 us), of 1024
// for the rest.
//
// A block lays out kPlanSessions sessions, and its share of the prefixes' units.  What
// it has to know of the rest -- the groups, and what the sessions before its own come
// to -- it works out from the requests itself (65535 of them are 64 a thread), so that
// one launch does without a word between blocks.  Whole numbers: the same plan
// whatever the order of the atomics.
template <int NT>
__global__ __launch_bounds__(NT) void plan_kernel(Sizes z, Requests r, PlanOf plan, nd_prefix_maps maps)
{
    constexpr int kMost = NT < 1024 ? NT : int(kMaxPrefixes);
    __shared__ uint32_t rows_s[kMost], from_s[kMost], before_s[kMost], end_s[kMost];
    __shared__ uint32_t first_s[kMost], units_s[kMost];
    __shared__ uint64_t room[2][NT / 64], weight_s;
    __shared__ __align__(16) uint32_t group_s[kPlanSessions];  // prefix and rows of a session
    __shared__ int there_s[kPlanSessions], at_s[kPlanSessions], used_s[kPlanSessions], len_s[kPlanSessions];
    __shared__ uint32_t runs_s[kPlanSessions], unit_s[kPlanSessions], units_at;
    const int t = threadIdx.x, lane = t & 63;
    const uint32_t R = uint32_t(z.H / z.KVH), P = z.prefixes, S = z.count;
    const uint32_t s0 = blockIdx.x * kPlanSessions, s1 = min(S, s0 + kPlanSessions), i0 = s0 + uint32_t(t);
    // this block's sessions, and of all the first kHeld a thread
    constexpr int kHeld = NT < 1024 ? 1 : 4;
    Given held[kHeld], here{-1, 0, 0};
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        held[k] = Given{-1, 0, 0};
        if (uint32_t(t + k * NT) < S) held[k] = given_of(z, r, uint32_t(t + k * NT));
    }
    if (t < kPlanSessions && i0 < s1) here = given_of(z, r, i0);
    for (uint32_t p = t; p < P; p += NT) {
        rows_s[p] = before_s[p] = 0, from_s[p] = 0xffffffffu;
        end_s[p] = uint32_t(r.prefix_len[p]);
    }
    if (t == 0) weight_s = 0, units_at = 0;
    __syncthreads();
    const Want mine = want_of(z, uint32_t(r.window), here, end_s);
    // f of every session before `end`
    auto sessions = [&](uint32_t end, auto f) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (uint32_t(t + k * NT) < end) f(uint32_t(t + k * NT), want_of(z, uint32_t(r.window), held[k], end_s));
        for (uint32_t i = uint32_t(t + kHeld * NT); i < end; i += NT) f(i, want_of(z, uint32_t(r.window), given_of(z, r, i), end_s));
    };
    auto tiles_of = [&](uint32_t rows) { return (rows * R + kCols - 1) / kCols; };
    auto own_chunks = [&](const Want &w) { return chunks_of(uint32_t(w.lo), uint32_t(w.span), uint32_t(z.cap)); };
    auto group_chunks = [&](uint32_t p) { return chunks_of(from_s[p], end_s[p] - from_s[p], uint32_t(z.pcap)); };
    // (at most 8 heads a kv head, so 2^21 tiles or less, of 2^19 + 1 chunks)
    auto add_weight = [&](uint64_t v) {
        v = ndl::last_lane(ndl::wave_scan(v));
        if (lane == 0 && v) atomicAdd(reinterpret_cast<unsigned long long *>(&weight_s), v);
    };

    // ---- the groups, and all walks ----
    uint64_t weight = 0;
    sessions(S, [&](uint32_t i, const Want &w) {
        const uint32_t m = uint32_t(w.rows());
        if (!m) return;
        weight += uint64_t(tiles_of(m)) * (own_chunks(w) + kExtra);
        if (w.prefix < 0) return;
        atomicAdd(&rows_s[w.prefix], m);
        atomicMin(&from_s[w.prefix], uint32_t(w.from));
        if (i < s0) atomicAdd(&before_s[w.prefix], m);
    });
    add_weight(weight);
    __syncthreads();
    weight = 0;
    for (uint32_t p = t; p < P; p += NT)
        if (rows_s[p]) weight += uint64_t(tiles_of(rows_s[p])) * (group_chunks(p) + kExtra);
    add_weight(weight);
    __syncthreads();
    // ---- the length of a run: each wave's share of all chunks, a unit counted as kExtra
    // more for its beginning and end (a run more: no more units than places and tiles).
    // The prefixes' units, the longest, come first, and short ones fill the gaps ----
    const double places = double(max(1u, kWaves / uint32_t(z.KVH)));
    const double share = double(weight_s) / places;
    const uint32_t each = uint32_t(fmin(fmax(share + 1.0, double(kLeast)), 1048576.0));

    // ---- where each group's rows and units begin ----
    uint32_t rows_all = 0, units_all = 0;
    for (uint32_t p0 = 0; p0 < P; p0 += NT) {
        const uint32_t p = p0 + t, rows = p < P ? rows_s[p] : 0;
        const uint32_t units = rows ? (tiles_of(rows) * runs_of(group_chunks(p), each) + 3) & ~3u : 0;
        uint64_t at, all;
        if (p0) __syncthreads();
        block_scan<NT>(uint64_t(rows) << 32 | units, at, all, room[0]);
        if (p < P) {
            first_s[p] = rows_all + uint32_t(at >> 32);
            units_s[p] = units_all + uint32_t(at);
            if (blockIdx.x == 0 && maps.first) maps.first[p] = int(first_s[p]);
        }
        rows_all += uint32_t(all >> 32);
        units_all += uint32_t(all);
    }
    if (blockIdx.x == 0 && t == 0 && maps.first) maps.first[P] = int(rows_all);

    // ---- what the sessions before this block's come to, and all ----
    uint32_t sum = 0;
    sessions(blockIdx.x ? s0 : S, [&](uint32_t, const Want &w) {
        const uint32_t m = uint32_t(w.rows());
        if (m) sum += tiles_of(m) * runs_of(own_chunks(w), each);
    });
    sum = ndl::last_lane(ndl::wave_scan(sum));
    if (lane == 0) atomicAdd(&units_at, sum);

    // ---- this block's sessions ----
    const uint32_t m = uint32_t(mine.rows()), tiles = tiles_of(m), chunks = m ? own_chunks(mine) : 0;
    const uint32_t runs = runs_of(chunks, each);
    if (t < kPlanSessions) group_s[t] = m && mine.prefix >= 0 ? uint32_t(mine.prefix) << 16 | m : 0xffff0000u;
    uint64_t at, all;
    block_scan<NT>(tiles * runs, at, all, room[1]);  // (a barrier: units_at, group_s)
    const uint32_t units0 = units_all + (blockIdx.x ? units_at : 0);
    if (blockIdx.x == 0 && t == 0)
        *plan.head() = Head{kPlanMagic, int(z.count), int(z.rows), int(P), z.H, z.KVH, z.cap, z.pcap,
                            int(units_all + units_at), r.window, {}};
    // a session's place among those of its prefix: four threads each
    if (t < 4 * kPlanSessions) {
        constexpr int kShare = 4;
        const int j = t / kShare, part = t % kShare, last = min(j | (64 / kShare - 1), int(s1 - s0) - 1);
        const uint32_t key = group_s[j] >> 16;
        uint32_t rank = 0;
        // (to the wave's last session, alike in all lanes: `last` is)
        for (int i = 4 * part; i <= last; i += 4 * kShare) {
            const uint4 g = *reinterpret_cast<const uint4 *>(&group_s[i]);
            const uint32_t gg[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) rank += i + e < j && gg[e] >> 16 == key ? gg[e] & 0xffffu : 0u;
        }
        rank += uint32_t(ndl::wave_xor_int<1>(int(rank)));
        rank += uint32_t(ndl::wave_xor_int<2>(int(rank)));
        if (part == 0) at_s[j] = int(rank);
    }
    __syncthreads();
    if (t < kPlanSessions && i0 < s1) {
        const uint32_t rank = (mine.prefix >= 0 ? before_s[mine.prefix] : 0) + uint32_t(at_s[t]);
        uint32_t unit = units0 + uint32_t(at);
        runs_s[t] = runs;
        unit_s[t] = unit;
        for (uint32_t q = 0; 4 * q < tiles; ++q)
            for (uint32_t k = 0; k < runs; ++k)
                for (uint32_t j = 4 * q; j < min(tiles, 4 * q + 4); ++j)
                    plan.unit()[unit++] = Unit{~int(i0), int(j), int(m), 0, int(k), int(runs),
                                               mine.lo, mine.span, mine.used, int(chunks), {}};
        there_s[t] = mine.bad ? ~mine.there : mine.there;
        at_s[t] = int(rank);
        used_s[t] = mine.used;
        len_s[t] = mine.prefix_len;
    }
    __syncthreads();

    // ---- their rows, and what lies behind the last of the order ----
    const uint32_t N = z.rows, total = (s1 > s0 ? s1 - s0 : 0) * N;
    for (uint32_t k = t; k < total; k += NT) {
        const uint32_t j = k / N, n = k - j * N, p = group_s[j] >> 16;
        const int row = int(s0 * N + k);
        int pos = -1, rot = -1, from = -1, lo = -1;
        Seats seats{};
        const bool bad = there_s[j] < 0;
        seats.is = bad && int(n) < ~there_s[j] ? 1 : -1;
        if (!bad && int(n) < there_s[j]) {
            // (the row's place in the whole is below 2^31)
            const int end = len_s[j] + used_s[j] + int(n), open = r.window ? max(end - r.window + 1, 0) : 0;
            pos = used_s[j] + int(n);
            rot = end;
            from = min(open, len_s[j]);
            lo = max(open - len_s[j], 0);
            if (p < P) {
                const uint32_t to = first_s[p] + uint32_t(at_s[j]) + n;
                plan.place()[to] = Place{row, from};
                if (maps.order) maps.order[to] = row;
                seats.prefix = Seat{int(units_s[p]), int(runs_of(group_chunks(p), each)), int(tiles_of(rows_s[p])),
                                    int((uint32_t(at_s[j]) + n) * R)};
            }
            seats.own = Seat{int(unit_s[j]), int(runs_s[j]), int(tiles_of(uint32_t(there_s[j]))), int(n * R)};
            seats.is = 0;
        }
        plan.seat()[row] = seats;
        if (maps.pos) maps.pos[row] = pos;
        if (maps.rot) maps.rot[row] = rot;
        if (maps.from) maps.from[row] = from;
        if (maps.lo) maps.lo[row] = lo;
    }
    const uint32_t thread = blockIdx.x * NT + t, threads = gridDim.x * NT;
    if (maps.order)
        for (uint32_t k = rows_all + thread; k < S * N; k += threads) maps.order[k] = -1;

    // ---- the groups' units, over all blocks ----
    for (uint32_t k = thread; k < units_all; k += threads) {
        uint32_t p = 0;  // the last group that begins at or before k
        for (uint32_t d = kMost / 2; d; d /= 2)
            if (p + d < P && units_s[p + d] <= k) p += d;
        const uint32_t i = k - units_s[p], rows = rows_s[p], tiles = tiles_of(rows), chunks = group_chunks(p);
        const uint32_t runs = runs_of(chunks, each), full = tiles / 4, rest = tiles % 4;
        uint32_t run = 0, tile = tiles;  // (past the last: a unit of no tile)
        if (i < 4 * full * runs) {
            const uint32_t q = i / (4 * runs);
            run = (i - q * 4 * runs) / 4;
            tile = 4 * q + i % 4;
        } else if (i < tiles * runs) {
            run = (i - 4 * full * runs) / rest;
            tile = 4 * full + (i - 4 * full * runs) % rest;
        }
        plan.unit()[k] = Unit{int(p), int(tile), int(rows), int(first_s[p]), int(run), int(runs),
                              int(from_s[p]), int(end_s[p] - from_s[p]), 0, int(chunks), {}};
    }
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

// Operands of a chunk that a block's waves share (of an fp32 query), twice: one is read
// while the next one is laid down.  K as f16, 16 positions after 16; V as f16, column
// 4 n + c of eight positions a lane.
struct Shared {
    uint32_t k[2][4][64][4], v[2][4][64][4];
};

template <int QK, bool QQ, bool TOGETHER>
__device__ __forceinline__ void walk(const Geom &gown, const Geom &gp, const Attend &at, const Head &hd, const Unit &un,
                                     uint32_t unit, uint32_t kvh, float *sc_s, Shared *sh_s)
{
    static_assert(!(QQ && TOGETHER), "of query codes each wave reads K for itself");
    constexpr int SL = QK / 4, KD = SL / 4;  // a lane's slice of a K row; its dwords (3 or 4)
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n = lane & 15, qd = lane >> 4;
    const uint32_t R = uint32_t(gown.H / gown.KVH);
    const bool own = !TOGETHER && un.source < 0;
    const uint32_t ncols = uint32_t(un.rows) * R, tile = uint32_t(un.tile);

    const uint32_t f = min(tile * kCols + uint32_t(n), ncols - 1), r = at.by_rep.quotient(f);
    Place pl{};
    if (!own) pl = at.plan.place()[uint32_t(un.first) + r];
    const uint32_t cap = uint32_t(own ? gown.cap : gp.cap);
    const uint8_t *blk = own ? at.kv + size_t(~un.source) * at.kv_stride : at.pkv + size_t(un.source) * at.pkv_stride;
    const size_t v_off = own ? gown.v_off : gp.v_off, ks_off = own ? gown.ks_off : gp.ks_off;
    const rows_t kb = rows_at(blk + size_t(kvh) * cap * QK, cap * QK);
    const rows_t vb = rows_at(blk + v_off + size_t(kvh) * cap * VD, cap * VD);
    // K scales, and vs_off - ks_off bytes on (KVH cap 4, below 2^32) the V scales
    const uint32_t to_vs = uint32_t((own ? gown.vs_off : gp.vs_off) - ks_off);
    const rows_t sb = rows_at(blk + ks_off + size_t(kvh) * cap * 4, to_vs + cap * 4);
    // ---- the walk: up to the ring's end, then from its start, in chunks of 32 (the
    // last of a part shorter).  It is no longer than the ring, so it wraps once ----
    const uint32_t span = uint32_t(un.span), begin = uint32_t(un.from), slo = begin % cap;
    const uint32_t n0 = min(span, cap - slo), n1 = span - n0;
    const int e0 = int((n0 + 31) / 32), nch = un.chunks, step = un.runs;
    struct Chunk {
        int ch, left, stop;  // its number; positions from p0 to the part's end, 0 behind the last; the part's last and one
        uint32_t s0, p0;     // its first slot and position
    } now, ahead;            // that whose scores come next, and together the one whose K and V do
    auto put = [=](Chunk &c, int i) {
        const bool second = i >= e0;
        const uint32_t off = 32u * uint32_t(second ? i - e0 : i);
        c.ch = i;
        c.s0 = i >= nch ? 0u : (second ? 0u : slo) + off;
        c.p0 = begin + (second ? n0 : 0u) + off;
        c.left = i >= nch ? 0 : int((second ? n1 : n0) - off);
        c.stop = second ? nch : min(e0, nch);
    };
    auto next = [=](Chunk &c) {
        if (c.ch + step < c.stop) [[likely]] {
            c.ch += step;
            c.s0 += 32u * uint32_t(step);
            c.p0 += 32u * uint32_t(step);
            c.left -= 32 * step;
        } else {
            asm volatile("");  // (a branch, not thirty selects in every chunk)
            put(c, c.ch + step);
        }
    };
    // alone: a wave's K rows and V; together: the part that it lays down for all, K
    // dwords of half `w & 1` of 16 positions `w >> 1`, V of positions 2 w, 2 w + 1 of
    // every eight
    uint32_t kr[2][KD], vr[TOGETHER ? 2 : 8];
    float scr = 0.0f;
    const uint32_t kl = TOGETHER ? uint32_t((16 * (w >> 1) + n) * QK + qd * SL + 8 * (w & 1)) : uint32_t(n * QK + qd * SL);
    const uint32_t vl = uint32_t((4 * qd + (TOGETHER ? 16 * (w >> 1) + 2 * (w & 1) : 0)) * VD + 4 * n);
    const uint32_t scl = (lane & 31) * 4 + (lane < 32 ? 0u : to_vs);
    // loads of K and V are never conditional: past the last chunk they read some slot
    auto load_k = [&](uint32_t s0) {
        const uint32_t o = here(kl + s0 * QK);
        if constexpr (TOGETHER) {
            if (KD == 3 && (w & 1)) {
                kr[0][0] = __builtin_amdgcn_raw_buffer_load_b32(kb, o, 0, 0);
            } else {
                const auto r = __builtin_amdgcn_raw_buffer_load_b64(kb, o, 0, 0);
                kr[0][0] = r[0], kr[0][1] = r[1];
            }
        } else {
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
        }
    };
    auto load_scales = [&](uint32_t s0) {
        scr = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(sb, scl + s0 * 4, 0, 0));
    };
    auto load_v = [&](uint32_t s0) {
        const uint32_t o = here(vl + s0 * VD);
#pragma unroll
        for (int j = 0; j < (TOGETHER ? 2 : 8); ++j)
            vr[j] = __builtin_amdgcn_raw_buffer_load_b32(vb, o + (16 * (j >> 2) + (j & 3)) * VD, 0, 0);
    };
    // the wave's part into buffer `to`
    auto lay_down = [&](int to) {
        u32x4_t *kk = reinterpret_cast<u32x4_t *>(sh_s->k[to][w][lane]);
        const uint32_t u0 = kr[0][0] ^ 0x80808080u;
        if (KD == 3 && (w & 1)) {  // (twice: the product that takes both pieces of the query)
            *kk = vec4<u32x4_t>(f16_pair<0>(u0), f16_pair<1>(u0), f16_pair<0>(u0), f16_pair<1>(u0));
        } else {
            const uint32_t u1 = kr[0][1] ^ 0x80808080u;
            *kk = vec4<u32x4_t>(f16_pair<0>(u0), f16_pair<1>(u0), f16_pair<0>(u1), f16_pair<1>(u1));
        }
        const uint32_t v0 = vr[0] ^ 0x80808080u, v1 = vr[1] ^ 0x80808080u;
        sh_s->v[to][0][lane][w] = f16_codes<0>(v0, v1);
        sh_s->v[to][1][lane][w] = f16_codes<1>(v0, v1);
        sh_s->v[to][2][lane][w] = f16_codes<2>(v0, v1);
        sh_s->v[to][3][lane][w] = f16_codes<3>(v0, v1);
    };
    // all waves' parts are there, and read
    auto meet = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };
    put(now, un.run);
    load_k(now.s0);
    load_scales(now.s0);
    load_v(now.s0);

    // ---- the wave's columns: what they see, and the query operand, asked for while
    // the first chunk is on its way.  A column past the end is a copy of the last ----
    uint32_t row, lo, hi;
    if (own) {
        const uint32_t end = uint32_t(un.used) + r;  // the row's own position, below 2^31
        row = uint32_t(~un.source) * at.z.rows + r;
        lo = hd.window && end + 1 > uint32_t(hd.window) ? end + 1 - uint32_t(hd.window) : 0;
        hi = end;
    } else {
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
    // the first position that all columns see, and the last
    uint32_t tlo = lo, thi = hi;
    auto both = [&](auto distance) {
        constexpr int D = decltype(distance)::value;
        tlo = max(tlo, uint32_t(ndl::wave_xor_int<D>(int(tlo))));
        if constexpr (!TOGETHER) thi = min(thi, uint32_t(ndl::wave_xor_int<D>(int(thi))));
    };
    both(std::integral_constant<int, 1>{});
    both(std::integral_constant<int, 2>{});
    both(std::integral_constant<int, 4>{});
    both(std::integral_constant<int, 8>{});
    tlo = __builtin_amdgcn_readfirstlane(tlo);
    thi = __builtin_amdgcn_readfirstlane(thi);

    // ---- the query operand, while the first chunk is on its way ----
    float cf0;                        // factor of a score, in bits, is |cf0| 2^(kexp - sh)
    int sh;
    intx4_t qi;                       // QQ: codes
    uint32_t qp[2][8];                // else: f16 pieces
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
        float nan = 0.0f;  // or NaN: of a NaN or an infinity
#pragma unroll
        for (int e = 0; e < SL; ++e) nan = __builtin_fmaf(v[e], 0.0f, nan);
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

    int buf = 0;
    if constexpr (TOGETHER) {
        lay_down(0);
        ahead = now;
        next(ahead);
        load_k(ahead.s0);
        load_v(ahead.s0);
        meet();
    }
    while (now.ch < nch) {
        const uint32_t p0 = now.p0;
        const int left = now.left;
        // ---- the positions each column sees ----
        const bool full = p0 >= tlo && left >= 32 && (TOGETHER || p0 + 31 <= thi);  // (thi of a prefix: all)
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
        sc_s[lane] = sc;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        floatx4_t ks[2], vs[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            ks[a] = *reinterpret_cast<const floatx4_t *>(&sc_s[16 * a + 4 * qd]);
            vs[a] = *reinterpret_cast<const floatx4_t *>(&sc_s[32 + 16 * a + 4 * qd]);
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
                uint32_t kp[8];  // qk 48: the last two twice
                if constexpr (TOGETHER) {
                    const u32x4_t lo4 = *reinterpret_cast<const u32x4_t *>(sh_s->k[buf][2 * a][lane]);
                    kp[0] = lo4[0], kp[1] = lo4[1], kp[2] = lo4[2], kp[3] = lo4[3];
                    const u32x4_t hi4 = *reinterpret_cast<const u32x4_t *>(sh_s->k[buf][2 * a + 1][lane]);
                    kp[4] = hi4[0], kp[5] = hi4[1], kp[6] = hi4[2], kp[7] = hi4[3];
                } else {
#pragma unroll
                    for (int d = 0; d < KD; ++d) {
                        const uint32_t u = kr[a][d] ^ 0x80808080u;
                        kp[2 * d] = f16_pair<0>(u);
                        kp[2 * d + 1] = f16_pair<1>(u);
                    }
                    if constexpr (KD == 3) kp[6] = kp[4], kp[7] = kp[5];
                }
                floatx4_t d{0.0f, 0.0f, 0.0f, 0.0f};
                auto add = [&](uint32_t k0, uint32_t k1, uint32_t k2, uint32_t k3, uint32_t q0, uint32_t q1,
                               uint32_t q2, uint32_t q3) {
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(vec4<f16x8_t>(k0, k1, k2, k3),
                                                               vec4<f16x8_t>(q0, q1, q2, q3), d, 0, 0, 0);
                };
                const uint32_t *qh = qp[0], *ql = qp[1];
                // the small pieces first; of qk 48 a lane's last four codes meet both
                // pieces in one product
                if constexpr (KD == 4) add(kp[4], kp[5], kp[6], kp[7], ql[4], ql[5], ql[6], ql[7]);
                add(kp[0], kp[1], kp[2], kp[3], ql[0], ql[1], ql[2], ql[3]);
                if constexpr (KD == 3)
                    add(kp[4], kp[5], kp[6], kp[7], ql[4], ql[5], qh[4], qh[5]);
                else
                    add(kp[4], kp[5], kp[6], kp[7], qh[4], qh[5], qh[6], qh[7]);
                add(kp[0], kp[1], kp[2], kp[3], qh[0], qh[1], qh[2], qh[3]);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[4 * a + i] = d[i] * ks[a][i];
            }
        }
        // the next chunk: its K lands during the softmax and the values; together, it has
        // landed, and the one after it does
        next(now);
        load_scales(now.s0);
        if constexpr (TOGETHER) {
            lay_down(buf ^ 1);
            next(ahead);
            load_k(ahead.s0);
            load_v(ahead.s0);
        } else {
            load_k(now.s0);
        }
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
                for (int c = 0; c < 4; ++c) {
                    float code;
                    if constexpr (TOGETHER)
                        code = float(reinterpret_cast<const _Float16 *>(sh_s->v[buf][c][lane])[j]);
                    else
                        code = i8_at(vr[j], c) * 0x1p-9f;
                    acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(code, wt[j], acc[c], 0, 0, 0);
                }
#pragma unroll
            for (int j = 0; j < 8; ++j) wt[j] = 0.0f;
        }
        {
            uint32_t ph[4], pl[4], u[TOGETHER ? 2 : 8];
#pragma unroll
            for (int j = 0; j < 4; ++j) split2(wt[2 * j], wt[2 * j + 1], ph[j], pl[j]);
            if constexpr (!TOGETHER) {
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] = vr[j] ^ 0x80808080u;
            }
            auto column = [&](auto cc) {
                constexpr int c = decltype(cc)::value;
                f16x8_t vf;
                if constexpr (TOGETHER)
                    vf = *reinterpret_cast<const f16x8_t *>(sh_s->v[buf][c][lane]);
                else
                    vf = vec4<f16x8_t>(f16_codes<c>(u[0], u[1]), f16_codes<c>(u[2], u[3]), f16_codes<c>(u[4], u[5]),
                                       f16_codes<c>(u[6], u[7]));
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
        if constexpr (TOGETHER) {
            meet();
            buf ^= 1;
        } else {
            load_v(now.s0);  // lands during the next scores
        }
    }

    // ---- the sums ----
    l_run += ndl::wave_xor<16>(l_run);
    l_run += ndl::wave_xor<32>(l_run);
    l_run = ((__float_as_int(cf0) < 0) & (l_run != 0.0f)) ? NAN : l_run;
    // left as 2^more of what has a weight of 1/2 to 1: of values near fp32's end the
    // sum may be beyond it, the mean is not
    const int more = __builtin_amdgcn_frexp_expf(l_run);
    // (from here on the maximum is in bits; -inf: sums are 0, or NaN where a score was.
    // m + more may be rounded, M with it; m - M is not)
    const float mb = m_run == -INFINITY ? -INFINITY : mu, M = mb + float(more);
    const float by = mb == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mb - M + float(more));
    const size_t to = (size_t(unit) * gown.KVH + kvh) * kCols + n;
    float *po = at.part_o + to * VD + 16 * qd;
    // lane (n, qd) holds V columns 16 qd + 4 i + c
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        floatx4_t o;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = __builtin_amdgcn_ldexpf(acc[c][i], vexp - 1 - more) * by;
        *reinterpret_cast<floatx4_t *>(po + 4 * i) = o;
    }
    if (qd == 0)
        *reinterpret_cast<floatx2_t *>(at.part_ml + to * 2) = floatx2_t{M, __builtin_amdgcn_ldexpf(l_run, -more) * by};
}

// A block's four units, each for itself: a wave turns its chunk's K and V into operands
// in its registers.  Or, of four tiles of a prefix over the same chunks, together: a wave
// turns a quarter of them, in LDS, and reads all back, two buffers in turn (four, and a
// meeting every other chunk: the same time).  512 rows over 2 kv heads, fp32 queries, together
// and alone (us): runs of 7 chunks 20.6, 19.3; 12 26.4, 27.0; 16 31.6, 33.1; 26 46.2, 50.3.
// Of query codes K needs no turning, and V's alone is not worth the meetings: 7 20.1, 18.3;
// 16 30.1, 29.8; 26 43.7, 43.8.
constexpr int kTogether = 10;  // chunks of a run

template <int QK, bool QQ>
__global__ __launch_bounds__(256, 4) void prefix_kernel(Geom gown, Geom gp, Attend at, uint32_t first)
{
    __shared__ __align__(16) float sc_s[4][64];
    const uint32_t w = uint32_t(__builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)));
    const uint32_t unit = 4 * (first + blockIdx.y) + w, kvh = blockIdx.x;
    // (both asked for at once: the list has as many places as the grid waves)
    const Head hd = *at.plan.head();
    const Unit un = at.plan.unit()[unit];
    if (!made_for(hd, at.z) || int(unit) >= hd.units) return;
    const uint32_t ncols = uint32_t(un.rows) * uint32_t(gown.H / gown.KVH), tile = uint32_t(un.tile);
    if (tile * kCols >= ncols) return;
    if constexpr (!QQ) {
        __shared__ __align__(16) Shared sh_s;
        // (a prefix's first unit is a multiple of four, and its full quads come first.  One
        // condition: as three branches the 46 us of the largest step are 48)
        if (int(un.source >= 0) & int((tile | 3) * kCols < ncols) & int(un.chunks >= kTogether * un.runs))
            walk<QK, QQ, true>(gown, gp, at, hd, un, unit, kvh, sc_s[w], &sh_s);
        else
            walk<QK, QQ, false>(gown, gp, at, hd, un, unit, kvh, sc_s[w], nullptr);
    } else {
        walk<QK, QQ, false>(gown, gp, at, hd, un, unit, kvh, sc_s[w], nullptr);
    }
}

constexpr int kAtOnce = 8;

// The sums of a (row, head) meet: a wave each, a lane a run of chunks, then a lane a
// column.  Four dependent reads, 3 to 7.5 us a call; the first sums are asked for ahead of
// their weights (one row of 8 runs: 3.9 -> 3.0 us).
__global__ __launch_bounds__(256) void prefix_join_kernel(Attend at, uint32_t first, uint32_t total)
{
    const uint32_t oh = blockIdx.x * 4 + uint32_t(__builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)));
    if (oh >= total) return;
    const int lane = threadIdx.x & 63;
    const uint32_t H = uint32_t(at.z.H), R = H / uint32_t(at.z.KVH), down = oh / H;
    const uint32_t row = first + down, head = oh - down * H, kvh = at.by_rep.quotient(head), r = head - kvh * R;
    float *out = at.out + (size_t(row) * H + head) * VD;
    const Head hd = *at.plan.head();
    const Seats seats = at.plan.seat()[row];
    if (!made_for(hd, at.z) || seats.is > 0) {
        out[lane] = NAN;
        return;
    }
    if (seats.is < 0) return;
    // the first run's sums, their number and how far apart they are (slots)
    uint32_t to[2], apart[2];
    int runs[2];
    auto find = [&](const Seat &s, int i) {
        const uint32_t f = uint32_t(s.column) + r, tile = f / kCols, q4 = tile & ~3u;
        runs[i] = s.runs;
        apart[i] = min(uint32_t(s.tiles) - q4, 4u) * uint32_t(at.z.KVH) * kCols;
        to[i] = ((uint32_t(s.unit) + q4 * uint32_t(s.runs) + (tile - q4)) * uint32_t(at.z.KVH) + kvh) * kCols + f % kCols;
    };
    find(seats.prefix, 0);
    find(seats.own, 1);
    const int all = runs[0] + runs[1];
    float M = -INFINITY, L = 0.0f, O = 0.0f;
    const float *own = at.part_o + size_t(to[1]) * VD, *po = runs[0] ? at.part_o + size_t(to[0]) * VD : own;
    size_t step = size_t(apart[runs[0] ? 0 : 1]) * VD;
    int left = runs[0];  // of the prefix
    for (int j0 = 0; j0 < all; j0 += 64) {
        const int j = j0 + lane, many = min(64, all - j0);
        // the sums of run e of these (the prefix's, then the own ones), eight a time; the
        // first are asked for ahead of what they are multiplied by
        float o[kAtOnce] = {};
        auto load = [&](int e0) {
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                if (j0 + e0 + k >= min(all, j0 + 64)) break;
                o[k] = po[lane];
                po += step;
                if (--left == 0) po = own, step = size_t(apart[1]) * VD;
            }
        };
        load(0);
        float m = -INFINITY, l = 0.0f;
        if (j < all) {
            const size_t p = j < runs[0] ? to[0] + size_t(j) * apart[0] : to[1] + size_t(j - runs[0]) * apart[1];
            const floatx2_t ml = *reinterpret_cast<const floatx2_t *>(at.part_ml + 2 * p);
            m = ml[0];
            l = ml[1];
        }
        // (a NaN among the weights is one of L; M is a number or -inf)
        const float top = fmaxf(M, wave_max(m)), by = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top);
        const float was = M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - top);
        M = top;
        // as means of what is there, so that no sum leaves the values' range
        const float now = L * was, sum = now + wave_sum(l * by);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum, share = by * inv;
        O *= now * inv;
        for (int e = 0;;) {
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k)
                if (e + k < many) O += o[k] * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(share), e + k));
            e += kAtOnce;
            if (e >= many) break;
            load(e);
        }
        L = sum;
    }
    out[lane] = L != L ? NAN : O;
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

size_t partial_floats(const Sizes &z) { return size_t(layout_of(z).units) * z.KVH * kCols * (VD + 2); }

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
    const bool small = count <= 256 && prefixes < 256;
    hipLaunchKernelGGL(small ? plan_kernel<256> : plan_kernel<1024>, dim3(blocks), dim3(small ? 256 : 1024), 0, ctx->stream, z,
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
    a.part_ml = a.part_o + size_t(a.plan.l.units) * a.z.KVH * kCols * VD;
    nd_kv_geom pg = *g;
    pg.cap = a.z.pcap;
    auto *fn = g->qk_head_dim == 48 ? (quant_query ? prefix_kernel<48, true> : prefix_kernel<48, false>)
                                    : (quant_query ? prefix_kernel<64, true> : prefix_kernel<64, false>);
    // HIP counts a launch's threads in 32 bits (and its second axis' blocks in 16): units
    // and rows beyond that go in further launches
    const uint32_t quads = a.plan.l.units / 4, each = std::min(65535u, ((1u << 24) - 1) / uint32_t(g->num_kv_heads));
    for (uint32_t first = 0; first < quads; first += each) {
        hipLaunchKernelGGL(fn, dim3(unsigned(g->num_kv_heads), std::min(each, quads - first)), dim3(256), 0, ctx->stream,
                           make_geom(g), make_geom(&pg), a, first);
        if (int rc = nd::check_launch("attend_prefix_i8")) return rc;
    }
    const size_t step = (size_t(1) << 25) / size_t(g->num_heads);
    for (size_t first = 0; first < count * rows; first += step) {
        const uint32_t total = uint32_t(std::min(step, count * rows - first) * g->num_heads);
        hipLaunchKernelGGL(prefix_join_kernel, dim3((total + 3) / 4), dim3(256), 0, ctx->stream, a, uint32_t(first), total);
        if (int rc = nd::check_launch("prefix_join")) return rc;
    }
    return ND_OK;
}

}  // extern "C"
