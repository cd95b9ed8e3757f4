"""A batch that shares its prompts: the plan's maps against plain whole numbers,
attention over shared prefixes against a plain 64-bit form.

Tolerance: that of tree attention (tests/test_gpu_tree.py), whose arithmetic it
is: 2e-5 for N(0, 1) keys, values and queries.  Sums over a prefix and over a
session's own positions meet by two more products, within the same bound.
"""
import numpy as np
import pytest
import torch

import needle_amd as nd
import prefix_ref as P
import tree_ref as R
from conftest import dev, host

pytestmark = pytest.mark.gpu
TOL = 2e-5
SHAPES = [(12, 2, 48), (12, 12, 64), (8, 4, 64), (16, 2, 64), (5, 1, 48), (3, 3, 48)]


def _i32(a):
    return None if a is None else dev(np.asarray(a, np.int32))


class Batch:
    """Blocks and requests: every live position holds an N(0, 1) row, the rest
    of a block is garbage."""

    def __init__(self, ctx, seed, shape, plen, used, which=None, length=None, rows=1, window=0, cap=None, pcap=None,
                 k_size=1.0, v_size=1.0, q_size=1.0):
        self.ctx, self.rng = ctx, np.random.default_rng(seed)
        self.H, self.KVH, self.QK = shape
        self.plen, self.used, self.which, self.length = plen, used, which, length
        self.rows, self.window, self.S, self.P = rows, window, len(used), len(plen)
        self.cap = cap or max(max(used, default=0), 0) + rows
        self.pcap = pcap or max(max(plen, default=1), 1)
        self.g = nd.kv_geom(self.H, self.KVH, self.QK, 64, self.cap)
        self.pg = nd.kv_geom(self.H, self.KVH, self.QK, 64, self.pcap)
        self.kv, self.nb = self._blocks(self.g, [u + rows for u in used], k_size, v_size)
        self.pkv, self.pnb = self._blocks(self.pg, plen, k_size, v_size)
        self.q = (q_size * self.rng.normal(size=(self.S, rows, self.H * self.QK))).astype(np.float32)
        self.there, self.bad, self.maps = P.layout(self.pcap, self.cap, plen, used, which, length, rows, window)

    def _blocks(self, g, ends, k_size, v_size):
        blk, nb = nd.kv_alloc(g, max(len(ends), 1))
        blk.fill_(0xff)
        for i, end in enumerate(ends):
            n = min(max(end, 0), g.cap)
            if not n or end > 1 << 25:
                continue
            at = torch.arange(end - n, end, dtype=torch.int32, device="cuda")
            k = (k_size * self.rng.normal(size=(n, g.num_kv_heads * g.qk_head_dim))).astype(np.float32)
            v = (v_size * self.rng.normal(size=(n, g.num_kv_heads * 64))).astype(np.float32)
            nd.kv_write(self.ctx, g, blk[i * nb:(i + 1) * nb], 0, at, dev(k), dev(v))
        return blk, nb

    def plan(self, **kw):
        return nd.prefix_plan(self.ctx, self.g, self.pcap, _i32(self.plen) if self.P else None, _i32(self.used),
                              prefix_of=_i32(self.which), length=_i32(self.length), rows=self.rows,
                              window=self.window, **kw)

    def attend(self, quant=False, scale=None, out=None, plan=None, **kw):
        plan = plan or self.plan()[0]
        return nd.attend_prefix_i8(self.ctx, self.g, self.kv, self.nb, self.pkv if self.P else None, self.pnb, plan,
                                   dev(self.q), scale=scale, quant_query=quant, out=out, **kw)

    def check(self, quant=False, scale=None, tol=TOL, sessions=None):
        _, maps = self.plan()
        for t, k in zip(maps, ("pos", "rot", "from", "lo", "order", "first")):
            assert np.array_equal(host(t), self.maps[k]), k
        out = torch.full((self.S, self.rows, self.H * 64), 7.0, device="cuda")
        got = host(self.attend(quant, scale, out=out)).reshape(self.S, self.rows, self.H, 64)
        own = {}
        for i in range(self.S):
            assert (got[i, self.there[i]:] == 7).all(), i
            mine = got[i, :self.there[i]]
            if self.bad[i]:
                assert np.isnan(mine).all(), i
                continue
            if sessions is not None and i not in sessions:
                assert np.isfinite(mine).all(), i
                continue
            p = (0 if self.P else -1) if self.which is None else self.which[i]
            blk = nd.kv_unpack(self.g, host(self.kv[i * self.nb:(i + 1) * self.nb]))
            if p >= 0 and p not in own:
                own[p] = nd.kv_unpack(self.pg, host(self.pkv[p * self.pnb:(p + 1) * self.pnb]))
            for n in range(self.there[i]):
                want = P.attend(self.H, blk, self.cap, own.get(p), self.pcap, self.plen[p] if p >= 0 else 0, self.maps,
                                i, n, self.q[i, n], quant, 1.0 / np.sqrt(self.QK) if scale is None else scale)
                err = np.abs(mine[n] - want).max()
                assert err <= tol, (i, n, err)


# ---- the plan -------------------------------------------------------------------

def _requests(rng, S, N, count, plen, used):
    which = rng.integers(-1, count, S) if count else None
    return (list(rng.integers(0, plen + 1, count)), list(rng.integers(0, used + 1, S)),
            None if which is None else list(which), list(rng.integers(0, N + 1, S)))


@pytest.mark.parametrize("window", [0, 1, 7, 100])
@pytest.mark.parametrize("S,N,count", [(1, 1, 1), (1, 1, 0), (3, 1, 2), (64, 1, 1), (255, 3, 5), (256, 1, 300),
                                       (257, 2, 9), (1000, 7, 40), (3001, 1, 2048), (5, 256, 3)])
def test_maps(ctx, S, N, count, window):
    rng = np.random.default_rng(S + N + window)
    plen, used, which, length = _requests(rng, S, N, count, 200, 90)
    cap, pcap = 90 + N, 201
    for kw in ({}, dict(length=None), dict(which=None)):
        w, m = kw.get("which", which), kw.get("length", length)
        _, maps = nd.prefix_plan(ctx, nd.kv_geom(12, 2, 48, 64, cap), pcap, _i32(plen) if count else None, _i32(used),
                                 prefix_of=_i32(w), length=_i32(m), rows=N, window=window)
        want = P.layout(pcap, cap, plen, used, w, m, N, window)[2]
        for t, k in zip(maps, ("pos", "rot", "from", "lo", "order", "first")):
            assert t.dtype == torch.int32 and np.array_equal(host(t), want[k]), k


def test_maps_of_numbers_that_cannot_be(ctx):
    top = 2 ** 31 - 1
    plen = [50, -1, 0, 80, top]
    used = [3, -1, 5, 5, 5, 5, 40, 2, 2, top - 50, top - 51, 0, 5, 5, 9, 9, top]
    which = [0, 0, 5, -7, 1, 2, 0, 0, 0, 0, 0, 4, 3, 3, -1, 0, 0]
    length = [1, 1, 1, 1, 1, 2, 2, 3, -1, 1, 1, 0, 1, 2, 2, 0, 0]
    for window in (0, 60, 1):
        for cap, pcap in ((20, 60), (41, 80), (3, 49)):
            _, maps = nd.prefix_plan(ctx, nd.kv_geom(12, 2, 48, 64, cap), pcap, _i32(plen), _i32(used),
                                     prefix_of=_i32(which), length=_i32(length), rows=2, window=window)
            _, _, want = P.layout(pcap, cap, plen, used, which, length, 2, window)
            for t, k in zip(maps, ("pos", "rot", "from", "lo", "order", "first")):
                assert np.array_equal(host(t), want[k]), (k, window, cap)


def test_maps_one_by_one_and_a_plan_of_the_callers(ctx):
    g, S, N, count = nd.kv_geom(12, 12, 64, 64, 30), 70, 2, 3
    rng = np.random.default_rng(5)
    plen, used, which, length = _requests(rng, S, N, count, 40, 20)
    args = dict(prefix_of=_i32(which), length=_i32(length), rows=N, window=9)
    _, want = nd.prefix_plan(ctx, g, 40, _i32(plen), _i32(used), **args)
    nb = nd.prefix_plan_bytes(g, S, N, count)
    room = torch.full((nb + 32,), 0x5a, dtype=torch.uint8, device="cuda")
    for one in range(6):
        maps = [torch.full_like(t, 99) if j == one else None for j, t in enumerate(want)]
        plan, got = nd.prefix_plan(ctx, g, 40, _i32(plen), _i32(used), plan=room[:nb], maps=maps, **args)
        assert torch.equal(got[one], want[one]) and plan.data.data_ptr() == room.data_ptr()
    plan, got = nd.prefix_plan(ctx, g, 40, _i32(plen), _i32(used), plan=plan, maps=False, **args)
    assert got is False and (host(room[nb:]) == 0x5a).all()
    _, none = nd.prefix_plan(ctx, g, 40, _i32(plen), _i32([]), rows=3)
    assert none[0].shape == (0, 3) and (host(none[5]) == 0).all()


# ---- attention --------------------------------------------------------------------

@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("S,plen,used", [(1, 1, 0), (1, 33, 5), (2, 31, 0), (3, 64, 31), (7, 100, 32), (17, 129, 64),
                                         (33, 300, 33), (4, 1000, 200)])
def test_one_prefix(ctx, shape, S, plen, used, quant):
    rng = np.random.default_rng(S)
    Batch(ctx, S + plen, shape, [plen], list(rng.integers(0, used + 1, S))).check(quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("shape", [(12, 2, 48), (12, 12, 64), (5, 1, 48)])
@pytest.mark.parametrize("S,N,count,plen,used,window", [(5, 1, 2, 90, 40, 0), (20, 3, 4, 70, 50, 0), (9, 33, 3, 200, 9, 0),
                                                        (40, 1, 6, 300, 100, 64), (12, 5, 3, 400, 300, 128), (3, 70, 2, 60, 10, 20),
                                                        (6, 2, 0, 0, 200, 50), (30, 1, 30, 40, 20, 1)])
def test_several_prefixes(ctx, shape, S, N, count, plen, used, window, quant):
    rng = np.random.default_rng(S + N + plen)
    lens, u, which, length = _requests(rng, S, N, count, plen, used)
    # blocks no larger than the windows need: rings that have wrapped
    cap = min(used, window) + N if window else None
    pcap = min(plen, window) if window and count else None
    Batch(ctx, S + N, shape, lens, u, which, length, N, window, cap, pcap).check(quant)


@pytest.mark.parametrize("quant", [False, True])
def test_sessions_that_see_none_of_their_prefix(ctx, quant):
    """A window behind the prefix's end, prefixes without positions, sessions
    without a prefix, sessions without rows, prefixes without sessions."""
    Batch(ctx, 1, (12, 2, 48), [50, 0, 20, 9], [70, 3, 0, 30, 12, 40], [0, 1, 1, -1, 2, 2], [1, 1, 1, 1, 0, 1], 1, 16,
          cap=40).check(quant)
    Batch(ctx, 2, (12, 12, 64), [0], [0, 0, 5]).check(quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("S,N,plen", [(130, 1, 500), (300, 1, 60), (600, 1, 900), (65, 4, 700), (40, 40, 300)])
def test_many_sessions(ctx, S, N, plen, quant):
    rng = np.random.default_rng(S)
    which = [int(i % 9 != 4) - 1 if i < S // 2 else 1 for i in range(S)]
    b = Batch(ctx, S, (12, 2, 48), [plen, plen // 2], list(rng.integers(0, 50, S)), which,
              list(rng.integers(0, N + 1, S)), N)
    b.check(quant, sessions={0, 1, 4, 13, S // 2, S - 2, S - 1})


@pytest.mark.parametrize("quant", [False, True])
def test_bad_sessions_between_good_ones(ctx, quant):
    Batch(ctx, 3, (12, 2, 48), [40, 500], [5, 30, 2, 7, 9, 11], [0, 0, 1, 2, 0, 0], [1, 2, 1, 1, 3, 2], 2, cap=31,
          pcap=64).check(quant)


def test_plans_of_other_sizes_give_nan(ctx):
    b = Batch(ctx, 4, (12, 2, 48), [40], [5, 7, 9])
    plan, _ = b.plan()
    other = nd.prefix_plan(ctx, b.g, b.pcap, _i32([40]), _i32([5, 7]))[0]
    room = torch.zeros(nd.prefix_plan_bytes(b.g, 3, 1, 1), dtype=torch.uint8, device="cuda")
    for data in (torch.cat([other.data, room])[:room.numel()], room, room + 0xff):
        stale = nd.PrefixPlan(data.contiguous(), plan.sizes)
        assert np.isnan(host(b.attend(plan=stale))).all()
    assert np.isfinite(host(b.attend(plan=plan))).all()


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("k_size,v_size", [(1e-6, 1e6), (30.0, 1e-12), (1e-30, 1e-30), (3.0, 1e30), (1e34, 1.0),
                                           (1e-38, 1e36)])
def test_sizes_of_values(ctx, k_size, v_size, quant):
    """Scores of N(0, 1) products whatever the keys' size; outputs to the same
    share of the values'."""
    Batch(ctx, 6, (12, 2, 48), [140], [0, 40, 33, 5], k_size=k_size, v_size=v_size,
          q_size=min(1 / k_size, 1e30)).check(quant, tol=TOL * v_size)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_any_scale(ctx, scale):
    for quant in (False, True):
        Batch(ctx, 7, (8, 4, 64), [70], [3, 40]).check(quant, scale=scale, tol=TOL * max(1, 8 * abs(scale)))


@pytest.mark.parametrize("quant", [False, True])
def test_queries_that_are_no_numbers(ctx, quant):
    b = Batch(ctx, 8, (12, 2, 48), [80, 30], [6, 7, 8, 9], [0, 1, 0, -1], rows=2)
    want = host(b.attend(quant)).reshape(4, 2, 12, 64)
    for i, n, h, bad in ((0, 0, 3, np.nan), (1, 1, 11, np.inf), (2, 0, 0, -np.inf), (3, 1, 5, np.nan)):
        b.q[i, n, h * 48 + 7] = bad
    got = host(b.attend(quant)).reshape(4, 2, 12, 64)
    hit = np.zeros((4, 2, 12), bool)
    hit[[0, 1, 2, 3], [0, 1, 0, 1], [3, 11, 0, 5]] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], want[~hit])


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("garbage", [np.nan, np.inf, -np.inf, 3e38, -1e-40])
def test_garbage_where_no_row_looks(ctx, quant, garbage):
    """Positions before a row's window, behind its own and of other rows."""
    b = Batch(ctx, 9, (12, 2, 48), [100, 90], [50, 20, 35], [0, 0, 1], [3, 1, 2], 3, 64, pcap=120, cap=80)
    want = host(b.attend(quant))
    for g, blk, nb, live in ((b.g, b.kv, b.nb, [(0, 53), (0, 21), (0, 37)]), (b.pg, b.pkv, b.pnb, [(100 - 43, 100), (90 - 28, 90)])):
        off = nd.kv_offsets(g)
        for i, (lo, hi) in enumerate(live):
            dead = torch.tensor([s for s in range(g.cap) if not lo <= s < hi], device="cuda")
            mine = blk[i * nb:(i + 1) * nb]
            for part in ("ks", "vs"):
                f = mine[off[part]:off[part] + 4 * g.num_kv_heads * g.cap].view(torch.float32).view(g.num_kv_heads, g.cap)
                f[:, dead] = garbage
    assert np.array_equal(host(b.attend(quant)), want, equal_nan=False)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_scales_that_are_no_numbers(ctx, quant, where):
    """A V scale that is no number makes none of the rows that see it, and of no others."""
    b = Batch(ctx, 10, (12, 2, 48), [70, 70], [20, 30, 10], [0, 1, 0])
    want = host(b.attend(quant)).reshape(3, 12, 64)
    g, blk, nb = (b.pg, b.pkv, b.pnb) if where == "prefix" else (b.g, b.kv, b.nb)
    off = nd.kv_offsets(g)["vs"]
    vs = blk[nb:2 * nb][off:off + 4 * g.num_kv_heads * g.cap].view(torch.float32).view(g.num_kv_heads, g.cap)
    vs[1, 7] = np.nan
    got = host(b.attend(quant)).reshape(3, 12, 64)
    assert np.isnan(got[1, 6:]).all()
    assert np.array_equal(got[1, :6], want[1, :6]) and np.array_equal(got[[0, 2]], want[[0, 2]])


def _positive(b, g, blk, nb, i, pos, k, v):
    nd.kv_write(b.ctx, g, blk[i * nb:(i + 1) * nb], 0, _i32(pos), dev(k.astype(np.float32)), dev(v.astype(np.float32)))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("sink", [1e-9, 1e-20, 0.0])
@pytest.mark.parametrize("ahead", [5, 15, 25, 60])
@pytest.mark.parametrize("S,shape", [(1, (12, 2, 48)), (70, (12, 2, 48)), (30, (4, 4, 64))])
def test_the_rest_behind_rows_of_next_to_no_values(ctx, S, shape, ahead, sink, quant):
    """A position of the prefix 2^ahead ahead of the others holds next to no
    values: the others' values, of one sign, decide.  The output is (2^ahead sink s +
    341 r) / (2^ahead + 341), s and r means of values of 1 to 2; every term of it
    is of that sign and off by a few 2^-23 of itself, its weight by the rounding of
    a score of 60 bits (60 2^-24): 2e-5 of the output's size is the bar."""
    H, KVH, QK = shape
    plen, own = 300, 40
    b = Batch(ctx, 11, shape, [plen], [own] * S, cap=own + 1)
    rng = np.random.default_rng(12)
    k = np.zeros((plen, KVH, QK))
    k[37, :, 0] = 1.0
    v = rng.uniform(1, 2, (plen, KVH * 64))
    v[37] = sink * rng.uniform(1, 2, KVH * 64)
    _positive(b, b.pg, b.pkv, b.pnb, 0, np.arange(plen), k.reshape(plen, -1), v)
    for i in range(S):
        _positive(b, b.g, b.kv, b.nb, i, np.arange(own + 1), np.zeros((own + 1, KVH * QK)),
                  rng.uniform(1, 2, (own + 1, KVH * 64)))
    b.q[:] = 0
    b.q.reshape(S, 1, H, QK)[..., 0] = ahead * np.log(2) * np.sqrt(QK)
    size = 1.5 * (341 + sink * 2.0 ** ahead) / (341 + 2.0 ** ahead)
    b.check(quant, tol=TOL * max(size, 2.0 ** -40) * 1.5, sessions={0, S // 2, S - 1})


@pytest.mark.parametrize("quant", [False, True])
def test_sums_of_large_values(ctx, quant):
    """Values near fp32's end: the mean is there where a sum is not."""
    b = Batch(ctx, 13, (12, 2, 48), [500], [100, 40])
    rng = np.random.default_rng(14)
    for g, blk, nb, i, n in ((b.pg, b.pkv, b.pnb, 0, 500), (b.g, b.kv, b.nb, 0, 101), (b.g, b.kv, b.nb, 1, 41)):
        _positive(b, g, blk, nb, i, np.arange(n), rng.normal(size=(n, 96)), rng.uniform(2.5e38, 3.3e38, (n, 128)))
    b.check(quant, tol=TOL * 3.3e38)


# ---- long runs of many rows, whose tiles lay K and V down for each other ------------

LONG = [(128, 128, 48), (256, 128, 64)]


def _long(seed, shape, ctx, S=70, plen=701, **kw):
    """70 sessions behind one prefix on 128 kv heads: runs of 10 chunks and more (a
    wave's share of the chunks of all tiles, three more a tile, and one)."""
    H, KVH, _ = shape
    b = Batch(ctx, seed, shape, [plen], [i * 7 % 40 for i in range(S)], **kw)
    tiles, chunks = -(-S * (H // KVH) // 16), -(-min(plen, kw.get("window") or plen) // 32)
    each = (tiles * (chunks + 3) + S * 4) // (4096 // KVH) + 1
    assert tiles >= 4 and chunks // -(-chunks // each) >= 10
    return b


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("shape", LONG)
@pytest.mark.parametrize("S,plen,window", [(64, 700, 0), (70, 673, 0), (79, 1409, 0), (70, 701, 690), (64, 1500, 740)])
def test_long_runs(ctx, shape, S, plen, window, quant):
    kw = dict(window=window, pcap=window + 1, cap=41) if window else {}
    _long(21, shape, ctx, S, plen, **kw).check(quant, sessions={0, 5, 17, S // 2, S - 1})


@pytest.mark.parametrize("shape", LONG)
@pytest.mark.parametrize("k_size,v_size", [(1e-6, 1e6), (30.0, 1e-12), (1e-30, 1e-30), (3.0, 1e30), (1e34, 1.0), (1e-38, 1e36)])
def test_long_runs_of_values_of_any_size(ctx, shape, k_size, v_size):
    _long(22, shape, ctx, k_size=k_size, v_size=v_size, q_size=min(1 / k_size, 1e30)).check(tol=TOL * v_size, sessions={0, 33, 69})


@pytest.mark.parametrize("shape", LONG)
@pytest.mark.parametrize("garbage", [np.nan, np.inf, 3e38, -1e-40])
def test_long_runs_and_what_is_no_number(ctx, shape, garbage):
    """Garbage where no row looks; then queries and a V scale that are no numbers."""
    H, KVH, QK = shape
    b = _long(23, shape, ctx, window=690, pcap=720)
    want = host(b.attend())
    off, first = nd.kv_offsets(b.pg), 701 + 1 - 690  # the earliest window begins there
    for part in ("ks", "vs"):
        f = b.pkv[off[part]:off[part] + 4 * KVH * 720].view(torch.float32).view(KVH, 720)
        f[:, :first] = garbage
        f[:, 701:] = garbage
    assert np.array_equal(host(b.attend()), want)
    b.q.reshape(70, H, QK)[3, 5, 1] = np.nan
    b.q.reshape(70, H, QK)[40, 64, 2] = garbage if not np.isfinite(garbage) else np.nan
    vs = b.pkv[off["vs"]:off["vs"] + 4 * KVH * 720].view(torch.float32).view(KVH, 720)
    vs[9, 300] = np.nan
    got, want = host(b.attend()).reshape(70, H, 64), want.reshape(70, H, 64)
    hit, R = np.zeros((70, H), bool), H // KVH
    hit[3, 5] = hit[40, 64] = True
    hit[:, 9 * R:10 * R] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], want[~hit])


@pytest.mark.parametrize("sink", [1e-9, 1e-20, 0.0])
@pytest.mark.parametrize("ahead", [5, 25, 60])
def test_long_runs_behind_a_row_of_next_to_no_values(ctx, ahead, sink):
    """As above (701 + 1 .. 40 other positions)."""
    shape = H, KVH, QK = LONG[0]
    b = _long(24, shape, ctx, cap=41)
    rng = np.random.default_rng(25)
    k = np.zeros((701, KVH, QK))
    k[337, :, 0] = 1.0
    v = rng.uniform(1, 2, (701, KVH * 64))
    v[337] = sink * rng.uniform(1, 2, KVH * 64)
    _positive(b, b.pg, b.pkv, b.pnb, 0, np.arange(701), k.reshape(701, -1), v)
    for i in range(70):
        _positive(b, b.g, b.kv, b.nb, i, np.arange(41), np.zeros((41, KVH * QK)), rng.uniform(1, 2, (41, KVH * 64)))
    b.q[:] = 0
    b.q.reshape(70, 1, H, QK)[..., 0] = ahead * np.log(2) * np.sqrt(QK)
    size = 1.5 * (741 + sink * 2.0 ** ahead) / (701 + 2.0 ** ahead)
    b.check(tol=TOL * max(size, 2.0 ** -40) * 1.5, sessions={0, 35, 69})


def test_long_runs_of_large_values(ctx):
    b = _long(26, LONG[0], ctx)
    rng = np.random.default_rng(27)
    _positive(b, b.pg, b.pkv, b.pnb, 0, np.arange(701), rng.normal(size=(701, 128 * 48)), rng.uniform(2.5e38, 3.3e38, (701, 128 * 64)))
    for i in range(70):
        n = b.used[i] + 1
        _positive(b, b.g, b.kv, b.nb, i, np.arange(n), rng.normal(size=(n, 128 * 48)), rng.uniform(2.5e38, 3.3e38, (n, 128 * 64)))
    b.check(tol=TOL * 3.3e38, sessions={0, 35, 69})


def test_sessions_over_one_block_and_strides(ctx):
    """kv_stride 0, and blocks further apart than they are large."""
    b = Batch(ctx, 15, (8, 4, 64), [60, 30], [9, 9], [0, 1])
    out = b.attend()
    wide = torch.zeros(2 * (b.nb + 512), dtype=torch.uint8, device="cuda")
    pwide = torch.zeros(2 * (b.pnb + 1024), dtype=torch.uint8, device="cuda")
    for i in range(2):
        wide[i * (b.nb + 512):][:b.nb] = b.kv[i * b.nb:(i + 1) * b.nb]
        pwide[i * (b.pnb + 1024):][:b.pnb] = b.pkv[i * b.pnb:(i + 1) * b.pnb]
    plan, _ = b.plan()
    got = nd.attend_prefix_i8(ctx, b.g, wide, b.nb + 512, pwide, b.pnb + 1024, plan, dev(b.q))
    assert torch.equal(got, out)
    b.kv[b.nb:] = b.kv[:b.nb]
    both = b.attend()
    got = nd.attend_prefix_i8(ctx, b.g, b.kv, 0, b.pkv, b.pnb, plan, dev(b.q))
    assert torch.equal(got, both)


def test_the_same_bits_whatever_shares_the_batch(ctx):
    """Twice the same call, and a step that repeats itself, give the same bits."""
    b = Batch(ctx, 16, (12, 2, 48), [700, 90], [33] * 50, [i % 2 for i in range(50)], rows=2)
    one = host(b.attend(True))
    for _ in range(3):
        assert np.array_equal(host(b.attend(True)), one)


def test_a_prefix_and_the_rest_are_one_context(ctx):
    """What decoding over one block that holds the whole context gives."""
    H, KVH, QK, L, u = 12, 2, 48, 333, 47
    rng = np.random.default_rng(17)
    k, v = rng.normal(size=(L + u + 1, KVH * QK)), rng.normal(size=(L + u + 1, KVH * 64))
    b = Batch(ctx, 17, (H, KVH, QK), [L], [u])
    _positive(b, b.pg, b.pkv, b.pnb, 0, np.arange(L), k[:L], v[:L])
    _positive(b, b.g, b.kv, b.nb, 0, np.arange(u + 1), k[L:], v[L:])
    whole = nd.kv_geom(H, KVH, QK, 64, L + u + 1)
    blk, nb = nd.kv_alloc(whole)
    nd.kv_write(ctx, whole, blk, 0, _i32(np.arange(L + u + 1)), dev(k.astype(np.float32)), dev(v.astype(np.float32)))
    for quant in (False, True):
        want = nd.attend_step_i8(ctx, whole, blk, 0, _i32([0]), _i32([L + u]), dev(b.q[0]), quant_query=quant)
        # each within TOL of the same sums
        assert np.abs(host(b.attend(quant))[0] - host(want)).max() <= 2 * TOL


def test_offsets_beyond_32_bits(ctx):
    """Blocks, queries and outputs more than 2^32 bytes apart."""
    g = nd.kv_geom(12, 12, 64, 64, 40)
    nb = nd.kv_block_bytes(g)
    far = (1 << 32) // 3 // 256 * 256 + 512
    kv = torch.zeros(4 * far + nb, dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(18)
    b = Batch(ctx, 18, (12, 12, 64), [30], [8] * 5, cap=40)
    for i in range(5):
        kv[i * far:i * far + nb] = b.kv[i * b.nb:(i + 1) * b.nb]
    pkv = torch.zeros(4 * far + b.pnb, dtype=torch.uint8, device="cuda")
    pkv[4 * far:] = b.pkv[:b.pnb]
    plan, _ = nd.prefix_plan(ctx, g, b.pcap, _i32([0, 0, 0, 0, 30]), _i32([8] * 5), prefix_of=_i32([4] * 5))
    got = nd.attend_prefix_i8(ctx, g, kv, far, pkv, far, plan, dev(b.q))
    assert torch.equal(got, b.attend()) and rng is not None


@pytest.mark.parametrize("H,KVH,S,rows", [(4096, 4096, 1100, 1), (1500, 1500, 3000, 1), (16, 2, 65535, 9)])
def test_many_heads_and_more_units_than_a_launch_holds(ctx, H, KVH, S, rows):
    """Sessions over one block give the bits of one session."""
    b = Batch(ctx, 19, (H, KVH, 48), [], [5], rows=rows)
    b.check()
    plan, _ = nd.prefix_plan(ctx, b.g, 1, None, _i32([5] * S), rows=rows)
    got = nd.attend_prefix_i8(ctx, b.g, b.kv, 0, None, 0, plan, dev(b.q).expand(S, -1, -1).contiguous())
    assert (got == b.attend()).all()


@pytest.mark.parametrize("quant", [False, True])
def test_positions_at_the_end_of_32_bits(ctx, quant):
    """Rings whose last position is 2^31 - 1: a session's, and a prefix's with a session behind it."""
    top = 2 ** 31 - 1
    b = Batch(ctx, 29, (12, 2, 48), [top - 70, 0], [67, top - 2, 2 ** 30], [0, 1, -1], rows=3, window=75, cap=80, pcap=77)
    rng = np.random.default_rng(30)
    for g, blk, nb, i, end in ((b.pg, b.pkv, b.pnb, 0, top - 70), (b.g, b.kv, b.nb, 1, top + 1), (b.g, b.kv, b.nb, 2, 2 ** 30 + 3)):
        pos = np.arange(end - 77, end)  # three windows of 75
        _positive(b, g, blk, nb, i, pos, rng.normal(size=(77, 96)), rng.normal(size=(77, 128)))
    assert not b.bad.any() and b.maps["rot"].max() == top
    b.check(quant)


def test_no_sessions(ctx):
    g = nd.kv_geom(12, 2, 48, 64, 8)
    kv, nb = nd.kv_alloc(g, 1)
    for plen in (None, [5, 0]):
        plan, maps = nd.prefix_plan(ctx, g, 8, _i32(plen), _i32([]))
        assert [t.numel() for t in maps] == [0, 0, 0, 0, 0, len(plen or []) + 1] and not host(maps[5]).any()
        out = nd.attend_prefix_i8(ctx, g, kv, nb, kv if plen else None, 0, plan, torch.zeros(0, 1, 576, device="cuda"))
        assert out.shape == (0, 1, 768)


def test_a_plan_without_the_room_of_its_sizes(ctx):
    b = Batch(ctx, 28, (12, 2, 48), [40], [5, 7, 9])
    plan, _ = b.plan()
    with pytest.raises(ValueError, match="plan"):
        b.attend(plan=nd.PrefixPlan(plan.data[:-64], plan.sizes))
    many = nd.PrefixPlan(plan.data, (300, *plan.sizes[1:]))
    with pytest.raises(ValueError, match="plan"):
        nd.attend_prefix_i8(ctx, b.g, b.kv, 0, b.pkv, 0, many, torch.zeros(300, 1, 576, device="cuda"))


# ---- the shipped geometry's long runs, thousands of sessions, far rows ---------------

@pytest.mark.parametrize("shape,S,N,plen,window", [((12, 2, 48), 300, 1, 6400, 0), ((12, 2, 48), 24, 33, 2500, 0), ((12, 2, 48), 40, 20, 2600, 2400),
                                                   ((16, 2, 64), 240, 1, 6001, 0), ((5, 1, 48), 1000, 1, 4500, 0), ((8, 4, 64), 120, 10, 3300, 3000)])
def test_long_runs_of_few_kv_heads(ctx, shape, S, N, plen, window):
    """fp32 queries whose tiles lay K and V down for each other, two to eight heads a kv head: a group of `S`
    sessions in runs of 10 chunks and more, a short prefix and sessions without one beside it."""
    rng = np.random.default_rng(S)
    H, KVH, _ = shape
    which = [0] * S + [1, -1, 1]
    used = list(rng.integers(0, 40, S + 3))
    length = [N] * (S - 1) + list(rng.integers(1, N + 1, 4))
    b = Batch(ctx, S, shape, [plen, 90], used, which, length, N, window, pcap=window + 50 if window else None)
    tiles, chunks = sum(length[:S]) * (H // KVH) // 16, (min(plen, window) if window else plen) // 32
    each = tiles * (chunks + 3) // (4096 // KVH) + 1
    assert tiles >= 8 and chunks // -(-chunks // each) >= 10
    b.check(sessions={0, 1, S // 2, S - 1, S, S + 1, S + 2})


@pytest.mark.parametrize("S,N,count,window", [(4097, 1, 1, 0), (4200, 3, 7, 50), (9000, 2, 300, 0), (65535, 1, 2048, 33), (65535, 16, 5, 0)])
def test_maps_of_thousands_of_sessions(ctx, S, N, count, window):
    """More sessions than a block's threads hold at once."""
    rng = np.random.default_rng(S + N)
    plen, used, which, length = _requests(rng, S, N, count, 200, 90)
    _, maps = nd.prefix_plan(ctx, nd.kv_geom(12, 2, 48, 64, 90 + N), 201, _i32(plen), _i32(used), prefix_of=_i32(which),
                             length=_i32(length), rows=N, window=window)
    want = P.layout(201, 90 + N, plen, used, which, length, N, window)[2]
    for t, k in zip(maps, ("pos", "rot", "from", "lo", "order", "first")):
        assert np.array_equal(host(t), want[k]), k


@pytest.mark.parametrize("quant", [False, True])
def test_attention_of_thousands_of_sessions(ctx, quant):
    S = 4500
    rng = np.random.default_rng(40)
    b = Batch(ctx, 41, (5, 1, 48), [130, 70, 0, 33], list(rng.integers(0, 12, S)), list(rng.integers(-1, 4, S)),
              list(rng.integers(0, 3, S)), 2)
    b.check(quant, sessions={0, 63, 64, 1023, 1024, 4095, 4096, 4097, 4200, S - 1})


@pytest.mark.parametrize("quant", [False, True])
def test_a_session_whatever_else_the_step_holds(ctx, quant):
    """The same session alone, behind others of its prefix and beside other prefixes: each time within the
    tolerance of the same 64-bit sums."""
    b = Batch(ctx, 42, (12, 2, 48), [700, 90], [33, 5, 20, 0, 12, 33, 7], [0, 0, 1, -1, 0, 1, 0], rows=2)
    whole = host(b.attend(quant))
    b.check(quant)
    for keep in ([0], [1, 0], [2, 3, 0, 5], [6, 5, 4, 0]):
        kv = torch.cat([b.kv[i * b.nb:(i + 1) * b.nb] for i in keep])
        plan, _ = nd.prefix_plan(ctx, b.g, b.pcap, _i32(b.plen), _i32([b.used[i] for i in keep]),
                                 prefix_of=_i32([b.which[i] for i in keep]), rows=2)
        got = host(nd.attend_prefix_i8(ctx, b.g, kv, b.nb, b.pkv, b.pnb, plan, dev(b.q[keep]), quant_query=quant))
        assert np.abs(got - whole[keep]).max() <= 2 * TOL


def test_queries_and_outputs_beyond_32_bits(ctx):
    """2^20 rows of 65 heads: 4.3e9 numbers of each.  Sessions over one block give the bits of seven."""
    S, N, H = 65535, 16, 65
    b = Batch(ctx, 43, (H, H, 64), [], [5], rows=N)
    base = torch.randn(7, H * 64, device="cuda")
    i, n = torch.arange(S, device="cuda")[:, None], torch.arange(N, device="cuda")
    q = base[(i * N + n).view(-1) % 7].view(S, N, H * 64)
    want = nd.attend_prefix_i8(ctx, b.g, b.kv, 0, None, 0, nd.prefix_plan(ctx, b.g, 1, None, _i32([5] * 7), rows=N)[0], q[:7].clone())
    plan, _ = nd.prefix_plan(ctx, b.g, 1, None, _i32([5] * S), rows=N)
    got = nd.attend_prefix_i8(ctx, b.g, b.kv, 0, None, 0, plan, q)
    assert torch.isfinite(want).all()
    for first in range(0, S, 7 * 1024):
        part = got[first:first + 7 * 1024]
        assert torch.equal(part, want.repeat(1025, 1, 1)[:len(part)])


# ---- refusals -----------------------------------------------------------------------

def test_refusals(ctx):
    g = nd.kv_geom(12, 2, 48, 64, 64)
    kv, nb = nd.kv_alloc(g, 2)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.zeros(2, 1, 576, device="cuda")

    def refused(what, f):
        with pytest.raises(nd.NeedleError) as e:
            f()
        assert e.value.code == nd.ND_ERR_ARG and what in str(e.value), str(e.value)

    some = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    for what, geom, pcap, plen, used, kw in (
            ("rows", g, 64, z(1), z(2), dict(rows=0)), ("rows", g, 64, z(1), z(2), dict(rows=257)),
            ("count", g, 64, z(1), z(65536), {}), ("sessions x", g, 64, z(1), z(65535), dict(rows=17)),
            ("prefixes", g, 64, z(2049), z(2), {}), ("window", g, 64, z(1), z(2), dict(window=-1)),
            ("prefix_cap", g, 0, z(1), z(2), {}), ("prefix_cap", g, (1 << 24) + 1, z(1), z(2), {}),
            ("num_heads", nd.kv_geom(5, 2, 48, 64, 64), 64, z(1), z(2), {})):
        refused(what, lambda: nd.prefix_plan(ctx, geom, pcap, plen, used, plan=some, maps=False, **kw))
    refused("plan holds", lambda: nd.prefix_plan(ctx, g, 64, z(1), z(2), plan=some[:64]))
    refused("aligned", lambda: nd.prefix_plan(ctx, g, 64, z(1), z(2), plan=some[8:]))
    assert nd.prefix_plan_bytes(g, 70000, 1, 1) == 0 and "count" in nd.last_error()
    plan, _ = nd.prefix_plan(ctx, g, 64, z(1), z(2))
    ok = lambda **kw: nd.attend_prefix_i8(ctx, g, kv, nb, kv, nb, plan, q, **kw)  # noqa: E731
    assert ok().shape == (2, 1, 768)
    for kw in (dict(prefix_of=z(1)), dict(length=z(1)), dict(maps=[z(1)] + [None] * 5), dict(prefix_of=z(2).long())):
        with pytest.raises(ValueError):
            nd.prefix_plan(ctx, g, 64, z(1), z(2), **kw)
    for bad in (lambda: nd.attend_prefix_i8(ctx, g, kv[:nb], nb, kv, nb, plan, q),
                lambda: nd.attend_prefix_i8(ctx, g, kv, nb, None, nb, plan, q),
                lambda: nd.attend_prefix_i8(ctx, g, kv, nb, kv[:-256], 2 * nb, nd.prefix_plan(ctx, g, 64, z(2), z(2))[0], q),
                lambda: nd.attend_prefix_i8(ctx, g, kv, nb, kv, nb, plan, q[:1]),
                lambda: nd.attend_prefix_i8(ctx, g, kv, nb, kv, nb, plan, q[..., :500].contiguous()),
                lambda: nd.attend_prefix_i8(ctx, g, kv, nb, kv, nb, plan, q.double()),
                lambda: nd.attend_prefix_i8(ctx, nd.kv_geom(12, 2, 48, 64, 32), kv, nb, kv, nb, plan, q),
                lambda: ok(out=q), lambda: ok(work=z(4))):
        with pytest.raises(ValueError):
            bad()
    refused("aligned", lambda: nd.attend_prefix_i8(ctx, g, kv[64:], 0, kv, nb, plan, q))
    refused("aligned", lambda: nd.attend_prefix_i8(ctx, g, kv, nb, kv[64:], 0, nd.PrefixPlan(plan.data, (2, 1, 1, 32, 12, 2, 64)), q))
    mha = nd.kv_geom(12, 12, 64, 64, 64)
    both = torch.zeros(6 * 768, device="cuda")
    plan, _ = nd.prefix_plan(ctx, mha, 64, None, z(2))
    kv, nb = nd.kv_alloc(mha, 2)
    for a, b in ((0, 0), (0, 1), (2, 1)):
        refused("overlaps", lambda: nd.attend_prefix_i8(ctx, mha, kv, nb, None, 0, plan, both[a * 768:][:1536].view(2, 1, 768),
                                                        out=both[b * 768:][:1536].view(2, 1, 768)))
    for shape in ((12, 2, 32, 64), (12, 2, 64, 128)):
        other = nd.kv_geom(*shape, 64)
        kv, nb = nd.kv_alloc(other, 2)
        plan, _ = nd.prefix_plan(ctx, other, 64, None, z(2))
        refused("no prefix attention", lambda: nd.attend_prefix_i8(ctx, other, kv, nb, None, 0, plan, torch.zeros(2, 1, 12 * 64, device="cuda"),
                                                                   out=torch.zeros(2, 1, 12 * 128, device="cuda")))
    none, _ = nd.prefix_plan(ctx, mha, 64, None, z(0))
    assert nd.attend_prefix_i8(ctx, mha, kv, nb, None, 0, none, torch.zeros(0, 1, 768, device="cuda")).shape == (0, 1, 768)
