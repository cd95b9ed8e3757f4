"""Attention of drafted trees over the int8 cache against a plain 64-bit form.

Tolerance.  A score is a dot of at most 64 products summed in fp32 and three
products: off by at most 67 * 2^-24 of the sum of the products' magnitudes,
which for these N(0, 1) draws stays below 64 * 0.8 = 51 before and 7.4 after
the scale, so below 3.0e-5, and by a root's share of that (4e-6) in any draw.
A weight is off by as much, by a few steps of its exponential (4 * 2^-24) and
by the 22 bits or more it is held in; an output, a mean of |v| < 5.5 under
such weights in numerator and sum, by 2 * (4e-6 + 5e-7) * 5.5 / 2 = 2.5e-5 at
the very most and in draws of many positions far less: 2e-5 is the bar, as
for the other int8 attention.  Larger or smaller values scale it.
"""
import numpy as np
import pytest
import torch

import needle_amd as nd
import tree_ref as R
from conftest import dev, host

pytestmark = pytest.mark.gpu
TOL = 2e-5


def _block(ctx, rng, H, KVH, QK, cap, upto, count, k_size=1.0, v_size=1.0):
    """Blocks that hold positions upto - cap .. upto - 1; the rest is garbage."""
    g = nd.kv_geom(H, KVH, QK, 64, cap)
    blk, nb = nd.kv_alloc(g, count)
    blk.fill_(0xff)
    for i in range(count):
        p0 = max(0, upto - cap)
        n = upto - p0
        k = (rng.normal(size=(n, KVH * QK)) * k_size).astype(np.float32)
        v = (rng.normal(size=(n, KVH * 64)) * v_size).astype(np.float32)
        nd.kv_write(ctx, g, blk[i * nb:(i + 1) * nb], 0, torch.arange(p0, upto, dtype=torch.int32, device="cuda"),
                    dev(k), dev(v))
    return g, blk, nb


def _parents(rng, count, nodes, branch=3):
    up = np.zeros((count, nodes), np.int64)
    for j in range(nodes):
        up[:, j] = -1 if j == 0 else np.maximum(j - 1 - rng.integers(0, branch + 1, count), -1)
    return up


def _want(g, blk, nb, base, length, lo, see, q, quant, scale=None):
    """[S][N][H * 64], NaN where a row is not to be compared."""
    S, N = lo.shape
    H, QK = g.num_heads, g.qk_head_dim
    scale = 1.0 / np.sqrt(QK) if scale is None else scale
    out = np.full((S, N, H * 64), np.nan)
    for i in range(S):
        k, ks, v, vs = nd.kv_unpack(g, blk[i * nb:(i + 1) * nb])
        m = N if length is None else int(length[i])
        for n in range(m):
            first = min(int(lo[i, n]), int(base[i]))
            pos = np.arange(first, base[i] + m)
            slot = pos % g.cap
            sees = np.concatenate([np.ones(int(base[i]) - first, bool), see[i, n, :m] != 0])
            used = np.where(sees, slot, 0)
            kk = k[used] * np.where(sees[:, None], ks[used], 1).astype(np.float64)[..., None]
            vv = v[used] * np.where(sees[:, None], vs[used], 1).astype(np.float64)[..., None]
            qq = q[i, n].reshape(H, QK)
            if quant:
                c, s = R.stand_for(qq)
                qq = c * s.astype(np.float64)[:, None]
            out[i, n] = R.attend(qq, kk, vv, sees, scale).reshape(-1)
    return out


def _check(ctx, g, blk, nb, base, lo, see, q, length=None, quant=False, scale=None, tol=TOL, rows=None):
    base, lo = np.asarray(base, np.int32), np.asarray(lo, np.int32)
    S, N = lo.shape
    out = torch.full((S, N, g.num_heads * 64), 7.0, device="cuda")
    args = (ctx, g, blk, nb, dev(base), dev(lo), dev(R.words_of(see)), dev(q.reshape(S, N, -1)))
    kw = dict(length=None if length is None else dev(np.asarray(length, np.int32)), quant_query=quant, scale=scale)
    got = host(nd.attend_tree_i8(*args, out=out, **kw))
    # the same call with its own workspace, bit for bit
    need = nd.attend_tree_i8_work(ctx, g, S, N)
    own = torch.full((need + 256,), 0xa5, dtype=torch.uint8, device="cuda")
    twice = torch.full_like(out, 7.0)
    nd.attend_tree_i8(*args, out=twice, work=own[:max(need, 16)], **kw)
    assert np.array_equal(host(twice), got, equal_nan=True) and (host(own)[max(need, 16):] == 0xa5).all()
    b = host(blk)
    pick = range(S) if rows is None else rows
    for i in pick:
        one = slice(i, i + 1)
        want = _want(g, b[i * nb:(i + 1) * nb] if nb else b, nb or len(b), base[one],
                     None if length is None else length[one], lo[one], see[one], q[one], quant, scale)[0]
        there = ~np.isnan(want)
        assert not np.isnan(got[i][there]).any(), i
        assert np.max(np.abs(got[i][there] - want[there]), initial=0) <= tol, (i, np.abs(got[i][there] - want[there]).max())
        assert (got[i][~there] == 7.0).all(), i  # rows behind the tree's end
    return got


SHAPES = [(12, 2, 48), (12, 12, 64), (16, 2, 64), (5, 1, 48), (7, 1, 64), (6, 2, 64), (4, 2, 48)]


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("H,KVH,QK", SHAPES)
@pytest.mark.parametrize("nodes,base,cap", [(1, 0, 1), (1, 5, 6), (2, 31, 33), (8, 32, 40), (16, 70, 129), (33, 0, 64),
                                            (31, 200, 700), (64, 1, 65), (13, 500, 513)])
def test_trees(ctx, H, KVH, QK, nodes, base, cap, quant):
    """Ragged trees and bases, rings below a tile and just large enough."""
    rng = np.random.default_rng(nodes * 100 + cap + H)
    S = 3
    g, blk, nb = _block(ctx, rng, H, KVH, QK, cap, base + nodes, S)
    bases = base - np.minimum(np.arange(S) * 7, base)
    length = np.maximum(nodes - np.arange(S) * 3, 0)
    see = R.bits_of(nd.tree_mask(_parents(rng, S, nodes)), nodes)
    # a ring holds its last `cap` positions: what a shorter base would read before them is not there
    lo = np.maximum(bases + length - cap, max(0, base + nodes - cap))[:, None] + np.zeros((1, nodes), int)
    q = rng.normal(size=(S, nodes, H * QK)).astype(np.float32)
    _check(ctx, g, blk, nb, bases, np.minimum(lo, bases[:, None] + 1), see, q, length, quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("H,KVH,QK", [(12, 2, 48), (12, 12, 64), (8, 1, 64)])
@pytest.mark.parametrize("nodes,base,cap,window", [(40, 5000, 1061, 1000), (21, 999, 300, 256), (7, 4097, 64, 50),
                                                   (100, 3001, 3200, 0), (256, 700, 1000, 0), (3, 9000, 9003, 0)])
def test_windows_and_wrapped_rings(ctx, H, KVH, QK, nodes, base, cap, window, quant):
    rng = np.random.default_rng(cap + nodes)
    g, blk, nb = _block(ctx, rng, H, KVH, QK, cap, base + nodes, 1)
    up = _parents(rng, 1, nodes)
    depth = np.zeros((1, nodes), int)
    for j in range(nodes):
        depth[0, j] = depth[0, up[0, j]] + 1 if up[0, j] >= 0 else 0
    lo = np.maximum(base + depth + 1 - window, 0) if window else np.zeros_like(depth)
    lo = np.maximum(lo, base + nodes - cap)
    see = R.bits_of(nd.tree_mask(up), nodes)
    q = rng.normal(size=(1, nodes, H * QK)).astype(np.float32)
    _check(ctx, g, blk, nb, [base], lo, see, q, quant=quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("H,KVH,QK", [(12, 2, 48), (12, 12, 64), (5, 1, 64)])
@pytest.mark.parametrize("nodes,base,cap,reach", [(40, 170, 100, 60), (64, 95, 128, 64), (256, 1900, 1000, 744),
                                                  (33, 40, 64, 31), (5, 62, 64, 59), (32, 32, 48, 16), (100, 50, 101, 1),
                                                  (97, 1097, 98, 1), (2, 63, 64, 0), (70, 999, 1000, 0)])
def test_a_tree_across_the_rings_end(ctx, H, KVH, QK, nodes, base, cap, reach, quant):
    """Trees whose nodes lie on both sides of the ring's end, in front of every
    part of a word of the mask."""
    rng = np.random.default_rng(nodes + base)
    assert base % cap + nodes > cap and reach + nodes <= cap
    g, blk, nb = _block(ctx, rng, H, KVH, QK, cap, base + nodes, 2)
    bases = np.array([base, base - 1])
    length = np.array([nodes, max(nodes - 2, 1)])
    see = np.concatenate([R.bits_of(nd.tree_mask(_parents(rng, 1, nodes)), nodes),
                          rng.integers(0, 2, (1, nodes, nodes)).astype(np.uint8)])
    lo = bases[:, None] - rng.integers(0, reach + 1, (2, nodes))
    lo[1] = np.maximum(lo[1], base + nodes - cap)  # what is there of the shorter one
    q = rng.normal(size=(2, nodes, H * QK)).astype(np.float32)
    _check(ctx, g, blk, nb, bases, lo, see, q, length, quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("sessions,nodes,base", [(65, 16, 300), (130, 5, 90), (300, 2, 40), (9, 30, 2000)])
def test_many_sessions(ctx, sessions, nodes, base, quant):
    """Every launch shape: few sessions with long spans, many with short ones."""
    rng = np.random.default_rng(sessions)
    g, blk, nb = _block(ctx, rng, 12, 2, 48, base + nodes, base + nodes, sessions)
    bases = base - np.arange(sessions) % 17
    see = R.bits_of(nd.tree_mask(_parents(rng, sessions, nodes)), nodes)
    length = nodes - np.arange(sessions) % 3 % nodes
    lo = np.zeros((sessions, nodes), int)
    q = rng.normal(size=(sessions, nodes, 12 * 48)).astype(np.float32)
    _check(ctx, g, blk, nb, bases, lo, see, q, length, quant, rows=sorted({0, 1, 7, sessions // 2, sessions - 1}))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("base", [0, 3, 100, 2100])
def test_any_mask_and_rows_that_see_nothing(ctx, base, quant):
    """Masks that are no tree, bits behind the tree's end, rows with nothing
    (zeros), with the committed positions alone, and with one node alone."""
    rng = np.random.default_rng(base)
    nodes, S = 37, 3
    g, blk, nb = _block(ctx, rng, 12, 2, 48, base + nodes, base + nodes, S)
    see = rng.integers(0, 2, (S, nodes, nodes)).astype(np.uint8)
    see[:, 4] = 0
    see[:, 5] = 0
    see[:, 6] = 0
    see[:, 6, 30] = 1
    length = np.array([nodes, 31, 6])
    lo = rng.integers(0, base + 1, (S, nodes))
    lo[:, [4, 6]] = base + np.array([0, 5])
    q = rng.normal(size=(S, nodes, 12 * 48)).astype(np.float32)
    got = _check(ctx, g, blk, nb, np.full(S, base), lo, see, q, length, quant)
    assert not got[:, 4].any() and got[0, 6].any() and not got[1, 6, 0] == 0


@pytest.mark.parametrize("quant", [False, True])
def test_garbage_in_places_no_row_reads(ctx, quant):
    """NaN and infinite scales before the window, behind the tree and in nodes
    outside a row's mask reach nobody but the rows that read them."""
    rng = np.random.default_rng(2)
    nodes, base, cap = 10, 90, 128
    g, blk, nb = _block(ctx, rng, 12, 2, 48, cap, base + nodes, 1)
    off = nd.kv_offsets(g)
    for part in ("ks", "vs"):
        s = blk[off[part]:off[part] + 4 * 2 * cap].view(torch.float32).view(2, cap)
        s[:, :20] = float("nan")
        s[:, 20:30] = float("inf")
        s[:, base + 7] = float("nan")  # node 7
        s[:, base + 8] = float("inf")  # node 8
        s[:, base + nodes:] = float("nan")
    see = R.bits_of(nd.tree_mask(_parents(rng, 1, nodes)), nodes).copy()
    see[:, :, 7:9] = 0
    see[0, 7, 7] = see[0, 8, 8] = 1
    q = rng.normal(size=(1, nodes, 12 * 48)).astype(np.float32)
    lo = np.full((1, nodes), 30)
    lo[0, 2] = 57
    clean = np.array([0, 1, 2, 3, 4, 5, 6, 9])
    args = (ctx, g, blk, nb, dev(np.array([base], np.int32)), dev(lo.astype(np.int32)), dev(R.words_of(see)), dev(q))
    got = host(nd.attend_tree_i8(*args, quant_query=quant))
    want = _want(g, host(blk), nb, [base], None, lo, see, q, quant)
    assert np.abs(got[0, clean] - want[0, clean]).max() <= TOL
    assert np.isnan(got[0, 7]).all()


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("k_size,v_size", [(1e-6, 1e6), (30.0, 1e-12), (1e-30, 1e-30), (3.0, 1e30), (1e34, 1.0),
                                           (1e37, 1e-30)])
def test_sizes_of_values(ctx, k_size, v_size, quant):
    """Values far from 1, and V rows of very different sizes in one span."""
    rng = np.random.default_rng(5)
    nodes, base = 16, 200
    g, blk, nb = _block(ctx, rng, 12, 2, 48, 256, base + nodes, 1, k_size, v_size)
    see = R.bits_of(nd.tree_mask(_parents(rng, 1, nodes)), nodes)
    q = (rng.normal(size=(1, nodes, 12 * 48)) / max(k_size, 1e-30)).astype(np.float32)
    if quant and k_size > 1e36:
        return  # a scale whose inverse is beyond fp32: there are no codes to compare
    _check(ctx, g, blk, nb, [base], np.zeros((1, nodes), int), see, q, quant=quant, tol=TOL * v_size)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("spread", [1e3, 1e6, 1e12])
def test_small_values_beside_large_ones(ctx, spread, quant):
    """Rows whose window holds small values only, beside rows that read large
    ones: each row's error is measured against its own values."""
    rng = np.random.default_rng(7)
    nodes, base = 24, 320
    g, blk, nb = _block(ctx, rng, 12, 2, 48, 400, base + nodes, 1)
    off = nd.kv_offsets(g)
    s = blk[off["vs"]:off["vs"] + 4 * 2 * 400].view(torch.float32).view(2, 400)
    s[:, :100] *= spread
    s[:, 150:200:3] /= spread
    see = R.bits_of(nd.tree_mask(_parents(rng, 1, nodes)), nodes)
    lo = np.where(np.arange(nodes) % 2, 100, 0)[None]
    q = rng.normal(size=(1, nodes, 12 * 48)).astype(np.float32)
    args = (ctx, g, blk, nb, dev(np.array([base], np.int32)), dev(lo.astype(np.int32)), dev(R.words_of(see)), dev(q))
    got = host(nd.attend_tree_i8(*args, quant_query=quant))
    want = _want(g, host(blk), nb, [base], None, lo, see, q, quant)
    assert np.abs(got[0, 1::2] - want[0, 1::2]).max() <= TOL
    assert np.abs(got[0, ::2] - want[0, ::2]).max() <= TOL * spread


@pytest.mark.parametrize("quant", [False, True])
def test_weight_on_a_row_of_small_values(ctx, quant):
    """Most of the weight on a position whose values are tiny (a sink): the
    rest, 2^-20 of the weight, decides the output."""
    rng = np.random.default_rng(9)
    nodes, base = 9, 200
    g, blk, nb = _block(ctx, rng, 12, 2, 48, 256, base + nodes, 1)
    off = nd.kv_offsets(g)
    q = np.abs(rng.normal(size=(1, nodes, 12 * 48))).astype(np.float32)
    kv = blk[:2 * 256 * 48].view(torch.int8).view(2, 256, 48)
    kv[:, 5] = 100
    blk[off["ks"]:off["ks"] + 4 * 512].view(torch.float32).view(2, 256)[:, 5] = 0.03
    blk[off["vs"]:off["vs"] + 4 * 512].view(torch.float32).view(2, 256)[:, 5] = 1e-9
    see = R.bits_of(nd.tree_mask(_parents(rng, 1, nodes)), nodes)
    lo = np.zeros((1, nodes), int)
    args = (ctx, g, blk, nb, dev(np.array([base], np.int32)), dev(lo.astype(np.int32)), dev(R.words_of(see)), dev(q))
    got = host(nd.attend_tree_i8(*args, quant_query=quant))
    want = _want(g, host(blk), nb, [base], None, lo, see, q, quant)
    # scores here reach 20: their fp32 steps, 20 * 67 * 2^-24 in the worst case, are a relative error of the weights
    assert np.linalg.norm(got - want) <= 8e-5 * np.linalg.norm(want)


@pytest.mark.parametrize("quant", [False, True])
def test_queries_that_are_no_numbers(ctx, quant):
    """A head with a NaN or an infinity gives NaN, its neighbours do not."""
    rng = np.random.default_rng(12)
    nodes, base = 5, 70
    g, blk, nb = _block(ctx, rng, 12, 2, 48, 80, base + nodes, 1)
    see = R.bits_of(nd.tree_mask(_parents(rng, 1, nodes)), nodes)
    q = rng.normal(size=(1, nodes, 12, 48)).astype(np.float32)
    q[0, 1, 3, 20], q[0, 2, 0, 0], q[0, 4, 11, 47] = np.nan, np.inf, -np.inf
    q[0, 3, 5] = 0.0
    args = (ctx, g, blk, nb, dev(np.array([base], np.int32)), dev(np.zeros((1, nodes), np.int32)), dev(R.words_of(see)))
    got = host(nd.attend_tree_i8(*args, dev(q.reshape(1, nodes, -1)), quant_query=quant)).reshape(nodes, 12, 64)
    gone = np.zeros((nodes, 12), bool)
    gone[1, 3] = gone[2, 0] = gone[4, 11] = True
    assert np.isnan(got[gone]).all()
    want = _want(g, host(blk), nb, [base], None, np.zeros((1, nodes), int), see,
                 np.where(gone[None, :, :, None], 0, q).reshape(1, nodes, -1), quant).reshape(nodes, 12, 64)
    assert np.abs(got[~gone] - want[~gone]).max() <= TOL


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_any_scale(ctx, scale):
    rng = np.random.default_rng(11)
    nodes, base = 12, 100
    g, blk, nb = _block(ctx, rng, 6, 2, 64, 128, base + nodes, 1)
    see = R.bits_of(nd.tree_mask(_parents(rng, 1, nodes)), nodes)
    q = rng.normal(size=(1, nodes, 6 * 64)).astype(np.float32)
    for quant in (False, True):
        # scores grow with the scale, their errors too (the bar is set for 1 / 8)
        _check(ctx, g, blk, nb, [base], np.zeros((1, nodes), int), see, q, quant=quant, scale=scale,
               tol=TOL * max(1, 8 * abs(scale)))


def test_wrong_numbers_give_nan(ctx):
    """Rows whose numbers cannot be, and only those."""
    rng = np.random.default_rng(4)
    nodes, cap = 4, 50
    g, blk, nb = _block(ctx, rng, 12, 2, 48, cap, 44, 7)
    see = np.repeat(np.eye(nodes, dtype=np.uint8)[None], 7, 0)
    base = np.array([40, -1, 40, 40, 40, 2 ** 31 - 3, 40], np.int32)
    length = np.array([4, 4, 5, -1, 0, 4, 4], np.int32)
    lo = np.zeros((7, nodes), np.int32)
    lo[0, 1], lo[6] = -1, -2 ** 31
    lo[5] = 2 ** 31 - 5
    q = rng.normal(size=(7, nodes, 12 * 48)).astype(np.float32)
    out = torch.full((7, nodes, 12 * 64), 7.0, device="cuda")
    got = host(nd.attend_tree_i8(ctx, g, blk, nb, dev(base), dev(lo), dev(R.words_of(see)), dev(q), length=dev(length),
                                 out=out))
    assert np.isnan(got[0, 1]).all() and np.isfinite(got[0, [0, 2, 3]]).all()
    for i in (1, 2, 3, 5, 6):
        assert np.isnan(got[i]).all(), i
    assert (got[4] == 7.0).all()
    # a span one longer than the ring (51 positions written: every slot holds one)
    g, blk, nb = _block(ctx, rng, 12, 2, 48, cap, 51, 1)
    lo = np.array([[0, 1, 0, 1]], np.int32)
    got = host(nd.attend_tree_i8(ctx, g, blk[:nb], nb, dev(np.array([47], np.int32)), dev(lo),
                                 dev(R.words_of(see[:1])), dev(q[:1])))
    assert np.isnan(got[0, [0, 2]]).all() and np.isfinite(got[0, [1, 3]]).all()


def test_sessions_over_one_block(ctx):
    """kv_stride 0: several trees tried over one session's cache."""
    rng = np.random.default_rng(6)
    nodes, base = 6, 77
    g, blk, nb = _block(ctx, rng, 12, 2, 48, 90, base + nodes, 1)
    see = R.bits_of(nd.tree_mask(_parents(rng, 3, nodes)), nodes)
    q = rng.normal(size=(3, nodes, 12 * 48)).astype(np.float32)
    _check(ctx, g, blk, 0, [base] * 3, np.zeros((3, nodes), int), see, q)


def test_a_tree_of_one_node_is_a_decode_step(ctx):
    """One node a session: nd_attend_step_i8's answer for the same span."""
    rng = np.random.default_rng(8)
    g, blk, nb = _block(ctx, rng, 12, 2, 48, 300, 300, 5)
    base = np.array([299, 0, 31, 32, 100], np.int32)
    q = dev(rng.normal(size=(5, 12 * 48)).astype(np.float32))
    zero = dev(np.zeros(5, np.int32))
    for quant in (False, True):
        a = nd.attend_step_i8(ctx, g, blk, nb, zero, dev(base), q, quant_query=quant)
        b = nd.attend_tree_i8(ctx, g, blk, nb, dev(base), zero.view(5, 1), dev(np.ones((5, 1, 1), np.int32)),
                              q.view(5, 1, -1), quant_query=quant)
        assert (a - b.view(5, -1)).abs().max().item() <= TOL


def test_offsets_beyond_32_bits(ctx):
    """A block of 4.4 GB, the window and the tree near its end."""
    g = nd.kv_geom(4, 2, 64, 64, 1 << 24)
    blk = torch.empty(nd.kv_block_bytes(g), dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(10)
    first, nodes = (1 << 24) - 80, 20
    k, v = (rng.normal(size=(100, 128)).astype(np.float32) for _ in range(2))
    pos = torch.arange(first, first + 100, dtype=torch.int32, device="cuda")  # wraps after 80
    nd.kv_write(ctx, g, blk, 0, pos, dev(k), dev(v))
    see = R.bits_of(nd.tree_mask(_parents(rng, 1, nodes)), nodes)
    q = rng.normal(size=(1, nodes, 256)).astype(np.float32)
    got = host(nd.attend_tree_i8(ctx, g, blk, 0, dev(np.array([first + 80], np.int32)),
                                 dev(np.full((1, nodes), first, np.int32)), dev(R.words_of(see)), dev(q)))
    kc, ks = R.stand_for(k.reshape(100, 2, 64))
    vc, vs = R.stand_for(v.reshape(100, 2, 64))
    for n in range(nodes):
        sees = np.concatenate([np.ones(80, bool), see[0, n] != 0])
        want = R.attend(q[0, n].reshape(4, 64), kc * ks[..., None].astype(np.float64),
                        vc * vs[..., None].astype(np.float64), sees, 0.125)
        assert np.abs(got[0, n] - want.reshape(-1)).max() <= TOL


def test_refusals(ctx):
    g = nd.kv_geom(12, 2, 48, 64, 64)
    blk, nb = nd.kv_alloc(g, 2)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.zeros(2, 4, 576, device="cuda")

    def refused(what, f):
        with pytest.raises(nd.NeedleError) as e:
            f()
        assert e.value.code == nd.ND_ERR_ARG and what in str(e.value), str(e.value)

    big = torch.zeros(1, 257, 576, device="cuda")
    refused("nodes", lambda: nd.attend_tree_i8(ctx, g, blk, nb, z(1), z(1, 257), z(1, 257, 9), big))
    refused("nodes", lambda: nd.attend_tree_i8(ctx, g, blk, nb, z(2), z(2, 1), z(2, 1, 1), q[:, :0]))
    for bad in (nd.kv_geom(12, 2, 32, 64, 64), nd.kv_geom(12, 2, 64, 128, 64), nd.kv_geom(18, 2, 48, 64, 64)):
        store, bb = nd.kv_alloc(nd.kv_geom(12, 2, 64, 128, 64), 2)
        refused("", lambda: nd.attend_tree_i8(ctx, bad, store, bb, z(2), z(2, 4), z(2, 4, 1),
                                              torch.zeros(2, 4, 18 * 64, device="cuda"),
                                              out=torch.zeros(2, 4, 18 * 128, device="cuda")))
    refused("aligned", lambda: nd.attend_tree_i8(ctx, g, blk[64:], nb, z(1), z(1, 4), z(1, 4, 1), q[:1]))
    huge = nd.kv_geom(96, 48, 48, 64, 1 << 24)
    rc = nd.lib().nd_attend_tree_i8(ctx.h, huge, blk.data_ptr(), 0, 1, 1, blk.data_ptr(), None, blk.data_ptr(),
                                    blk.data_ptr(), q.data_ptr(), 1.0, 0, q.data_ptr(), None, 0)
    assert rc == nd.ND_ERR_ARG and "2^29" in nd.last_error()
    ok = (z(2), z(2, 4), z(2, 4, 1), q)
    assert nd.attend_tree_i8(ctx, g, blk, nb, *ok).shape == (2, 4, 768)
    for args, kw in (((z(1), *ok[1:]), {}), ((ok[0], z(2, 3), *ok[2:]), {}), ((*ok[:2], z(2, 3, 1), q), {}),
                     ((*ok[:3], q.view(8, 576)), {}), ((*ok[:3], q.double()), {}), (ok, dict(out=q)),
                     (ok, dict(length=z(1))), ((*ok[:3], q.cpu()), {}), ((ok[0].long(), *ok[1:]), {}),
                     (ok, dict(work=z(4)))):
        with pytest.raises(ValueError):
            nd.attend_tree_i8(ctx, g, blk, nb, *args, **kw)
    with pytest.raises(ValueError):
        nd.attend_tree_i8(ctx, g, blk[:nb], nb, *ok)  # two sessions, one block
    assert nd.attend_tree_i8(ctx, g, blk, nb, z(0), z(0, 4), z(0, 4, 1), q[:0]).shape == (0, 4, 768)


def test_an_output_over_the_queries_is_refused(ctx):
    g = nd.kv_geom(12, 12, 64, 64, 64)
    blk, nb = nd.kv_alloc(g, 2)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    both = torch.zeros(4 * 4 * 768, device="cuda")
    part = lambda at: both[at * 4 * 768:][:2 * 4 * 768].view(2, 4, 768)  # noqa: E731
    args = ctx, g, blk, nb, z(2), z(2, 4), z(2, 4, 1)
    for q_at, out_at in ((0, 0), (0, 1), (2, 1)):
        with pytest.raises(nd.NeedleError, match="overlaps"):
            nd.attend_tree_i8(*args, part(q_at), out=part(out_at))
    for q_at, out_at in ((0, 2), (2, 0)):
        nd.attend_tree_i8(*args, part(q_at), out=part(out_at))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("sessions,base", [(1, 0), (3, 70), (1, 3000), (300, 200)])
def test_nothing_to_see_for_a_query_that_is_no_number(ctx, sessions, base, quant):
    """A node that attends to nothing gets zeros whatever its query holds and
    whatever the nodes beside it read, and with a scale that is no number."""
    rng = np.random.default_rng(base)
    nodes = 5
    g, blk, _ = _block(ctx, rng, 12, 2, 48, base + nodes, base + nodes, 1)
    see = np.repeat(np.tril(np.ones((nodes, nodes), np.uint8))[None], sessions, 0)
    see[:, [1, 3]] = 0
    lo = np.zeros((sessions, nodes), np.int32)
    lo[:, 1], lo[:, 3] = base, base + 9
    q = rng.normal(size=(sessions, nodes, 12, 48)).astype(np.float32)
    q[:, 1, :, 7], q[:, 3, ::2, 40], q[:, 3, 1::2, 0] = np.nan, np.inf, -np.inf
    q[:, 2, 4, 47] = np.nan  # sees what the root sees
    args = (ctx, g, blk, 0, dev(np.full(sessions, base, np.int32)), dev(lo), dev(R.words_of(see)),
            dev(q.reshape(sessions, nodes, -1)))
    got = host(nd.attend_tree_i8(*args, quant_query=quant)).reshape(sessions, nodes, 12, 64)
    assert not got[:, [1, 3]].any()
    assert np.isnan(got[:, 2, 4]).all()
    assert np.isfinite(got[:, [0, 4]]).all() and np.isfinite(np.delete(got[:, 2], 4, 1)).all()
    got = host(nd.attend_tree_i8(*args, quant_query=quant, scale=float("nan")))
    assert not got[:, [1, 3]].any() and np.isnan(got[:, [0, 2, 4]]).all()


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("sessions", [1, 300])
def test_sums_of_large_values(ctx, sessions, quant):
    """Thousands of values near fp32's end: their mean is there, their sum is not."""
    rng = np.random.default_rng(15)
    nodes, base = 2, 4000
    g, blk, nb = _block(ctx, rng, 12, 2, 48, base + nodes, base + nodes, 1, 0.05, 5e37)
    off = nd.kv_offsets(g)
    v = blk[off["v"]:off["v"] + 2 * (base + nodes) * 64].view(torch.int8)
    v.copy_(v.abs())
    see = np.repeat(np.tril(np.ones((nodes, nodes), np.uint8))[None], sessions, 0)
    q = rng.normal(size=(sessions, nodes, 12 * 48)).astype(np.float32)
    lo = np.zeros((sessions, nodes), np.int32)
    got = host(nd.attend_tree_i8(ctx, g, blk, 0, dev(np.full(sessions, base, np.int32)), dev(lo),
                                 dev(R.words_of(see)), dev(q), quant_query=quant))
    want = _want(g, host(blk), nb, [base], None, lo[:1], see[:1], q[:1], quant)
    assert np.abs(got[0] - want[0]).max() <= TOL * 5e37


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("sink", [1e-9, 1e-20, 0.0])
@pytest.mark.parametrize("ahead", [5, 15, 20, 25, 30, 60])
@pytest.mark.parametrize("sessions,H,KVH,QK", [(1, 12, 2, 48), (300, 12, 2, 48), (70, 4, 4, 64)])
def test_the_rest_behind_rows_of_next_to_no_values(ctx, sessions, H, KVH, QK, ahead, sink, quant):
    """Positions that take all but 2^-ahead of the weight and hold values next to
    zero, or zeros (of scale 1), one in each of the first 32 chunks, so that each
    wave meets one before most of its walk: the rest decides the output.

    Tolerance, of each head by itself.  A head's error is at most delta sum(w |v|)
    / sum(w), delta the relative error of a weight: a score's fp32 sum, 67 * 2^-24
    of the sum of the products' magnitudes (these queries are a quarter of N(0, 1),
    keys N(0, 1): below 67 * 2^-24 * 13 / 6.9 = 7.5e-6); its distance from the
    maximum, less than ahead + 12 bits, of ln 2 each, off by seven roundings (the
    scale, its product with log2 e, the query's scale, the key's, the product, the
    difference, the sums' scaling): 5 * 2^-24 (ahead + 12); the weight itself and
    its sums, 8 * 2^-24.
    """
    rng = np.random.default_rng(ahead)
    nodes, base, cap = 2, 5000, 5100
    g, blk, nb = _block(ctx, rng, H, KVH, QK, cap, base + nodes, 1)
    off = nd.kv_offsets(g)
    part = lambda at, n: blk[at:at + n]  # noqa: E731
    kc = part(0, KVH * cap * QK).view(torch.int8).view(KVH, cap, QK)
    vc = part(off["v"], KVH * cap * 64).view(torch.int8).view(KVH, cap, 64)
    ks, vs = (part(off[s], 4 * KVH * cap).view(torch.float32).view(KVH, cap) for s in ("ks", "vs"))
    at = torch.arange(32, device="cuda") * 32 + 5
    kc[:, :, 0] = 0
    kc[:, at] = 0
    kc[:, at, 0] = 127
    vc[:] = vc.abs()  # all of one sign: the rest does not average out
    vc[:, at] = 100 if sink else 0
    vs[:, at] = sink if sink else 1.0
    q = rng.normal(size=(sessions, nodes, H, QK)).astype(np.float32) / 4
    q[..., 0] = 4.0
    bits = 1 / np.sqrt(QK) / np.log(2)
    # the rest: about 5000 weights of 2^0 on average, 2^12.3 together
    ks[:, at] = (ahead + 12.3 - 5) / (127 * 4 * bits)
    see = np.repeat(np.tril(np.ones((nodes, nodes), np.uint8))[None], sessions, 0)
    lo = np.zeros((sessions, nodes), np.int32)
    got = host(nd.attend_tree_i8(ctx, g, blk, 0, dev(np.full(sessions, base, np.int32)), dev(lo),
                                 dev(R.words_of(see)), dev(q.reshape(sessions, nodes, -1)), quant_query=quant))
    delta = 7.5e-6 + 2.0 ** -24 * (8 + 5 * (ahead + 12))
    b = host(blk)
    for i in {0, sessions // 2, sessions - 1}:
        one = (g, b, nb, [base], None, lo[i:i + 1], see[i:i + 1], q[i:i + 1].reshape(1, nodes, -1), quant)
        want = _want(*one)[0].reshape(nodes, H, 64)
        # with values of one sign sum(w |v|) / sum(w) is the output itself
        err = np.linalg.norm(got[i].reshape(nodes, H, 64) - want, axis=-1) / np.linalg.norm(want, axis=-1)
        assert err.max() <= delta, err.max()


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("seed", range(6))
def test_rows_far_ahead_of_any_size_anywhere(ctx, seed, quant):
    """Positions up to 2^60 ahead of the others, at any distance from one another,
    with values of 10^-12 to 1 of theirs, or zeros, among values of sizes that change
    along the cache.  The tolerance is the one above: values of one sign, the error
    of a weight."""
    rng = np.random.default_rng(seed)
    S, nodes, base, cap, H, KVH, QK = (1, 1, 130, 400)[seed % 4], 3, 6000, 6200, 12, 2, 48
    g, blk, nb = _block(ctx, rng, H, KVH, QK, cap, base + nodes, 1)
    off = nd.kv_offsets(g)
    part = lambda at, n: blk[at:at + n]  # noqa: E731
    kc = part(0, KVH * cap * QK).view(torch.int8).view(KVH, cap, QK)
    vc = part(off["v"], KVH * cap * 64).view(torch.int8).view(KVH, cap, 64)
    ks, vs = (part(off[s], 4 * KVH * cap).view(torch.float32).view(KVH, cap) for s in ("ks", "vs"))
    vc[:] = vc.abs()
    vs *= dev(10.0 ** np.repeat(rng.uniform(-2, 2, cap // 200), 200)).float()
    at = np.cumsum(rng.integers(1, (20, 90, 300)[seed % 3], base))
    at = dev(at[at < base])
    kc[:, :, 0] = 0
    kc[:, at] = 0
    kc[:, at, 0] = 127
    bits = 1 / np.sqrt(QK) / np.log(2)
    ks[:, at] = dev(rng.uniform(0, 60, len(at)) / (127 * 4 * bits)).float()
    vs[:, at] *= dev(10.0 ** rng.uniform(-12, 0, len(at))).float()
    none = at[dev(rng.random(len(at)) < 0.3)]
    vc[:, none], vs[:, none] = 0, 1.0
    q = rng.normal(size=(S, nodes, H, QK)).astype(np.float32) / 4
    q[..., 0] = 4.0
    see = np.repeat(np.tril(np.ones((nodes, nodes), np.uint8))[None], S, 0)
    lo = rng.integers(0, 400, (S, nodes)).astype(np.int32)
    got = host(nd.attend_tree_i8(ctx, g, blk, 0, dev(np.full(S, base, np.int32)), dev(lo),
                                 dev(R.words_of(see)), dev(q.reshape(S, nodes, -1)), quant_query=quant))
    delta = 7.5e-6 + 2.0 ** -24 * (8 + 5 * 72)
    b = host(blk)
    for i in {0, S // 2, S - 1}:
        want = _want(g, b, nb, [base], None, lo[i:i + 1], see[i:i + 1], q[i:i + 1].reshape(1, nodes, -1), quant)
        want = want[0].reshape(nodes, H, 64)
        err = np.linalg.norm(got[i].reshape(nodes, H, 64) - want, axis=-1) / np.linalg.norm(want, axis=-1)
        assert err.max() <= delta, err.max()


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("garbage", [3e38, -3e38, -np.inf, 1e30, -1e-40])
def test_scales_of_nodes_no_row_names(ctx, garbage, quant):
    """A node of the tree that no mask names need not have been written: whatever
    numbers lie there, the others' outputs are what they were."""
    rng = np.random.default_rng(14)
    nodes, base, cap = 40, 900, 1000
    g, blk, nb = _block(ctx, rng, 12, 2, 48, cap, base + nodes, 1, 1.0, 1e-3)
    see = np.tril(np.ones((nodes, nodes), np.uint8))[None].copy()
    see[:, :, [3, 33, 38]] = 0
    q = rng.normal(size=(1, nodes, 12 * 48)).astype(np.float32)
    off = nd.kv_offsets(g)
    for part in ("ks", "vs"):
        s = blk[off[part]:off[part] + 4 * 2 * cap].view(torch.float32).view(2, cap)
        s[:, [base + 3, base + 33, base + 38]] = garbage
    lo = np.zeros((1, nodes), int)
    got = host(nd.attend_tree_i8(ctx, g, blk, nb, dev(np.array([base], np.int32)), dev(lo.astype(np.int32)),
                                 dev(R.words_of(see)), dev(q), quant_query=quant))
    want = _want(g, host(blk), nb, [base], None, lo, see, q, quant)
    assert np.abs(got - want).max() <= 1e-3 * TOL


def test_work_of_sizes_that_are_refused(ctx):
    g = nd.kv_geom(12, 2, 48, 64, 4096)
    assert nd.attend_tree_i8_work(ctx, g, 1, 4) > 0
    for bad, count, nodes in ((nd.kv_geom(2, 4, 48, 64, 4096), 1, 4), (nd.kv_geom(18, 2, 48, 64, 4096), 1, 4),
                              (nd.kv_geom(12, 5, 48, 64, 4096), 1, 4), (nd.kv_geom(12, 2, 32, 64, 4096), 1, 4),
                              (nd.kv_geom(12, 2, 48, 64, (1 << 24) + 1), 1, 4), (g, 65536, 4), (g, 1 << 63, 4),
                              (g, 1, 0), (g, 0, 4), (g, 1, 257), (g, 1, 1 << 62)):
        assert nd.attend_tree_i8_work(ctx, bad, count, nodes) == 0


def test_more_sessions_than_a_launch_holds(ctx):
    """Sessions on both sides of the border between two launches."""
    rng = np.random.default_rng(17)
    S, base, KVH = 50000, 6, 12
    first = (1 << 18) // KVH  # of the second launch
    g, blk, nb = _block(ctx, rng, KVH, KVH, 64, base + 1, base + 1, 1)
    bases = np.arange(S) % (base + 1)
    length = (np.arange(S) % 11 != 3).astype(np.int32)
    lo = np.minimum(np.arange(S)[:, None] % 3, bases[:, None])
    see = (np.arange(S) % 5 != 1).astype(np.uint8).reshape(S, 1, 1)
    q = rng.normal(size=(S, 1, KVH * 64)).astype(np.float32)
    rows = sorted({0, 1, 3, S - 1, *(first + np.arange(-12, 12)), *(2 * first + np.arange(-12, 12))})
    _check(ctx, g, blk, 0, bases, lo, see, q, length, rows=rows)


def test_query_codes_of_a_subnormal_scale(ctx):
    """A query whose scale's inverse is beyond fp32: codes of 127, -128 and (of
    0 times infinity) no number, as the quantiser's steps give them."""
    rng = np.random.default_rng(16)
    nodes, base = 16, 200
    g, blk, nb = _block(ctx, rng, 12, 2, 48, 256, base + nodes, 1, 1e37, 1.0)
    see = R.bits_of(nd.tree_mask(_parents(rng, 1, nodes)), nodes)
    q = (rng.normal(size=(1, nodes, 12, 48)) * 1e-37).astype(np.float32)
    q[0, 5, 7, 3] = 0.0
    args = (ctx, g, blk, nb, dev(np.array([base], np.int32)), dev(np.zeros((1, nodes), np.int32)),
            dev(R.words_of(see)), dev(q.reshape(1, nodes, -1)))
    got = host(nd.attend_tree_i8(*args, quant_query=True)).reshape(nodes, 12, 64)
    assert np.isnan(got[5, 7]).all()
    q[0, 5, 7, 3] = 1e-37
    want = _want(g, host(blk), nb, [base], None, np.zeros((1, nodes), int), see, q.reshape(1, nodes, -1), True)
    there = np.ones((nodes, 12), bool)
    there[5, 7] = False
    # every element counts 127 or 128 times qs, 2.5 |q| and more here: scores up to 20, of 48 equal codes
    assert np.abs(got - want.reshape(nodes, 12, 64))[there].max() <= 8 * TOL
