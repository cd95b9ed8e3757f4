"""Rotary rows, the cache written with rotation and the cache read back,
against plain 64-bit forms.

Tolerances.  A turned element is worked out in fp64 and rounded to fp32 once:
half a step, 2^-24 of it, and what fp64 leaves of the angle pos f: f's power
and the product are each off by 2^-53 of the angle, which is at most pos (f <=
1 here), sine and cosine by about 2^-53: together below pos 2^-51 of the
pair's larger element, taken as 2^-50 (pos + 4).  A code follows from the
turned value times 1 / scale (both fp32): off by 127 steps of 2^-24 three
times over at most, 2.3e-5 of a code, so a code is the plain form's unless the
plain value lies within 1e-4 of the border between two codes.
"""
import numpy as np
import pytest
import torch

import needle_amd as nd
import tree_ref as R
from conftest import dev, host

pytestmark = pytest.mark.gpu

SCALINGS = {"plain": {}, "linear": dict(scaling="linear", factor=4.0),
            "parts": dict(scaling="parts", factor=8.0, trained=2048, turns=(1.0, 20.0))}


def _spec(rot, layout, how, theta=10000.0, gain=1.0):
    kw = SCALINGS[how]
    return nd.rope(rot, theta=theta, layout=layout, gain=gain, **kw), R.freqs(rot, theta, **kw)


def _near(got, want, x, pos, gain=1.0):
    tol = 2.0 ** -24 * np.abs(want) + 2.0 ** -50 * (np.asarray(pos, np.float64)[:, None, None] + 4) * abs(gain) * \
        2 * np.abs(x).max()
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


@pytest.mark.parametrize("how", list(SCALINGS))
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("rows,heads,dim,rot", [(1, 1, 2, 2), (1, 12, 48, 48), (7, 3, 64, 48), (33, 5, 30, 10),
                                                (65, 2, 256, 256), (300, 12, 64, 64), (5, 40, 128, 2), (9, 3, 17, 6)])
def test_rope_rows(ctx, rows, heads, dim, rot, layout, how):
    rng = np.random.default_rng(rows * dim + rot)
    r, f = _spec(rot, layout, how, gain=1.25)
    x = rng.normal(size=(rows, heads, dim)).astype(np.float32)
    pos = rng.integers(0, 100000, rows).astype(np.int32)
    pos[0] = 0
    y = host(nd.rope_rows(ctx, r, dev(x.reshape(rows, -1)), dev(pos), heads)).reshape(x.shape)
    _near(y, R.turned(x, pos, f, layout, 1.25), x, pos, 1.25)
    assert np.array_equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_rope_far_positions(ctx, layout):
    rng = np.random.default_rng(1)
    r, f = _spec(64, layout, "plain", theta=1e6)
    pos = np.array([2 ** 24 - 1, 10 ** 7 + 1, 2 ** 31 - 1, 999983], np.int32)
    x = rng.normal(size=(4, 2, 64)).astype(np.float32)
    y = host(nd.rope_rows(ctx, r, dev(x.reshape(4, -1)), dev(pos), 2)).reshape(x.shape)
    _near(y, R.turned(x, pos, f, layout), x, pos)


@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("dim,rot,off", [(48, 48, 0), (48, 40, 1), (30, 30, 3), (64, 16, 2)])
def test_rope_strided_in_place_and_padding(ctx, dim, rot, off, layout):
    """Rows apart at any alignment; in place; rows of negative position and the
    elements between rows stay as they are."""
    rng = np.random.default_rng(dim + off)
    r, f = _spec(rot, layout, "plain")
    rows, heads = 50, 3
    buf = rng.normal(size=(rows, off + heads * dim + 5)).astype(np.float32)
    pos = rng.integers(0, 5000, rows).astype(np.int32)
    pos[[0, 7, 49]] = -1, -5, -1
    want = buf.copy().astype(np.float64)
    x = buf[:, off:off + heads * dim].reshape(rows, heads, dim)
    want[:, off:off + heads * dim] = np.where((pos < 0)[:, None], x.reshape(rows, -1),
                                              R.turned(x, np.maximum(pos, 0), f, layout).reshape(rows, -1))
    t = dev(buf)
    view = t[:, off:off + heads * dim]
    other = torch.full((rows, heads * dim + 3), 7.0, device="cuda")
    nd.rope_rows(ctx, r, view, dev(pos), heads, out=other[:, :heads * dim])
    o = host(other)
    assert (o[pos < 0] == 7.0).all() and (o[:, heads * dim:] == 7.0).all()
    nd.rope_rows(ctx, r, view, dev(pos), heads, out=view)
    got = host(t)
    _near(got[:, None], want[:, None], buf, np.maximum(pos, 0))
    same = np.ones(buf.shape, bool)
    same[pos >= 0, off:off + heads * dim] = False
    assert np.array_equal(got[same], buf[same])
    assert np.array_equal(o[pos >= 0, :heads * dim], got[pos >= 0, off:off + heads * dim])


def test_rope_of_the_forward_layout(ctx):
    """Position 0 turns nothing, and turning by a then b is turning by a + b."""
    r, _ = _spec(48, "halves", "plain")
    x = torch.randn(10, 12 * 48, device="cuda")
    zero = torch.zeros(10, dtype=torch.int32, device="cuda")
    assert torch.equal(nd.rope_rows(ctx, r, x, zero, 12), x)
    a = nd.rope_rows(ctx, r, nd.rope_rows(ctx, r, x, zero + 100, 12), zero + 23, 12)
    b = nd.rope_rows(ctx, r, x, zero + 123, 12)
    assert (a - b).abs().max().item() <= 2 * 2.0 ** -23 * x.abs().max().item() * 1.5


def _blocks(g, count):
    blk, nb = nd.kv_alloc(g, count)
    blk.fill_(0x5a)
    return blk, nb


def _near_codes(got, scale, want):
    """Codes and scales against the exact turned rows."""
    codes, ref = R.stand_for(want)
    assert (np.abs(scale.astype(np.float64) - ref) <= 2.0 ** -22 * ref).all()
    y = np.abs(want / ref[..., None].astype(np.float64))
    border = np.abs(y - np.floor(y) - 0.5) < 1e-4
    off = got.astype(int) - codes
    assert (off[~border] == 0).all() and (np.abs(off) <= 1).all()


@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("H,KVH,QK,VD,rot", [(12, 2, 48, 64, 48), (12, 12, 64, 64, 40), (5, 1, 16, 32, 2),
                                             (4, 2, 256, 128, 256), (6, 3, 96, 16, 34)])
@pytest.mark.parametrize("blocks,per,cap", [(1, 1, 1), (3, 5, 17), (2, 130, 200)])
def test_write_rope(ctx, H, KVH, QK, VD, rot, blocks, per, cap, layout):
    """Wrapped rings, several rows a block, fused projections, padding."""
    rng = np.random.default_rng(QK + per)
    r, f = _spec(rot, layout, "plain")
    g = nd.kv_geom(H, KVH, QK, VD, cap)
    blk, nb = _blocks(g, blocks)
    n = blocks * per
    pos = (1000 + np.arange(n) % per).astype(np.int32)
    turn = rng.integers(0, 9000, n).astype(np.int32)
    if per > 2:
        pos[[1, n - 1]] = -1
    buf = rng.normal(size=(n, (H + KVH) * QK + KVH * VD + 3)).astype(np.float32)
    buf[0, H * QK:H * QK + QK] = 0.0  # a key of zeros
    t = dev(buf)
    q, k, v = t[:, :H * QK], t[:, H * QK:(H + KVH) * QK], t[:, (H + KVH) * QK:(H + KVH) * QK + KVH * VD]
    out = torch.full((n, H * QK), 7.0, device="cuda")
    before = host(blk)
    nd.kv_write_rope(ctx, g, r, blk, nb, dev(pos), k, v, q=q, q_out=out, rot_pos=dev(turn), per_block=per)
    there = pos >= 0
    x = buf[:, :H * QK].reshape(n, H, QK)
    o = host(out).reshape(n, H, QK)
    _near(o[there], R.turned(x, turn, f, layout)[there], x, turn[there])
    assert (o[~there] == 7.0).all()
    kw = R.turned(buf[:, H * QK:(H + KVH) * QK].reshape(n, KVH, QK), turn, f, layout)
    vw = buf[:, (H + KVH) * QK:(H + KVH) * QK + KVH * VD].reshape(n, KVH, VD)
    b = host(blk)
    touched = np.zeros_like(b, bool)
    for i in range(blocks):
        kc, ks, vc, vs = nd.kv_unpack(g, b[i * nb:(i + 1) * nb])
        rows = np.flatnonzero(there & (np.arange(n) // per == i))
        slot = pos[rows] % cap
        _near_codes(kc[slot], ks[slot], kw[rows])
        _near_codes(vc[slot], vs[slot], vw[rows].astype(np.float64))
        off = nd.kv_offsets(g)
        for s in slot:
            for h in range(KVH):
                for start, width in ((0, QK), (off["v"], VD), (off["ks"], 4), (off["vs"], 4)):
                    a = i * nb + start + (h * cap + s) * width
                    touched[a:a + width] = True
    assert np.array_equal(b[~touched], before[~touched])  # nothing else is written
    # the same rows through rope_rows and kv_write, bit for bit
    two, _ = _blocks(g, blocks)
    kt = nd.rope_rows(ctx, r, k, dev(turn), KVH)
    for i in range(blocks):
        a = slice(i * per, (i + 1) * per)
        nd.kv_write(ctx, g, two[i * nb:(i + 1) * nb], 0, dev(pos[a]), kt[a], v[a].contiguous())
    assert torch.equal(two, blk)
    # in place, and without queries
    again, _ = _blocks(g, blocks)
    nd.kv_write_rope(ctx, g, r, again, nb, dev(pos), k, v, rot_pos=dev(turn), per_block=per)
    assert torch.equal(again, blk)
    nd.kv_write_rope(ctx, g, r, again, nb, dev(pos), k, v, q=q, q_out=q, rot_pos=dev(turn), per_block=per)
    assert torch.equal(again, blk) and np.array_equal(host(q)[there], host(out)[there])
    assert np.array_equal(host(t)[:, H * QK:], buf[:, H * QK:])


@pytest.mark.parametrize("H,KVH,QK,VD", [(12, 2, 48, 64), (3, 3, 96, 128), (2, 1, 256, 16)])
def test_write_of_values_that_are_no_numbers(ctx, H, KVH, QK, VD):
    """NaN, infinities, zeros and values next to fp32's ends: the codes and scales
    that kv_write stores for the same turned rows, bit for bit."""
    rng = np.random.default_rng(QK)
    n = 9
    k, v = (rng.normal(size=(n, KVH * d)).astype(np.float32) for d in (QK, VD))
    for x in (k, v):
        x[0, 3], x[1, 5], x[2, 0], x[3, :] = np.nan, np.inf, -np.inf, 0.0
        x[4] *= 1e38
        x[5] *= 1e-38
        x[6] *= 1e-44
        x[7, :4] = [3e38, -3e38, 1e-45, 0.0]
    r, g = nd.rope(QK - 16 if QK > 48 else 48, layout="pairs"), nd.kv_geom(H, KVH, QK, VD, 16)
    a, _ = _blocks(g, 1)
    b, _ = _blocks(g, 1)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    nd.kv_write_rope(ctx, g, r, a, 0, pos, dev(k), dev(v), rot_pos=pos + 70, per_block=n)
    nd.kv_write(ctx, g, b, 0, pos, nd.rope_rows(ctx, r, dev(k), pos + 70, KVH), dev(v))
    assert torch.equal(a, b)


@pytest.mark.parametrize("H,KVH,QK,VD", [(12, 2, 48, 64), (12, 12, 64, 64), (5, 1, 16, 256), (6, 3, 96, 16)])
@pytest.mark.parametrize("blocks,per,cap", [(1, 1, 1), (3, 5, 17), (2, 301, 400)])
def test_read_back(ctx, H, KVH, QK, VD, blocks, per, cap):
    """Codes times scale, to the bit; zeros at negative positions; the same
    position twice."""
    rng = np.random.default_rng(cap)
    g = nd.kv_geom(H, KVH, QK, VD, cap)
    blk, nb = nd.kv_alloc(g, blocks)
    b = rng.integers(0, 256, blocks * nb, dtype=np.uint8)
    off = nd.kv_offsets(g)
    for i in range(blocks):
        for part in ("ks", "vs"):
            s = rng.lognormal(size=KVH * cap).astype(np.float32)
            b[i * nb + off[part]:i * nb + off[part] + s.nbytes] = s.view(np.uint8)
    blk.copy_(dev(b))
    n = blocks * per
    pos = rng.integers(0, 3 * cap, n).astype(np.int32)
    pos[rng.random(n) < 0.2] = -1
    k, v = nd.kv_read(ctx, g, blk, nb, dev(pos), per_block=per)
    k, v = host(k).reshape(n, KVH, QK), host(v).reshape(n, KVH, VD)
    blocks_of = [nd.kv_unpack(g, b[i * nb:(i + 1) * nb]) for i in range(blocks)]
    for i in range(n):
        if pos[i] < 0:
            assert not k[i].any() and not v[i].any()
            continue
        kc, ks, vc, vs = blocks_of[i // per]
        s = pos[i] % cap
        assert np.array_equal(k[i], kc[s].astype(np.float32) * ks[s][:, None]), i
        assert np.array_equal(v[i], vc[s].astype(np.float32) * vs[s][:, None]), i


def test_offsets_beyond_32_bits(ctx):
    """A block of 4.4 GB: rows near its end, in every head."""
    g = nd.kv_geom(4, 2, 64, 64, 1 << 24)
    blk = torch.empty(nd.kv_block_bytes(g), dtype=torch.uint8, device="cuda")
    assert blk.numel() > 1 << 32
    pos = torch.tensor([(1 << 24) - 1, (1 << 24) - 5, (1 << 25) - 2, 3], dtype=torch.int32, device="cuda")
    r, f = _spec(64, "pairs", "plain")
    x = np.random.default_rng(0).normal(size=(4, 256)).astype(np.float32)
    t = dev(x)
    nd.kv_write_rope(ctx, g, r, blk, 0, pos, t[:, :128], t[:, 128:], per_block=4)
    k, v = nd.kv_read(ctx, g, blk, 0, pos, per_block=4)
    want = R.turned(x[:, :128].reshape(4, 2, 64), host(pos), f, "pairs")
    for got, ref in ((host(k), want), (host(v), x[:, 128:].reshape(4, 2, 64))):
        codes, scale = R.stand_for(ref)
        assert np.abs(got.reshape(4, 2, 64) - codes * scale[..., None]).max() <= 1.01 * scale.max()
        assert np.abs(got.reshape(4, 2, 64) - ref).max() <= 0.51 * scale.max()


def test_no_rows(ctx):
    r, g = nd.rope(48), nd.kv_geom(12, 2, 48, 64, 16)
    blk, nb = nd.kv_alloc(g, 1)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    e = lambda w: torch.empty(0, w, device="cuda")  # noqa: E731
    assert nd.rope_rows(ctx, r, e(576), none, 12).shape == (0, 576)
    assert nd.kv_write_rope(ctx, g, r, blk, nb, none, e(96), e(128), q=e(576)).shape == (0, 576)
    assert nd.kv_read(ctx, g, blk, nb, none)[0].shape == (0, 96)


def test_refusals(ctx):
    x = torch.zeros(4, 96, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")

    def refused(what, code, f):
        with pytest.raises(nd.NeedleError) as e:
            f()
        assert e.value.code == code and what in str(e.value), str(e.value)

    for r, what in ((nd.rope(47), "rot_dim"), (nd.rope(0), "rot_dim"), (nd.rope(258), "rot_dim"),
                    (nd.rope(48, theta=0.0), "theta"), (nd.rope(48, theta=float("nan")), "theta"),
                    (nd.rope(48, gain=float("inf")), "gain"), (nd.rope(48, scaling="linear", factor=0.0), "factor"),
                    (nd.rope(48, scaling="parts", factor=2.0), "trained"),
                    (nd.rope(48, scaling="parts", factor=2.0, trained=9, turns=(2.0, 2.0)), "turns"),
                    (nd.rope(64), "dim 48")):
        refused(what, nd.ND_ERR_ARG, lambda: nd.rope_rows(ctx, r, x, pos, 2))
    r = nd.rope(48)
    both = torch.zeros(4 * 96 + 8, device="cuda")
    refused("overlaps", nd.ND_ERR_ARG, lambda: nd.rope_rows(ctx, r, both[:384].view(4, 96), pos, 2,
                                                            out=both[8:392].view(4, 96)))
    g = nd.kv_geom(2, 2, 48, 64, 8)
    blk, nb = nd.kv_alloc(g, 1)
    v = torch.zeros(4, 128, device="cuda")
    refused("rot_dim", nd.ND_ERR_ARG, lambda: nd.kv_write_rope(ctx, g, nd.rope(64), blk, 0, pos, x, v, per_block=4))
    refused("overlaps", nd.ND_ERR_ARG, lambda: nd.kv_write_rope(ctx, g, r, blk, 0, pos, x, v, q=torch.zeros(4, 96, device="cuda"),
                                                                q_out=x, per_block=4))
    refused("aligned", nd.ND_ERR_ARG, lambda: nd.kv_write_rope(ctx, g, r, nd.kv_alloc(g, 2)[0][16:], 0, pos, x, v, per_block=4))
    for f in (lambda: nd.rope_rows(ctx, r, x, pos, 5), lambda: nd.rope_rows(ctx, r, x, pos[:3], 2),
              lambda: nd.rope_rows(ctx, r, x.double(), pos, 2), lambda: nd.rope_rows(ctx, r, x, pos.long(), 2),
              lambda: nd.rope_rows(ctx, r, x.cpu(), pos, 2), lambda: nd.rope_rows(ctx, r, x, pos, 2, out=x[:, :48]),
              lambda: nd.rope_rows(ctx, r, x.t().contiguous().t(), pos, 2),
              lambda: nd.rope_rows(ctx, r, x[:1].expand(4, 96), pos, 2),
              lambda: nd.kv_write_rope(ctx, g, r, blk, nb, pos, x, v),  # four blocks, one there
              lambda: nd.kv_write_rope(ctx, g, r, blk, nb, pos, x, x, per_block=4),
              lambda: nd.kv_write_rope(ctx, g, r, blk, nb, pos, x, v, per_block=0),
              lambda: nd.kv_write_rope(ctx, g, r, blk, nb, pos, x, v, q_out=x, per_block=4),
              lambda: nd.kv_read(ctx, g, blk, nb, pos), lambda: nd.kv_read(ctx, g, blk, nb, pos, per_block=4, k=x[:3])):
        with pytest.raises(ValueError):
            f()
