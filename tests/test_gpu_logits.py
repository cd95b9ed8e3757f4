"""Logits under rules and the pick, against a plain 64-bit form.

Tolerance: a logit goes through at most six fp32 roundings (the quotient or
product of the repeat penalty, count times frequency, its subtraction, the
presence's, and the bias's sum), each half a step, 2^-24 of a value that is
at most the sum of the magnitudes that went in: 6 * 2^-24 of that sum, and
2^-24 more for each further bias of the same token.
"""
import numpy as np
import pytest
import torch

import needle_amd as nd
import tree_ref as R
from conftest import dev, host

pytestmark = pytest.mark.gpu


def _plain(x, c):
    """(y, magnitudes) in 64 bits, row by row."""
    y = x.astype(np.float64)
    size = np.abs(y)
    rows, n = x.shape
    for i in range(rows):
        if c.get("hist") is not None:
            h = c["hist"][i]
            m = min(max(c["hist_len"][i], 0), len(h)) if "hist_len" in c else len(h)
            start = max(c["out_from"][i], 0) if "out_from" in c else 0
            ok = lambda a: a[(a >= 0) & (a < n)]  # noqa: E731
            ever = np.unique(ok(h[:m]))
            made = np.bincount(ok(h[start:m]), minlength=n)
            if "repeat" in c:
                r = float(c["repeat"][i])
                z = y[i, ever]
                y[i, ever] = np.where(z > 0, z / r, z * r)
                size[i, ever] = np.maximum(size[i, ever], np.abs(y[i, ever]))
            if "frequency" in c:
                y[i] -= made * float(c["frequency"][i])
                size[i] += np.abs(made * float(c["frequency"][i]))
            if "presence" in c:
                y[i] -= (made > 0) * float(c["presence"][i])
                size[i] += (made > 0) * abs(float(c["presence"][i]))
        if "bias" in c:
            m = min(max(c["bias_len"][i], 0), c["bias"].shape[1]) if "bias_len" in c else c["bias"].shape[1]
            for t, b in zip(c["bias_id"][i, :m], c["bias"][i, :m]):
                if 0 <= t < n:
                    y[i, t] += float(b)
                    size[i, t] += 1.2 * abs(float(b))
        if "mask" in c:
            row = c["mask_row"][i] if "mask_row" in c else i
            if 0 <= row < len(c["mask"]):
                y[i, R.bits_of(c["mask"][row], n) == 0] = -np.inf
    return y, size


def _first(row):
    best, at = -np.inf, -1
    for i in np.flatnonzero(row > -np.inf):
        if row[i] > best:
            best, at = row[i], i
    return at


def _run(ctx, x, c, **kw):
    return nd.logits_adjust(ctx, x if torch.is_tensor(x) else dev(x), **{k: dev(v) for k, v in c.items()}, **kw)


def _check(ctx, x, c):
    out, nxt = _run(ctx, x, c, pick=True)
    out, nxt = host(out), host(nxt)
    want, size = _plain(x, c)
    gone = np.isneginf(want)
    assert np.array_equal(np.isneginf(out), gone)
    assert (np.abs(out - want)[~gone] <= 6 * 2.0 ** -24 * size[~gone]).all(), np.abs(out - want)[~gone].max()
    assert nxt.tolist() == [_first(r) for r in out]
    assert np.array_equal(host(_run(ctx, x, c, write=False)), nxt)
    t = dev(x)
    assert np.array_equal(host(_run(ctx, t, c, out=t)), out)  # in place
    return out, nxt


def _case(rng, rows, n, hist=50, biases=9, states=5):
    c = dict(hist=rng.integers(-2, n + 2 if n < 64 else max(2, n // 8), (rows, hist)).astype(np.int32),
             hist_len=rng.integers(-1, hist + 3, rows).astype(np.int32),
             out_from=rng.integers(-1, hist + 1, rows).astype(np.int32),
             repeat=rng.uniform(0.8, 2, rows).astype(np.float32), frequency=rng.uniform(-0.2, 0.6, rows).astype(np.float32),
             presence=rng.uniform(0, 1, rows).astype(np.float32),
             bias_id=rng.integers(-1, n + 1, (rows, biases)).astype(np.int32),
             bias=rng.normal(size=(rows, biases)).astype(np.float32),
             bias_len=rng.integers(-1, biases + 2, rows).astype(np.int32),
             mask=R.words_of(rng.integers(0, 2, (states, n))), mask_row=rng.integers(-1, states + 1, rows).astype(np.int32))
    return (3 * rng.normal(size=(rows, n))).astype(np.float32), c


@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (2, 31), (5, 33), (4, 255), (3, 1024), (2, 4095), (2, 4096),
                                    (3, 4097), (2, 8192), (70, 8192), (3, 8195), (2, 100003), (1, 262145)])
def test_all_rules(ctx, rows, n):
    rng = np.random.default_rng(n)
    _check(ctx, *_case(rng, rows, n))


@pytest.mark.parametrize("keep", [(), ("repeat",), ("frequency",), ("presence",), ("bias",), ("mask",), ("mask", "bias"),
                                  ("repeat", "presence")])
def test_each_rule_alone(ctx, keep):
    rng = np.random.default_rng(len(keep))
    x, c = _case(rng, 4, 5000)
    names = set(keep) | ({"hist"} if set(keep) & {"repeat", "frequency", "presence"} else set())
    names |= {"bias_id"} if "bias" in keep else set()
    c = {k: v for k, v in c.items() if k in names}
    if "mask" in c:
        c["mask"] = c["mask"][:4]
    out, _ = _check(ctx, x, c)
    if not keep:
        assert np.array_equal(out, x)


@pytest.mark.parametrize("hist", [0, 1, 3000, 40000])
def test_history_lengths(ctx, hist):
    rng = np.random.default_rng(hist)
    x, c = _case(rng, 3, 8192, hist=hist)
    c["hist_len"][:] = hist
    _check(ctx, x, c)


def test_one_token_over_and_over(ctx):
    """Counts beyond 16 bits, of one token, in every lane at once."""
    n, m = 8192, 70000
    c = dict(hist=np.full((2, m), 77, np.int32), frequency=np.array([0.001, 1.0], np.float32),
             repeat=np.array([2.0, 0.5], np.float32), out_from=np.array([3, 69999], np.int32))
    x = np.random.default_rng(0).normal(size=(2, n)).astype(np.float32)
    out, _ = _check(ctx, x, c)
    r = x[0, 77] / np.float32(2) if x[0, 77] > 0 else x[0, 77] * np.float32(2)
    assert out[0, 77] == np.float32(r - np.float32(69997) * np.float32(0.001))


@pytest.mark.parametrize("n,biases", [(50, 300), (8192, 1000), (9000, 3)])
def test_the_same_bias_twice(ctx, n, biases):
    """Biases of one token add up in the list's order, whatever lanes they meet in."""
    rng = np.random.default_rng(n)
    ids = rng.integers(0, 40, (3, biases)).astype(np.int32)
    bias = (10.0 ** rng.uniform(-4, 4, (3, biases)) * rng.choice([-1, 1], (3, biases))).astype(np.float32)
    x = rng.normal(size=(3, n)).astype(np.float32)
    out = host(_run(ctx, x, dict(bias_id=ids, bias=bias)))
    for i in range(3):
        for t in range(40):
            s = None
            for b in bias[i, ids[i] == t]:
                s = b if s is None else np.float32(s + b)
            assert out[i, t] == (x[i, t] if s is None else np.float32(x[i, t] + s)), (i, t)
    for _ in range(3):
        assert np.array_equal(host(_run(ctx, x, dict(bias_id=ids, bias=bias))), out)


@pytest.mark.parametrize("n", [20, 5000, 20000])
def test_masks_that_leave_one_or_none(ctx, n):
    bits = np.zeros((4, n), np.uint8)
    bits[1, n - 1] = bits[2, 0] = 1
    bits[3, [5, n - 3]] = 1
    x = np.zeros((4, n), np.float32)
    x[:, 7] = 100.0
    x[3, n - 3] = 1.0
    out, nxt = _check(ctx, x, dict(mask=R.words_of(bits)))
    assert nxt.tolist() == [-1, n - 1, 0, n - 3]
    assert np.isneginf(out[0]).all()
    # garbage behind the last token's bit is not read as a token
    w = R.words_of(bits)
    if n % 32:
        w[:, -1] |= np.int32(-1) << np.int32(n % 32)
    assert _check(ctx, x, dict(mask=w))[1].tolist() == nxt.tolist()


def test_nan_and_infinite_logits(ctx):
    """NaN and infinities stay, under a mask too; a NaN is never picked."""
    n = 9000
    x = np.random.default_rng(3).normal(size=(6, n)).astype(np.float32)
    x[0, 100] = x[1, 8999] = np.nan
    x[2] = np.nan
    x[3] = -np.inf
    x[4, [4200, 300]] = np.inf
    x[5, 50] = np.inf
    bits = np.ones((6, n), np.uint8)
    bits[5, 50] = bits[1, 8999] = 0
    out, nxt = (host(t) for t in _run(ctx, x, dict(mask=R.words_of(bits)), pick=True))
    want = np.where(bits == 1, x, -np.inf)
    assert np.array_equal(out, want, equal_nan=True)
    clean = np.where(np.isnan(want), -np.inf, want)
    assert nxt.tolist() == [_first(r) for r in clean] and nxt[2] == -1 and nxt[3] == -1 and nxt[4] == 300


@pytest.mark.parametrize("n", [100, 4096, 8200, 30001])
def test_ties_go_to_the_lowest_token(ctx, n):
    rng = np.random.default_rng(n)
    x = rng.integers(-2, 3, (40, n)).astype(np.float32)
    x[0] = 1.0
    x[1, :] = -3.0
    x[1, [n - 1, n - 2]] = 4.0
    _, nxt = _run(ctx, x, {}, pick=True)
    assert host(nxt).tolist() == x.argmax(1).tolist()


@pytest.mark.parametrize("off", [0, 1, 2, 3])
def test_rows_apart_at_any_alignment(ctx, off):
    rng = np.random.default_rng(off)
    x, c = _case(rng, 5, 8191)
    buf = torch.full((5, 8200), 3.0, device="cuda")
    buf[:, off:off + 8191] = dev(x)
    want = host(_run(ctx, x, c))
    out = torch.full((5, 8204), 5.0, device="cuda")
    got = _run(ctx, buf[:, off:off + 8191], c, out=out[:, 3 - off:3 - off + 8191])
    assert np.array_equal(host(got), want)
    o = host(out)
    assert (o[:, :3 - off] == 5.0).all() and (o[:, 3 - off + 8191:] == 5.0).all()


def test_no_rows_and_refusals(ctx):
    x = torch.zeros(2, 5000, device="cuda")
    assert nd.logits_adjust(ctx, x[:0]).shape == (0, 5000)

    def refused(what, f):
        with pytest.raises(nd.NeedleError) as e:
            f()
        assert e.value.code == nd.ND_ERR_ARG and what in str(e.value), str(e.value)

    words = torch.zeros(1, 157, dtype=torch.int32, device="cuda")
    refused("mask rows", lambda: nd.logits_adjust(ctx, x, mask=words))
    refused("bias", lambda: nd.logits_adjust(ctx, x, bias=torch.zeros(2, 3, device="cuda")))
    b = torch.zeros(10004, device="cuda")
    refused("overlaps", lambda: nd.logits_adjust(ctx, b[:10000].view(2, 5000), out=b[4:].view(2, 5000)))
    refused("work", lambda: nd.logits_adjust(ctx, torch.zeros(2, 50000, device="cuda"), pick=True,
                                             work=torch.zeros(16, dtype=torch.uint8, device="cuda")))
    ids = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for kw in (dict(mask=words[:, :100]), dict(hist=ids[:1]), dict(hist=ids.long()), dict(hist=ids, repeat=x[0, :1]),
               dict(bias_id=ids, bias=x[:, :2]), dict(out=x[:, :10]), dict(hist=ids.cpu()),
               dict(mask=torch.zeros(2, 157, dtype=torch.int64, device="cuda")), dict(mask_row=ids[0, :1])):
        with pytest.raises(ValueError):
            nd.logits_adjust(ctx, x, **kw)


@pytest.mark.parametrize("count,n", [(1 << 23, 1), ((1 << 23) + 5, 3)])
def test_more_rows_than_a_launch_holds(ctx, count, n):
    """Rows of every launch, up to the last one."""
    x = torch.arange(count * n, device="cuda").view(count, n).remainder(1000).float()
    out, nxt = nd.logits_adjust(ctx, x, repeat=torch.full((count,), 2.0, device="cuda"),
                                hist=torch.zeros(count, 1, dtype=torch.int32, device="cuda"), pick=True)
    want = x.clone()
    want[:, 0] /= 2
    assert torch.equal(out, want)
    best = torch.zeros(count, dtype=torch.int32, device="cuda")
    for j in range(1, n):
        best = torch.where(want[:, j] > want.gather(1, best[:, None].long())[:, 0], j, best).int()
    assert torch.equal(nxt, best)


@pytest.mark.parametrize("n,biases,tokens", [(9000, 20000, 9000), (8192, 30000, 3), (20, 5000, 20), (20001, 4001, 4000)])
def test_long_lists_of_biases(ctx, n, biases, tokens):
    """Lists of many entries, a few tokens or all of them listed again and again."""
    rng = np.random.default_rng(biases)
    ids = rng.integers(0, tokens, (2, biases)).astype(np.int32)
    if tokens == 4000:
        ids[:, :4000] = rng.permutation(4000)  # a single token twice
    bias = (10.0 ** rng.uniform(-4, 4, (2, biases)) * rng.choice([-1, 1], (2, biases))).astype(np.float32)
    x = rng.normal(size=(2, n)).astype(np.float32)
    hist = rng.integers(0, tokens, (2, 50)).astype(np.int32)
    out, nxt = (host(t) for t in _run(ctx, x, dict(bias_id=ids, bias=bias, hist=hist,
                                                   presence=np.array([0.5, 1.0], np.float32)), pick=True))
    want = x.copy()
    for i in range(2):
        want[i, np.unique(hist[i])] -= np.float32(0.5 + 0.5 * i)
        total = {}
        for t, b in zip(ids[i].tolist(), bias[i]):
            total[t] = np.float32(total[t] + b) if t in total else b
        for t, b in total.items():
            want[i, t] += b
    assert np.array_equal(out, want)
    assert nxt.tolist() == want.argmax(1).tolist()
