"""Tokens drawn from rows of logits against a plain 64-bit form.

A pick is the border's: it has to be the plain form's wherever the draw is
further than 1e-11 of the sum from falling otherwise.  Both sides are that
exact: a weight is off by a few 2^-53 of itself and, on the device, by half a
unit, of which a row's sum has 2^61 or more, so 2^17 of them by 3e-14 of the sum;
the plain form's running sum is off by 2^17 2^-53 = 1.5e-11 of itself at the very
most and by a root's share of that (4e-14) in draws.  Rows of equal logits have
equal weights, and are drawn by exact fractions.  A chance is one rounding to
fp32 (2^-24 of it) of a quotient that is 1e-12 exact.
"""
import numpy as np
import pytest
import torch

import needle_amd as nd
import prefix_ref as P
from conftest import dev, host

pytestmark = pytest.mark.gpu
RULES = [dict(), dict(temperature=0.6), dict(temperature=1.9), dict(top_k=1), dict(top_k=40), dict(top_k=700, temperature=3.0),
         dict(top_p=0.9), dict(top_p=0.3, temperature=2.5), dict(min_p=0.05), dict(min_p=0.001, temperature=1.4),
         dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.02), dict(temperature=5.0, top_k=3000, top_p=0.999)]
SIZES = [1, 2, 3, 63, 64, 65, 511, 512, 513, 1000, 1025, 2048, 4097, 8191, 8192, 8193, 16384, 20001, 32768, 50000, 100003, 131072]
F32, I32 = ("temperature", "top_p", "min_p"), ("top_k",)


def _run(ctx, x, u, rules, **kw):
    x = np.asarray(x, np.float32)
    rows = len(x)
    full = {k: dev(np.full(rows, v, np.int32 if k in I32 else np.float32) if np.isscalar(v) else
                   np.asarray(v, np.int32 if k in I32 else np.float32)) for k, v in rules.items()}
    return [host(t) for t in nd.sample_rows(ctx, dev(x), dev(np.asarray(u, np.float32)), **full, **kw)]


def _check(ctx, x, u, rules, least=0.97):
    got, prob = _run(ctx, x, u, rules)
    clear = 0
    for i in range(len(x)):
        mine = {k: v if np.isscalar(v) else v[i] for k, v in rules.items()}
        want, chance, room = P.draw(x[i], u[i], **mine)
        if room > 1e-11:
            clear += 1
            assert got[i] == want, (i, got[i], want, room)
            assert abs(float(prob[i]) - chance) <= 2.0 ** -24 * chance + 1e-12, (i, prob[i], chance)
    assert clear >= least * len(x)


def _logits(rng, rows, n):
    x = 2 * rng.normal(size=(rows, n))
    x[:, rng.integers(0, n, min(n, 20))] += 6
    return x.astype(np.float32)


@pytest.mark.parametrize("rules", RULES)
@pytest.mark.parametrize("n", SIZES)
def test_draws(ctx, n, rules):
    rng = np.random.default_rng(n)
    rows = 9 if n > 20000 else 24
    _check(ctx, _logits(rng, rows, n), rng.random(rows).astype(np.float32), rules)


@pytest.mark.parametrize("rows", [300, 1100, 5000])
def test_many_rows_of_their_own_rules(ctx, rows):
    rng = np.random.default_rng(rows)
    n = 700
    rules = dict(temperature=rng.choice([0.0, 0.5, 1.0, 2.0], rows), top_k=rng.choice([0, 1, 5, 100, 699, 700, 9000], rows),
                 top_p=rng.choice([0.1, 0.8, 0.99, 1.0], rows), min_p=rng.choice([0.0, 0.01, 0.3], rows))
    _check(ctx, _logits(rng, rows, n), rng.random(rows).astype(np.float32), rules)


@pytest.mark.parametrize("rules", RULES)
@pytest.mark.parametrize("n", [700, 8192, 30000])
@pytest.mark.parametrize("step", [0.25, 2.0, 16.0])
def test_logits_of_a_few_levels(ctx, n, step, rules):
    """Thousands of equal logits: the lower number comes first."""
    rng = np.random.default_rng(n)
    x = (np.round(_logits(rng, 8, n) / step) * step).astype(np.float32)
    _check(ctx, x, rng.random(8).astype(np.float32), rules)


@pytest.mark.parametrize("n", [5, 512, 513, 1000, 8192, 8193, 70001])
@pytest.mark.parametrize("top_k,top_p", [(0, 1.0), (0, 0.37), (600, 1.0), (600, 0.5), (3, 0.999), (0, 2.0 ** -20)])
def test_equal_logits(ctx, n, top_k, top_p):
    us = np.array([0.0, 1 / 3, 0.5, 0.7499, 0.99, 1 - 2.0 ** -24, 2.0 ** -24, 0.25], np.float32)
    x = np.full((len(us), n), -3.25, np.float32)
    got, prob = _run(ctx, x, us, dict(top_k=top_k, top_p=top_p, temperature=0.3))
    kept = min(n, top_k or n)
    for u, g in zip(us, got):
        assert g == P.draw_in_whole_numbers([1] * kept, u, top_p), (u, g)
    if top_p < 1:
        kept = max(1, int(np.ceil(float(np.float32(top_p)) * kept)))
    assert (prob == np.float32(1 / kept)).all()


@pytest.mark.parametrize("rules", [dict(), dict(top_k=5000), dict(top_p=0.6), dict(top_k=9000, top_p=0.9)])
@pytest.mark.parametrize("n", [1000, 20000])
def test_neighbouring_floats(ctx, n, rules):
    """Every logit one step of fp32 from the next, in any order."""
    rng = np.random.default_rng(1)
    base = np.float32(3.0).view(np.int32)
    x = np.stack([(base - rng.permutation(n)).astype(np.int32).view(np.float32) for _ in range(6)])
    _check(ctx, x, rng.random(6).astype(np.float32), rules)


@pytest.mark.parametrize("n", [900, 8192, 40000])
@pytest.mark.parametrize("rules", RULES)
def test_lowest_values_and_masks(ctx, n, rules):
    """Tokens at fp32's lowest value, at -1e30, at -inf and NaN beside ordinary ones."""
    rng = np.random.default_rng(n + 1)
    x = _logits(rng, 10, n)
    for i, v in enumerate([np.finfo(np.float32).min, -1e30, -np.inf, np.nan, -1e5] * 2):
        hit = rng.random(n) < (0.5 if i < 5 else 0.995)
        hit[rng.integers(0, n)] = False
        x[i, hit] = v
    _check(ctx, x, rng.random(10).astype(np.float32), rules)


@pytest.mark.parametrize("n", [600, 10000, 33000])
def test_rows_without_tokens_and_infinite_ones(ctx, n):
    x = np.full((6, n), -np.inf, np.float32)
    x[1] = np.nan
    x[2, n // 2] = -200.0
    x[3, [3, n - 2, n // 3]] = np.inf
    x[3, 7] = 5
    x[4, n - 1] = np.finfo(np.float32).min
    x[5] = np.inf
    u = np.array([0.3, 0.3, 0.9, 0.5, 0.99, 0.5], np.float32)
    for rules in (dict(), dict(temperature=0.0), dict(top_k=2, top_p=0.6, min_p=0.5), dict(temperature=np.inf)):
        got, prob = _run(ctx, x, u, rules)
        greedy = rules.get("temperature") == 0
        assert got[:3].tolist() == [-1, -1, n // 2] and got[4] == n - 1
        assert prob[:3].tolist() == [0, 0, 1] and prob[4] == 1
        two = rules.get("top_k") == 2
        assert got[3] == (3 if greedy else sorted([3, n - 2, n // 3])[1])
        assert got[5] == (0 if greedy else 1 if two else n // 2)


def test_random_numbers_at_the_ends(ctx):
    rng = np.random.default_rng(3)
    us = np.array([0.0, -0.0, -1.0, np.nan, 1e-40, 1 - 2.0 ** -24, 1.0, 2.0, np.inf], np.float32)
    for n in (10, 800, 9000, 50000):
        x = np.repeat(_logits(rng, 1, n), len(us), 0)
        for rules in (dict(top_k=7), dict(top_p=0.5), dict(min_p=0.1)):
            got, _ = _run(ctx, x, us, rules)
            last = P.draw(x[0], 1.0, **rules)[0]
            assert (got[:5] == np.argmax(x[0])).all() and (got[5:] == last).all()


def test_rules_at_the_ends(ctx):
    rng = np.random.default_rng(4)
    for n in (40, 3000, 20000):
        x, u = _logits(rng, 16, n), rng.random(16).astype(np.float32)
        first = np.argmax(x, 1)
        free = _run(ctx, x, u, dict())
        for rules in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=np.nan), dict(temperature=1e-30),
                      dict(temperature=1e-45), dict(top_k=1), dict(top_p=0.0), dict(top_p=-3.0), dict(top_p=1e-44),
                      dict(min_p=1.0), dict(min_p=7.0), dict(min_p=np.inf)):
            got, prob = _run(ctx, x, u, rules)
            assert (got == first).all() and (prob == 1).all(), rules
        for rules in (dict(temperature=1.0), dict(top_k=0), dict(top_k=-4), dict(top_k=n), dict(top_k=2 ** 31 - 1),
                      dict(top_p=1.0), dict(top_p=3.0), dict(top_p=np.nan), dict(min_p=0.0), dict(min_p=-1.0),
                      dict(min_p=np.nan), dict(min_p=1e-44)):
            got = _run(ctx, x, u, rules)
            assert np.array_equal(got[0], free[0]) and np.array_equal(got[1], free[1]), rules
        for t in (np.inf, 1e38):  # every token alike
            got, prob = _run(ctx, x, u, dict(temperature=t))
            by = np.argsort(-x, 1, kind="stable")
            want = [by[i, P.draw_in_whole_numbers([1] * n, u[i])] for i in range(16)] if t == np.inf else got
            assert got.tolist() == list(want) and np.allclose(prob, 1 / n, rtol=2.0 ** -23)


def test_every_logit_at_its_size(ctx):
    """Logits of any size: far below one, and hundreds apart."""
    rng = np.random.default_rng(5)
    for size in (1e-38, 1e-3, 50.0, 1e4, 1e37):
        x = (size * rng.normal(size=(12, 5000))).astype(np.float32)
        for rules in (dict(temperature=min(size, 1e30)), dict(temperature=0.1 * min(size, 1e30), top_k=60), dict(top_p=0.7)):
            _check(ctx, x, rng.random(12).astype(np.float32), rules)


def test_ties_of_both_zeros(ctx):
    x = np.full((4, 2000), -9.0, np.float32)
    x[:, [5, 900]] = 0.0
    x[:, [3, 1500]] = -0.0
    got, _ = _run(ctx, x, [0.0, 0.3, 0.6, 0.9], dict(top_k=4))
    assert got.tolist() == [3, 5, 900, 1500]


@pytest.mark.parametrize("n", [333, 8192, 25001])
def test_rows_apart_and_unaligned(ctx, n):
    """Rows of a wider tensor that begin anywhere: the same bits; nothing else is written."""
    rng = np.random.default_rng(6)
    x, u = _logits(rng, 7, n), rng.random(7).astype(np.float32)
    want = _run(ctx, x, u, dict(top_p=0.9, temperature=1.1))
    for pad, at in ((1, 0), (5, 1), (64, 3)):
        wide = torch.full((7, n + pad), 50.0, device="cuda")
        view = wide[:, at:at + n] if at + n <= n + pad else wide[:, :n]
        view.copy_(dev(x))
        before = wide.clone()
        out, prob = torch.full((9,), 77, dtype=torch.int32, device="cuda"), torch.full((9,), 7.0, device="cuda")
        nd.sample_rows(ctx, view, dev(u), temperature=torch.full((7,), 1.1, device="cuda"),
                       top_p=torch.full((7,), 0.9, device="cuda"), out=out[:7], prob=prob[:7])
        assert np.array_equal(host(out[:7]), want[0]) and np.array_equal(host(prob[:7]), want[1])
        assert (host(out[7:]) == 77).all() and (host(prob[7:]) == 7).all() and torch.equal(wide, before)


def test_a_row_alone_is_the_row_in_a_batch(ctx):
    rng = np.random.default_rng(7)
    for n in (1000, 9001, 60000):
        x, u = _logits(rng, 40, n), rng.random(40).astype(np.float32)
        rules = dict(temperature=1.3, top_k=300, top_p=0.97)
        want = _run(ctx, x, u, rules)
        for _ in range(2):
            again = _run(ctx, x, u, rules)
            assert np.array_equal(want[0], again[0]) and np.array_equal(want[1], again[1])
        for i in (0, 17, 39):
            one = _run(ctx, x[i:i + 1], u[i:i + 1], rules)
            assert one[0][0] == want[0][i] and one[1][0] == want[1][i]


@pytest.mark.parametrize("rules", [dict(temperature=1.3), dict(top_k=300, top_p=0.97), dict(top_k=2000, top_p=0.9), dict(min_p=0.2)])
@pytest.mark.parametrize("n", [700, 8192])
def test_few_rows_are_the_rows_of_many(ctx, n, rules):
    """Ordinary rows, equal and neighbouring logits, infinite ones and none, in 600 rows and in threes."""
    rng = np.random.default_rng(n)
    x, u = _logits(rng, 600, n), rng.random(600).astype(np.float32)
    x[1::8] = 2.5
    x[2::8] = np.float32(3) + rng.integers(0, 3, (75, n)).astype(np.float32) * np.float32(2.0 ** -22)
    x[3::8, ::3] = np.inf
    x[4::8] = np.nan
    x[5::8, 1:] = -np.inf
    x[6::8] = -3.4028235e38
    want = _run(ctx, x, u, rules)
    for i in range(0, 48, 3):
        got = _run(ctx, x[i:i + 3], u[i:i + 3], rules)
        assert np.array_equal(got[0], want[0][i:i + 3]) and np.array_equal(got[1], want[1][i:i + 3]), i
    assert (want[0][4::8] == -1).all() and (want[0][5::8] == 0).all() and (want[0][3::8] % 3 == 0).all()


def test_the_largest_row(ctx):
    n = 1 << 24
    x = torch.full((2, n), -5.0, device="cuda")
    x[0, n - 1] = 3.0
    u = torch.tensor([0.0, 0.75], device="cuda")
    got, prob = (host(t) for t in nd.sample_rows(ctx, x, u))
    assert got.tolist() == [n - 1, n // 4 * 3] and prob[1] == 2.0 ** -24
    want = np.exp(8.0) / (np.exp(8.0) + n - 1)
    assert abs(float(prob[0]) - want) <= 2.0 ** -24 * want + 1e-8


def test_more_rows_than_a_launch_holds(ctx):
    rows = (1 << 32) // 512 + 9
    x = torch.zeros(rows, 2, device="cuda")
    x[:, 1] = torch.arange(rows, device="cuda") % 3 - 1.0
    got, _ = nd.sample_rows(ctx, x, torch.zeros(rows, device="cuda"))
    assert torch.equal(got, (torch.arange(rows, device="cuda") % 3 == 2).int())


def test_rows_beyond_32_bits_of_offset(ctx):
    n, rows = 1 << 20, 1100
    x = torch.zeros(rows, n, device="cuda")
    x[:, 12345] = 30.0
    x[rows - 1, n - 2] = 60.0
    got, _ = nd.sample_rows(ctx, x, torch.full((rows,), 0.5, device="cuda"), top_k=torch.full((rows,), 3, dtype=torch.int32, device="cuda"))
    assert got[-1].item() == n - 2 and (got[:-1] == 12345).all()


def test_no_rows(ctx):
    for n in (5, 20000):
        token, chance = nd.sample_rows(ctx, torch.zeros(0, n, device="cuda"), torch.zeros(0, device="cuda"))
        assert token.shape == chance.shape == (0,)


def test_refusals(ctx):
    x, u = torch.zeros(3, 100, device="cuda"), torch.zeros(3, device="cuda")
    for bad in (lambda: nd.sample_rows(ctx, x.double(), u), lambda: nd.sample_rows(ctx, x.cpu(), u),
                lambda: nd.sample_rows(ctx, x, u[:2]), lambda: nd.sample_rows(ctx, x, u.double()),
                lambda: nd.sample_rows(ctx, x, u, temperature=u[:1]), lambda: nd.sample_rows(ctx, x, u, top_k=u),
                lambda: nd.sample_rows(ctx, x, u, top_p=u.int()), lambda: nd.sample_rows(ctx, x, u, out=u),
                lambda: nd.sample_rows(ctx, x.t(), u), lambda: nd.sample_rows(ctx, x, u, prob=u.int()),
                lambda: nd.sample_rows(ctx, x, u, work=u)):
        with pytest.raises(ValueError):
            bad()
    L, p, q = nd.lib(), x.data_ptr(), u.data_ptr()
    for what, args in (("n 0", (p, 100, 3, 0, None, q, q, None)), ("2^24", (p, 1 << 25, 1, (1 << 24) + 1, None, q, q, None)),
                       ("stride", (p, 99, 3, 100, None, q, q, None)), ("null", (None, 100, 3, 100, None, q, q, None)),
                       ("null", (p, 100, 3, 100, None, None, q, None)), ("null", (p, 100, 3, 100, None, q, None, None)),
                       ("count", (p, 100, 1 << 31, 100, None, q, q, None))):
        assert L.nd_sample_rows(ctx.h, *args, None, 0) == nd.ND_ERR_ARG and what in nd.last_error(), nd.last_error()
    assert L.nd_sample_rows(ctx.h, None, 0, 0, 5, None, None, None, None, None, 0) == nd.ND_OK
    assert L.nd_sample_rows(ctx.h, p, 0, 1, 100, None, q, q, None, None, 0) == nd.ND_OK  # one row: any stride
    torch.cuda.synchronize()


@pytest.mark.parametrize("rules", [dict(), dict(top_p=0.5), dict(top_k=600), dict(top_k=900, top_p=0.8)])
@pytest.mark.parametrize("rows,n,width", [(40, 2000, 0.3), (40, 8192, 0.1), (600, 2000, 0.3), (600, 5000, 0.02), (40, 30000, 0.3),
                                          (40, 30000, 0.02)])
def test_bins_of_many_tokens(ctx, rows, n, width, rules):
    """Targets in bins (of 2^(1/16)) of 65 to 512 tokens, and of thousands, which are listed twice: every row's
    weights but the largest lie within `width` of another."""
    rng = np.random.default_rng(rows + n)
    x = (-4 - width * rng.random((rows, n))).astype(np.float32)
    x[:, n // 3] = 0.0
    x[:, n // 2] = -60.0
    _check(ctx, x, (0.2 + 0.79 * rng.random(rows)).astype(np.float32), rules)


@pytest.mark.parametrize("n", [5, 900, 9000, 30000])
def test_an_infinite_temperature_with_min_p(ctx, n):
    """exp(d / inf) is 1 for every finite d, which a min_p of 1 or less lets stay; above 1 the first maximum alone."""
    rng = np.random.default_rng(n)
    x, u = _logits(rng, 8, n), rng.random(8).astype(np.float32)
    x[1::2, 1::3] = -np.inf
    x[2] = np.where(rng.random(n) < 0.5, 3e38, -3e38)
    for kw in (dict(), dict(top_p=0.5), dict(top_k=600)):
        for min_p in (1.0, 1 - 2.0 ** -24, 1e-44):
            got, prob = _run(ctx, x, u, dict(temperature=np.inf, min_p=min_p, **kw))
            for i in range(8):
                by = np.argsort(-x[i], kind="stable")[:np.isfinite(x[i]).sum()]
                by = by[:kw.get("top_k")]
                kept = int(np.ceil(kw["top_p"] * len(by))) if "top_p" in kw else len(by)
                assert got[i] == by[P.draw_in_whole_numbers([1] * kept, u[i])] and prob[i] == np.float32(1 / kept), (i, min_p)
        got, prob = _run(ctx, x, u, dict(temperature=np.inf, min_p=1 + 2.0 ** -23, **kw))
        assert (got == np.argmax(x, 1)).all() and (prob == 1).all()


@pytest.mark.parametrize("rules", [dict(), dict(top_p=0.4), dict(top_k=20000)])
@pytest.mark.parametrize("n", [8192, 33000, 70001, 300000])
def test_the_lowest_temperature_over_equal_and_neighbouring_logits(ctx, n, rules):
    """1 / T beyond fp32: more ties than 64 bits hold in units of 2^-49, and logits as far apart as T, which weigh 1 / e."""
    t = float(np.float32(1e-45))
    rng = np.random.default_rng(n)
    u = rng.random(6).astype(np.float32)
    got, prob = _run(ctx, np.full((6, n), 2.0), u, dict(temperature=t, **rules))
    kept = min(n, rules.get("top_k", n))
    kept = int(np.ceil(float(np.float32(rules["top_p"])) * kept)) if "top_p" in rules else kept
    for i in range(6):
        assert got[i] == P.draw_in_whole_numbers([1] * kept, u[i]) and prob[i] == np.float32(1 / kept)
    _check(ctx, (-rng.integers(0, 5, (6, n)) * t).astype(np.float32), u, dict(temperature=t, **rules), least=0.8)


@pytest.mark.parametrize("rules", [dict(), dict(top_p=0.7), dict(top_k=200000, top_p=0.9), dict(min_p=0.01)])
@pytest.mark.parametrize("temperature", [3e38, 1.5e38, 3.4028235e38])
def test_logits_further_apart_than_the_largest_number(ctx, temperature, rules):
    """The largest logit and the rest at both ends of fp32, at a temperature under which the rest weighs as much."""
    n, rng = 300000, np.random.default_rng(31)
    x = np.full((4, n), -3e38, np.float32)
    x[1:] = -(1.5e38 + 1.9e38 * rng.random((3, n)))
    x[np.arange(4), [7, n // 2, n - 1, 8192]] = 3e38
    x[3] = (6.8e38 * (rng.random(n) - 0.5)).astype(np.float32)
    _check(ctx, x, (0.02 + 0.97 * rng.random(4)).astype(np.float32), dict(temperature=temperature, **rules), least=0.7)


@pytest.mark.parametrize("rules", [dict(), dict(top_p=0.9), dict(top_k=6000000, top_p=0.5)])
def test_a_long_rows_unit_is_one(ctx, rules):
    """Rows of 1500 slices of 8192 whose bound on the sum lies at a power of two: added up in another order
    (of these seeds, of 1024 threads instead of 512) it rounds to the other side, and the unit is twice or half of it."""
    n, infinite = 1500 * 8192, torch.tensor([float("inf")], device="cuda")
    there = int(2 ** 23 / (1.001 * float(np.float32(1.0001)) ** 2))
    for seed in (1, 2, 4, 12, 13):
        rng = np.random.default_rng(seed)
        x = np.full(n, -np.inf, np.float32)
        ids = rng.permutation(n)[:there]
        x[ids] = 20 * rng.random(there) - 10
        x = dev(x)[None]
        by = torch.sort(x[0], descending=True, stable=True)[1]
        kept = min(there, rules.get("top_k", there))
        kept = int(np.ceil(float(np.float32(rules["top_p"])) * kept)) if "top_p" in rules else kept
        full = {k: torch.tensor([v], dtype=torch.int32 if k in I32 else torch.float32, device="cuda") for k, v in rules.items()}
        for u in (0.125, 0.515625, 0.875):  # (u kept is exact in fp64)
            got, prob = nd.sample_rows(ctx, x, torch.tensor([u], device="cuda"), temperature=infinite, **full)
            assert got.item() == by[int(u * kept)].item() and host(prob)[0] == np.float32(1 / kept), (seed, u)


@pytest.mark.parametrize("temperature", [1e30, 1e38, 3.4028235e38])
@pytest.mark.parametrize("n", [40, 3000, 20000])
def test_tokens_alike_at_a_very_high_temperature(ctx, n, temperature):
    """Logits less than 100 apart weigh 1 - 1e-28 or more of each other: as many units."""
    rng = np.random.default_rng(n)
    x, u = _logits(rng, 12, n), rng.random(12).astype(np.float32)
    by = np.argsort(-x, 1, kind="stable")
    for kw, kept in ((dict(), n), (dict(top_k=17), 17), (dict(top_k=2000), min(n, 2000)), (dict(top_p=0.25), n // 4)):
        got, prob = _run(ctx, x, u, dict(temperature=temperature, **kw))
        assert got.tolist() == [by[i, P.draw_in_whole_numbers([1] * kept, u[i])] for i in range(12)], kw
        assert (prob == np.float32(1 / kept)).all(), kw
