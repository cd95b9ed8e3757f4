"""The host side of the shared-prefix operators and of sampling: plan sizes,
structures, what is refused without a GPU, and the plain forms themselves."""
import ctypes as C

import numpy as np
import pytest

import needle_amd as nd
import prefix_ref as P


def test_null_arguments():
    L = nd.lib()
    assert L.nd_prefix_plan(None, None, 1, 1, 1, 1, None, None, None, None, 0, None, 0, None) == nd.ND_ERR_ARG
    assert L.nd_attend_prefix_i8(None, None, None, 0, 1, 1, None, 0, 1, 1, None, None, 1.0, 0, None, None, 0) == nd.ND_ERR_ARG
    assert L.nd_sample_rows(None, None, 0, 1, 1, None, None, None, None, None, 0) == nd.ND_ERR_ARG
    assert "context" in nd.last_error()
    assert L.nd_attend_prefix_i8_work(None, nd.kv_geom(12, 2, 48, 64, 8), 1, 1, 1) == 0


@pytest.mark.parametrize("count,rows,prefixes", [(65536, 1, 1), (1, 0, 1), (1, 257, 1), (65535, 17, 1), (1, 1, 2049)])
def test_plan_sizes_refused(count, rows, prefixes):
    assert nd.prefix_plan_bytes(nd.kv_geom(12, 2, 48, 64, 8), count, rows, prefixes) == 0
    assert nd.last_error()


def test_plan_sizes():
    g = nd.kv_geom(12, 2, 48, 64, 8)
    sizes = [nd.prefix_plan_bytes(g, *a) for a in ((0, 1, 0), (1, 1, 0), (1, 1, 1), (64, 1, 1), (64, 9, 5), (65535, 16, 2048))]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert nd.prefix_plan_bytes(nd.kv_geom(12, 5, 48, 64, 8), 1, 1, 1) == 0 and "multiple" in nd.last_error()


def test_structures_match_the_header():
    assert C.sizeof(nd.PrefixMaps) == 6 * 8 and C.sizeof(nd.Sampling) == 4 * 8


def test_the_plain_draw_in_whole_numbers_and_in_64_bits():
    rng = np.random.default_rng(1)
    for _ in range(300):
        n = int(rng.integers(1, 40))
        u, p = np.float32(rng.random()), np.float32(rng.uniform(0.05, 1.2))
        got, chance, room = P.draw(np.zeros(n, np.float32), u, top_p=p)
        if room > 1e-9:
            assert got == P.draw_in_whole_numbers([1] * n, u, p)
        assert 0 < chance <= 1


def test_the_plain_draw_keeps_what_the_rules_say():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.25, 0.05], np.float32))
    order = [1, 3, 2, 0, 4]
    for u, want in ((0.0, 1), (0.39, 1), (0.41, 3), (0.66, 2), (0.86, 0), (0.96, 4)):
        assert P.draw(x, u)[0] == want
    assert [P.draw(x, 0.999, top_k=k)[0] for k in range(1, 6)] == order
    assert [P.draw(x, 0.999, top_p=p)[0] for p in (0.3, 0.6, 0.8, 0.9, 0.99)] == order
    assert [P.draw(x, 0.999, min_p=p)[0] for p in (0.9, 0.6, 0.4, 0.2, 0.1)] == order
    assert P.draw(x, 0.9, temperature=0.0)[:2] == (1, 1.0) and P.draw(x * np.inf, 0.5)[0] == -1
