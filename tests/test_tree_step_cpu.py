"""The host side of the drafted-tree operators: frequencies, tree masks, and
what is refused before anything reaches a GPU."""
import ctypes as C

import numpy as np
import pytest

import needle_amd as nd
import tree_ref as R


@pytest.mark.parametrize("rot", [2, 6, 48, 64, 256])
@pytest.mark.parametrize("theta", [10000.0, 500000.0, 7.5])
@pytest.mark.parametrize("kw", [{}, dict(scaling="linear", factor=4.0),
                                dict(scaling="parts", factor=8.0, trained=4096, turns=(1.0, 32.0)),
                                dict(scaling="parts", factor=0.5, trained=10, turns=(0.0, 0.001))])
def test_frequencies(rot, theta, kw):
    """A power of theta, off by a step or two of fp64 in either form."""
    got = nd.rope_freqs(nd.rope(rot, theta=theta, **kw))
    want = R.freqs(rot, theta, **kw)
    assert np.allclose(got, want, rtol=1e-14, atol=0)


@pytest.mark.parametrize("r", [nd.rope(0), nd.rope(3), nd.rope(-2), nd.rope(258), nd.rope(48, theta=-1.0),
                               nd.rope(48, theta=float("inf")), nd.rope(48, gain=float("nan")),
                               nd.rope(48, scaling="linear", factor=-1.0), nd.rope(48, scaling="linear", factor=float("nan")),
                               nd.rope(48, scaling="parts", factor=2.0, trained=0),
                               nd.rope(48, scaling="parts", factor=2.0, trained=8, turns=(3.0, 1.0)),
                               nd.rope(48, scaling="parts", factor=2.0, trained=8, turns=(float("nan"), 1.0)),
                               nd.rope(48, scaling="linear", factor=1e-4), nd.rope(256, theta=1e-300),
                               nd.Rope(2, 0, 48, 1e4, 1, 0, 0, 1, 1), nd.Rope(0, 3, 48, 1e4, 1, 0, 0, 1, 1)])
def test_frequencies_refused(r):
    with pytest.raises(nd.NeedleError) as e:
        nd.rope_freqs(r)
    assert e.value.code == nd.ND_ERR_ARG


def test_names_refused():
    for kw in (dict(layout="half"), dict(scaling="none")):
        with pytest.raises(ValueError):
            nd.rope(48, **kw)


def test_null_arguments():
    L = nd.lib()
    assert L.nd_rope_freqs(None, None) == nd.ND_ERR_ARG
    assert L.nd_rope_rows(None, None, 1, None, 1, 48, None, 48, None, 48) == nd.ND_ERR_ARG
    assert L.nd_kv_read(None, None, None, 0, 1, 1, None, None, None) == nd.ND_ERR_ARG
    assert L.nd_kv_write_rope(None, None, None, None, 0, 1, 1, None, None, None, 0, None, 0, None, 0, None, 0) == nd.ND_ERR_ARG
    assert L.nd_attend_tree_i8(None, None, None, 0, 1, 1, None, None, None, None, None, 1.0, 0, None, None, 0) == nd.ND_ERR_ARG
    assert L.nd_logits_adjust(None, None, 0, 1, 1, None, None, 0, None, None, 0) == nd.ND_ERR_ARG
    assert "context" in nd.last_error()


@pytest.mark.parametrize("n", [1, 5, 31, 32, 33, 100, 256])
def test_tree_masks(n):
    rng = np.random.default_rng(n)
    up = np.array([[rng.integers(-1, j) if j else -1 for j in range(n)] for _ in range(3)])
    got = R.bits_of(nd.tree_mask(up), n)
    assert nd.tree_mask(up).shape == (3, n, (n + 31) // 32) and nd.tree_mask(up[0]).shape == (n, (n + 31) // 32)
    for i in range(3):
        for j in range(n):
            want, a = np.zeros(n, np.uint8), j
            while a >= 0:
                want[a] = 1
                a = up[i, a]
            assert np.array_equal(got[i, j], want)


@pytest.mark.parametrize("up", [[0], [-1, 1], [-1, 0, 5], []])
def test_tree_masks_refused(up):
    with pytest.raises(ValueError):
        nd.tree_mask(up)


def test_structures_match_the_header():
    """The sizes a C compiler gives the structures."""
    assert C.sizeof(nd.Rope) == 64 and nd.Rope.theta.offset == 16
    assert C.sizeof(nd.LogitsRules) == 15 * 8
