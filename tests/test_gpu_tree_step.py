"""The drafted-tree operators together, as a server calls them: keys and
queries of every node turned and appended, the trees attended, the logits
ruled and picked, the accepted path committed -- eagerly, on a stream of its
own, and captured into graphs.

Tolerances are those of the operators' own tests (tests/test_gpu_tree.py).
"""
import numpy as np
import pytest
import torch

import needle_amd as nd
import tree_ref as R
from conftest import dev, host

pytestmark = pytest.mark.gpu
H, KVH, QK, VD, N, S, VOCAB = 12, 2, 48, 64, 9, 3, 9001
UP = np.array([[-1, 0, 0, 1, 1, 2, 3, 6, 4], [-1, 0, 1, 2, 3, 4, 5, 6, 7], [-1, 0, 0, 0, 0, 0, 0, 0, 0]])


def _depth():
    d = np.zeros((S, N), np.int32)
    for j in range(1, N):
        d[:, j] = d[np.arange(S), UP[:, j]] + 1
    return d


class Step:
    """The buffers of a step and its calls."""

    def __init__(self, ctx, seed, base=(40, 133, 7)):
        rng = np.random.default_rng(seed)
        self.ctx, self.base = ctx, np.array(base, np.int32)
        self.geom = nd.kv_geom(H, KVH, QK, VD, 150)
        self.rope = nd.rope(QK)
        self.kv, self.nb = nd.kv_alloc(self.geom, S)
        for i in range(S):
            n = int(base[i])
            t = dev(np.arange(n, dtype=np.int32))
            nd.kv_write_rope(ctx, self.geom, self.rope, self.kv[i * self.nb:(i + 1) * self.nb], 0, t,
                             dev(rng.normal(size=(n, KVH * QK)).astype(np.float32)),
                             dev(rng.normal(size=(n, KVH * VD)).astype(np.float32)), per_block=max(n, 1))
        self.pos = dev((self.base[:, None] + np.arange(N)).astype(np.int32).reshape(-1))
        self.turn = dev((self.base[:, None] + _depth()).astype(np.int32).reshape(-1))
        self.mask = dev(nd.tree_mask(UP))
        self.based, self.lo = dev(self.base), dev(np.zeros((S, N), np.int32))
        self.qkv = torch.empty(S * N, (H + KVH) * QK + KVH * VD, device="cuda")
        self.head = dev(rng.normal(size=(H * VD, VOCAB)).astype(np.float32))
        self.hist = dev(rng.integers(0, VOCAB, (S * N, 20)).astype(np.int32))
        self.repeat = torch.full((S * N,), 1.3, device="cuda")
        self.grammar = dev(R.words_of(rng.integers(0, 2, (S * N, VOCAB))))
        self.q = torch.empty(S * N, H * QK, device="cuda")
        self.out = torch.empty(S, N, H * VD, device="cuda")
        self.logits = torch.empty(S * N, VOCAB, device="cuda")
        self.work = torch.empty(max(16, nd.attend_tree_i8_work(ctx, self.geom, S, N),
                                    nd.logits_adjust_work(ctx, S * N, VOCAB)), dtype=torch.uint8, device="cuda")
        self.next = None
        self.fill(seed)

    def fill(self, seed):
        self.qkv.copy_(dev(np.random.default_rng(1000 + seed).normal(size=self.qkv.shape).astype(np.float32)))

    def run(self, work=True):
        c, g, w = self.ctx, self.geom, self.work if work else None
        q, k, v = self.qkv.split([H * QK, KVH * QK, KVH * VD], 1)
        nd.kv_write_rope(c, g, self.rope, self.kv, self.nb, self.pos, k, v, q=q, q_out=self.q, rot_pos=self.turn,
                         per_block=N)
        nd.attend_tree_i8(c, g, self.kv, self.nb, self.based, self.lo, self.mask, self.q.view(S, N, -1),
                          quant_query=True, out=self.out, work=w)
        torch.mm(self.out.view(S * N, -1), self.head, out=self.logits)
        _, self.next = nd.logits_adjust(c, self.logits, hist=self.hist, repeat=self.repeat, mask=self.grammar,
                                        out=self.logits, pick=True, work=w)
        return self.out, self.logits, self.next


def _state(st):
    torch.cuda.synchronize()
    return [host(t).copy() for t in (st.q, st.out, st.logits, st.next, st.kv)]


def test_a_node_is_its_path_decoded(ctx):
    """Each node's attention is that of its ancestors decoded one after
    another, and the accepted path, committed, is what decoding it stores."""
    st = Step(ctx, 1)
    out, logits, nxt = (host(t).copy() for t in st.run())
    qkv = host(st.qkv).copy()
    for i in range(S):
        for n in (0, 4, 7, 8):
            path, a = [], n
            while a >= 0:
                path.append(a)
                a = UP[i, a]
            path = path[::-1]
            blk = st.kv[i * st.nb:(i + 1) * st.nb].clone()
            rows = dev(qkv[i * N + np.array(path)])
            q, k, v = (t.contiguous() for t in rows.split([H * QK, KVH * QK, KVH * VD], 1))
            at = dev((st.base[i] + np.arange(len(path))).astype(np.int32))
            nd.kv_write(ctx, st.geom, blk, 0, at, nd.rope_rows(ctx, st.rope, k, at, KVH), v)
            one = nd.attend_step_i8(ctx, st.geom, blk, 0, at[-1:] * 0, at[-1:], nd.rope_rows(ctx, st.rope, q, at, H)[-1:],
                                    quant_query=True)
            assert np.abs(host(one)[0] - out[i, n]).max() <= 2e-5, (i, n)
            # commit the path over the drafted slots
            mine = st.kv[i * st.nb:(i + 1) * st.nb].clone()
            nd.kv_write_rope(ctx, st.geom, st.rope, mine, 0, at, k, v, per_block=len(path))
            for a, b in zip(nd.kv_read(ctx, st.geom, mine, 0, at, per_block=len(path)),
                            nd.kv_read(ctx, st.geom, blk, 0, at, per_block=len(path))):
                assert torch.equal(a, b)
    allowed = R.bits_of(host(st.grammar), VOCAB) == 1
    assert np.array_equal(np.isneginf(logits), ~allowed)
    assert nxt.tolist() == [int(np.argmax(r)) for r in logits]
    raw = out.reshape(S * N, -1).astype(np.float64) @ host(st.head).astype(np.float64)
    for r, h in zip(raw, host(st.hist)):
        t = np.unique(h)
        r[t] = np.where(r[t] > 0, r[t] / np.float32(1.3), r[t] * np.float32(1.3))
    # a product of 768 terms in fp32, summed in any order, and one quotient
    tol = 770 * 2.0 ** -24 * (np.abs(out.reshape(S * N, -1)) @ np.abs(host(st.head)))
    assert (np.abs(logits - raw) <= 1.31 * tol)[allowed].all()


def test_with_and_without_work_on_two_streams():
    """A context of another stream than the current one: outputs of its own,
    the same bits."""
    ctx = nd.Ctx(0)
    want = _state(_ran(Step(ctx, 2)))
    side = torch.cuda.Stream()
    other = nd.Ctx(0, stream=side)
    st = Step(ctx, 2)
    torch.cuda.synchronize()
    g, c = st.geom, other
    q, k, v = st.qkv.split([H * QK, KVH * QK, KVH * VD], 1)
    q = nd.kv_write_rope(c, g, st.rope, st.kv, st.nb, st.pos, k, v, q=q, rot_pos=st.turn, per_block=N)
    out = nd.attend_tree_i8(c, g, st.kv, st.nb, st.based, st.lo, st.mask, q.view(S, N, -1), quant_query=True)
    with torch.cuda.stream(side):
        torch.mm(out.view(S * N, -1), st.head, out=st.logits)
    logits, nxt = nd.logits_adjust(c, st.logits, hist=st.hist, repeat=st.repeat, mask=st.grammar, pick=True)
    torch.cuda.synchronize()
    for a, b in zip(want, (q, out, logits, nxt, st.kv)):
        assert np.array_equal(a, host(b).reshape(a.shape))
    other.close()
    ctx.close()


def _ran(st):
    st.run()
    return st


def test_captured_and_replayed():
    """Two graphs of one context, replayed in turn with other inputs and eager
    work between: every replay's results are the eager ones."""
    side = torch.cuda.Stream()
    ctx = nd.Ctx(0, stream=side)
    with torch.cuda.stream(side):
        a, b = Step(ctx, 3), Step(ctx, 4, (0, 20, 141))
        eager = Step(ctx, 3)
        graphs = []
        for st in (a, b):
            st.run()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                st.run()
            graphs.append(g)
        for turn in range(4):
            for st, g in ((a, graphs[0]), (b, graphs[1])):
                st.fill(10 * turn)
                g.replay()
                got = _state(st)
                ref = Step(ctx, 3 if st is a else 4, tuple(st.base))
                ref.fill(10 * turn)
                want = _state(_ran(ref))
                for x, y in zip(got, want):
                    assert np.array_equal(x, y), turn
            eager.fill(turn)
            eager.run(work=False)
    torch.cuda.synchronize()
    ctx.close()


def test_capture_without_work_is_refused():
    side = torch.cuda.Stream()
    ctx = nd.Ctx(0, stream=side)
    x = torch.zeros(2, 60000, device="cuda")
    torch.cuda.synchronize()
    assert nd.logits_adjust_work(ctx, 2, 60000) > 0
    g = torch.cuda.CUDAGraph()
    y = torch.empty_like(x)
    with torch.cuda.graph(g, stream=side):
        with pytest.raises(nd.NeedleError) as e:
            nd.logits_adjust(ctx, x, pick=True, out=y)
        nd.logits_adjust(ctx, x, out=y)
    assert "work" in str(e.value)
    x += 1
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, y)
    ctx.close()
