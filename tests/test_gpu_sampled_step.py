"""Sampled decoding of a batch that shares its prompts, as a server runs it: the
step laid out, keys and queries turned and appended, the prefixes and the
sessions' own positions attended, the next tokens drawn -- eagerly, on a
stream of its own, and captured into graphs; and the model's own loop with
drawn tokens.

Tolerances are those of the operators' own tests (tests/test_gpu_prefix.py).
"""
import numpy as np
import pytest
import torch

import needle_amd as nd
import prefix_ref as P
import v3_synth as V
from conftest import dev, host

pytestmark = pytest.mark.gpu
H, KVH, QK, VD, VOCAB = 12, 2, 48, 64, 9001


def _i32(a):
    return dev(np.asarray(a, np.int32))


class Step:
    """The buffers of a step of up to `rows` tokens a session, and its calls."""

    def __init__(self, ctx, seed, plen=(70, 133), used=(0, 21, 5, 40), which=(0, 1, 1, -1), length=(2, 3, 1, 2), rows=3, window=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.rows, self.window = ctx, rows, window
        self.plen, self.used, self.which, self.length = (np.array(a, np.int32) for a in (plen, used, which, length))
        self.S, self.cap, self.pcap = len(used), 60, max(plen)
        self.g, self.pg = nd.kv_geom(H, KVH, QK, VD, self.cap), nd.kv_geom(H, KVH, QK, VD, self.pcap)
        self.rope = nd.rope(QK)
        self.pkv, self.pnb = nd.kv_alloc(self.pg, len(plen))
        self.kv, self.nb = nd.kv_alloc(self.g, self.S)
        for i, n in enumerate(plen):
            self._put(self.pg, self.pkv[i * self.pnb:(i + 1) * self.pnb], rng, np.arange(n), np.arange(n))
        for i, n in enumerate(used):
            at = np.arange(n)
            self._put(self.g, self.kv[i * self.nb:(i + 1) * self.nb], rng, at, at + (plen[which[i]] if which[i] >= 0 else 0))
        n = self.S * rows
        self.d = [dev(a) for a in (self.plen, self.used, self.which, self.length)]
        self.plan = torch.empty(nd.prefix_plan_bytes(self.g, self.S, rows, len(plen)), dtype=torch.uint8, device="cuda")
        self.maps = [torch.empty(self.S, rows, dtype=torch.int32, device="cuda") for _ in range(4)] + [None, None]
        self.qkv = torch.empty(n, (H + KVH) * QK + KVH * VD, device="cuda")
        self.q, self.out = torch.empty(n, H * QK, device="cuda"), torch.zeros(self.S, rows, H * VD, device="cuda")
        self.head = dev((0.4 * rng.normal(size=(H * VD, VOCAB))).astype(np.float32))
        self.logits = torch.empty(n, VOCAB, device="cuda")
        self.u, self.temperature = torch.empty(n, device="cuda"), torch.full((n,), 0.8, device="cuda")
        self.top_k, self.top_p = torch.full((n,), 40, dtype=torch.int32, device="cuda"), torch.full((n,), 0.9, device="cuda")
        self.top_k[1::3] = 0
        self.next, self.prob = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda")
        self.work = torch.empty(max(nd.attend_prefix_i8_work(ctx, self.g, self.S, rows, len(plen)),
                                    nd.sample_rows_work(ctx, n, VOCAB)), dtype=torch.uint8, device="cuda")
        self.fill(seed)

    def _put(self, g, blk, rng, at, turn):
        if len(at):
            nd.kv_write_rope(self.ctx, g, self.rope, blk, 0, _i32(at), dev(rng.normal(size=(len(at), KVH * QK)).astype(np.float32)),
                             dev(rng.normal(size=(len(at), KVH * VD)).astype(np.float32)), rot_pos=_i32(turn), per_block=len(at))

    def fill(self, seed, used=None):
        rng = np.random.default_rng(1000 + seed)
        self.qkv.copy_(dev(rng.normal(size=self.qkv.shape).astype(np.float32)))
        self.u.copy_(dev(rng.random(len(self.u)).astype(np.float32)))
        if used is not None:
            self.used = np.array(used, np.int32)
            self.d[1].copy_(dev(self.used))

    def run(self, work=True):
        c, w = self.ctx, self.work if work else None
        plan, _ = nd.prefix_plan(c, self.g, self.pcap, self.d[0], self.d[1], prefix_of=self.d[2], length=self.d[3], rows=self.rows,
                                 window=self.window, plan=self.plan, maps=self.maps)
        q, k, v = self.qkv.split([H * QK, KVH * QK, KVH * VD], 1)
        nd.kv_write_rope(c, self.g, self.rope, self.kv, self.nb, self.maps[0].view(-1), k, v, q=q, q_out=self.q,
                         rot_pos=self.maps[1].view(-1), per_block=self.rows)
        nd.attend_prefix_i8(c, self.g, self.kv, self.nb, self.pkv, self.pnb, plan, self.q.view(self.S, self.rows, -1),
                            quant_query=True, out=self.out, work=w)
        torch.mm(self.out.view(self.S * self.rows, -1), self.head, out=self.logits)
        nd.sample_rows(c, self.logits, self.u, temperature=self.temperature, top_k=self.top_k, top_p=self.top_p, out=self.next,
                       prob=self.prob, work=w)
        return self

    def state(self):
        torch.cuda.synchronize()
        there = np.arange(self.rows)[None] < self.length[:, None]
        return [host(t).copy() for t in (self.out, self.logits, self.next, self.prob, self.kv)] + \
            [host(self.q).reshape(self.S, self.rows, -1)[there].copy()]


@pytest.mark.parametrize("window", [0, 50])
def test_a_row_is_its_context_decoded(ctx, window):
    """Each row's attention is that of one block that holds its whole context, and
    its token the plain draw from its logits."""
    st = Step(ctx, 1, window=window).run()
    out, logits, nxt, prob, _, _ = st.state()
    for i in range(st.S):
        p = st.which[i]
        L = int(st.plen[p]) if p >= 0 else 0
        u, m = int(st.used[i]), int(st.length[i])
        whole = nd.kv_geom(H, KVH, QK, VD, L + u + m)
        blk, _ = nd.kv_alloc(whole)
        parts = [(st.pkv[p * st.pnb:(p + 1) * st.pnb], st.pg, 0, L)] if p >= 0 else []
        parts.append((st.kv[i * st.nb:(i + 1) * st.nb], st.g, L, u + m))
        for b, g, at, n in parts:
            k, v = nd.kv_read(ctx, g, b, 0, _i32(np.arange(n)), per_block=n)
            nd.kv_write(ctx, whole, blk, 0, _i32(at + np.arange(n)), k, v)
        for n in range(m):
            end = L + u + n
            lo = max(0, end + 1 - window) if window else 0
            one = nd.attend_step_i8(ctx, whole, blk, 0, _i32([lo]), _i32([end]), st.q[i * st.rows + n][None], quant_query=True)
            # rows read back and written again keep their codes (the largest is 127), and a scale
            # that is rounded once more is off by 2^-23: 1e-6 of a weight, 1e-5 of an output, and
            # either side is within 2e-5 of its sums
            assert np.abs(host(one)[0] - out[i, n]).max() <= 5e-5, (i, n)
            want = P.draw(logits[i * st.rows + n], float(host(st.u)[i * st.rows + n]), temperature=0.8,
                          top_k=int(host(st.top_k)[i * st.rows + n]), top_p=0.9)
            assert want[2] > 1e-11 and nxt[i * st.rows + n] == want[0], (i, n)
            assert abs(prob[i * st.rows + n] - want[1]) <= 2.0 ** -24 * want[1] + 1e-12


def test_a_prompt_in_one_step_or_token_by_token(ctx):
    """Rows of one step, or as many steps of a row: the same cache and the same
    outputs, within the attention's tolerance."""
    a = Step(ctx, 2, length=(3, 3, 3, 3)).run()
    out = a.state()[0]
    b = Step(ctx, 2, length=(1, 1, 1, 1), rows=1)
    qkv = a.qkv.view(a.S, 3, -1)
    for n in range(3):
        b.qkv.copy_(qkv[:, n])
        b.d[1].copy_(dev(a.used + n))
        b.run()
        assert np.abs(host(b.out)[:, 0] - out[:, n]).max() <= 2 * 2e-5, n
    assert torch.equal(a.kv, b.kv)


def test_without_work_on_a_stream_of_its_own():
    """A context of another stream than the current one, its own workspace and
    outputs: the same bits."""
    ctx = nd.Ctx(0)
    want = Step(ctx, 3).run().state()
    side = torch.cuda.Stream()
    other = nd.Ctx(0, stream=side)
    st = Step(ctx, 3)
    torch.cuda.synchronize()
    st.ctx = other
    plan, maps = nd.prefix_plan(other, st.g, st.pcap, st.d[0], st.d[1], prefix_of=st.d[2], length=st.d[3], rows=st.rows)
    q, k, v = st.qkv.split([H * QK, KVH * QK, KVH * VD], 1)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pos, rot = maps[0].reshape(-1), maps[1].reshape(-1)
    q = nd.kv_write_rope(other, st.g, st.rope, st.kv, st.nb, pos, k, v, q=q, rot_pos=rot, per_block=st.rows)
    out = nd.attend_prefix_i8(other, st.g, st.kv, st.nb, st.pkv, st.pnb, plan, q.view(st.S, st.rows, -1), quant_query=True)
    with torch.cuda.stream(side):
        torch.mm(out.view(st.S * st.rows, -1), st.head, out=st.logits)
    nxt, prob = nd.sample_rows(other, st.logits, st.u, temperature=st.temperature, top_k=st.top_k, top_p=st.top_p)
    torch.cuda.synchronize()
    for a, b in zip(want, (out, st.logits, nxt, prob, st.kv)):
        assert np.array_equal(a, host(b).reshape(a.shape))
    other.close()
    ctx.close()


def test_captured_and_replayed():
    """Two graphs of one context that share a workspace, replayed in turn with other
    inputs, lengths and eager work between: every replay's results are the eager
    ones."""
    side = torch.cuda.Stream()
    ctx = nd.Ctx(0, stream=side)
    with torch.cuda.stream(side):
        kw = dict(plen=(44,), used=(3, 9), which=(0, 0), length=(1, 1), rows=1)
        a, b = Step(ctx, 4), Step(ctx, 5, **kw)
        if a.work.numel() < b.work.numel():
            a.work = b.work
        b.work = a.work
        eager, graphs = Step(ctx, 4), []
        for st in (a, b):
            st.run()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                st.run()
            graphs.append(g)
        blocks = [a.kv.clone(), b.kv.clone()]
        for turn in range(4):
            for st, g, kv, seed, more in ((a, graphs[0], blocks[0], 4, {}), (b, graphs[1], blocks[1], 5, kw)):
                base = np.array(more.get("used", (0, 21, 5, 40)))
                st.kv.copy_(kv)
                st.fill(10 * turn, base + turn)
                g.replay()
                got = st.state()
                ref = Step(ctx, seed, **more)
                ref.kv.copy_(kv)
                ref.fill(10 * turn, base + turn)
                for x, y in zip(got, ref.run().state()):
                    assert np.array_equal(x, y), turn
            eager.fill(turn)
            eager.run(work=False)
    torch.cuda.synchronize()
    ctx.close()


def test_capture_without_work_is_refused():
    side = torch.cuda.Stream()
    ctx = nd.Ctx(0, stream=side)
    with torch.cuda.stream(side):
        st = Step(ctx, 6).run()
        torch.cuda.synchronize()
        big = torch.zeros(2, 60000, device="cuda")
        u = torch.zeros(2, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            plan = nd.PrefixPlan(st.plan, (st.S, st.rows, 2, st.pcap, H, KVH, st.cap))
            for f in (lambda: nd.attend_prefix_i8(ctx, st.g, st.kv, st.nb, st.pkv, st.pnb, plan, st.q.view(st.S, st.rows, -1), out=st.out),
                      lambda: nd.sample_rows(ctx, big, u, out=st.next, prob=st.prob)):
                with pytest.raises(nd.NeedleError, match="work"):
                    f()
            nd.sample_rows(ctx, st.logits[:, :8192], st.u, out=st.next, prob=st.prob)  # rows of one slice need none
        g.replay()
    torch.cuda.synchronize()
    ctx.close()


def test_work_that_is_too_small(ctx):
    st = Step(ctx, 7)
    for f in (lambda w: nd.attend_prefix_i8(ctx, st.g, st.kv, st.nb, st.pkv, st.pnb, st.run() and nd.PrefixPlan(
                st.plan, (st.S, st.rows, 2, st.pcap, H, KVH, st.cap)), st.q.view(st.S, st.rows, -1), work=w),
              lambda w: nd.sample_rows(ctx, st.logits, st.u, work=w)):
        for w in (st.work[:64], st.work[8:]):
            with pytest.raises(nd.NeedleError, match="work"):
                f(w)


# ---- the model's loop ----------------------------------------------------------------

def _model(ctx, sessions, steps):
    g, recs = V.build_records(V.small_geometry(4), seed=5)
    dm = nd.V3Model(ctx, g, recs, V.CODEBOOK)
    prompts = np.stack([V.prompt_tokens(20, 40 + i) for i in range(sessions)])
    batches = []
    for _ in range(2):
        b = nd.V3Batch(dm, sessions, max_len=20 + steps + 8, max_chunk=20)
        batches.append((b, b.prefill(prompts)))
    return dm, batches


def test_a_drawn_loop_is_its_steps_drawn(ctx):
    sessions, steps = 3, 30
    dm, ((a, first), (b, same)) = _model(ctx, sessions, steps)
    assert np.array_equal(first, same)
    u = torch.rand(steps, sessions, device="cuda")
    rules = dict(temperature=torch.tensor([0.7, 1.0, 1.6], device="cuda"), top_k=torch.tensor([20, 0, 0], dtype=torch.int32, device="cuda"),
                 top_p=torch.tensor([1.0, 0.8, 0.95], device="cuda"), min_p=torch.tensor([0.0, 0.0, 0.05], device="cuda"))
    got = b.sampled(first, u, **rules)
    logits = torch.empty(sessions, dm.rows, device="cuda")
    tok = first
    for k in range(steps):
        a.step(tok, logits=logits, want_next=False)
        drawn, _ = nd.sample_rows(ctx, logits, u[k], **rules)
        tok = host(drawn)
        assert np.array_equal(tok, got[:, k]), k
    assert len(np.unique(got)) > 3 and np.array_equal(a.positions(), b.positions())
    # and both go on from the same state
    assert np.array_equal(a.step(got[:, -1]), b.step(got[:, -1]))
    a.close(), b.close(), dm.close()


def test_a_drawn_loop_over_a_long_vocabulary(ctx):
    """Logits of several slices, whose workspace is the context's."""
    g = V.small_geometry(4)
    g.update(vocab_size=20000, out_vocab=20000)
    g, recs = V.build_records(g, seed=6)
    dm = nd.V3Model(ctx, g, recs, V.CODEBOOK)
    assert dm.rows == 20000
    sessions, steps = 2, 8
    a, b = (nd.V3Batch(dm, sessions, max_len=40, max_chunk=20) for _ in range(2))
    prompts = np.stack([V.prompt_tokens(20, 50 + i) for i in range(sessions)])
    first = a.prefill(prompts)
    assert np.array_equal(first, b.prefill(prompts))
    u = torch.rand(steps, sessions, device="cuda")
    rules = dict(temperature=torch.tensor([0.9, 1.5], device="cuda"), top_k=torch.tensor([900, 0], dtype=torch.int32, device="cuda"),
                 top_p=torch.tensor([0.9, 0.95], device="cuda"))
    got = b.sampled(first, u, **rules)
    logits, tok = torch.empty(sessions, dm.rows, device="cuda"), first
    for k in range(steps):
        a.step(tok, logits=logits, want_next=False)
        tok = host(nd.sample_rows(ctx, logits, u[k], **rules)[0])
        assert np.array_equal(tok, got[:, k]), k
    assert len(np.unique(got)) > 3
    a.close(), b.close(), dm.close()


def test_a_cold_loop_is_the_greedy_one(ctx):
    dm, ((a, first), (b, _)) = _model(ctx, 2, 12)
    want = a.greedy(first, 12)
    u = torch.rand(12, 2, device="cuda")
    assert np.array_equal(b.sampled(first, u, temperature=torch.zeros(2, device="cuda")), want)
    for bad in (u[:, :1], u.double(), u.view(-1)):
        with pytest.raises(ValueError):
            b.sampled(first, bad)
    with pytest.raises(nd.NeedleError):
        b.sampled(first, torch.rand(40, 2, device="cuda"))
    a.close(), b.close(), dm.close()
