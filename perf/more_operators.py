"""Sampled decoding of a batch that shares its prompts, as measurable cases.

A server whose sessions begin with the same text (a set of tool descriptions)
holds that text's keys and values once.  Each step it lays out the batch's rows
from the requests' lengths, appends them to the sessions' own blocks, lets every
row attend to its session's prefix and to the session's own positions, and draws
each session's next token:

  plan     positions, angles and windows of every row, and the rows grouped by
           prefix, from the requests' lengths
  attend   attention of the batch over its shared prefixes and its own blocks
  sample   temperature, min-p, top-k and top-p on rows of logits, and the draw

With `own` false `run` computes them in their plain form; with `own` true it
makes the calls of needle-rs_amd/needle_amd.py.  Sizes are the shipped
Needle-3 geometry's (12 query heads on 2 kv heads, qk 48, v 64, windows of 1024,
8192 tokens of vocabulary), the benchmark's 12 x 64 cache, and generic ones.
"""
import math
import os
import sys

import numpy as np
import torch

own = False


def listed():
    v3 = dict(heads=12, kv_heads=2, qk=48)
    mha = dict(heads=12, kv_heads=12, qk=64)
    return [
        # the rows of a small batch's step: the smallest call
        dict(name="plan_few", kind="plan", sessions=5, rows=1, prefixes=1, prefix=300, used=40, window=0, **v3),
        # a windowed layer's rows of thousands of requests over many prompts, some tokens each
        dict(name="plan_many", kind="plan", sessions=4001, rows=5, prefixes=90, prefix=3000, used=900, window=1024, **v3),
        # a few completions of one short prompt: latency
        dict(name="attend_few", kind="attend", sessions=4, rows=1, prefixes=1, prefix=301, used=60, window=0,
             quant_query=True, **v3),
        # 64 sessions behind 2000 tokens of tool descriptions
        dict(name="attend_64", kind="attend", sessions=64, rows=1, prefixes=1, prefix=2000, used=120, window=0,
             quant_query=True, **v3),
        # 200 sessions of the 12 x 64 cache behind seven prompts of their own lengths, fp32 queries
        dict(name="attend_groups", kind="attend", sessions=200, rows=1, prefixes=7, prefix=4000, used=500, window=0,
             quant_query=False, **mha),
        # the windowed layers of 128 sessions: part of the prompt has left the window, own rings have wrapped
        dict(name="attend_window", kind="attend", sessions=128, rows=1, prefixes=3, prefix=1501, used=1300, window=1024,
             quant_query=True, **v3),
        # 24 sessions' own prompts of up to 33 tokens, prefilled behind the tool descriptions in one step
        dict(name="attend_chunk", kind="attend", sessions=24, rows=33, prefixes=2, prefix=2500, used=10, window=0,
             quant_query=True, **v3),
        # 512 completions behind a full context: the scores
        dict(name="attend_large", kind="attend", sessions=512, rows=1, prefixes=1, prefix=8000, used=100, window=0,
             quant_query=False, **v3),
        # one session's token, every rule: latency
        dict(name="sample_one", kind="sample", rows=1, n=8192, temperature=0.7, top_k=40, top_p=0.95, min_p=0.02),
        # a large batch, the usual nucleus
        dict(name="sample_batch", kind="sample", rows=1024, n=8192, temperature=0.8, top_k=0, top_p=0.9, min_p=0.0),
        # the whole distribution, hot
        dict(name="sample_flat", kind="sample", rows=320, n=8191, temperature=1.7, top_k=0, top_p=1.0, min_p=0.0),
        # a large odd vocabulary, rows that are not aligned
        dict(name="sample_wide", kind="sample", rows=200, n=100003, temperature=1.0, top_k=50, top_p=0.95, min_p=0.0),
    ]


# ---- drawn cases ------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "attend", "attend", "attend", "sample", "sample"])
    heads, kv_heads, qk = rng.choice([(12, 2, 48), (12, 2, 48), (12, 12, 64), (8, 4, 64), (16, 2, 64), (5, 1, 48)])
    geom = dict(heads=heads, kv_heads=kv_heads, qk=qk)
    window = rng.choice([0, 0, 256, 1024])
    if kind == "plan":
        rows = rng.choice([1, 1, 1, _log(rng, 2, 64)])
        sessions = _log(rng, 1, 20000 // rows)
        return dict(kind=kind, sessions=sessions, rows=rows, prefixes=_log(rng, 1, min(200, sessions)),
                    prefix=_log(rng, 1, 8000), used=_log(rng, 1, 4000), window=window, **geom)
    if kind == "attend":
        rows = rng.choice([1, 1, 1, _log(rng, 2, 64)])
        prefix, used = _log(rng, 1, 8000), _log(rng, 1, 2000)
        span = prefix + used + rows
        span = min(span, window + rows) if window else span
        most = min(1.0e8 / (span * rows * heads), 2.0e8 / ((used + rows) * kv_heads * (qk + 64)))
        sessions = _log(rng, 1, max(1, min(600, int(most) // 2)))
        return dict(kind=kind, sessions=sessions, rows=rows, prefixes=_log(rng, 1, min(16, sessions)), prefix=prefix,
                    used=used, window=window, quant_query=rng.random() < 0.5, **geom)
    n = 8192 if rng.random() < 0.4 else _log(rng, 300, 150000)
    return dict(kind=kind, rows=_log(rng, 1, max(2, min(4096, 20000000 // n))), n=n,
                temperature=rng.uniform(0.3, 2.0), top_k=rng.choice([0, 0, _log(rng, 1, min(n, 4000))]),
                top_p=rng.choice([1.0, rng.uniform(0.1, 0.999)]), min_p=rng.choice([0.0, 0.0, 10 ** rng.uniform(-4, -0.5)]))


# ---- sizes that the case alone fixes ----------------------------------------

def _requests(case):
    """Each session's prefix (-1: none), own positions so far and rows of this
    step, and each prefix's length (all ragged)."""
    s, rows, count = case["sessions"], case["rows"], case["prefixes"]
    i, p = np.arange(s), np.arange(count)
    which = (i * 7 + i // 5) % count
    if count > 1:
        which = np.where(i % 11 == 10, -1, which)
    used = case["used"] - (i * 37) % (case["used"] // 2 + 1)
    length = rows - (i * 5) % (rows // 2 + 1)
    plen = case["prefix"] - (p * 53) % (case["prefix"] // 3 + 1)
    return [a.astype(np.int32) for a in (which, used, length, plen)]


def _caps(case):
    """Positions that an own block and a prefix's block hold."""
    most = case["used"] + case["rows"]
    if case["window"]:  # rings
        return min(most, case["window"] + case["rows"] + 5), min(case["prefix"], case["window"] + 7)
    return most + 3, case["prefix"] + 1


def _rows(case):
    """Per (session, row), for a host's reckoning: whether it is there, the first
    and the number of its prefix's and of its own positions."""
    which, used, length, plen = _requests(case)
    n = np.arange(case["rows"])[None]
    there = n < length[:, None]
    before = np.where(which >= 0, plen[np.maximum(which, 0)], 0)[:, None]
    at = before + used[:, None] + n
    start = np.maximum(at + 1 - case["window"], 0) if case["window"] else np.zeros_like(at)
    first, lo = np.minimum(start, before), np.maximum(start - before, 0)
    return which, there, first, before - first, lo, used[:, None] + n + 1 - lo


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- the cache's bytes -------------------------------------------------------

def _parts(case, cap):
    """Byte offsets of a block's parts (k, v, k scales, v scales) and its size."""
    kvh, at = case["kv_heads"], [0]
    for size in (kvh * cap * case["qk"], kvh * cap * 64, 4 * kvh * cap, 4 * kvh * cap):
        at.append(at[-1] + -(-size // 256) * 256)
    return at


def _views(case, kv, cap):
    """The blocks' parts as tensors [blocks][KVH][cap](..)."""
    at, kvh, qk = _parts(case, cap), case["kv_heads"], case["qk"]
    b = kv.view(-1, at[4])
    s = len(b)
    k = b[:, :kvh * cap * qk].view(torch.int8).view(s, kvh, cap, qk)
    v = b[:, at[1]:at[1] + kvh * cap * 64].view(torch.int8).view(s, kvh, cap, 64)
    ks = b[:, at[2]:at[2] + 4 * kvh * cap].view(torch.float32).view(s, kvh, cap)
    vs = b[:, at[3]:at[3] + 4 * kvh * cap].view(torch.float32).view(s, kvh, cap)
    return k, v, ks, vs


def _quant(x):
    """Codes and scales of the last axis, in the cache's own 32-bit steps."""
    top = x.abs().amax(-1, keepdim=True)
    one = torch.ones_like(top)  # tensor by tensor: the rounded quotient, no product with 1/127
    scale = torch.where(top > 0, torch.div(top, one * 127), one)
    y = x * torch.div(one, scale)
    r = torch.sign(y) * torch.floor(y.abs().double() + 0.5).float()
    return r.clamp(-128, 127), scale


def _filled(case, blocks, cap, g):
    """Blocks whose every slot holds a quantised N(0, 1) row."""
    kv = torch.zeros(blocks * _parts(case, cap)[4], dtype=torch.uint8, device="cuda")
    k, v, ks, vs = _views(case, kv, cap)
    for part, scales in ((k, ks), (v, vs)):
        codes, scale = _quant(_randn(g, *part.shape))
        part.copy_(codes.to(torch.int8))
        scales.copy_(scale[..., 0])
    return kv


# ---- inputs -----------------------------------------------------------------

def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "sample":
        return _prepare_sample(case, g)
    which, used, length, plen = _requests(case)
    if kind == "plan":  # the same requests, in another order
        p = np.random.default_rng(int(seed)).permutation(len(which))
        which, used, length = which[p], used[p], length[p]
    st = dict(case=case, which=_cuda(which), used=_cuda(used), length=_cuda(length), plen=_cuda(plen))
    cap, pcap = _caps(case)
    st["cap"], st["pcap"] = cap, pcap
    if kind == "plan":
        return st
    s, rows = case["sessions"], case["rows"]
    st["kv"], st["stride"] = _filled(case, s, cap, g), _parts(case, cap)[4]
    st["pkv"], st["pstride"] = _filled(case, case["prefixes"], pcap, g), _parts(case, pcap)[4]
    st["q"] = 2 * _randn(g, s, rows, case["heads"] * case["qk"])
    st["out"] = _randn(g, s, rows, case["heads"] * 64)  # rows past a session's end stay as they are
    if own:  # one plan serves a step's layers
        nd, ctx = _needle()
        st["plan"] = _plan(nd, ctx, case, st)[0]
    return st


def _prepare_sample(case, g):
    rows, n = case["rows"], case["n"]
    x = 2 * _randn(g, rows, n)
    # a few tokens stand out, as a trained model's do (no token twice: the seed alone decides)
    likely = (torch.randint(0, n, (rows, 1), generator=g, device="cuda") + torch.arange(24, device="cuda") * (n // 24)) % n
    x.scatter_(1, likely, 7 + 2.5 * _randn(g, rows, 24))
    i = torch.arange(rows, device="cuda")
    # rows under a grammar have lost half of their tokens
    gone = torch.randint(0, 2, (n,), generator=g, device="cuda") == 1
    x.masked_fill_((i % 5 == 3)[:, None] & gone[None], -math.inf)
    st = dict(case=case, x=x, u=torch.rand(rows, generator=g, device="cuda"))
    # every request has its own settings; some are greedy, some leave a rule out
    vary = 0.75 + 0.5 * torch.rand(rows, generator=g, device="cuda")
    st["temperature"] = torch.where(i % 16 == 7, 0.0, case["temperature"] * vary)
    st["top_k"] = torch.where(i % 6 == 4, 0, (case["top_k"] * vary).long().clamp(min=1)).int() if case["top_k"] else None
    st["top_p"] = torch.where(i % 7 == 5, 1.0, (case["top_p"] * (1.1 - 0.2 * vary)).clamp(max=1.0)) \
        if case["top_p"] < 1 else None
    st["min_p"] = torch.where(i % 8 == 6, 0.0, case["min_p"] * vary) if case["min_p"] > 0 else None
    return st


# ---- one pass ---------------------------------------------------------------

_HAND = {}


def _needle():
    """The package and the context of the current stream, as a server holds them."""
    device = torch.cuda.current_device()
    key = device, torch._C._cuda_getCurrentRawStream(device)  # (current_stream() takes a microsecond)
    if key not in _HAND:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "needle-rs_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import needle_amd
        _HAND[key] = needle_amd, needle_amd.Ctx(device)
    return _HAND[key]


def run(st):
    case = st["case"]
    return {"plan": _run_plan, "attend": _run_attend, "sample": _run_sample}[case["kind"]](case, st)


def _plan(nd, ctx, case, st):
    geom = nd.kv_geom(case["heads"], case["kv_heads"], case["qk"], 64, st["cap"])
    return nd.prefix_plan(ctx, geom, st["pcap"], st["plen"], st["used"], prefix_of=st["which"], length=st["length"],
                          rows=case["rows"], window=case["window"])


def _maps(case, st):
    """pos, rot, from, lo [S][N]; order [S N]; first [P + 1], all in whole numbers."""
    n = torch.arange(case["rows"], device="cuda")[None]
    which, used, count = st["which"].long(), st["used"].long()[:, None], case["prefixes"]
    before = torch.where(which >= 0, st["plen"].long()[which.clamp(min=0)], 0)[:, None]
    rot = before + used + n
    start = (rot + 1 - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(rot)
    there = n < st["length"][:, None]
    maps = [torch.where(there, m, -1).int() for m in (used + n, rot, torch.minimum(start, before), (start - before).clamp(min=0))]
    key = torch.where(there & (which >= 0)[:, None], which[:, None], count).reshape(-1)
    order = torch.argsort(key, stable=True)
    grouped = key[order]
    order = torch.where(grouped < count, order, -1).int()
    first = (key[None] < torch.arange(count + 1, device="cuda")[:, None]).sum(1).int()
    return maps + [order, first]


def _run_plan(case, st):
    if own:
        nd, ctx = _needle()
        return _plan(nd, ctx, case, st)[1]
    return _maps(case, st)


def _run_attend(case, st):
    h, kvh, qk, rows, s = case["heads"], case["kv_heads"], case["qk"], case["rows"], case["sessions"]
    cap, pcap, rep = st["cap"], st["pcap"], h // kvh
    if own:
        nd, ctx = _needle()
        geom = nd.kv_geom(h, kvh, qk, 64, cap)
        return nd.attend_prefix_i8(ctx, geom, st["kv"], st["stride"], st["pkv"], st["pstride"], st["plan"], st["q"],
                                   quant_query=case["quant_query"], out=st["out"])
    q = st["q"].reshape(s, rows, h, qk)
    if case["quant_query"]:
        codes, scale = _quant(q)
        q = codes * scale
    q = q.reshape(s, rows, kvh, rep, qk).permute(0, 2, 1, 3, 4).reshape(s, kvh, rows * rep, qk)
    _, _, first, lo, _, _ = _maps(case, st)
    # the sessions' own positions: the last of the ring up to the step's end
    k, v, ks, vs = _views(case, st["kv"], cap)
    back = min(cap, case["used"] + rows)
    end = (st["used"] + rows).long()[:, None]
    pos = end - back + torch.arange(back, device="cuda")
    slot = (pos % cap)[:, None, :].expand(s, kvh, back)
    kf = torch.gather(k, 2, slot[..., None].expand(s, kvh, back, qk)).float() * torch.gather(ks, 2, slot)[..., None]
    vf = torch.gather(v, 2, slot[..., None].expand(s, kvh, back, 64)).float() * torch.gather(vs, 2, slot)[..., None]
    n = torch.arange(rows, device="cuda")[None, :, None]
    sees = (pos[:, None] >= lo.long()[..., None]) & (pos[:, None] <= st["used"].long()[:, None, None] + n) & (pos[:, None] >= 0)
    sees = sees[:, None, :, None].expand(s, 1, rows, rep, back).reshape(s, 1, rows * rep, back)
    t = torch.matmul(q, kf.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(qk))
    t = t.masked_fill(~sees, -math.inf)
    top = t.amax(-1, keepdim=True)
    w = torch.exp(t - torch.where(top == -math.inf, 0.0, top))
    total, o = w.sum(-1, keepdim=True), torch.matmul(w, vf)
    # the prefixes, one after another, each for the rows of its sessions at once
    k, v, ks, vs = _views(case, st["pkv"], pcap)
    which, used, length, plen = _requests(case)
    for p in range(case["prefixes"]):
        mine = _cuda(np.flatnonzero(which == p))
        if not len(mine):
            continue
        m, back = len(mine), min(pcap, int(plen[p]))
        pos = int(plen[p]) - back + torch.arange(back, device="cuda")
        slot = pos % pcap
        kf = k[p][:, slot].float() * ks[p][:, slot, None]
        vf = v[p][:, slot].float() * vs[p][:, slot, None]
        qp = q[mine].transpose(0, 1).reshape(kvh, m * rows * rep, qk)
        sees = pos >= first[mine].long().reshape(-1, 1)
        sees = sees[:, None].expand(m * rows, rep, back).reshape(1, m * rows * rep, back)
        t = torch.matmul(qp, kf.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(qk))
        t = t.masked_fill(~sees, -math.inf)
        more = t.amax(-1, keepdim=True)
        w = torch.exp(t - torch.where(more == -math.inf, 0.0, more))

        def back_to(a):
            return a.reshape(kvh, m, rows * rep, -1).transpose(0, 1)
        more, sums, values = back_to(more), back_to(w.sum(-1, keepdim=True)), back_to(torch.matmul(w, vf))
        both = torch.maximum(top[mine], more)
        at = torch.where(both == -math.inf, 0.0, both)
        a, b = torch.exp(top[mine] - at), torch.exp(more - at)
        total[mine], o[mine] = total[mine] * a + sums * b, o[mine] * a + values * b
    o = o / torch.where(total == 0, 1.0, total)
    o = o.reshape(s, kvh, rows, rep, 64).permute(0, 2, 1, 3, 4).reshape(s, rows, h * 64)
    there = torch.arange(rows, device="cuda")[None] < st["length"][:, None]
    return torch.where(there[..., None], o, st["out"])


def _run_sample(case, st):
    if own:
        nd, ctx = _needle()
        return nd.sample_rows(ctx, st["x"], st["u"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                              min_p=st["min_p"])
    n = case["n"]
    x, at = torch.sort(st["x"], dim=1, descending=True, stable=True)
    t = st["temperature"].double()[:, None]
    w = torch.exp((x.double() - x[:, :1].double()) / torch.where(t > 0, t, 1.0))
    keep = x > -math.inf
    if st["min_p"] is not None:
        keep = keep & (w >= st["min_p"].double()[:, None])
    if st["top_k"] is not None:
        k = st["top_k"].long()[:, None]
        keep = keep & ((torch.arange(n, device="cuda")[None] < k) | (k <= 0))
    w = torch.where(keep, w, 0.0)
    upto = torch.cumsum(w, 1)
    if st["top_p"] is not None:
        p = st["top_p"].double()[:, None]
        w = torch.where((upto - w < p * upto[:, -1:]) | (p >= 1), w, 0.0)
        upto = torch.cumsum(w, 1)
    drawn = (upto <= st["u"].double()[:, None] * upto[:, -1:]).sum(1, keepdim=True)
    drawn = torch.where(t > 0, drawn, 0)
    prob = torch.where(t > 0, torch.gather(w, 1, drawn) / upto[:, -1:], 1.0)
    return torch.gather(at, 1, drawn)[:, 0].int(), prob[:, 0].float()


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "plan":
        s, rows = case["sessions"], case["rows"]
        return dict(bytes=12 * s + 4 * case["prefixes"] + 20 * s * rows + 4 * (case["prefixes"] + 1), flops=8 * s * rows)
    if kind == "attend":
        which, there, first, old, lo, new = _rows(case)
        h, kvh, qk = case["heads"], case["kv_heads"], case["qk"]
        span = 0
        for p in range(case["prefixes"]):
            mine = (which == p)[:, None] & there
            span += int((old * mine).max()) if mine.any() else 0
        end = (lo + new) * there
        span += int((end.max(1) - lo[:, 0]).sum())
        pairs, rows = int(((old + new) * there).sum()), int(there.sum())
        return dict(bytes=span * kvh * (qk + 64 + 8) + 4 * rows * h * (qk + 64), flops=2 * pairs * h * (qk + 64))
    return dict(bytes=case["rows"] * (4 * case["n"] + 28), flops=4 * case["rows"] * case["n"])


# ---- the same in 64 bits ----------------------------------------------------

def _stands_for(q):
    codes, scale = _quant(q)
    return codes.double() * scale.double()


def _exact_attend(case, st):
    """Row by row of each session: its prefix's positions and its own, side by side."""
    h, kvh, qk = case["heads"], case["kv_heads"], case["qk"]
    which, there, first, old, lo, new = _rows(case)
    blocks = _views(case, st["kv"], st["cap"]), _views(case, st["pkv"], st["pcap"])
    out = st["out"].double()
    for i in range(case["sessions"]):
        m, p = int(there[i].sum()), int(which[i])
        parts, sees = [], []
        if p >= 0 and old[i, :m].max() > 0:
            begin, end = int(first[i, :m].min()), int(first[i, 0] + old[i, 0])
            at = np.arange(begin, end)
            parts.append((blocks[1], p, at % st["pcap"]))
            sees.append(at[None] >= first[i, :m, None])
        at = np.arange(int(lo[i, 0]), int(lo[i, m - 1] + new[i, m - 1]))
        parts.append((blocks[0], i, at % st["cap"]))
        sees.append((at[None] >= lo[i, :m, None]) & (at[None] < (lo + new)[i, :m, None]))
        k, v = (torch.cat([b[c][j][:, _cuda(slot)].double() * b[c + 2][j][:, _cuda(slot), None].double()
                           for b, j, slot in parts], 1).repeat_interleave(h // kvh, 0) for c in (0, 1))
        q = st["q"][i, :m].reshape(m, h, qk)
        q = (_stands_for(q) if case["quant_query"] else q.double()).transpose(0, 1)
        t = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(qk)
        w = torch.softmax(t.masked_fill(~_cuda(np.concatenate(sees, 1))[None], -math.inf), -1)
        out[i, :m] = torch.matmul(w, v).transpose(0, 1).reshape(m, -1)
    return out


def _exact_sample(case, st):
    """By thresholds instead of positions: each rule as the lowest logit it keeps."""
    x, rows = st["x"].cpu().numpy().astype(np.float64), case["rows"]
    get = {k: (st[k].cpu().numpy().astype(np.float64) if st[k] is not None else None)
           for k in ("u", "temperature", "top_k", "top_p", "min_p")}
    nxt, prob = np.zeros(rows, np.int32), np.ones(rows)
    for i in range(rows):
        t = get["temperature"][i]
        if not t > 0:
            nxt[i] = int(np.argmax(x[i]))
            continue
        ids = np.flatnonzero(x[i] > -np.inf)
        z = (x[i, ids] - x[i].max()) / t
        if get["min_p"] is not None and get["min_p"][i] > 0:
            some = z >= math.log(get["min_p"][i])
            ids, z = ids[some], z[some]
        by = np.lexsort((ids, -z))
        if get["top_k"] is not None and get["top_k"][i] > 0:
            by = by[:int(get["top_k"][i])]
        ids, w = ids[by], np.exp(z[by])
        if get["top_p"] is not None and get["top_p"][i] < 1:
            sums = np.add.accumulate(w)
            end = int(np.searchsorted(sums, get["top_p"][i] * sums[-1], side="left")) + 1
            ids, w = ids[:end], w[:end]
        sums = np.add.accumulate(w)
        j = int(np.searchsorted(sums, get["u"][i] * sums[-1], side="right"))
        nxt[i], prob[i] = ids[j], w[j] / sums[-1]
    return torch.from_numpy(nxt), torch.from_numpy(prob)


def _exact_plan(case, st):
    """Request by request, each row put to the end of its prefix's group."""
    rows, count = case["rows"], case["prefixes"]
    groups = [[] for _ in range(count)]
    maps = [[], [], [], []]
    plen = st["plen"].tolist()
    for i, (p, used, m) in enumerate(zip(st["which"].tolist(), st["used"].tolist(), st["length"].tolist())):
        before = plen[p] if p >= 0 else 0
        for n in range(rows):
            at = before + used + n
            start = max(at + 1 - case["window"], 0) if case["window"] else 0
            row = (used + n, at, min(start, before), max(start - before, 0)) if n < m else (-1, -1, -1, -1)
            for out, value in zip(maps, row):
                out.append(value)
            if n < m and p >= 0:
                groups[p].append(i * rows + n)
    order = [row for group in groups for row in group]
    order += [-1] * (len(maps[0]) - len(order))
    first = np.cumsum([0] + [len(group) for group in groups])
    as32 = [torch.tensor(m, dtype=torch.int32) for m in maps + [order, first.tolist()]]
    return [m.reshape(-1, rows) for m in as32[:4]] + as32[4:]


def exact(case, seed):
    if case["kind"] == "plan":
        return _exact_plan(case, prepare(case, seed))
    if case["kind"] == "sample" and case["rows"] * case["n"] > 60000000:
        return None
    st = prepare(case, seed)
    return _exact_attend(case, st) if case["kind"] == "attend" else _exact_sample(case, st)
