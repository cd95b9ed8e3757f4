"""The operators of a drafted-tree serving step, as measurable cases.

A server that verifies a tree of drafted tokens a session in one step rotates
the tree's queries and keys, appends keys and values to the int8 cache, lets
every node attend to the committed positions and to its ancestors, and picks
from each node's logits under the request's rules:

  rope     rotary positions of a stack of rows
  write    rows appended to the cache, queries and keys rotated on the way,
           then read back
  read     committed positions of the cache as fp32 rows
  tree     attention of every session's drafted tree over its int8 block
  logits   penalties, biases and grammar masks on rows of logits, and the pick

With `own` false `run` computes them in their plain form; with `own` true it
makes the calls of needle-rs_amd/needle_amd.py.  Sizes are the shipped
Needle-3 geometry's (12 query heads on 2 kv heads, qk 48, v 64, 8192 tokens
of vocabulary), the benchmark's 12 x 64 cache, and generic ones.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

HALVES, PAIRS = "halves", "pairs"


def listed():
    v3 = dict(heads=12, kv_heads=2, qk=48)
    mha = dict(heads=12, kv_heads=12, qk=64)
    return [
        # the queries of one session's eight drafted tokens: the smallest call
        dict(name="rope_one", kind="rope", rows=8, heads=12, dim=48, rot=48, layout=HALVES, scaling="plain",
             theta=10000.0, factor=1.0, trained=0, gain=1.0, far=8192),
        # a prompt's queries, interleaved, 48 of 64 elements rotated, stretched past the trained length
        dict(name="rope_prompt", kind="rope", rows=6001, heads=12, dim=64, rot=48, layout=PAIRS, scaling="parts",
             theta=500000.0, factor=8.0, trained=8192, gain=1.125, far=1000000),
        # 64 sessions' trees of 16 nodes appended in one call
        dict(name="write_trees", kind="write", sessions=64, per=16, cap=2111, ctx=2000, rot=48, layout=HALVES,
             scaling="plain", factor=1.0, **v3),
        # eight prompts of 1000 tokens into the 12 x 64 cache
        dict(name="write_prompts", kind="write", sessions=8, per=1000, cap=2048, ctx=1100, rot=64, layout=PAIRS,
             scaling="linear", factor=4.0, **mha),
        # a long conversation handed on: the live window of a wrapped ring, read back
        dict(name="read_ring", kind="read", sessions=16, per=8001, cap=8192, ctx=20000, **v3),
        # one session's tree of eight nodes over a short prompt: latency
        dict(name="tree_one", kind="tree", sessions=1, nodes=8, cap=512, ctx=301, window=0, branch=3,
             quant_query=True, **v3),
        # 64 sessions near 2000 tokens, 16 nodes each
        dict(name="tree_64", kind="tree", sessions=64, nodes=16, cap=2111, ctx=2000, window=0, branch=3,
             quant_query=True, **v3),
        # the same 64 sessions in a windowed layer's wrapped ring, odd trees, fp32 queries
        dict(name="tree_window", kind="tree", sessions=64, nodes=21, cap=1061, ctx=5000, window=1024, branch=2,
             quant_query=False, **v3),
        # 64 sessions of the 12 x 64 cache: the HBM stream
        dict(name="tree_mha", kind="tree", sessions=64, nodes=13, cap=2112, ctx=2048, window=0, branch=4,
             quant_query=False, **mha),
        # one row of logits, a short history, a grammar state: latency
        dict(name="logits_one", kind="logits", rows=1, n=8192, hist=300, biases=8, states=4),
        # 16 nodes of 64 sessions, long histories
        dict(name="logits_trees", kind="logits", rows=1024, n=8192, hist=2000, biases=20, states=40),
        # a large odd vocabulary, rows that are not aligned
        dict(name="logits_wide", kind="logits", rows=200, n=100003, hist=4001, biases=300, states=16),
    ]


# ---- drawn cases ------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "write", "read", "tree", "tree", "tree", "logits", "logits"])
    heads, kv_heads, qk = rng.choice([(12, 2, 48), (12, 2, 48), (12, 12, 64), (8, 4, 64), (16, 2, 64), (5, 1, 48)])
    geom = dict(heads=heads, kv_heads=kv_heads, qk=qk)
    turn = dict(layout=rng.choice([HALVES, PAIRS]), scaling=rng.choice(["plain", "linear", "parts"]))
    if kind == "rope":
        dim = 16 * rng.randint(1, 12)
        heads = _log(rng, 1, 32)
        return dict(kind=kind, rows=_log(rng, 1, max(2, 4600000 // (heads * dim))), heads=heads, dim=dim,
                    rot=2 * rng.randint(1, dim // 2), theta=10.0 ** rng.uniform(3, 6), factor=rng.uniform(1, 32),
                    trained=_log(rng, 1024, 32768), gain=rng.uniform(1, 1.4), far=_log(rng, 64, 1000000), **turn)
    if kind in ("write", "read"):
        sessions = _log(rng, 1, 128)
        per = _log(rng, 1, max(1, min(4000, 6000000 // (kv_heads * (qk + 64) * sessions))))
        cap = per + _log(rng, 1, 1024)
        case = dict(kind=kind, sessions=sessions, per=per, cap=cap, ctx=_log(rng, per, 40000), **geom)
        return case if kind == "read" else dict(case, rot=2 * rng.randint(1, qk // 2), factor=rng.uniform(1, 16), **turn)
    if kind == "tree":
        nodes = _log(rng, 1, 128)
        ctx = _log(rng, 1, 12000)
        window = rng.choice([0, 0, 256, 1024])
        cap = (min(window, ctx) if window else ctx) + nodes + rng.randint(0, 300)
        most = min(2.0e8 / (cap * kv_heads * (qk + 64)), 2.5e7 / (cap * nodes * heads))
        return dict(kind=kind, sessions=_log(rng, 1, max(1, min(128, int(most)))), nodes=nodes, cap=cap, ctx=ctx,
                    window=window, branch=rng.randint(1, 5), quant_query=rng.random() < 0.5, **geom)
    n = 8192 if rng.random() < 0.4 else _log(rng, 300, 150000)
    return dict(kind=kind, rows=_log(rng, 1, max(2, min(4096, 20000000 // n))), n=n, hist=_log(rng, 1, 5000),
                biases=_log(rng, 1, min(300, n)), states=_log(rng, 1, 64))


# ---- sizes that the case alone fixes ----------------------------------------

def _bases(case):
    """Committed positions of each session (ragged) and its rows in this call."""
    i = np.arange(case["sessions"])
    base = case["ctx"] - (i * 37) % (case["ctx"] // 4 + 1)
    return base.astype(np.int32), i


def _tree(case):
    """Per session: committed positions, nodes, each node's first position, and
    the nodes it attends to (its ancestors and itself) as 0/1 [S][N][N]."""
    n, window = case["nodes"], case["window"]
    base, i = _bases(case)
    length = (n - (i * 5) % (n // 4 + 1)).astype(np.int32)
    see = np.zeros((len(i), n, n), np.uint8)
    depth = np.zeros((len(i), n), np.int32)
    for j in range(n):
        if j:
            up = j - 1 - (j * 5 + i * 3) % min(j, case["branch"])
            see[:, j] = see[i, up]
            depth[:, j] = depth[i, up] + 1
        see[:, j, j] = 1
    lo = np.maximum(base[:, None] + depth + 1 - window, 0) if window else np.zeros_like(depth)
    return base, length, lo.astype(np.int32), see


def _words(bits):
    """0/1 [..][n] as 32-bit words, bit t % 32 of word t / 32 (int32 patterns)."""
    n = bits.shape[-1]
    pad = np.zeros(bits.shape[:-1] + (-n % 32,), np.uint8)
    packed = np.packbits(np.concatenate([bits, pad], -1), axis=-1, bitorder="little")
    return np.ascontiguousarray(packed).view(np.int32)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- the cache's bytes -------------------------------------------------------

def _parts(case):
    """Byte offsets of a block's parts (k, v, k scales, v scales) and its size."""
    kvh, cap = case["kv_heads"], case["cap"]
    at = [0]
    for size in (kvh * cap * case["qk"], kvh * cap * 64, 4 * kvh * cap, 4 * kvh * cap):
        at.append(at[-1] + -(-size // 256) * 256)
    return at


def _views(case, kv):
    """The blocks' parts as tensors [S][KVH][cap](..)."""
    at, s, kvh, cap, qk = _parts(case), case["sessions"], case["kv_heads"], case["cap"], case["qk"]
    b = kv.view(s, at[4])
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


def _filled(case, g):
    """Blocks whose every slot holds a quantised N(0, 1) row."""
    at = _parts(case)
    kv = torch.zeros(case["sessions"] * at[4], dtype=torch.uint8, device="cuda")
    k, v, ks, vs = _views(case, kv)
    for part, scales in ((k, ks), (v, vs)):
        codes, scale = _quant(_randn(g, *part.shape))
        part.copy_(codes.to(torch.int8))
        scales.copy_(scale[..., 0])
    return kv


# ---- inputs -----------------------------------------------------------------

def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "rope":
        rows = case["rows"]
        return dict(case=case, x=_randn(g, rows, case["heads"] * case["dim"]),
                    pos=torch.randint(0, case["far"], (rows,), generator=g, device="cuda", dtype=torch.int32))
    if kind in ("write", "read"):
        s, per = case["sessions"], case["per"]
        base, _ = _bases(case)
        st = dict(case=case, kv=_filled(case, g), stride=_parts(case)[4])
        if kind == "read":  # the last `per` committed positions
            first = np.maximum(base - per, 0)
            st["pos"] = _cuda((first[:, None] + np.arange(per)).astype(np.int32).reshape(-1))
            return st
        pos = base[:, None] + np.arange(per)  # slots one after another, angles by depth
        st["pos"] = _cuda(pos.astype(np.int32).reshape(-1))
        st["turn"] = _cuda((base[:, None] + np.arange(per) * 2 // 3).astype(np.int32).reshape(-1))
        h, kvh, qk = case["heads"], case["kv_heads"], case["qk"]
        # one projection's rows: q, k and v side by side
        st["qkv"] = _randn(g, s * per, (h + kvh) * qk + kvh * 64)
        return st
    if kind == "tree":
        base, length, lo, see = _tree(case)
        s, n = lo.shape
        st = dict(case=case, kv=_filled(case, g), stride=_parts(case)[4], base=_cuda(base), length=_cuda(length),
                  lo=_cuda(lo), mask=_cuda(_words(see)))
        st["q"] = 2 * _randn(g, s, n, case["heads"] * case["qk"])
        st["out"] = _randn(g, s, n, case["heads"] * 64)  # rows past a tree's end stay as they are
        return st
    rows, n, hist = case["rows"], case["n"], case["hist"]
    i = torch.arange(rows, device="cuda")
    st = dict(case=case, x=4 * _randn(g, rows, n))
    # tokens repeat: drawn from an eighth of the vocabulary
    st["hist"] = torch.randint(0, max(1, n // 8), (rows, hist), generator=g, device="cuda", dtype=torch.int32)
    st["hist_len"] = (hist - (i * 13) % (hist // 2 + 1)).int()
    st["out_from"] = (st["hist_len"] // 3).int()
    st["repeat"] = 1 + torch.rand(rows, generator=g, device="cuda")
    st["presence"], st["frequency"] = (torch.rand(2, rows, generator=g, device="cuda") * 0.5).unbind(0)
    start = torch.randint(0, n, (rows, 1), generator=g, device="cuda")
    b = torch.arange(case["biases"], device="cuda")
    st["bias_id"] = ((start + b * max(1, n // case["biases"])) % n).int()  # no token twice
    st["bias"] = 4 * _randn(g, rows, case["biases"])
    st["bias_len"] = (case["biases"] - i % (case["biases"] // 2 + 1)).int()
    bits = np.random.default_rng(int(seed)).integers(0, 2, size=(case["states"], n), dtype=np.uint8)
    st["mask"] = _cuda(_words(bits))
    st["mask_row"] = torch.where(i % 3 == 1, -1, i % case["states"]).int()  # some rows have no grammar
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


def _spec(case, nd):
    return nd.rope(case["rot"], theta=case.get("theta", 10000.0), layout=case["layout"], scaling=case["scaling"],
                   factor=case["factor"], trained=case.get("trained", 4096), turns=(1.0, 32.0),
                   gain=case.get("gain", 1.0))


def run(st):
    case = st["case"]
    return {"rope": _run_rope, "write": _run_write, "read": _run_read, "tree": _run_tree,
            "logits": _run_logits}[case["kind"]](case, st)


def _turned(case, x, pos, heads, dim):
    """Rows of heads turned by their positions; angles and products in 64 bits,
    as far positions and codes next to a border need."""
    half = case["rot"] // 2
    e = -2.0 * torch.arange(half, device=x.device, dtype=torch.float64) / case["rot"]
    f = torch.pow(case.get("theta", 10000.0), e)
    if case["scaling"] == "linear":
        f = f / case["factor"]
    if case["scaling"] == "parts":
        turns = f * (case.get("trained", 4096) / (2 * math.pi))
        keep = ((turns - 1.0) / 31.0).clamp(0, 1)
        f = f * (keep + (1 - keep) / case["factor"])
    a = (pos.double()[:, None] * f)[:, None]
    c, s = torch.cos(a), torch.sin(a)
    x = x.reshape(len(pos), heads, dim)
    if case["layout"] == PAIRS:
        u, w = x[..., 0:2 * half:2].double(), x[..., 1:2 * half:2].double()
    else:
        u, w = x[..., :half].double(), x[..., half:2 * half].double()
    u, w = case.get("gain", 1.0) * (u * c - w * s), case.get("gain", 1.0) * (u * s + w * c)
    turned = torch.stack([u, w], -1 if case["layout"] == PAIRS else -2).reshape(len(pos), heads, 2 * half)
    return torch.cat([turned.float(), x[..., 2 * half:]], -1).reshape(len(pos), heads * dim)


def _run_rope(case, st):
    if own:
        nd, ctx = _needle()
        return nd.rope_rows(ctx, _spec(case, nd), st["x"], st["pos"], case["heads"])
    return _turned(case, st["x"], st["pos"], case["heads"], case["dim"])


def _rows_of(case, st):
    """(block, slot) of every row of a write or read."""
    block = torch.arange(st["pos"].numel(), device="cuda") // case["per"]
    return block, st["pos"].long() % case["cap"]


def _read_plain(case, st):
    k, v, ks, vs = _views(case, st["kv"])
    block, slot = _rows_of(case, st)
    return [(part[block, :, slot].float() * scale[block, :, slot][..., None]).reshape(len(slot), -1)
            for part, scale in ((k, ks), (v, vs))]


def _run_write(case, st):
    h, kvh, qk = case["heads"], case["kv_heads"], case["qk"]
    q, k, v = st["qkv"].split([h * qk, kvh * qk, kvh * 64], 1)
    if own:
        nd, ctx = _needle()
        geom = nd.kv_geom(h, kvh, qk, 64, case["cap"])
        q = nd.kv_write_rope(ctx, geom, _spec(case, nd), st["kv"], st["stride"], st["pos"], k, v, q=q,
                             rot_pos=st["turn"], per_block=case["per"])
        return q, nd.kv_read(ctx, geom, st["kv"], st["stride"], st["pos"], per_block=case["per"])
    block, slot = _rows_of(case, st)
    kc, vc, ks, vs = _views(case, st["kv"])
    q = _turned(case, q, st["turn"], h, qk)
    codes, scale = _quant(_turned(case, k, st["turn"], kvh, qk).reshape(-1, kvh, qk))
    kc[block, :, slot], ks[block, :, slot] = codes.to(torch.int8), scale[..., 0]
    codes, scale = _quant(v.reshape(-1, kvh, 64))
    vc[block, :, slot], vs[block, :, slot] = codes.to(torch.int8), scale[..., 0]
    return q, _read_plain(case, st)


def _run_read(case, st):
    if own:
        nd, ctx = _needle()
        geom = nd.kv_geom(case["heads"], case["kv_heads"], case["qk"], 64, case["cap"])
        return nd.kv_read(ctx, geom, st["kv"], st["stride"], st["pos"], per_block=case["per"])
    return _read_plain(case, st)


def _run_tree(case, st):
    h, kvh, qk, n = case["heads"], case["kv_heads"], case["qk"], case["nodes"]
    if own:
        nd, ctx = _needle()
        geom = nd.kv_geom(h, kvh, qk, 64, case["cap"])
        return nd.attend_tree_i8(ctx, geom, st["kv"], st["stride"], st["base"], st["lo"], st["mask"], st["q"],
                                 length=st["length"], quant_query=case["quant_query"], out=st["out"])
    k, v, ks, vs = _views(case, st["kv"])
    s, rep = case["sessions"], h // kvh
    # the last positions of the ring up to the tree's end, oldest first
    back = min(case["cap"], case["ctx"] + n)
    pos = st["base"].long()[:, None] + n - back + torch.arange(back, device="cuda")
    slot = (pos % case["cap"])[:, None, :].expand(s, kvh, back)
    kf = torch.gather(k, 2, slot[..., None].expand(s, kvh, back, qk)).float() * torch.gather(ks, 2, slot)[..., None]
    vf = torch.gather(v, 2, slot[..., None].expand(s, kvh, back, 64)).float() * torch.gather(vs, 2, slot)[..., None]
    node = pos - st["base"].long()[:, None]  # below 0: committed
    at = node.clamp(0, n - 1)[:, None].expand(s, n, back)
    bit = torch.gather(st["mask"], 2, at // 32) >> (at % 32) & 1
    node, pos = node[:, None], pos[:, None]
    sees = torch.where(node < 0, pos >= st["lo"].long()[..., None].clamp(min=0),
                       (bit != 0) & (node < st["length"].long()[:, None, None]))
    q = st["q"].reshape(s, n, h, qk)
    if case["quant_query"]:
        codes, scale = _quant(q)
        q = codes * scale
    q = q.reshape(s, n, kvh, rep, qk).permute(0, 2, 1, 3, 4).reshape(s, kvh, n * rep, qk)
    sees = sees[:, None, :, None].expand(s, 1, n, rep, back).reshape(s, 1, n * rep, back)
    t = (q @ kf.transpose(2, 3)) * (1.0 / math.sqrt(qk))
    t = t.masked_fill(~sees, -math.inf)
    top = t.amax(-1, keepdim=True)
    w = torch.exp(t - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    o = (w @ vf) / torch.where(total == 0, 1.0, total)
    o = o.reshape(s, kvh, n, rep, 64).permute(0, 2, 1, 3, 4).reshape(s, n, h * 64)
    there = torch.arange(n, device="cuda")[None] < st["length"][:, None]
    return torch.where(there[..., None], o, st["out"])


def _run_logits(case, st):
    if own:
        nd, ctx = _needle()
        return nd.logits_adjust(ctx, st["x"], hist=st["hist"], hist_len=st["hist_len"], out_from=st["out_from"],
                                repeat=st["repeat"], presence=st["presence"], frequency=st["frequency"],
                                bias_id=st["bias_id"], bias=st["bias"], bias_len=st["bias_len"], mask=st["mask"],
                                mask_row=st["mask_row"], pick=True)
    x, n, rows = st["x"], case["n"], case["rows"]
    at = torch.arange(case["hist"], device="cuda")[None]
    here = at < st["hist_len"][:, None]
    tok = torch.where(here, st["hist"], n).long()
    new = torch.where(at >= st["out_from"][:, None], tok, n)
    count = torch.zeros(2, rows, n + 1, device="cuda")
    one = torch.ones_like(tok, dtype=torch.float32)
    count[0].scatter_add_(1, tok, one)
    count[1].scatter_add_(1, new, one)
    ever, made = count[0, :, :n] > 0, count[1, :, :n]
    r = st["repeat"][:, None].expand_as(x)
    y = torch.where(ever, torch.where(x > 0, torch.div(x, r), x * r), x)
    y = y - made * st["frequency"][:, None]
    y = y - torch.where(made > 0, st["presence"][:, None], 0.0)
    there = torch.arange(case["biases"], device="cuda")[None] < st["bias_len"][:, None]
    bias = torch.zeros(rows, n + 1, device="cuda")
    bias.scatter_(1, torch.where(there, st["bias_id"], n).long(), st["bias"])
    y = y + bias[:, :n]
    t = torch.arange(n, device="cuda")
    bit = st["mask"][st["mask_row"].clamp(min=0).long()][:, t // 32] >> (t % 32) & 1
    y = torch.where((bit != 0) | (st["mask_row"] < 0)[:, None], y, -math.inf)
    top = y.amax(1, keepdim=True)
    first = torch.where(y == top, t[None], n).amin(1)
    return y, torch.where(top[:, 0] == -math.inf, -1, first).int()


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "rope":
        values = case["rows"] * case["heads"] * case["dim"]
        turned = case["rows"] * case["heads"] * case["rot"]
        return dict(bytes=8 * values + 4 * case["rows"], flops=3 * turned)
    if kind in ("write", "read"):
        rows, h, kvh, qk = case["sessions"] * case["per"], case["heads"], case["kv_heads"], case["qk"]
        cached, scales = kvh * (qk + 64), 8 * kvh
        if kind == "read":
            return dict(bytes=rows * (5 * cached + scales + 4), flops=rows * cached)
        return dict(bytes=rows * (8 * h * qk + 4 * cached + cached + scales + 8 + 4 * cached),
                    flops=rows * (3 * (h + kvh) * case["rot"] + 3 * cached))
    if kind == "tree":
        base, length, lo, see = _tree(case)
        h, kvh, qk = case["heads"], case["kv_heads"], case["qk"]
        there = np.arange(case["nodes"])[None] < length[:, None]
        first = np.where(there, np.minimum(lo, base[:, None]), base[:, None]).min(1)
        span = int((base + length - first).sum())
        pairs = int((np.maximum(base[:, None] - lo, 0) * there).sum()) + int((see * there[..., None]).sum())
        rows = int(length.sum())
        return dict(bytes=span * kvh * (qk + 64 + 8) + 4 * rows * (h * (qk + 64) + 1 + see.shape[2] // 32 + 1),
                    flops=2 * pairs * h * (qk + 64))
    rows, n = case["rows"], case["n"]
    some = min(case["states"], rows)
    return dict(bytes=8 * rows * n + rows * (4 * case["hist"] + 8 * case["biases"] + 40) + some * (-(-n // 32)) * 4,
                flops=3 * rows * n)


# ---- the same in 64 bits ----------------------------------------------------

def _exact_turned(case, x, pos, heads, dim):
    """Each pair as a complex number times gain e^(i pos f)."""
    rot, theta = case["rot"], case.get("theta", 10000.0)
    freq = []
    for j in range(rot // 2):
        f = theta ** (-2.0 * j / rot)
        if case["scaling"] == "linear":
            f /= case["factor"]
        elif case["scaling"] == "parts":
            keep = min(max((case.get("trained", 4096) * f / (2 * math.pi) - 1.0) / 31.0, 0.0), 1.0)
            f *= keep + (1 - keep) / case["factor"]
        freq.append(f)
    angle = pos.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
    x = x.double().reshape(len(pos), heads, dim).clone()
    j = torch.arange(rot // 2, device="cuda")
    a, b = (2 * j, 2 * j + 1) if case["layout"] == PAIRS else (j, j + rot // 2)
    z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.full_like(angle, case.get("gain", 1.0)), angle)
    x[..., a], x[..., b] = z.real, z.imag
    return x.reshape(len(pos), heads * dim)


def _stands_for(x, width):
    """What the cache holds of rows of heads: codes (by 32-bit steps) times scale."""
    codes, scale = _quant(x.float().reshape(len(x), -1, width))
    return (codes.double() * scale.double()).reshape(len(x), -1)


def _exact_tree(case, st):
    k, v, ks, vs = _views(case, st["kv"])
    base, length, lo, see = _tree(case)
    h, kvh, qk, n = case["heads"], case["kv_heads"], case["qk"], case["nodes"]
    out = st["out"].double()
    for i in range(case["sessions"]):
        b, m = int(base[i]), int(length[i])
        first = int(lo[i, :m].min())
        slot = torch.arange(min(first, b), b + m, device="cuda") % case["cap"]
        kd = k[i][:, slot].double() * ks[i][:, slot, None].double()
        vd = v[i][:, slot].double() * vs[i][:, slot, None].double()
        q = st["q"][i, :m].reshape(m, h, qk)
        if case["quant_query"]:
            codes, scale = _quant(q)
            q = codes.double() * scale.double()
        old = torch.arange(min(first, b), b, device="cuda")[None] >= _cuda(lo[i, :m])[:, None]
        sees = torch.cat([old, _cuda(see[i, :m, :m]) != 0], 1)
        q = q.double().transpose(0, 1)
        t = torch.matmul(q, kd.repeat_interleave(h // kvh, 0).transpose(1, 2).contiguous()) / math.sqrt(qk)
        w = torch.softmax(t.masked_fill(~sees[None], -math.inf), -1)
        out[i, :m] = torch.matmul(w, vd.repeat_interleave(h // kvh, 0)).transpose(0, 1).reshape(m, -1)
    return out


def _exact_logits(case, st):
    rows, n = case["rows"], case["n"]
    y = st["x"].double()
    hist, bias_id = st["hist"].cpu().numpy(), st["bias_id"].cpu().numpy()
    ends, starts, biases = (st[k].tolist() for k in ("hist_len", "out_from", "bias_len"))
    made = np.zeros((rows, n), np.int64)
    ever = np.zeros((rows, n), bool)
    for i in range(rows):
        ever[i, hist[i, :ends[i]]] = True
        made[i] = np.bincount(hist[i, starts[i]:ends[i]], minlength=n)
    made, ever = _cuda(made), _cuda(ever)
    r = st["repeat"].double()[:, None]
    y = torch.where(ever, torch.where(y > 0, y / r, y * r), y)
    y = y - made * st["frequency"].double()[:, None] - (made > 0) * st["presence"].double()[:, None]
    for i in range(rows):
        m = biases[i]
        y[i, _cuda(bias_id[i, :m]).long()] += st["bias"][i, :m].double()
    bits = np.unpackbits(st["mask"].cpu().numpy().view(np.uint8), axis=-1, bitorder="little")[:, :n]
    banned = (_cuda(bits)[st["mask_row"].clamp(min=0).long()] == 0) & (st["mask_row"] >= 0)[:, None]
    return y.masked_fill(banned, -math.inf), None


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "rope":
        return _exact_turned(case, st["x"], st["pos"], case["heads"], case["dim"])
    if kind == "write":
        h, kvh, qk = case["heads"], case["kv_heads"], case["qk"]
        q, k, v = st["qkv"].split([h * qk, kvh * qk, kvh * 64], 1)
        k = _exact_turned(case, k, st["turn"], kvh, qk)
        return _exact_turned(case, q, st["turn"], h, qk), [_stands_for(k, qk), _stands_for(v, 64)]
    if kind == "read":
        k, v, ks, vs = _views(case, st["kv"])
        block, slot = _rows_of(case, st)
        return [(part.double() * scale.double()[..., None])[block, :, slot].reshape(len(slot), -1)
                for part, scale in ((k, ks), (v, vs))]
    return _exact_tree(case, st) if kind == "tree" else _exact_logits(case, st)
