"""Plain 64-bit forms of the drafted-tree operators, for their tests (numpy)."""
import numpy as np


def freqs(rot, theta=10000.0, scaling="plain", factor=1.0, trained=0, turns=(1.0, 32.0)):
    f = np.array([theta ** (-2.0 * j / rot) for j in range(rot // 2)])
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        g = np.clip((trained * f / (2 * np.pi) - turns[0]) / (turns[1] - turns[0]), 0, 1)
        f = f * (g + (1 - g) / factor)
    return f


def turned(x, pos, f, layout, gain=1.0):
    """x [rows][heads][dim] turned by pos [rows], in 64 bits."""
    y = np.array(x, np.float64)
    half = len(f)
    j = np.arange(half)
    a, b = (2 * j, 2 * j + 1) if layout == "pairs" else (j, j + half)
    z = (y[..., a] + 1j * y[..., b]) * (gain * np.exp(1j * np.asarray(pos, np.float64)[:, None, None] * f))
    y[..., a], y[..., b] = z.real, z.imag
    return y


def stand_for(x):
    """(codes, scales) of the rows of the last axis, by the cache's 32-bit steps."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(-1)
    scale = np.where(top > 0, top / np.float32(127), np.float32(1)).astype(np.float32)
    y = x * (np.float32(1) / scale)[..., None]
    r = np.sign(y) * np.floor(np.abs(y.astype(np.float64)) + 0.5)
    return np.clip(r, -128, 127).astype(np.int8), scale


def attend(q, k, v, sees, scale):
    """q [H][QK], k [P][KVH][QK], v [P][KVH][VD], sees [P]: [H][VD] in 64 bits."""
    H, KVH = q.shape[0], k.shape[1]
    out = np.zeros((H, v.shape[2]))
    at = np.flatnonzero(sees)
    if not len(at):
        return out
    for h in range(H):
        kk, vv = k[at, h // (H // KVH)].astype(np.float64), v[at, h // (H // KVH)].astype(np.float64)
        s = kk @ q[h].astype(np.float64) * scale
        w = np.exp(s - s.max())
        out[h] = (w / w.sum()) @ vv
    return out


def bits_of(words, n):
    """0/1 [..][n] of words [..][ceil(n / 32)]."""
    w = np.ascontiguousarray(words).view(np.uint8)
    return np.unpackbits(w, axis=-1, bitorder="little")[..., :n]


def words_of(bits):
    bits = np.asarray(bits, np.uint8)
    pad = np.zeros(bits.shape[:-1] + (-bits.shape[-1] % 32,), np.uint8)
    return np.ascontiguousarray(np.packbits(np.concatenate([bits, pad], -1), axis=-1, bitorder="little")).view(np.int32)
