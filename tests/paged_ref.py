"""The paged 4-bit cache and the rotary positions in plain numpy, 64 bits: what
the operators of moe_infer_amd.paged compute, from their definitions."""
import math

import numpy as np

D, ROWS, TILE = 256, 32, 9216

_r, _c = np.meshgrid(np.arange(ROWS), np.arange(D), indexing="ij")
_sub, _m, _g = _r // 16, _r % 16, _c // 64
# byte-free addresses within a tile: word and nibble of a code, halves of the scales
K_WORD = ((2 * _sub + _g // 2) * 64 + 16 * (_c // 16 % 4) + _m) * 4 + 2 * (_g % 2) + _c // 8 % 2
K_NIB = _c % 8
V_WORD = 1024 + (64 * _g + 16 * (_m // 4) + _c % 64 // 4) * 4 + _c % 4
V_NIB = _m % 4 + 4 * _sub
K_SO = 4096 + 2 * (4 * _r + _g)
V_SO = 4352 + (4 * _g + _m // 4) * 16 + 2 * (_m % 4) + _sub


def tile_rows(tile):
    """(K, V) [32, 256] f64 of one tile's 9216 bytes."""
    w, h = tile.view(np.uint32).astype(np.int64), tile.view(np.float16).astype(np.float64)
    out = []
    with np.errstate(invalid="ignore", over="ignore"):
        for word, nib, so, step in ((K_WORD, K_NIB, K_SO, 1), (V_WORD, V_NIB, V_SO, 8)):
            code = (w[word] >> (4 * nib)) & 15
            out.append(((16 + code) * h[so] + h[so + step]).astype(np.float16).astype(np.float64))
    return out


def sequence_rows(pages, table_row, rows, head):
    """(K, V) [rows, 256] of a sequence's first rows; NaN where a page is not there."""
    per = pages.shape[2]
    ks, vs = [], []
    for t in range(-(-rows // ROWS)):
        j = t // per
        page = int(table_row[j]) if j < len(table_row) else -1
        if 0 <= page < pages.shape[0]:
            k, v = tile_rows(pages[page, head, t % per])
        else:
            k = v = np.full((ROWS, D), np.nan)
        ks.append(k)
        vs.append(v)
    if not ks:
        return np.zeros((0, D)), np.zeros((0, D))
    return np.concatenate(ks)[:rows], np.concatenate(vs)[:rows]


def rotated(x, pos, rope, norm_w=None, eps=1e-6):
    """x [n, heads, 256] (f64) normed and rotated at pos [n]."""
    x = np.asarray(x, np.float64)
    if norm_w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(norm_w, np.float64)
    y, rot = x.copy(), rope.rotary_dim
    t = np.asarray(pos, np.float64)[:, None, None] * np.asarray(rope.frequencies)
    if rope.layout == "half":
        ia, ib = np.arange(rot // 2), rot // 2 + np.arange(rot // 2)
    else:
        ia, ib = np.arange(0, rot, 2), np.arange(1, rot, 2)
    a, b = x[..., ia], x[..., ib]
    y[..., ia] = rope.factor * (a * np.cos(t) - b * np.sin(t))
    y[..., ib] = rope.factor * (b * np.cos(t) + a * np.sin(t))
    return y


def quantised(x):
    """(values f16, distance of the nearest code border in codes) of x [..., 256] f64."""
    g = np.asarray(x, np.float64).reshape(-1, 64)
    with np.errstate(all="ignore"):
        lo, hi = g.min(1, keepdims=True), g.max(1, keepdims=True)
        s = ((hi - lo) / 15).astype(np.float16).astype(np.float64)
        o = (lo - 16 * s).astype(np.float16).astype(np.float64)
        pos = np.where(s > 0, (g - o) / s - 16, 0.0)
        code = np.clip(np.rint(pos), 0, 15)
        val = ((16 + code) * s + o).astype(np.float16)
        bad = ~(np.isfinite(g).all(1, keepdims=True) & np.isfinite(s) & np.isfinite(o))
        border = np.abs(pos - np.floor(pos) - 0.5)
    val = np.where(bad, np.float16(np.nan), val)
    border = np.where(bad | (pos < -0.4) | (pos > 15.4), 1.0, border)
    return val.reshape(np.shape(x)), border.reshape(np.shape(x))


def attend(q, k, v, first, gate=None):
    """(out, bound) [n, R, 256] f64 of q [n, R, 256] over k, v [rows, 256], token i
    seeing rows 0 .. first + i.  bound: how far an f16 kernel's output may be:
      weights in f16 for the product: half a step, 2^-11 of each, and 2^-25 of the
        largest where they are subnormal;
      scores and exponentials in f32: a dot of 256 products is off by 256 * 2^-24 of
        its absolute sum at most, a weight by twice that and 2^-16 (scores to 2^6 in
        base 2, times 2^-23; the exponential's last bits; the sums');
      the output's own rounding, 2^-11, after a gate that is off by 2^-20 of itself."""
    q, n = np.asarray(q, np.float64), len(q)
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        rows = first + i + 1
        if rows <= 0:
            continue
        kk, vv = k[:rows], v[:rows]
        s = q[i] @ kk.T / math.sqrt(D)
        ds = (np.abs(q[i]) @ np.abs(kk).T).max() / math.sqrt(D) * 256 * 2.0 ** -24
        p = np.exp(s - s.max(-1, keepdims=True))
        total = p.sum(-1, keepdims=True)
        out[i] = p / total @ vv
        bound[i] = (p / total @ np.abs(vv)) * (2.0 ** -11 + 2.0 ** -16 + 2 * ds) + \
            2.0 ** -25 * np.abs(vv).sum(0) / total
    if gate is not None:
        sg = 1 / (1 + np.exp(-np.asarray(gate, np.float64)))
        out, bound = out * sg, bound * sg + np.abs(out * sg) * 2.0 ** -20
    return out, bound + np.abs(out) * 2.0 ** -11 + 2.0 ** -25
