"""Values at the end of f16's range in the paged 4-bit cache."""
import numpy as np
import pytest
import torch

import moe_infer_amd as m

from . import paged_ref as R
from .gpu_util import announce
from .test_gpu_paged import D, Pool, f64, gen, i32, near, poison_tail, randn

pytestmark = pytest.mark.gpu


def cu_of(new):
    return i32(np.concatenate([[0], np.cumsum(new)]))


# ----------------------------------------------------------------- append --

def stored(x):
    """What 4 bits keep of x [n, 64] (f64): paged_ref's rule, with an offset that leaves code
    15 within f16, and no group with a value past it."""
    lo, hi = x.min(1, keepdims=True), x.max(1, keepdims=True)
    with np.errstate(all="ignore"):
        s = ((hi - lo) / 15).astype(np.float16).astype(np.float64)
        o = (lo - 16 * s).astype(np.float16).astype(np.float64)
        most = 65504 - 31 * s
        step = 2.0 ** (np.maximum(np.frexp(most)[1], -13) - 11)
        o = np.where(31 * s + o >= 65520, np.floor(most / step) * step, o)
        code = np.clip(np.where(s > 0, np.rint((x - o) / s) - 16, 0), 0, 15)
        val = ((16 + code) * s + o).astype(np.float16)
    return np.where((hi < 65520) & (np.abs(o) < 65520), val, np.float16(np.nan)), s


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ragged", [False, True])
def test_finite_values_read_back_finite(dtype, ragged):
    """Groups whose largest value is among f16's last: the nearest code of one scale and
    offset may stand for a value past 65504.  Off by half a step at most, but for
    the ends of the range: the least code stands for 16 scales past an offset that is rounded
    by 16 at most, the largest for 65504 less the offset's step of 32 at most (and a value
    may be 65520), and the value itself is rounded by 16."""
    announce(f"large values {dtype} {ragged}")
    rng = np.random.default_rng(1)
    n = 40
    lo = np.exp(rng.uniform(np.log(2200), np.log(65000), (n, 2, 4, 1)))
    hi = rng.uniform(np.maximum(lo, 64000), 65519, lo.shape)
    x = lo + (hi - lo) * rng.random((n, 2, 4, 64))
    x[..., 0], x[..., 1] = lo[..., 0], hi[..., 0]
    x[0, :, :, :] = 60000.0
    x[0, :, :, 7] = 65504.0
    if dtype == torch.float32:
        x[1, 0, 0, 9], x[2, 1, 3, 20] = 65520.0, 80000.0  # not in f16's range: their groups are no numbers
    if dtype == torch.bfloat16:
        x = np.minimum(x, 65280.0)
    k = torch.from_numpy(x.reshape(n, 2, D)).to(dtype).cuda()
    k = torch.where(k.isinf(), torch.full_like(k, 65504.0), k)
    v = -k.flip(0)
    v[3, 1, 70] = k[5, 0, 11]  # a group from one end of the range to the other
    pool = Pool(2, [1] * n if not ragged else [n], fill=False)
    cu = cu_of([n]) if ragged else None
    m.paged_append(pool.pages, pool.t, pool.len, k, v, cu_q=cu)
    # (most groups of v have an offset past f16, 16 scales below their least value)
    for name, got, src in zip("kv", m.paged_read(pool.pages, pool.t, pool.len, cu, n), (k, v)):
        src = f64(src).reshape(-1, 64)
        want, s = stored(src)
        got = f64(got).reshape(-1, 64)
        assert np.array_equal(got, want.astype(np.float64), equal_nan=True), name
        fine = ~np.isnan(want).any(1)
        assert np.all(np.isfinite(got[fine])) and (name == "v" or fine.mean() > 0.95)
        assert np.all(np.abs(got - src)[fine] <= (np.maximum(0.5 * s, 64) + 16)[fine]), name


# -------------------------------------------------------------- attention --

def large_group(pool, s, row, head, group, col):
    """V of a row's group: 16 scales of 1000 past 40000, but for column `col`, 31 of them."""
    page, t, w = pool.table[s][row // pool.page_rows], row % pool.page_rows // 32, row % 32
    tile = pool.host[page, head, t]
    h, words = tile.view(np.float16), tile.view(np.uint32)
    so = R.V_SO[w][64 * group]
    h[so], h[so + 8] = 1000.0, 40000.0
    for c in range(64 * group, 64 * group + 64):
        word, nib = R.V_WORD[w][c], int(R.V_NIB[w][c])
        words[word] = np.uint32((int(words[word]) & ~(15 << (4 * nib))) | ((15 << (4 * nib)) if c == col else 0))


@pytest.mark.parametrize("new,past", [(2, 62), (3, 62), (16, 56), (60, 40), (100, 40), (100, 3000)])
def test_large_values_do_not_reach_those_before_them(new, past):
    """A value past f16's range in a row that the later tokens see and the earlier do not: its
    scale and offset are finite, its product with a weight of 0 is not."""
    announce(f"{new} tokens behind {past}")
    lens = [new + past, 70]
    pool = Pool(3, lens, page_rows=32)
    poison_tail(pool, lens)
    q = randn(gen(4), new + 2, 16, D)
    ref, limit = pool.reference(q, [new, 2])
    row, group, col = past + new - 1 if new < 16 else past + new // 2, 2, 2 * 64 + 5
    seen = row - past
    large_group(pool, 0, row, 1, group, col)
    pool.put()
    for bound in (max(lens), 1 << 24):
        out = f64(m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu_of([new, 2]), q, new, bound))
        near(out[:seen], ref[:seen], limit[:seen], "tokens before it")
        near(out[:, :8], ref[:, :8], limit[:, :8], "the other KV head")
        near(out[new:], ref[new:], limit[new:], "the other sequence")
        rest = np.r_[0:128, 192:256]
        near(out[seen:new, 8:][..., rest], ref[seen:new, 8:][..., rest], limit[seen:new, 8:][..., rest], "other groups")
        assert not np.any(np.isfinite(out[seen:new, 8:, col])), "tokens that see it"


@pytest.mark.parametrize("bound", [100, 6000])  # an item to a workgroup, and split
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_without_keys_are_zero_whatever_their_gate(bound, dtype):
    """A padded batch: empty sequences and tokens without a row, whose gates nobody wrote."""
    lens, new = [0, 70, 3, 64], [2, 2, 5, 200]
    pool = Pool(5, [0, 70, 3, 64])
    g = gen(6)
    for count in (1, 2, 5, 200):
        take = [min(a, count) for a in new]
        n = sum(take)
        q, gate = randn(g, n, 16, D), randn(g, n, 16, D, dtype=dtype)
        first = np.concatenate([[r - a + i for i in range(a)] for r, a in zip(lens, take)])
        none = torch.from_numpy(first < 0).cuda()
        gate[none] = float("nan")
        out = f64(m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu_of(take), q, count, bound, gate=gate))
        gate[none] = 0.0
        ref, limit = pool.reference(q, take, gate)
        near(out, ref, limit, f"at most {count} tokens")
        assert np.all(out[first < 0] == 0)
