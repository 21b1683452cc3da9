"""Attention over the paged cache where its lengths or its scores are large: contexts
beyond 65536 rows, bounds on the lengths that take the other form of a call, and scores
of which one wins.  Against the definition in 64 bits (paged_ref.attend and its bound)."""
import math

import numpy as np
import pytest
import torch

import moe_infer_amd as m

from .gpu_util import announce
from .test_gpu_paged import D, LENS, Pool, f64, gen, i32, near, poison_tail, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,G", [(16, 2), (8, 1), (32, 8), (4, 4), (15, 3), (16, 1), (7, 1)])
def test_a_larger_bound_takes_another_form(H, G):
    """The same lengths with bounds that give a workgroup an item, split it in chunks, and cut
    the line of all tiles; each form repeats its own bits."""
    announce(f"{H}/{G}")
    pool = Pool(H * 17 + G, LENS, G=G)
    poison_tail(pool, LENS)
    q = randn(gen(1), len(LENS), H, D)
    ref, limit = pool.reference(q, [1] * len(LENS))
    for bound in (300, 5000, 1 << 20):
        out = m.attn_decode_paged(pool.pages, pool.t, pool.len, q, bound)
        near(out, ref, limit, f"bound {bound}")
        assert torch.equal(out, m.attn_decode_paged(pool.pages, pool.t, pool.len, q, bound))


@pytest.mark.parametrize("new", [1, 2, 9])
def test_one_row_wins(new):
    """Scores to some thousands: where the best is well ahead of the second, the output is its
    row of V.  A score is off by 256 * 2^-24 of its absolute sum (ds) at most, so a row that
    is 2 ds + 30 behind weighs less than e^-30 of the best and all of them less than 2^-30.
    The best's own weight is 2^(x - m) for a reference m that is up to 8 below it, or a
    rounded x itself, so it is no power of two: its product is off by f16's half step of it, 2^-11,
    while the sum holds it in f32, and the output rounds by 2^-11 again."""
    lens = [70, 300, 1500]
    pool = Pool(2, lens)
    q = 1000 * randn(gen(3), new * len(lens), 16, D)
    cu = i32(np.arange(0, new * len(lens) + 1, new))
    checked = 0
    for bound in (1500, 1 << 24):
        out = f64(m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, q, new, bound))
        assert np.all(np.isfinite(out))
        for s, rows in enumerate(lens):
            for h in range(16):
                k, v = pool.seq(s, h // 8)
                for i in range(new):
                    seen = rows - new + i + 1
                    x = f64(q[s * new + i, h])
                    score = k[:seen] @ x / math.sqrt(D)
                    ds = (np.abs(k[:seen]) @ np.abs(x)).max() / math.sqrt(D) * 256 * 2.0 ** -24
                    best, second = np.argmax(score), np.partition(score, -2)[-2]
                    if score[best] - second < 2 * ds + 30:
                        continue
                    limit = (2 * 2.0 ** -11 + 2.0 ** -20) * np.abs(v[best]) + 2.0 ** -29 * np.abs(v[:seen]).max() + 2.0 ** -25
                    near(out[s * new + i, h], v[best], limit, f"sequence {s} token {i} head {h}")
                    checked += 1
    assert checked > 0.8 * 2 * 16 * new * len(lens)


@pytest.mark.parametrize("new", [1, 3, 20])
def test_long_contexts(new):
    lens = [70001, 45]
    announce(f"{new} tokens behind {lens}")
    pool = Pool(4, lens, page_rows=256)
    poison_tail(pool, lens)
    g = gen(5)
    q, gate = 3 * randn(g, 2 * new, 16, D), randn(g, 2 * new, 16, D)
    ref, limit = pool.reference(q, [new, new], gate)
    out = m.attn_prefill_paged(pool.pages, pool.t, pool.len, i32([0, new, 2 * new]), q, new, 70001, gate=gate)
    near(out, ref, limit, "long")
