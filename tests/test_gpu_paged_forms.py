"""The forms that attention over the paged cache takes, each against the definition
in 64 bits (paged_ref.attend and its bound) at the sizes where it is taken: one
workgroup to an item and split walks of decode steps, short and long blocks of
prompts, blocks whose keys several workgroups share; and what must not depend on
the form: unseen rows, lost pages, replays of a captured call."""
import numpy as np
import pytest
import torch

import moe_infer_amd as m
from moe_infer_amd.paged import TILE_BYTES

from . import paged_ref as R
from .gpu_util import announce
from .test_gpu_paged import D, Pool, f64, gen, i32, near, poison_tail, randn

pytestmark = pytest.mark.gpu


def cu_of(new):
    return i32(np.concatenate([[0], np.cumsum(new)]))


@pytest.mark.parametrize("tokens", [1, 3])
@pytest.mark.parametrize("bound", [400, 6000])  # an item to a workgroup, and split
def test_decode_forms(tokens, bound):
    lens = [300, 400, 3, 129, 256, 31, 370, 65]
    announce(f"{tokens} tokens of {lens}, bound {bound}")
    pool = Pool(1, lens)
    poison_tail(pool, lens)
    new, g = [tokens] * len(lens), gen(2)
    q, gate = randn(g, sum(new), 16, D), randn(g, sum(new), 16, D)
    out = m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu_of(new), q, tokens, bound, gate=gate)
    ref, limit = pool.reference(q, new, gate)
    near(out, ref, limit, "lengths")
    # lost pages, lengths that cannot be, an empty sequence
    pool.table[3, 1], pool.table[6, 5] = -1, pool.num
    bad = list(lens)
    bad[0], bad[1], bad[2] = -5, bound + 1, 0
    out = f64(m.attn_prefill_paged(pool.pages, i32(pool.table), i32(bad), cu_of(new), q, tokens, bound,
                                   gate=gate)).reshape(len(lens), tokens, -1)
    assert np.all(np.isnan(out[[0, 1, 3, 6]])) and np.all(out[2] == 0)
    near(out[[4, 5, 7]], ref.reshape(out.shape)[[4, 5, 7]], limit.reshape(out.shape)[[4, 5, 7]], "the others")


@pytest.mark.parametrize("G,R_", [(2, 8), (1, 16), (3, 5)])
def test_decode_forms_agree_for_many(G, R_):
    """More sequences than a workgroup has threads, with both bounds."""
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 120, 600).tolist()
    pool = Pool(4, lens, G=G, page_rows=32)
    q = randn(gen(5), 600, G * R_, D)
    ref, limit = pool.reference(q, [1] * 600)
    for bound in (120, 30000):
        near(m.attn_decode_paged(pool.pages, pool.t, pool.len, q, bound), ref, limit, f"bound {bound}")


@pytest.mark.parametrize("H,G", [(16, 2), (16, 1), (9, 3), (4, 4)])
@pytest.mark.parametrize("rows", [128, 129, 256, 300])  # of the longest sequence, a KV head
@pytest.mark.parametrize("past", [0, 2500])
def test_prompt_forms(H, G, rows, past):
    ratio = H // G
    new = [-(-rows // ratio), 1, 7]
    lens = [new[0] + past, 1 + past // 3, 7]
    announce(f"{H}/{G}: {new} behind {past}")
    pool = Pool(6, lens, G=G, page_rows=32)
    poison_tail(pool, lens)
    g = gen(7)
    q, gate = randn(g, sum(new), H, D), randn(g, sum(new), H, D)
    ref, limit = pool.reference(q, new)
    for bound in (max(lens), 1 << 24):  # the size of a call goes by its bounds
        near(m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu_of(new), q, max(new), bound), ref, limit, "no gate")
    for gt in (gate, gate.float()):
        ref, limit = pool.reference(q, new, gt)
        out = m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu_of(new), q, max(new), max(lens), gate=gt)
        near(out, ref, limit, f"gate {gt.dtype}")
        again = m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu_of(new), q, max(new), max(lens), gate=gt)
        assert torch.equal(out, again)


def test_prompts_of_many_sequences():
    """More sequences than shares, of 0 to 40 tokens, some with more tokens than rows."""
    rng = np.random.default_rng(8)
    new = rng.integers(0, 41, 330).tolist()
    past = rng.integers(-3, 90, 330).tolist()
    lens = [max(0, a + b) for a, b in zip(new, past)]
    pool = Pool(9, lens, G=1, page_rows=32)
    q = randn(gen(10), sum(new), 8, D)
    ref, limit = pool.reference(q, new)
    for bound in (max(lens), 1 << 24):
        out = m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu_of(new), q, 40, bound)
        near(out, ref, limit, f"330 sequences, bound {bound}")


def test_prompts_beside_what_is_refused():
    """Sequences that give NaN (lengths that cannot be, too many tokens, a lost page far
    from a block's first piece) and empty ones leave the others as they are."""
    new = [70, 40, 33, 0, 64, 50]
    lens = [5000, 40, 900, 700, 64, 3000]
    pool = Pool(11, lens)
    q = randn(gen(12), sum(new), 16, D)
    ref, limit = pool.reference(q, new)
    at = np.concatenate([[0], np.cumsum(new)])
    pool.table[0, 70] = -1       # rows 4480 ..
    table, kv = i32(pool.table), i32([5000, -1, 900, 700, 64, 6000])
    out = f64(m.attn_prefill_paged(pool.pages, table, kv, cu_of(new), q, 70, 5000))
    for s, gone in enumerate([True, True, False, False, False, True]):
        got = out[at[s]:at[s + 1]]
        if gone:
            assert np.all(np.isnan(got)), s
        elif new[s]:
            near(got, ref[at[s]:at[s + 1]], limit[at[s]:at[s + 1]], f"sequence {s}")
    out = f64(m.attn_prefill_paged(pool.pages, table, kv, cu_of(new), q, 45, 5000))
    for s, gone in enumerate([True, True, False, False, True, True]):
        assert np.all(np.isnan(out[at[s]:at[s + 1]])) if gone else np.all(np.isfinite(out[at[s]:at[s + 1]])), s


def test_prompts_behind_values_that_are_not_numbers():
    """A V scale that is not finite in a row that a long block's later tokens see and its
    earlier do not.  (An infinite one, which no append writes: the weighted sum is infinite,
    or not a number in a tile that a mask cuts, and finite nowhere.)"""
    new, lens = [60], [4060]
    pool = Pool(13, lens)
    q = randn(gen(14), 60, 16, D)
    ref, limit = pool.reference(q, new)
    h = pool.host.view(np.float16)
    row = 4030
    h[pool.table[0, row // 64], 1, row % 64 // 32, R.V_SO[row % 32][0]] = np.inf
    pool.put()
    out = f64(m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu_of(new), q, 60, 4060))
    near(out[:30], ref[:30], limit[:30], "tokens that do not see it")
    near(out[:, :8], ref[:, :8], limit[:, :8], "the other KV head")
    assert not np.any(np.isfinite(out[30:, 8:, :64]))
    near(out[30:, 8:, 64:], ref[30:, 8:, 64:], limit[30:, 8:, 64:], "the other groups")


def test_captured_prompts_share_a_workspace():
    """Two captured calls of both forms, in turn over one workspace, as the program moves
    the lengths on and cuts the blocks elsewhere; eager work in between."""
    big = [9000, 700]
    pool = Pool(15, big)
    kv, g = i32([2100, 200]), gen(16)
    long, short = [100, 200], [9, 16]
    q1, q2 = randn(g, 300, 16, D), randn(g, 25, 16, D)
    c1, c2 = cu_of(long), cu_of(short)
    ws = m.paged_workspace(2, 300, 200, 9000)
    o1, o2 = torch.empty_like(q1), torch.empty_like(q2)

    def both(a, b, w):
        m.attn_prefill_paged(pool.pages, pool.t, kv, c1, q1, 200, 9000, out=a, workspace=w)
        m.attn_prefill_paged(pool.pages, pool.t, kv, c2, q2, 16, 9000, out=b, workspace=w)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both(o1, o2, ws)
    torch.cuda.current_stream().wait_stream(s)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        both(o1, o2, ws)
    with torch.cuda.graph(g2):
        both(o1, o2, ws)
    for i, rows in enumerate([(2100, 200), (9000, 700), (100, 201), (4097, 640)]):
        kv.copy_(i32(rows))
        q1.copy_(randn(g, 300, 16, D))
        o1.zero_(), o2.zero_()
        (g1 if i % 2 else g2).replay()
        torch.cuda.synchronize()
        w1, w2 = torch.empty_like(q1), torch.empty_like(q2)
        both(w1, w2, m.paged_workspace(2, 300, 200, 9000))
        assert torch.equal(o1, w1) and torch.equal(o2, w2), f"replay {i}"
        pool.rows = list(rows)
        for q, new, o in ((q1, long, o1), (q2, short, o2)):
            ref, limit = pool.reference(q, new)
            near(o, ref, limit, f"replay {i}")


def test_prompts_of_pages_past_32_bits():
    """Both forms over a pool of more than 4 GiB whose last pages they read."""
    per = 2 * 2 * TILE_BYTES
    num = (1 << 32) // per + 40
    pages = torch.empty((num, 2, 2, TILE_BYTES), dtype=torch.uint8, device="cuda")
    pool = Pool(17, [150], spare=0)
    table = np.array([[num - 1, num - 5, num - 2]], np.int32)
    for j in range(3):
        pages[table[0, j]] = pool.pages[pool.table[0, j]]
    for n in (10, 60):
        q = randn(gen(18 + n), n, 16, D)
        want = m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu_of([n]), q, n, 150)
        assert torch.equal(m.attn_prefill_paged(pages, i32(table), pool.len, cu_of([n]), q, n, 150), want)
    del pages


def test_two_prompts_at_once():
    """Calls on two streams, each with its own workspace, over the same pages."""
    pool = Pool(19, [3000, 2500])
    new = [90, 33]
    cu, g = cu_of(new), gen(20)
    qs = [randn(g, sum(new), 16, D) for _ in range(2)]
    want = [m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, q, 90, 3000) for q in qs]
    ws = [m.paged_workspace(2, sum(new), 90, 3000) for _ in range(2)]
    out = [torch.empty_like(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        for s, q, o, w in zip(streams, qs, out, ws):
            with torch.cuda.stream(s):
                m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, q, 90, 3000, out=o, workspace=w)
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("new,past", [(3, 62), (16, 56), (20, 50), (100, 40), (100, 3000)])
def test_a_lost_page_is_lost_to_those_that_see_it(new, past):
    """Every form: the tokens before the first row of a page that is not there are whole."""
    lens = [new + past, 70]
    pool = Pool(21, lens, page_rows=32)
    q = randn(gen(22), new + 2, 16, D)
    cu = cu_of([new, 2])
    ref, limit = pool.reference(q, [new, 2])
    gone = (past // 32 + 1) * 32  # a page's first row, within the new ones
    assert past < gone < new + past
    pool.table[0, gone // 32] = -1
    for bound in (max(lens), 1 << 24):
        out = f64(m.attn_prefill_paged(pool.pages, i32(pool.table), pool.len, cu, q, new, bound))
        seen = gone - past
        near(out[:seen], ref[:seen], limit[:seen], "before it")
        assert np.all(np.isnan(out[seen:new]))
        near(out[new:], ref[new:], limit[new:], "the other sequence")


@pytest.mark.parametrize("H,G", [(16, 2), (9, 3)])
def test_prompts_of_long_blocks(H, G):
    """Calls that fill the card: blocks of 256 rows, cut and whole, every kind of row in
    them."""
    new, past = [530, 3, 257, 0, 64], [1500, 700, 0, 30, 2]
    lens = [a + b for a, b in zip(new, past)]
    pool = Pool(23, lens, G=G, page_rows=32)
    poison_tail(pool, lens)
    g = gen(24)
    q, gate = randn(g, sum(new), H, D), randn(g, sum(new), H, D)
    ref, limit = pool.reference(q, new, gate)
    for gt in (gate, gate.float()):
        for bound in (max(lens), 9000):
            out = m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu_of(new), q, max(new), bound, gate=gt)
            near(out, ref, limit, f"bound {bound}")
    # a NaN scale of V in a row that only the later tokens of a block see, and a lost page
    h = pool.host.view(np.float16)
    row = 1600
    h[pool.table[0, row // 32], 0, 0, R.V_SO[row % 32][64]] = np.nan
    pool.put()
    pool.table[0, 1856 // 32] = -1
    out = f64(m.attn_prefill_paged(pool.pages, i32(pool.table), pool.len, cu_of(new), q, max(new), 9000, gate=gate))
    ratio = H // G
    near(out[:100], ref[:100], limit[:100], "before both")
    near(out[:356, ratio:], ref[:356, ratio:], limit[:356, ratio:], "the other KV heads before the page")
    assert np.all(np.isnan(out[100:356, :ratio, 64:128])) and np.all(np.isnan(out[356:530]))
    rest = np.r_[0:64, 128:256]
    near(out[100:356, :ratio][..., rest], ref[100:356, :ratio][..., rest], limit[100:356, :ratio][..., rest], "other groups")
    near(out[530:], ref[530:], limit[530:], "the other sequences")
