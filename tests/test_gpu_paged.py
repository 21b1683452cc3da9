"""The paged 4-bit cache and the rotary positions on the GPU against their
definitions in 64 bits (paged_ref.py).

Tolerances.  Rotated outputs: the arithmetic is f32 over exactly reduced angles
(an angle's f32 residue is off by 2^-25 rad, sine and cosine by 2^-23, the norm's
sum of 256 squares by less than 2^-18 of itself, a rotation by three roundings):
2^-18 of the head's largest value, plus half a step of the output's type.  Stored
codes: 64-bit arithmetic, equal unless the value lies within 1e-9 of a step of a
border.  Attention: paged_ref.attend's bound."""
import numpy as np
import pytest
import torch

import moe_infer_amd as m
from moe_infer_amd.paged import TILE_BYTES

from . import paged_ref as R
from .gpu_util import announce

pytestmark = pytest.mark.gpu
D = 256
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def f64(t):
    return t.detach().double().cpu().numpy()


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float16):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def norm_weights(g):
    return (1 + 0.2 * randn(g, D, dtype=torch.float32)).to(torch.bfloat16)


def near(out, ref, bound, what):
    o = f64(out) if isinstance(out, torch.Tensor) else out
    assert o.shape == ref.shape, what
    off = np.abs(o - ref) - bound
    at = np.unravel_index(np.argmax(np.where(np.isnan(off), np.inf, off)), off.shape)
    assert np.all(off <= 0), f"{what}: {o[at]} for {ref[at]} at {at}, bound {np.broadcast_to(bound, off.shape)[at]}"


class Pool:
    """Pages of random codes and sensible scales, and tables over them in no order."""

    def __init__(self, seed, rows, G=2, page_rows=64, spare=2, fill=True):
        rng = np.random.default_rng(seed)
        need = [-(-r // page_rows) for r in rows]
        self.G, self.page_rows, self.rows = G, page_rows, list(rows)
        self.num = sum(need) + spare
        order = rng.permutation(self.num)[:sum(need)]
        self.table = np.full((len(rows), max(1, max(need))), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        p = rng.integers(0, 256, (self.num, G, page_rows // 32, TILE_BYTES), dtype=np.uint8)
        if fill:
            h = p.view(np.float16)
            scale = rng.uniform(0.2, 0.4, p.shape[:3] + (256,)).astype(np.float16)
            low = (-23.5 * scale.astype(np.float64) + rng.uniform(-0.3, 0.3, scale.shape)).astype(np.float16)
            h[..., 4096:4352] = np.stack([scale[..., :128], low[..., :128]], -1).reshape(p.shape[:3] + (256,))
            vs = scale[..., 128:].reshape(p.shape[:3] + (16, 1, 8))
            vo = low[..., 128:].reshape(p.shape[:3] + (16, 1, 8))
            h[..., 4352:] = np.concatenate([vs, vo], -2).reshape(p.shape[:3] + (256,))
        self.host = p
        self.pages = torch.from_numpy(p).cuda()
        self.t, self.len = i32(self.table), i32(self.rows)

    def put(self):
        self.pages.copy_(torch.from_numpy(self.host))

    def seq(self, s, head, rows=None):
        return R.sequence_rows(self.host, self.table[s], self.rows[s] if rows is None else rows, head)

    def reference(self, q, new, gate=None, H=None):
        """attend() of every sequence's last tokens; q [n, H, D]."""
        q = f64(q)
        out, bound = np.zeros(q.shape), np.zeros(q.shape)
        at, ratio = 0, q.shape[1] // self.G
        for s, (r, n) in enumerate(zip(self.rows, new)):
            for h in range(self.G):
                k, v = self.seq(s, h)
                sl = (slice(at, at + n), slice(h * ratio, (h + 1) * ratio))
                out[sl], bound[sl] = R.attend(q[sl], k, v, r - n, None if gate is None else f64(gate)[sl])
            at += n
        return out, bound


# -------------------------------------------------------------- rotations --

@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rot", [0, 8, 64, 136, 256])
@pytest.mark.parametrize("tin,tout", [(torch.float32, torch.float16), (torch.float16, torch.float16),
                                      (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                      (torch.float16, torch.float32), (torch.bfloat16, torch.float16)])
def test_rope_apply(layout, rot, tin, tout):
    announce(f"rope {layout} {rot} {tin} {tout}")
    g = gen(rot + 1)
    rope = m.Rope(rot, 1e6, layout, {"type": "yarn", "factor": 4.0, "original_max_position": 8192} if rot == 64 else None)
    x = randn(g, 7, 5, 2 * D, dtype=tin)[..., :D]  # strided, as beside a gate
    pos = [0, 1, 31, 4097, 131071, 1048575, 2 ** 31 - 1]
    w = norm_weights(g)
    for weights in (None, w):
        out = m.rope_apply(x, torch.tensor(pos, device="cuda"), rope, norm_w=weights, out_dtype=tout)
        ref = R.rotated(f64(x), pos, rope, None if weights is None else f64(weights))
        top = np.abs(ref).max(-1, keepdims=True)
        assert out.dtype == tout
        near(out, ref, 2.0 ** -18 * top + HALF_STEP[tout] * np.abs(ref) + 2.0 ** -25, f"{layout} {rot}")
    again = m.rope_apply(x, i32(pos), rope, norm_w=w, out_dtype=tout)
    assert torch.equal(out, again)


def test_rope_apply_in_place_one_token_and_negative():
    g = gen(5)
    rope = m.Rope(64, 1e4, "half")
    x = randn(g, 1, 3, D)
    want = m.rope_apply(x, i32([77]), rope)
    assert m.rope_apply(x, i32([77]), rope, out=x) is x and torch.equal(x, want)
    back = m.rope_apply(want, i32([-77]), rope, out_dtype=torch.float32)
    first = m.rope_apply(want, i32([0]), rope, out_dtype=torch.float32)
    assert torch.equal(first, want.float())
    near(back, R.rotated(f64(want), [-77], rope), 2.0 ** -16, "negative")
    with pytest.raises(ValueError):
        m.rope_apply(x, i32([1, 2]), rope)
    with pytest.raises(ValueError):
        y = randn(g, 2, 3, D)
        m.rope_apply(y.transpose(0, 1), i32([1, 2, 3]), rope, out=y)
    with pytest.raises(ValueError):
        m.rope_apply(x[..., ::2], i32([1]), rope)
    with pytest.raises(TypeError):
        m.rope_apply(x.double(), i32([1]), rope)


# ----------------------------------------------------------------- append --

def check_append(pool, new, k, v, rope, kw, cu, what):
    """The rows of the call hold the codes of the definition, all other bytes are as they were."""
    before = pool.host.copy()
    now = pool.pages.cpu().numpy()
    pos = np.concatenate([np.arange(r - n, r) for r, n in zip(pool.rows, new)]) if sum(new) else np.zeros(0)
    kr = R.rotated(f64(k)[:len(pos)], pos, rope, None if kw is None else f64(kw))
    vr = f64(v)[:len(pos)]
    touched = np.zeros(before.shape, bool)
    at = 0
    for s, (r, n) in enumerate(zip(pool.rows, new)):
        for h in range(pool.G):
            k_now, v_now = R.sequence_rows(now, pool.table[s], r, h)
            for i in range(n):
                row = r - n + i
                if row < 0:
                    continue
                for name, got, ref in (("k", k_now, kr), ("v", v_now, vr)):
                    val, border = R.quantised(ref[at + i, h])
                    same = (got[row] == val.astype(np.float64)) | (np.isnan(got[row]) & np.isnan(val))
                    assert np.all(same | (border < 1e-9)), f"{what}: {name} of sequence {s} row {row}"
                # bytes that the row owns (a byte of V codes is shared by two rows)
                page, t = pool.table[s][row // pool.page_rows], row % pool.page_rows // 32
                own = touched[page, h, t]
                w = row % 32
                for word, nib in ((R.K_WORD[w], R.K_NIB[w]),
                                  (R.V_WORD[w], R.V_NIB[w])):
                    own[word * 4 + nib // 2] = True
                for so, step in ((R.K_SO[w], 1), (R.V_SO[w], 8)):
                    for x in (so, so + step):
                        own[2 * x] = own[2 * x + 1] = True
        at += n
    assert np.array_equal(now[~touched], before[~touched]), f"{what}: bytes of other rows changed"
    # nibbles of V that share a byte with the call's
    for s, r in enumerate(pool.rows):
        for h in range(pool.G):
            old = R.sequence_rows(before, pool.table[s], r, h)
            new_ = R.sequence_rows(now, pool.table[s], r, h)
            keep = max(r - new[s], 0)
            for a, b in zip(old, new_):
                assert np.array_equal(a[:keep], b[:keep], equal_nan=True), f"{what}: a row before the call's changed"


APPEND_ONE = [1, 32, 33, 64, 65, 0, 100, 17, 16, 128]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout,rot,norm", [("half", 64, True), ("interleaved", 256, False), ("half", 136, False),
                                             ("interleaved", 0, True)])
def test_append_one_token(dtype, layout, rot, norm):
    announce(f"append one {dtype} {layout} {rot}")
    pool = Pool(1, APPEND_ONE, G=3, page_rows=32)
    g, B = gen(2), len(APPEND_ONE)
    rope = m.Rope(rot, 1e6, layout)
    q, k, v = randn(g, B, 6, D, dtype=dtype), 3 * randn(g, B, 3, D, dtype=dtype), randn(g, B, 3, D, dtype=dtype)
    qw, kw = (norm_weights(g), norm_weights(g)) if norm else (None, None)
    qo = m.paged_append(pool.pages, pool.t, pool.len, k, v, rope=rope, q=q, q_norm_w=qw, k_norm_w=kw)
    new = [1] * B
    check_append(pool, [0 if r == 0 else 1 for r in pool.rows], torch.cat([k[:5], k[6:]]), torch.cat([v[:5], v[6:]]),
                 rope, kw, None, "one token")
    ref = R.rotated(f64(q), [r - 1 for r in pool.rows], rope, None if qw is None else f64(qw))
    near(qo, ref, 2.0 ** -18 * np.abs(ref).max(-1, keepdims=True) + 2.0 ** -11 * np.abs(ref) + 2.0 ** -25, "q")
    rk, rv = m.paged_read(pool.pages, pool.t, pool.len)
    now = pool.pages.cpu().numpy()
    for s, r in enumerate(pool.rows):
        for h in range(3):
            a, b = R.sequence_rows(now, pool.table[s], r, h)
            assert np.array_equal(f64(rk)[s, h], a[-1] if r else np.zeros(D))
            assert np.array_equal(f64(rv)[s, h], b[-1] if r else np.zeros(D))


@pytest.mark.parametrize("new,past,page", [([1], [0], 32), ([33, 1, 0, 64], [0, 31, 40, 32], 32),
                                           ([100, 3, 29, 2], [5, 61, 3, 127], 64), ([257], [15], 256),
                                           ([0, 0, 7], [0, 9, 0], 128)])
@pytest.mark.parametrize("layout,rot,norm,dtype", [("half", 64, True, torch.float32),
                                                   ("interleaved", 192, False, torch.float16)])
def test_append_ragged(new, past, page, layout, rot, norm, dtype):
    announce(f"append ragged {new} {past} {page} {layout}")
    pool = Pool(3, [a + b for a, b in zip(new, past)], G=2, page_rows=page)
    g, n, extra = gen(4), sum(new), 3
    rope = m.Rope(rot, 1e6, layout, {"type": "linear", "factor": 2.0})
    proj = randn(g, n + extra, 4, 2 * D, dtype=dtype)
    k, v = randn(g, n + extra, 2, D, dtype=dtype), randn(g, 2, n + extra, D, dtype=dtype).transpose(0, 1)
    qw, kw = (norm_weights(g), norm_weights(g)) if norm else (None, None)
    cu = i32(np.concatenate([[0], np.cumsum(new)]))
    qo = torch.full((n + extra, 4, D), 7.0, dtype=torch.float16, device="cuda")
    m.paged_append(pool.pages, pool.t, pool.len, k, v, rope=rope, cu_q=cu, q=proj[..., :D], q_norm_w=qw, k_norm_w=kw,
                   q_out=qo)
    check_append(pool, new, k, v, rope, kw, cu, f"ragged {new}")
    pos = np.concatenate([np.arange(r - a, r) for r, a in zip(pool.rows, new)])
    ref = R.rotated(f64(proj[:n, :, :D]), pos, rope, None if qw is None else f64(qw))
    near(qo[:n], ref, 2.0 ** -18 * np.abs(ref).max(-1, keepdims=True) + 2.0 ** -11 * np.abs(ref) + 2.0 ** -25, "q")
    assert torch.all(qo[n:] == 7.0), "tokens behind the last sequence"
    out = [torch.full((n + extra, 2, D), 5.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    rk, rv = m.paged_read(pool.pages, pool.t, pool.len, cu, n + extra, out=out)
    now, at = pool.pages.cpu().numpy(), 0
    for s, a in enumerate(new):
        for h in range(2):
            for got, want in zip((rk, rv), R.sequence_rows(now, pool.table[s], pool.rows[s], h)):
                assert np.array_equal(f64(got)[at:at + a, h], want[pool.rows[s] - a:], equal_nan=True)
        at += a
    assert torch.all(rk[n:] == 5.0) and torch.all(rv[n:] == 5.0)


def test_append_odd_values():
    """Constant groups, NaN, infinities, values past f16, subnormal ranges."""
    pool = Pool(5, [40], G=1)
    x = torch.randn(40, 1, D, device="cuda", generator=gen(6))
    x[0] = 0.0
    x[1] = -3.0
    x[2, 0, 5] = float("nan")
    x[3, 0, 70] = float("inf")
    x[4, 0, 140] = -float("inf")
    x[5, 0, 200] = 70000.0
    x[6, 0, :64] = torch.linspace(0, 2e-7, 64)
    x[7, 0, 64:128] = 1000.0 + torch.linspace(0, 0.01, 64)
    x[8, 0] = torch.arange(256).cuda() * 64.0
    x[9, 0, :64] = 40000.0 * torch.sign(x[9, 0, :64])  # 16 scales below the least is past f16
    cu = i32([0, 40])
    m.paged_append(pool.pages, pool.t, pool.len, x, x, cu_q=cu)
    check_append(pool, [40], x, x, m.Rope(0), None, cu, "odd values")
    k, v = m.paged_read(pool.pages, pool.t, pool.len, cu, 40)
    assert torch.equal(torch.isnan(k), torch.isnan(v))
    bad = torch.isnan(k[:, 0]).view(40, 4, 64)
    want = torch.zeros_like(bad)
    want[2, 0] = want[3, 1] = want[4, 2] = want[5, 3] = want[9, 0] = True
    assert torch.equal(bad, want)
    assert torch.all(k[0] == 0) and torch.all(k[1] == -3)


def test_append_and_read_bound_by_the_tables():
    """Rows without a page are not written and read as NaN; a sequence shorter than its
    tokens reads as zero; page numbers past the pool are no pages."""
    pool = Pool(7, [100, 3, 70], G=2, page_rows=32)
    pool.table[0, 1] = -1
    pool.table[2, 0] = pool.num
    pool.t = i32(pool.table)
    new, cu = [100, 5, 70], i32([0, 100, 105, 175])
    g = gen(8)
    k, v = randn(g, 175, 2, D), randn(g, 175, 2, D)
    m.paged_append(pool.pages, pool.t, pool.len, k, v, cu_q=cu)
    rk, rv = m.paged_read(pool.pages, pool.t, pool.len, cu, 175)
    for got, x in ((rk, k), (rv, v)):
        got, want = f64(got), R.quantised(f64(x))[0].astype(np.float64)
        assert np.all(np.isnan(got[32:64])) and np.array_equal(got[:32], want[:32])
        assert np.all(got[100:102] == 0) and np.array_equal(got[102:105], want[102:105])
        assert np.all(np.isnan(got[105:137])) and np.array_equal(got[137:], want[137:])
    spare = sorted(set(range(pool.num)) - set(pool.table.ravel().tolist()))
    now = pool.pages.cpu().numpy()
    assert np.array_equal(now[spare], pool.host[spare])
    # a table with fewer columns than the rows need
    m.paged_append(pool.pages, pool.t[:, :1].contiguous(), pool.len, k, v, cu_q=cu)
    assert np.array_equal(pool.pages.cpu().numpy()[pool.table[0, 2:]], now[pool.table[0, 2:]])


# ---------------------------------------------------------------- decode --

LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 97, 128, 255, 300]


@pytest.mark.parametrize("H,G", [(16, 2), (8, 1), (32, 8), (4, 4), (15, 3), (16, 1), (7, 1)])
@pytest.mark.parametrize("page", [32, 256])
def test_decode_heads_and_lengths(H, G, page):
    announce(f"decode {H}/{G} pages of {page}")
    pool = Pool(H * 31 + G, LENS, G=G, page_rows=page)
    g = gen(9)
    q, gate = randn(g, len(LENS), H, D), randn(g, len(LENS), H, D, dtype=torch.float32)
    for gt in (None, gate, gate.half()):
        out = m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 300, gate=gt)
        ref, bound = pool.reference(q, [1] * len(LENS), gt)
        near(out, ref, bound, f"{H}/{G}")
    assert torch.all(out[0] == 0), "an empty sequence"
    # the same bits again, also with a larger max_len's own split
    assert torch.equal(out, m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 300, gate=gate.half()))


@pytest.mark.parametrize("lens", [[4000], [9000, 1], [2500, 2500, 3, 0, 700]])
def test_decode_long(lens):
    announce(f"decode {lens}")
    pool = Pool(10, lens, page_rows=128)
    g = gen(11)
    q = 2 * randn(g, len(lens), 16, D)  # sharper weights
    out = m.attn_decode_paged(pool.pages, pool.t, pool.len, q, max(lens))
    ref, bound = pool.reference(q, [1] * len(lens))
    near(out, ref, bound, f"{lens}")
    ws = m.paged_workspace(len(lens), len(lens), 1, 40000)
    out2 = m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 40000, workspace=ws)
    near(out2, ref, bound, f"{lens}, a larger bound on the lengths")


def test_decode_many_short_sequences():
    rng = np.random.default_rng(12)
    lens = rng.integers(0, 90, 700).tolist()
    pool = Pool(12, lens, G=1, page_rows=32)
    q = randn(gen(13), 700, 8, D)
    out = m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 90)
    ref, bound = pool.reference(q, [1] * 700)
    near(out, ref, bound, "700 sequences")


def poison_tail(pool, rows):
    """Not-a-number scales in every row from rows[s] on of the sequences' pages."""
    h = pool.host.view(np.float16)
    for s, r in enumerate(rows):
        for row in range(r, pool.page_rows * int((pool.table[s] >= 0).sum())):
            page, t, w = pool.table[s][row // pool.page_rows], row % pool.page_rows // 32, row % 32
            for so, step in ((R.K_SO[w], 1), (R.V_SO[w], 8)):
                h[page, :, t, so] = np.nan
                h[page, :, t, so + step] = np.inf
    pool.put()


def test_rows_out_of_sight_do_not_count():
    """Stale rows behind the end, and rows that a prompt's earlier tokens do not see,
    may hold anything; the tokens that do see a NaN give NaN."""
    lens = [5, 33, 64, 95, 200]
    pool = Pool(14, lens)
    poison_tail(pool, lens)
    g = gen(15)
    q = randn(g, len(lens), 16, D)
    ref, bound = pool.reference(q, [1] * len(lens))
    near(m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 200), ref, bound, "decode")
    new = [5, 20, 1, 60, 130]
    cu = i32(np.concatenate([[0], np.cumsum(new)]))
    q = randn(g, sum(new), 16, D)
    ref, bound = pool.reference(q, new)
    near(m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, q, 130, 200), ref, bound, "prefill")
    # rows 150 on of the last sequence: V of group 1 only, then K
    h, base = pool.host.view(np.float16), sum(new[:4])
    for what in ("v", "k"):
        for row in range(150, 153):
            page, t, w = pool.table[4][row // 64], row % 64 // 32, row % 32
            so = R.V_SO[w][64] if what == "v" else R.K_SO[w][64]
            h[page, 0, t, so] = np.nan
        pool.put()
        out = f64(m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, q, 130, 200))
        assert np.all(np.isfinite(out[:base + 80])), what
        near(out[:base + 80], ref[:base + 80], bound[:base + 80], what)
        near(out[:, 8:], ref[:, 8:], bound[:, 8:], what)
        seen = out[base + 80:, :8]
        if what == "v":
            assert np.all(np.isnan(seen[..., 64:128]))
            rest = np.r_[0:64, 128:256]
            near(seen[..., rest], ref[base + 80:, :8][..., rest], bound[base + 80:, :8][..., rest], what)
        else:
            assert np.all(np.isnan(seen))


def test_masks_of_lowest_values():
    """Scores near the f16 range, equal scores, and one row far above all others."""
    pool = Pool(16, [70, 300])
    q = torch.zeros(2, 16, D, dtype=torch.float16, device="cuda")
    out = m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 300)
    ref, bound = pool.reference(q, [1, 1])
    near(out, ref, bound, "equal weights")
    q = 1000 * randn(gen(17), 2, 16, D)
    out = f64(m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 300))
    ref, _ = pool.reference(q, [1, 1])
    assert np.all(np.isfinite(out)) and np.abs(out - ref).max() < 4  # one row wins: values to 3.5
    picks = (np.abs(out - ref).max(-1) < 0.01).mean()
    assert picks > 0.9


def test_bad_tables_give_nan():
    lens = [40, 100, 64, 90]
    pool = Pool(18, lens, page_rows=32)
    q = randn(gen(19), 4, 16, D)
    want = f64(m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 100))
    pool.table[1, 2] = -1
    pool.table[3, 1] = pool.num + 7
    out = f64(m.attn_decode_paged(pool.pages, i32(pool.table), pool.len, q, 100))
    assert np.all(np.isnan(out[[1, 3]])) and np.array_equal(out[[0, 2]], want[[0, 2]])
    out = f64(m.attn_decode_paged(pool.pages, pool.t, i32([40, 101, -1, 90]), q, 100))
    assert np.all(np.isnan(out[[1, 2]])) and np.array_equal(out[[0, 3]], want[[0, 3]])
    # more tokens than max_q
    q = randn(gen(20), 9, 16, D)
    out = f64(m.attn_prefill_paged(pool.pages, pool.t, pool.len, i32([0, 2, 7, 8, 9]), q, 2, 100))
    assert np.all(np.isnan(out[2:7])) and np.all(np.isfinite(out[:2])) and np.all(np.isfinite(out[7:]))


def test_pages_past_32_bits():
    """A pool of more than 4 GiB: the last page lies behind 2^32 bytes."""
    per = 2 * 2 * TILE_BYTES
    num = (1 << 32) // per + 40
    pages = torch.empty((num, 2, 2, TILE_BYTES), dtype=torch.uint8, device="cuda")
    pool = Pool(21, [100], spare=0)
    table = np.array([[num - 1, num - 5]], np.int32)
    for j in range(2):
        pages[table[0, j]] = pool.pages[pool.table[0, j]]
    q = randn(gen(22), 1, 16, D)
    want = m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 100)
    assert torch.equal(m.attn_decode_paged(pages, i32(table), pool.len, q, 100), want)
    k, v = randn(gen(23), 1, 2, D), randn(gen(24), 1, 2, D)
    m.paged_append(pages, i32(table), pool.len, k, v)
    m.paged_append(pool.pages, pool.t, pool.len, k, v)
    assert torch.equal(pages[table[0, 1]], pool.pages[pool.table[0, 1]])
    a, b = m.paged_read(pages, i32(table), pool.len), m.paged_read(pool.pages, pool.t, pool.len)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    del pages


# --------------------------------------------------------------- prefill --

@pytest.mark.parametrize("new,past", [([1], [0]), ([2], [0]), ([8], [0]), ([9], [23]), ([33], [31]), ([64], [0]),
                                      ([130], [0]), ([200], [77]), ([257], [0]),
                                      ([1, 40, 0, 3, 17], [100, 0, 9, 64, 15]), ([4, 4, 4], [1000, 31, 0]),
                                      ([130, 1, 260], [300, 700, 12])])
@pytest.mark.parametrize("H,G", [(16, 2), (12, 4), (5, 1)])
def test_prefill(new, past, H, G):
    announce(f"prefill {new} after {past}, {H}/{G}")
    lens = [a + b for a, b in zip(new, past)]
    pool = Pool(25, lens, G=G)
    g, n = gen(26), sum(new)
    cu = i32(np.concatenate([[0], np.cumsum(new)]))
    q = randn(g, n + 2, H, D)
    gate = randn(g, n + 2, H, 2 * D, dtype=torch.float32)[..., D:]
    out = torch.full((n + 2, H, D), 3.0, dtype=torch.float16, device="cuda")
    m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, q, max(new), max(lens), gate=gate, out=out)
    ref, bound = pool.reference(q[:n], new, gate[:n])
    near(out[:n], ref, bound, f"{new} after {past}")
    assert torch.all(out[n:] == 3.0), "tokens behind the last sequence"
    # larger bounds than needed
    out2 = m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, q, max(new) + 100, max(lens) + 5000)
    ref, bound = pool.reference(q[:n], new)
    near(out2[:n], ref, bound, "larger bounds")


def test_prefill_more_tokens_than_rows():
    """A sequence shorter than its tokens: the tokens without a row attend nothing."""
    pool = Pool(27, [3, 40])
    q = randn(gen(28), 7 + 40, 16, D)
    out = m.attn_prefill_paged(pool.pages, pool.t, pool.len, i32([0, 7, 47]), q, 40, 40)
    ref, bound = pool.reference(q, [7, 40])
    near(out, ref, bound, "short")
    assert torch.all(out[:4] == 0)


def test_prefill_of_one_token_is_a_decode_step():
    pool = Pool(29, [500, 64, 1])
    q = randn(gen(30), 3, 16, D)
    a = m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 500)
    b = m.attn_prefill_paged(pool.pages, pool.t, pool.len, i32([0, 1, 2, 3]), q, 1, 500)
    assert torch.equal(a, b)


# ------------------------------------------------- buffers, streams, graphs --

@pytest.mark.parametrize("lens,new", [([700, 33], [1, 1]), ([700, 90], [40, 90]), ([6000], [200])])
def test_out_may_be_q_or_gate(lens, new):
    pool = Pool(31, lens)
    g, n = gen(32), sum(new)
    q, gate = randn(g, n, 16, D), randn(g, n, 16, D)
    cu = i32(np.concatenate([[0], np.cumsum(new)]))
    want = m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, q, max(new), max(lens), gate=gate)
    q2, g2 = q.clone(), gate.clone()
    m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, q2, max(new), max(lens), gate=gate, out=q2)
    m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, q, max(new), max(lens), gate=g2, out=g2)
    assert torch.equal(q2, want) and torch.equal(g2, want)
    wide = torch.empty(n, 17, D, dtype=torch.float16, device="cuda")
    wide[:, 1:] = q
    got = m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, wide[:, 1:], max(new), max(lens), gate=gate)
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="overlaps"):
        m.attn_prefill_paged(pool.pages, pool.t, pool.len, cu, wide[:, 1:], max(new), max(lens),
                             out=wide.view(-1)[:n * 16 * D].view(n, 16, D))


def test_python_refusals():
    pool = Pool(33, [40, 50])
    q = randn(gen(34), 2, 16, D)
    k = randn(gen(35), 2, 2, D)
    dec = lambda **kw: m.attn_decode_paged(**{**dict(pages=pool.pages, block_table=pool.t, kv_len=pool.len,  # noqa: E731
                                                     q=q, max_len=50), **kw})
    for kw in (dict(pages=pool.pages[..., :9000]), dict(pages=pool.pages[:, :, ::2]), dict(block_table=pool.t[:1]),
               dict(block_table=pool.t.view(-1)), dict(kv_len=pool.len[:1]), dict(q=q[:1]), dict(q=q[..., :128]),
               dict(q=q.cpu()), dict(gate=q[:, :8]), dict(out=q[:1]), dict(q=q[:, :15]), dict(max_len=-1),
               dict(workspace=torch.empty(0, dtype=torch.uint8, device="cuda"), max_len=90000)):
        with pytest.raises(ValueError):
            dec(**kw)
    for kw in (dict(pages=pool.pages.int()), dict(kv_len=pool.len.long()), dict(q=q.float()), dict(gate=q.bfloat16()),
               dict(out=q.float()), dict(q=None)):
        with pytest.raises(TypeError):
            dec(**kw)
    app = lambda **kw: m.paged_append(**{**dict(pages=pool.pages, block_table=pool.t, kv_len=pool.len, k=k, v=k),  # noqa: E731
                                         **kw})
    for kw in (dict(k=k[:1]), dict(v=k[:, :1]), dict(k=k[..., 1:]), dict(q_out=q), dict(q=q[:1]),
               dict(k_norm_w=torch.ones(255, dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises(ValueError):
            app(**kw)
    for kw in (dict(v=k.float()), dict(q=q.float()), dict(rope=1.0), dict(k_norm_w=torch.ones(256, device="cuda"))):
        with pytest.raises(TypeError):
            app(**kw)
    with pytest.raises(ValueError):
        m.paged_read(pool.pages, pool.t, pool.len, cu_q=i32([0, 1, 2]))
    with pytest.raises(TypeError):
        m.attn_prefill_paged(pool.pages, pool.t, pool.len, None, q, 1, 50)
    with pytest.raises((ValueError, TypeError)):
        m.paged_append(pool.pages, pool.t, pool.len, k.transpose(1, 2), k)


def test_another_stream():
    pool = Pool(36, [3000, 70])
    q = randn(gen(37), 2, 16, D)
    want = m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 3000)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = m.attn_decode_paged(pool.pages, pool.t, pool.len, q, 3000)
        rot = m.rope_apply(q, pool.len, m.Rope(64))
    s.synchronize()
    assert torch.equal(out, want) and torch.equal(rot, m.rope_apply(q, pool.len, m.Rope(64)))


def test_captured_step_follows_its_tables():
    """A captured append + decode, replayed as the program moves the lengths on, against
    the same calls made eagerly; two graphs that share a workspace, in turn."""
    rope, B = m.Rope(64, 1e6), 3
    g = gen(38)
    start = [30, 62, 1500]
    a, b = Pool(39, [r + 10 for r in start]), Pool(39, [r + 10 for r in start])
    kv = i32(start)
    k, v, q = randn(g, B, 2, D), randn(g, B, 2, D), randn(g, B, 16, D)
    ws = m.paged_workspace(B, B, 1, 2000)
    qo, out, out2 = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)

    def step(pool, lens, o):
        m.paged_append(pool.pages, pool.t, lens, k, v, rope=rope, q=q, q_out=qo)
        m.attn_decode_paged(pool.pages, pool.t, lens, qo, 2000, out=o, workspace=ws)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(a, kv, out)  # eager once, in both pools
        step(b, kv, out)
    torch.cuda.current_stream().wait_stream(s)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        step(a, kv, out)
    with torch.cuda.graph(g2):
        m.attn_decode_paged(a.pages, a.t, kv, q, 2000, out=out2, workspace=ws)
    for i in range(5):
        kv.add_(1)
        k.copy_(randn(g, B, 2, D))
        q.copy_(randn(g, B, 16, D))
        g1.replay()
        g2.replay()
        got, got2 = out.clone(), out2.clone()
        torch.cuda.synchronize()
        want = torch.empty_like(out)
        m.paged_append(b.pages, b.t, i32([r + 1 + i for r in start]), k, v, rope=rope, q=q, q_out=qo)
        lens = i32([r + 1 + i for r in start])
        m.attn_decode_paged(b.pages, b.t, lens, qo, 2000, out=want)
        assert torch.equal(got, want), f"replay {i}"
        assert torch.equal(got2, m.attn_decode_paged(b.pages, b.t, lens, q, 2000)), f"replay {i}"


def test_sequences_may_share_pages_that_are_read():
    pool = Pool(40, [128, 64])
    table = pool.table.copy()
    table[1, 0] = table[0, 0]  # a shared prefix
    q = randn(gen(41), 2, 16, D)
    out = f64(m.attn_decode_paged(pool.pages, i32(table), pool.len, q, 128))
    pool.table = table
    ref, bound = pool.reference(q, [1, 1])
    near(out, ref, bound, "shared prefix")


# --------------------------------------------------------------- together --

def test_prompt_steps_and_rollback_together():
    """A server's run over two layers: prompts, decode steps, a draft that is partly
    rejected, another sequence in the freed pages, against one attention over all rows as
    stored."""
    rope = m.Rope(64, 1e7, "half", {"type": "yarn", "factor": 2.0, "original_max_position": 128})
    cache = m.PagedCache(num_layers=2, num_q_heads=16, num_kv_heads=2, num_pages=24, page_rows=32)
    g = gen(42)
    w = [(norm_weights(g), norm_weights(g)) for _ in range(2)]
    a, b = cache.add(), cache.add()

    def step(seqs, new):
        t = cache.batch(seqs, new)
        for layer in cache.full_layers:
            proj, k, v = (randn(g, t.n, h, d, dtype=torch.float32) for h, d in ((16, 2 * D), (2, D), (2, D)))
            qw, kw = w[layer]
            pages = cache.pages(layer)
            q = m.paged_append(pages, t.block_table, t.kv_len, k, v, rope=rope, cu_q=t.cu_q, q=proj[..., :D],
                               q_norm_w=qw, k_norm_w=kw)
            ref_q = m.rope_apply(proj[..., :D], t.positions, rope, norm_w=qw, out_dtype=torch.float16)
            assert torch.equal(q, ref_q)
            gate = proj[..., D:]
            if t.cu_q is None:
                o = m.attn_decode_paged(pages, t.block_table, t.kv_len, q, t.max_len, gate=gate)
            else:
                o = m.attn_prefill_paged(pages, t.block_table, t.kv_len, t.cu_q, q, t.max_q, t.max_len, gate=gate)
            host, table = pages.cpu().numpy(), t.block_table.cpu().numpy()
            rows = t.kv_len.tolist()
            counts = [1] * len(seqs) if t.cu_q is None else np.diff(t.cu_q.cpu().numpy()).tolist()
            at = 0
            for s, (r, n) in enumerate(zip(rows, counts)):
                for h in range(2):
                    kk, vv = R.sequence_rows(host, table[s], r, h)
                    sl = (slice(at, at + n), slice(8 * h, 8 * h + 8))
                    ref, bound = R.attend(f64(q)[sl], kk, vv, r - n, f64(gate)[sl])
                    near(f64(o)[sl], ref, bound, f"layer {layer} sequence {s}")
                at += n

    step([a, b], [70, 129])
    for _ in range(3):
        step([b, a], 1)
    step([a, b], [5, 1])       # a draft for a
    cache.truncate(a, 75)      # three of five taken back
    step([a], [1])
    c = cache.add()
    cache.remove(b)
    step([c, a], [40, 2])
    assert cache.len(a) == 78 and cache.len(c) == 40
