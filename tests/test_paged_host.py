"""Host side of the paged cache and the rotary positions: rotation plans, the
page allocator, and the refusals of the C entries and the Python layer (no GPU:
every call here fails before any HIP call)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import moe_infer_amd as m
from moe_infer_amd import _lib
from moe_infer_amd.paged import TILE_BYTES

from . import paged_ref as R


# ------------------------------------------------------------- rotations --

def test_plain_frequencies():
    r = m.Rope(64, 1e7)
    want = [1e7 ** (-2 * i / 64) for i in range(32)]
    assert np.allclose(r.frequencies, want, rtol=1e-15) and r.factor == 1.0


@pytest.mark.parametrize("dim", [8, 64, 256])
def test_scaled_frequencies(dim):
    base = np.array(m.Rope(dim, 1e6).frequencies)
    lin = m.Rope(dim, 1e6, scaling={"type": "linear", "factor": 4.0})
    assert np.allclose(lin.frequencies, base / 4, rtol=1e-15)
    ntk = np.array(m.Rope(dim, 1e6, scaling={"type": "ntk", "factor": 4.0}).frequencies)
    assert ntk[0] == 1.0  # the fastest pair stays, the slowest goes 4 times slower
    assert math.isclose(ntk[-1], base[-1] / 4, rel_tol=1e-12)
    y = m.Rope(dim, 1e6, scaling={"type": "yarn", "factor": 4.0, "original_max_position": 4096})
    f = np.array(y.frequencies)
    turns = 4096 * base / (2 * math.pi)
    assert np.allclose(f[turns >= 32], base[turns >= 32], rtol=1e-15)
    assert np.allclose(f[turns <= 1], base[turns <= 1] / 4, rtol=1e-15)
    assert np.all((f <= base * (1 + 1e-15)) & (f >= base / 4 * (1 - 1e-15)))
    assert math.isclose(y.factor, 0.1 * math.log(4) + 1)
    one = m.Rope(dim, 1e6, scaling={"type": "yarn", "factor": 1.0, "original_max_position": 4096})
    assert np.allclose(one.frequencies, base, rtol=1e-15) and one.factor == 1.0


def test_rope_from_config():
    c = {"head_dim": 256, "partial_rotary_factor": 0.25, "rope_theta": 1e7,
         "rope_scaling": {"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 32768}}
    r = m.Rope.from_config(c)
    assert r.frequencies == m.Rope(64, 1e7, scaling={"type": "yarn", "factor": 2.0,
                                                     "original_max_position": 32768}).frequencies
    c["rope_scaling"] = {"rope_type": "default"}
    assert m.Rope.from_config(c, "interleaved").frequencies == m.Rope(64, 1e7).frequencies
    assert m.Rope.from_config(None).rotary_dim == 64


@pytest.mark.parametrize("kw", [
    dict(rotary_dim=12), dict(rotary_dim=264), dict(rotary_dim=-8), dict(layout="neox"),
    dict(theta=0.0), dict(theta=float("inf")), dict(scaling={"type": "other", "factor": 2}),
    dict(scaling={"type": "linear"}), dict(scaling={"type": "linear", "factor": 0.5}),
    dict(scaling={"type": "linear", "factor": 2, "beta_fast": 3}), dict(scaling={"factor": 2}),
    dict(scaling={"type": "yarn", "factor": 2}),
    dict(scaling={"type": "yarn", "factor": 2, "original_max_position": 0}),
    dict(scaling={"type": "yarn", "factor": 2, "original_max_position": 9, "beta_fast": 1}),
    dict(frequencies=[1.0] * 31), dict(frequencies=[float("nan")] * 32),
    dict(frequencies=[1.0] * 32, scaling={"type": "linear", "factor": 2}),
    dict(factor=float("inf"))])
def test_rope_refusals(kw):
    with pytest.raises(ValueError):
        m.Rope(**kw)


# -------------------------------------------------------------- allocator --

def cache(**kw):
    kw = {"num_layers": 1, "num_pages": 6, "page_rows": 32, "num_kv_heads": 1, "num_q_heads": 8,
          "device": "cpu", **kw}
    return m.PagedCache(**kw)


def test_pages_are_dealt_once_and_come_back():
    c = cache()
    a, b = c.add(), c.add()
    step = c.batch([a, b], [33, 64])
    assert step.n == 97 and step.max_q == 64 and step.max_len == 64 and c.free_pages == 2
    assert step.kv_len.tolist() == [33, 64] and step.cu_q.tolist() == [0, 33, 97]
    assert step.positions.tolist() == list(range(33)) + list(range(64))
    ids = step.block_table[0].tolist() + step.block_table[1].tolist()
    assert len(set(ids)) == 4 and all(0 <= i < 6 for i in ids)
    step = c.batch([b, a])
    assert step.cu_q is None and step.kv_len.tolist() == [65, 34]
    assert step.positions.tolist() == [64, 33] and step.block_table.shape == (2, 3)
    assert step.block_table[1, 2] == -1
    c.truncate(b, 64)
    assert c.free_pages == 2 and c.len(b) == 64
    c.truncate(b, 32)
    assert c.free_pages == 3
    c.remove(a)
    assert c.free_pages == 5
    with pytest.raises(ValueError):
        c.len(a)


def test_a_batch_that_does_not_fit_takes_nothing():
    c = cache()
    a, b = c.add(), c.add()
    c.extend(a, 10)
    with pytest.raises(MemoryError):
        c.batch([a, b], [30, 200])
    assert c.len(a) == 10 and c.len(b) == 0 and c.free_pages == 5
    for seqs, new in (([a, a], 1), ([], 1), ([a], [1, 2]), ([a], [-1]), ([a], [0]), ([a, 99], 1)):
        with pytest.raises(ValueError):
            c.batch(seqs, new)
    assert c.len(a) == 10
    with pytest.raises(ValueError):
        c.truncate(a, 11)
    with pytest.raises(ValueError):
        c.extend(a, -1)


def test_layers_follow_the_config():
    c = m.PagedCache({"num_hidden_layers": 8, "num_attention_heads": 16, "num_key_value_heads": 2,
                      "head_dim": 256, "linear_num_value_heads": 32, "linear_num_key_heads": 16},
                     num_pages=1, page_rows=32, device="cpu")
    assert c.full_layers == [3, 7] and c.pages(7).shape == (1, 2, 1, TILE_BYTES)
    with pytest.raises(ValueError):
        c.pages(0)
    for kw in (dict(page_rows=48), dict(page_rows=16), dict(page_rows=2048), dict(num_pages=0),
               dict(head_dim=128), dict(num_q_heads=9, num_kv_heads=2)):
        with pytest.raises(ValueError):
            cache(**kw)


# --------------------------------------------------------------- refusals --

def test_the_layout_is_a_permutation():
    """Every nibble and every scale of a tile is used once."""
    for word, nib in ((R.K_WORD, R.K_NIB), (R.V_WORD - 1024, R.V_NIB)):
        assert sorted((word * 8 + nib).ravel()) == list(range(8192))
    ks = np.unique(np.stack([R.K_SO, R.K_SO + 1]))
    vs = np.unique(np.stack([R.V_SO, R.V_SO + 8]))
    assert ks.tolist() == list(range(4096, 4352)) and vs.tolist() == list(range(4352, 4608))


FAKE = 1 << 20  # never dereferenced: the checks come first
F64 = (C.c_double * 128)(*([1.0] * 128))


def view(**kw):
    a = dict(pages=FAKE, num_pages=4, page_rows=64, table=FAKE, cols=2, kv_len=FAKE, cu_q=None, batch=2)
    a.update({k: v for k, v in kw.items() if k in a})
    return list(a.values())


def append(**kw):
    a = dict(n=2, H=16, G=2, D=256, type=1, q=None, q_ts=0, q_hs=0, k=FAKE, k_ts=512, k_hs=256, v=FAKE,
             v_ts=512, v_hs=256, qw=None, kw=None, eps=1e-6, f=F64, rot=64, ilv=0, factor=1.0,
             q_out=None, stream=None)
    a.update({k: v for k, v in kw.items() if k in a})
    return _lib.lib().mi_paged_append(*view(**kw), *a.values())


def attend(**kw):
    a = dict(n=2, max_q=1, max_len=100, H=16, G=2, D=256, q=FAKE, q_ts=4096, q_hs=256, gate=None, g_type=1,
             g_ts=0, g_hs=0, out=FAKE + (1 << 20), ws=FAKE, ws_bytes=1 << 40, stream=None)
    a.update({k: v for k, v in kw.items() if k in a})
    return _lib.lib().mi_attn_paged(*view(**kw), *a.values())


def read(**kw):
    a = dict(n=2, G=2, D=256, k_out=FAKE, v_out=FAKE + (1 << 20), stream=None)
    a.update({k: v for k, v in kw.items() if k in a})
    return _lib.lib().mi_paged_read(*view(**kw), *a.values())


def rope(**kw):
    a = dict(x=FAKE, type=1, ts=4096, hs=256, n=2, heads=16, D=256, pos=FAKE, pos64=0, w=None, eps=1e-6,
             f=F64, rot=64, ilv=0, factor=1.0, out=FAKE + (1 << 20), out_type=1, stream=None)
    a.update({k: v for k, v in kw.items() if k in a})
    return _lib.lib().mi_rope_apply(*a.values())


INV, UNS, RANGE = _lib.MI_ERR_INVALID_ARG, _lib.MI_ERR_UNSUPPORTED, _lib.MI_ERR_OUT_OF_RANGE
SHARED = [(dict(pages=None), INV), (dict(pages=FAKE + 8), INV), (dict(num_pages=0), INV),
          (dict(page_rows=16), INV), (dict(page_rows=96), INV), (dict(page_rows=2048), INV),
          (dict(table=None), INV), (dict(cols=0), INV), (dict(kv_len=None), INV), (dict(batch=0), INV),
          (dict(batch=70000, n=70000), UNS), (dict(D=128), UNS), (dict(n=0), INV), (dict(n=3), INV),
          (dict(G=0), INV)]


@pytest.mark.parametrize("call", [append, attend, read])
@pytest.mark.parametrize("kw,status", SHARED)
def test_shared_refusals(call, kw, status):
    assert call(**kw) == status and _lib.lib().mi_last_error()


@pytest.mark.parametrize("call,kw,status", [
    (append, dict(k=None), INV), (append, dict(v=FAKE + 2), INV), (append, dict(k_ts=500), INV),
    (append, dict(k_hs=128), INV), (append, dict(type=3), INV), (append, dict(rot=12), INV),
    (append, dict(rot=264), INV), (append, dict(f=None), INV), (append, dict(eps=-1.0), INV),
    (append, dict(factor=math.nan), INV), (append, dict(q=FAKE, q_ts=4096, q_hs=256), INV),
    (append, dict(q=FAKE, q_ts=4096, q_hs=256, q_out=FAKE + 512), INV),
    (append, dict(q=FAKE, q_ts=8192, q_hs=512, q_out=FAKE), INV),  # in place, but not in its strides
    (append, dict(q=FAKE, type=0, q_ts=4096, q_hs=256, q_out=FAKE), INV),
    (append, dict(q=FAKE << 1, q_ts=4096, q_hs=256, q_out=FAKE), INV),  # q_out over k
    (attend, dict(q=None), INV), (attend, dict(out=None), INV), (attend, dict(out=FAKE + 512), INV),
    (attend, dict(gate=FAKE << 2, g_type=2, g_ts=4096, g_hs=256), INV),
    (attend, dict(gate=FAKE + (1 << 20) + 512, g_ts=4096, g_hs=256), INV),
    (attend, dict(max_q=2), INV), (attend, dict(max_q=0, cu_q=FAKE), INV), (attend, dict(max_len=-1), INV),
    (attend, dict(max_len=2 ** 31 - 1), RANGE), (attend, dict(H=15), INV), (attend, dict(H=64, q_ts=16384), UNS),
    (attend, dict(ws=None), INV), (attend, dict(ws=FAKE + 4), INV), (attend, dict(ws_bytes=0, max_len=9000), INV),
    (read, dict(k_out=None), INV), (read, dict(v_out=FAKE), INV), (read, dict(v_out=FAKE + 8), INV),
    (rope, dict(x=None), INV), (rope, dict(pos=None), INV), (rope, dict(out=None), INV), (rope, dict(n=0), INV),
    (rope, dict(D=64), UNS), (rope, dict(out_type=5), INV), (rope, dict(out=FAKE + 512), INV),
    (rope, dict(out=FAKE, out_type=2), INV), (rope, dict(heads=0), INV), (rope, dict(eps=math.nan), INV)])
def test_refusals(call, kw, status):
    assert call(**kw) == status and _lib.lib().mi_last_error()


def test_workspace_size():
    ws = _lib.lib().mi_attn_paged_workspace_size
    assert ws(1, 1, 1, 32768, 16, 2) > 0
    for bad in ((0, 1, 1, 10, 16, 2), (1, 0, 1, 10, 16, 2), (1, 1, 0, 10, 16, 2), (1, 1, 1, -1, 16, 2),
                (1, 1, 1, 10, 16, 3), (1, 1, 1, 10, 64, 2)):
        assert ws(*bad) == 0
    with pytest.raises(ValueError):
        m.paged_workspace(1, 1, 1, 10, 16, 3)


def test_python_layer_takes_gpu_tensors_only():
    c = cache()
    a = c.add()
    s = c.batch([a], 4)
    k = torch.zeros(4, 1, 256, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        m.paged_append(c.pages(0), s.block_table, s.kv_len, k, k, cu_q=s.cu_q)
    with pytest.raises(ValueError, match="GPU"):
        m.rope_apply(k, s.positions, m.Rope(64))
    with pytest.raises(ValueError, match="GPU"):
        m.attn_decode_paged(c.pages(0), s.block_table, s.kv_len, k, 4)
    with pytest.raises(ValueError, match="GPU"):
        m.paged_read(c.pages(0), s.block_table, s.kv_len, s.cu_q, 4)
