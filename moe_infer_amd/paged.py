"""Rotary positions, and a paged KV cache in 4 bits for batches of sequences.

A server of many sequences keeps their rows in pages of one pool per layer
instead of one region each, and in 4 bits instead of 16 (288 bytes a row and KV
head instead of 1024).  A layer of a step is

    q = paged_append(pages, table, kv_len, k, v, rope=rope, cu_q=cu_q, q=q_proj,
                     q_norm_w=qw, k_norm_w=kw)      # norm, rotation, append
    o = attn_prefill_paged(pages, table, kv_len, cu_q, q, max_q, max_len, gate=gate)

and of a decode step (one token per sequence) the same without cu_q, through
attn_decode_paged.  The tables live on the device and the kernels read them, so
a captured step follows them as the program updates them in place.

PagedCache owns the pages of all layers and deals them to sequences;
PagedCache.batch() makes the tables of a step, new tensors each time: for a captured
step, copy them into its own (the block table into the first of its columns).  The functions take tensors, so
a program with an allocator of its own needs only the layout (include/mi_attn.h).

Beside the single-sequence Cache / qk_norm_rope_append / attn_prefill and the
ragged decode over whole regions (attention.py).  The reference keeps one f32
cache for one sequence (src/cache.rs:45-128).
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

import torch

from . import _lib
from .attention import HEAD_DIM, _device, _stream
from .kv_cache import _cfg_get

TILE_ROWS = 32
TILE_BYTES = 9216
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_HALF = (torch.float16,)
_GATES = (torch.float16, torch.float32)


class Rope:
    """A rotation plan: frequencies (64 bits) of the first rotary_dim columns,
    the layout of the pairs, and the factor on the rotated columns.

    layout: "half" pairs columns (i, i + rotary_dim / 2), "interleaved" (2i, 2i + 1).
    Without scaling, frequency i is theta^(-2i / rotary_dim).  scaling, a dict with
    "type" and "factor" s (>= 1), stretches it for a context s times longer:
      "linear"  every frequency / s
      "ntk"     theta * s^(rotary_dim / (rotary_dim - 2)) in theta's place
      "yarn"    frequency i * (1 - g + g / s), g = (i - first) / (last - first) held to
                [0, 1], first and last the pairs that make "beta_fast" (32) and "beta_slow"
                (1) turns r over "original_max_position" rows L,
                rotary_dim ln(L / (2 pi r)) / (2 ln theta), rounded down and up (not with
                "truncate" false): what a config.json means; and the rotated columns
                times "attention_factor" (default 0.1 ln s + 1).  "ramp": "turns" instead
                of "pairs": a line in the turns, g = (beta_fast - r) / (beta_fast - beta_slow)
    frequencies: a sequence of rotary_dim / 2 numbers instead of all that."""

    def __init__(self, rotary_dim: int = 64, theta: float = 1e7, layout: str = "half",
                 scaling: dict | None = None, frequencies=None, factor: float | None = None):
        rotary_dim = int(rotary_dim)
        if rotary_dim < 0 or rotary_dim % 8 or rotary_dim > HEAD_DIM:
            raise ValueError(f"rotary_dim {rotary_dim}: a multiple of 8, at most {HEAD_DIM}")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout {layout!r}: 'half' or 'interleaved'")
        turned = 1.0
        if frequencies is None:
            if not (theta > 0 and math.isfinite(theta)):
                raise ValueError(f"theta {theta}")
            frequencies, turned = _scaled(rotary_dim, float(theta), dict(scaling or {}))
        elif scaling:
            raise ValueError("frequencies are taken as they are: no scaling beside them")
        f = [float(x) for x in frequencies]
        if len(f) != rotary_dim // 2 or not all(math.isfinite(x) for x in f):
            raise ValueError(f"{rotary_dim // 2} finite frequencies are wanted")
        self.rotary_dim = rotary_dim
        self.layout = layout
        self.frequencies = tuple(f)
        self.factor = float(turned if factor is None else factor)
        if not math.isfinite(self.factor):
            raise ValueError(f"factor {self.factor}")
        self._pack()

    def _pack(self) -> None:
        """The C arguments: frequencies, rotary_dim, interleaved, factor."""
        self._f = (C.c_double * max(1, len(self.frequencies)))(*self.frequencies)
        self._args = (C.addressof(self._f), self.rotary_dim, int(self.layout == "interleaved"), self.factor)

    # A copy makes its own: the address in _args is of this object's _f.
    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_f", "_args")}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state)
        self._pack()

    @classmethod
    def from_config(cls, config, layout: str = "half") -> "Rope":
        """From a model's config.json dict: rope_theta, partial_rotary_factor,
        rope_scaling ({"rope_type" or "type": ..., "factor": ..., ...}; yarn's first context is
        "original_max_position_embeddings" rows, or the config's max_position_embeddings), or
        rope_parameters, which holds all three."""
        s = _cfg_get(config, "rope_scaling", None) or _cfg_get(config, "rope_parameters", None) or {}
        s = {k: v for k, v in s.items() if v is not None}
        if any(isinstance(v, dict) for v in s.values()):
            raise ValueError(f"rope_parameters of {sorted(s)}: give one layer type's")
        theta = _cfg_get(config, "rope_theta", s.pop("rope_theta", 1e7))
        part = _cfg_get(config, "partial_rotary_factor", s.pop("partial_rotary_factor", 0.25))
        dim = int(round(float(part) * int(_cfg_get(config, "head_dim", HEAD_DIM))))
        kind = s.pop("rope_type", None) or s.get("type", "default")
        if kind == "default":
            s = None
        else:
            s["type"] = kind
            rows = s.pop("original_max_position_embeddings", None)
            if kind == "yarn":
                _yarn_keys(s, rows or _cfg_get(config, "max_position_embeddings", None))
        return cls(dim, float(theta), layout, s)


def _yarn_keys(s: dict, rows) -> None:
    """A config's keys of yarn as Rope's.  mscale and mscale_all_dim: the factor is
    their ratio as 0.1 k ln s + 1 each; one of them alone (but for an mscale of 1) is read in
    two ways, so it is refused."""
    if rows is not None:
        s["original_max_position"] = rows
    a, b = s.pop("mscale", None), s.pop("mscale_all_dim", None)
    if "attention_factor" in s or not (a or b) or (a == 1 and not b):
        return
    if not (a and b):
        raise ValueError(f"yarn: mscale {a} with mscale_all_dim {b}: give attention_factor")
    log = 0.1 * math.log(float(s.get("factor", 1.0)))
    s["attention_factor"] = (a * log + 1.0) / (b * log + 1.0)


def _scaled(dim: int, theta: float, scaling: dict):
    """(frequencies, factor) of Rope's docstring."""
    kind = scaling.pop("type", "none")
    if kind == "none":
        if scaling:
            raise ValueError(f"scaling has no type but {sorted(scaling)}")
        return [theta ** (-2.0 * i / dim) for i in range(dim // 2)], 1.0
    known = {"linear": set(), "ntk": set(),
             "yarn": {"original_max_position", "beta_fast", "beta_slow", "ramp", "truncate", "attention_factor"}}
    if kind not in known:
        raise ValueError(f"scaling type {kind!r}: one of {sorted(known)}")
    if "factor" not in scaling:
        raise ValueError("scaling needs a factor")
    s = float(scaling.pop("factor"))
    if not (s >= 1.0 and math.isfinite(s)):
        raise ValueError(f"scaling factor {s}: at least 1")
    if set(scaling) - known[kind]:
        raise ValueError(f"scaling {kind!r} does not know {sorted(set(scaling) - known[kind])}")
    if kind == "ntk":
        theta *= s ** (dim / (dim - 2.0))
    f = [theta ** (-2.0 * i / dim) for i in range(dim // 2)]
    if kind == "linear":
        return [x / s for x in f], 1.0
    if kind == "ntk":
        return f, 1.0
    if "original_max_position" not in scaling:
        raise ValueError("yarn needs original_max_position")
    rows = float(scaling["original_max_position"])
    slow, fast = float(scaling.get("beta_slow", 1.0)), float(scaling.get("beta_fast", 32.0))
    ramp = scaling.get("ramp", "pairs")
    if not (rows > 0 and fast > slow) or (ramp == "pairs" and not (slow > 0 and theta > 1)):
        raise ValueError(f"yarn: original_max_position {rows}, beta_slow {slow}, beta_fast {fast}, theta {theta}")
    if ramp == "turns":
        share = [(fast - rows * x / (2 * math.pi)) / (fast - slow) for x in f]
    elif ramp == "pairs":
        pair = [dim * math.log(rows / (2 * math.pi * r)) / (2 * math.log(theta)) for r in (fast, slow)]
        if scaling.get("truncate", True):
            pair = [math.floor(pair[0]), math.ceil(pair[1])]
        first, last = max(pair[0], 0), min(pair[1], dim - 1)
        if first > last and dim:
            raise ValueError(f"yarn: no pair of {dim} columns makes {slow} to {fast} turns in {rows} rows")
        share = [(i - first) / max(last - first, 0.001) for i in range(dim // 2)]
    else:
        raise ValueError(f"yarn: ramp {ramp!r}: 'pairs' or 'turns'")
    factor = scaling.get("attention_factor")
    return ([x * (1.0 - g + g / s) for x, g in zip(f, (min(1.0, max(0.0, g)) for g in share))],
            0.1 * math.log(s) + 1.0 if factor is None else float(factor))


_NO_ROPE = Rope(0)


# ----------------------------------------------------------------- checks --
#
# A small call is a few us of GPU work and what the host spends decides how fast
# it goes: each check is one expression while nothing is wrong (0.2 to 0.5 us a
# tensor against 0.6 to 1.1 one by one), and only then looks for what is.

def _current() -> int:
    """The current device; -2, which no tensor is on, where there is none."""
    try:
        return _device()
    except (RuntimeError, AssertionError):
        return -2


def _check_rows(name: str, t, n: int | None, heads: int | None, dtypes, dev: int):
    """[n, heads, 256] on device dev, its columns contiguous: (tokens, heads, token
    stride, head stride)."""
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and t.dim() == 3 and t.get_device() == dev:
        (rows, h, d), (ts, hs, cs) = t.shape, t.stride()
        if h == 1:
            hs = HEAD_DIM
        if rows == 1:
            ts = h * hs
        size = t.element_size()
        if (d == HEAD_DIM and cs == 1 and (n is None or rows == n) and (heads is None or h == heads)
                and not (t.data_ptr() | ts * size | hs * size) & 15 and hs >= d and ts >= d):
            return rows, h, ts, hs
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    if t.dim() != 3 or t.shape[2] != HEAD_DIM:
        raise ValueError(f"{name} must be [tokens, heads, {HEAD_DIM}], got {tuple(t.shape)}")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{name} has {t.shape[0]} tokens, expected {n}")
    if heads is not None and t.shape[1] != heads:
        raise ValueError(f"{name} has {t.shape[1]} heads, expected {heads}")
    _refuse_device(name, t, dev)
    if t.stride(2) != 1:
        raise ValueError(f"{name}: its {HEAD_DIM} columns must be contiguous")
    if t.numel() == 0:
        raise ValueError(f"{name} is empty")
    if hs < HEAD_DIM or ts < HEAD_DIM:
        raise ValueError(f"{name}: rows overlap (strides {ts}, {hs})")
    raise ValueError(f"{name}: every row must be 16-byte aligned")


def _refuse_device(name: str, t: torch.Tensor, dev: int) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor, got {t.device}")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, the current device is cuda:{dev}")


def _check_table(name: str, t, numel: int | None, dtype, dev: int, aligned: int = 0) -> None:
    """A contiguous tensor of `dtype` on device dev; aligned: 15 for whole 16 bytes."""
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev and t.is_contiguous()
            and (numel is None or t.numel() == numel) and not t.data_ptr() & aligned):
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    _refuse_device(name, t, dev)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} has {t.numel()} elements, expected {numel}")
    raise ValueError(f"{name} must be 16-byte aligned")


def _check_pages(pages, block_table, kv_len, cu_q, dev: int):
    """The C arguments of the cache: pages .. batch; the batch; and the KV heads."""
    _check_table("pages", pages, None, torch.uint8, dev, 15)
    _check_table("block_table", block_table, None, torch.int32, dev)
    if pages.dim() != 4 or pages.shape[3] != TILE_BYTES or not pages.numel():
        raise ValueError(f"pages must be [pages, KV heads, page rows / {TILE_ROWS}, {TILE_BYTES}], "
                         f"got {tuple(pages.shape)}")
    if block_table.dim() != 2 or not block_table.numel():
        raise ValueError(f"block_table must be [batch, pages of a sequence], got "
                         f"{tuple(block_table.shape)}")
    (num, G, tiles, _), (batch, cols) = pages.shape, block_table.shape
    _check_table("kv_len", kv_len, batch, torch.int32, dev)
    if cu_q is not None:
        _check_table("cu_q", cu_q, batch + 1, torch.int32, dev)
    return (pages.data_ptr(), num, tiles * TILE_ROWS, block_table.data_ptr(), cols, kv_len.data_ptr(),
            None if cu_q is None else cu_q.data_ptr(), batch), batch, G


def _check_norm(name: str, w, dev: int):
    if w is None:
        return None
    _check_table(name, w, HEAD_DIM, torch.bfloat16, dev, 15)
    return w.data_ptr()


def _check_out(name: str, out, n: int, heads: int, dtype, dev: int):
    if out is None:
        return torch.empty((n, heads, HEAD_DIM), dtype=dtype, device=dev)
    _check_table(name, out, n * heads * HEAD_DIM, dtype, dev, 15)
    return out


# -------------------------------------------------------------- operators --

def rope_apply(x: torch.Tensor, positions: torch.Tensor, rope: Rope,
               norm_w: torch.Tensor | None = None, eps: float = 1e-6,
               out: torch.Tensor | None = None, out_dtype=None) -> torch.Tensor:
    """x [n, heads, 256] (f32, f16 or bf16, any token and head stride) rotated
    at positions [n] (int32 or int64), after an RMS norm with norm_w (bf16 [256])
    if given.  Returns [n, heads, 256] of out_dtype (default x's); out may be x."""
    dev = _current()
    n, heads, ts, hs = _check_rows("x", x, None, None, _DTYPES, dev)
    wide = isinstance(positions, torch.Tensor) and positions.dtype is torch.int64
    _check_table("positions", positions, n, torch.int64 if wide else torch.int32, dev)
    if not isinstance(rope, Rope):
        raise TypeError("rope must be a Rope")
    w = _check_norm("norm_w", norm_w, dev)
    dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    if dtype not in _DTYPES:
        raise TypeError(f"out_dtype {dtype}")
    out = _check_out("out", out, n, heads, dtype, dev)
    _lib.check(_lib.lib().mi_rope_apply(
        x.data_ptr(), _DTYPES[x.dtype], ts, hs, n, heads, HEAD_DIM, positions.data_ptr(), wide, w, eps,
        *rope._args, out.data_ptr(), _DTYPES[dtype], _stream()))
    return out


def paged_append(pages: torch.Tensor, block_table: torch.Tensor, kv_len: torch.Tensor,
                 k: torch.Tensor, v: torch.Tensor, rope: Rope | None = None,
                 cu_q: torch.Tensor | None = None, q: torch.Tensor | None = None,
                 q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None,
                 eps: float = 1e-6, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Appends n tokens' k, v [n, G, 256] as the last rows of their sequences:
    K normed (k_norm_w) and rotated at its row, both quantised to 4 bits.  kv_len
    counts the rows after the call; token i of sequence s (cu_q[s] + i) is row
    kv_len[s] - tokens of s + i; without cu_q each sequence brings one token.
    With q [n, H, 256] returns it normed and rotated, [n, H, 256] f16 (q_out; may
    be q).  q, k, v: one of f32, f16, bf16, any token and head stride (a view of a
    projection).  No rope: no rotation."""
    dev = _current()
    head, batch, G = _check_pages(pages, block_table, kv_len, cu_q, dev)
    n, _, kts, khs = _check_rows("k", k, None, G, _DTYPES, dev)
    if cu_q is None and n != batch:
        raise ValueError(f"{n} tokens for {batch} sequences without cu_q")
    same = (k.dtype,)
    _, _, vts, vhs = _check_rows("v", v, n, G, same, dev)
    if rope is None:
        rope = _NO_ROPE
    elif not isinstance(rope, Rope):
        raise TypeError("rope must be a Rope")
    H = qts = qhs = 0
    qp = None
    if q is not None:
        _, H, qts, qhs = _check_rows("q", q, n, None, same, dev)
        q_out = _check_out("q_out", q_out, n, H, torch.float16, dev)
        qp = q.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    _lib.check(_lib.lib().mi_paged_append(
        *head, n, H, G, HEAD_DIM, _DTYPES[k.dtype], qp, qts, qhs, k.data_ptr(), kts, khs, v.data_ptr(),
        vts, vhs, _check_norm("q_norm_w", q_norm_w, dev), _check_norm("k_norm_w", k_norm_w, dev), eps,
        *rope._args, None if q is None else q_out.data_ptr(), _stream()))
    return q_out


def paged_read(pages: torch.Tensor, block_table: torch.Tensor, kv_len: torch.Tensor,
               cu_q: torch.Tensor | None = None, n: int | None = None,
               out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """(k, v), each [n, G, 256] f16: the last cu_q[s + 1] - cu_q[s] rows of each
    sequence (without cu_q the last row), as stored.  n: their number, cu_q[-1];
    with cu_q it must be given, so that the call need not wait for the GPU."""
    dev = _current()
    head, batch, G = _check_pages(pages, block_table, kv_len, cu_q, dev)
    if n is None:
        if cu_q is not None:
            raise ValueError("n must be given with cu_q")
        n = batch
    n = int(n)
    k, v = out if out is not None else (None, None)
    k = _check_out("k", k, n, G, torch.float16, dev)
    v = _check_out("v", v, n, G, torch.float16, dev)
    _lib.check(_lib.lib().mi_paged_read(*head, n, G, HEAD_DIM, k.data_ptr(), v.data_ptr(), _stream()))
    return k, v


def paged_workspace(batch: int, n: int, max_q: int, max_len: int, num_q_heads: int = 16,
                    num_kv_heads: int = 2, device="cuda") -> torch.Tensor:
    """Workspace of attn_decode_paged / attn_prefill_paged for steps of these
    sizes (n tokens in all, at most max_q and max_len rows a sequence) and smaller
    ones; 135 MB where a sequence brings more than 32 tokens times heads of a group.
    Calls that may run at the same time need one each."""
    nbytes = _lib.lib().mi_attn_paged_workspace_size(batch, n, max_q, max_len, num_q_heads,
                                                     num_kv_heads)
    if not nbytes:
        raise ValueError(f"no workspace for batch {batch}, {n} tokens, max_q {max_q}, max_len "
                         f"{max_len}, heads {num_q_heads} / {num_kv_heads}")
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _attend(pages, block_table, kv_len, cu_q, q, max_q, max_len, gate, out, workspace):
    dev = _current()
    head, batch, G = _check_pages(pages, block_table, kv_len, cu_q, dev)
    n, H, qts, qhs = _check_rows("q", q, None, None, _HALF, dev)
    if cu_q is None and n != batch:
        raise ValueError(f"{n} tokens for {batch} sequences")
    if H % G:
        raise ValueError(f"{H} query heads for {G} KV heads")
    gp = None
    g_type = gts = ghs = 0
    if gate is not None:
        _, _, gts, ghs = _check_rows("gate", gate, n, H, _GATES, dev)
        g_type = _DTYPES[gate.dtype]
        gp = gate.data_ptr()
    out = _check_out("out", out, n, H, torch.float16, dev)
    if workspace is None:
        workspace = paged_workspace(batch, n, max_q, max_len, H, G, q.device)
    else:
        _check_table("workspace", workspace, None, torch.uint8, dev, 15)
    _lib.check(_lib.lib().mi_attn_paged(
        *head, n, max_q, max_len, H, G, HEAD_DIM, q.data_ptr(), qts, qhs, gp, g_type, gts, ghs,
        out.data_ptr(), workspace.data_ptr(), workspace.numel(), _stream()))
    return out


def attn_decode_paged(pages: torch.Tensor, block_table: torch.Tensor, kv_len: torch.Tensor,
                      q: torch.Tensor, max_len: int, gate: torch.Tensor | None = None,
                      out: torch.Tensor | None = None,
                      workspace: torch.Tensor | None = None) -> torch.Tensor:
    """A decode step: q [batch, H, 256] f16, sequence s over its kv_len[s] rows
    (at most max_len).  gate [batch, H, 256] f16 or f32: out *= sigmoid(gate).  An
    empty sequence gives zeros.  out may be q or gate itself."""
    return _attend(pages, block_table, kv_len, None, q, 1, int(max_len), gate, out, workspace)


def attn_prefill_paged(pages: torch.Tensor, block_table: torch.Tensor, kv_len: torch.Tensor,
                       cu_q: torch.Tensor, q: torch.Tensor, max_q: int, max_len: int,
                       gate: torch.Tensor | None = None, out: torch.Tensor | None = None,
                       workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of a ragged batch, its rows already appended: q [n, H, 256]
    f16, tokens cu_q[s] .. cu_q[s + 1] - 1 the last rows of sequence s (at most
    max_q tokens and max_len rows).  Prompts, chunks behind cached rows, drafts to
    verify.  gate and out as for attn_decode_paged; tokens from cu_q[-1] on are not
    written."""
    if cu_q is None:
        raise TypeError("cu_q must be a torch.Tensor")
    return _attend(pages, block_table, kv_len, cu_q, q, int(max_q), int(max_len), gate, out, workspace)


# -------------------------------------------------------------- the cache --

@dataclass
class PagedBatch:
    """The tables of one step, for every layer: PagedCache.batch()."""
    block_table: torch.Tensor     # int32 [batch, pages]
    kv_len: torch.Tensor          # int32 [batch]
    cu_q: torch.Tensor | None     # int32 [batch + 1]; None: one token each
    positions: torch.Tensor       # int32 [n], the row of every token
    n: int
    max_q: int
    max_len: int


class PagedCache:
    """Pages of every full-attention layer, dealt to sequences.

    Sequences are numbers that add() gives.  extend(seq, n) makes room for n more
    rows, truncate(seq, rows) takes a rejected draft back (rows past it stay in
    place and are overwritten), remove(seq) gives its pages back.  A page number
    means the same rows in every layer.  Not thread-safe, like Cache."""

    def __init__(self, config=None, *, num_layers: int | None = None, num_q_heads: int = 16,
                 num_kv_heads: int = 2, head_dim: int = HEAD_DIM, num_pages: int = 256,
                 page_rows: int = 64, device="cuda"):
        from .kv_cache import FULL_ATTN_INTERVAL
        n_hidden = int(_cfg_get(config, "num_hidden_layers", num_layers or 1))
        self.num_q_heads = int(_cfg_get(config, "num_attention_heads", num_q_heads))
        self.num_kv_heads = int(_cfg_get(config, "num_key_value_heads", num_kv_heads))
        if int(_cfg_get(config, "head_dim", head_dim)) != HEAD_DIM:
            raise ValueError(f"head_dim must be {HEAD_DIM}")
        if self.num_kv_heads <= 0 or self.num_q_heads % self.num_kv_heads:
            raise ValueError(f"{self.num_q_heads} query heads for {self.num_kv_heads} KV heads")
        if page_rows < TILE_ROWS or page_rows > 1024 or page_rows & (page_rows - 1):
            raise ValueError(f"page_rows {page_rows}: a power of two, 32 to 1024")
        if num_pages <= 0:
            raise ValueError(f"num_pages {num_pages}")
        linear = (_cfg_get(config, "linear_num_value_heads", 0) or 0) > 0 and \
                 (_cfg_get(config, "linear_num_key_heads", 0) or 0) > 0
        self.full_layers = [i for i in range(n_hidden)
                            if not linear or (i + 1) % FULL_ATTN_INTERVAL == 0]
        self.page_rows = int(page_rows)
        self.num_pages = int(num_pages)
        self.device = torch.device(device)
        # zeros: a fresh page's rows are 0 * code + 0
        self._pages = {layer: torch.zeros((self.num_pages, self.num_kv_heads,
                                           self.page_rows // TILE_ROWS, TILE_BYTES),
                                          dtype=torch.uint8, device=self.device)
                       for layer in self.full_layers}
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._rows: dict[int, int] = {}
        self._table: dict[int, list[int]] = {}
        self._next = 0

    def pages(self, layer: int) -> torch.Tensor:
        """The pages of model layer `layer`."""
        try:
            return self._pages[layer]
        except KeyError:
            raise ValueError(f"layer {layer} is not a full-attention layer") from None

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def add(self) -> int:
        seq = self._next
        self._next += 1
        self._rows[seq], self._table[seq] = 0, []
        return seq

    def _known(self, seq: int) -> None:
        if seq not in self._rows:
            raise ValueError(f"no sequence {seq}")

    def len(self, seq: int) -> int:
        self._known(seq)
        return self._rows[seq]

    def extend(self, seq: int, rows: int) -> int:
        """Room for `rows` more rows; the sequence's rows.  Takes nothing where
        the free pages do not suffice (MemoryError)."""
        self._known(seq)
        if rows < 0:
            raise ValueError(f"rows {rows}")
        total = self._rows[seq] + rows
        need = -(-total // self.page_rows) - len(self._table[seq])
        if need > len(self._free):
            raise MemoryError(f"{need} pages wanted, {len(self._free)} of {self.num_pages} free")
        for _ in range(need):
            self._table[seq].append(self._free.pop())
        self._rows[seq] = total
        return total

    def truncate(self, seq: int, rows: int) -> None:
        self._known(seq)
        if not 0 <= rows <= self._rows[seq]:
            raise ValueError(f"{rows} rows of a sequence of {self._rows[seq]}")
        keep = -(-rows // self.page_rows)
        self._free.extend(reversed(self._table[seq][keep:]))
        del self._table[seq][keep:]
        self._rows[seq] = rows

    def remove(self, seq: int) -> None:
        self.truncate(seq, 0)
        del self._rows[seq], self._table[seq]

    def batch(self, seqs, new=1) -> PagedBatch:
        """Extends each of seqs by its new rows (a number for all, or one each)
        and makes the step's tables.  All of them or, on an error, none."""
        seqs = list(seqs)
        counts = [int(new)] * len(seqs) if isinstance(new, int) else [int(x) for x in new]
        if not seqs or len(counts) != len(seqs) or len(set(seqs)) != len(seqs):
            raise ValueError("a batch is one or more different sequences, each with its new rows")
        for s, c in zip(seqs, counts):
            self._known(s)
            if c < 0:
                raise ValueError(f"rows {c}")
        if not sum(counts):
            raise ValueError("no sequence has a new row")
        before = [self._rows[s] for s in seqs]
        try:
            for s, c in zip(seqs, counts):
                self.extend(s, c)
        except MemoryError:
            for s, b in zip(seqs, before):
                self.truncate(s, b)
            raise
        n, B = sum(counts), len(seqs)
        M = max(1, max(len(self._table[s]) for s in seqs))
        host = [i for s in seqs for i in self._table[s] + [-1] * (M - len(self._table[s]))]
        host += [self._rows[s] for s in seqs]
        at = [0]
        for c in counts:
            at.append(at[-1] + c)
        host += at
        for b, c in zip(before, counts):
            host += range(b, b + c)
        # one copy for all of the step's tables
        t = torch.tensor(host, dtype=torch.int32).to(self.device)
        table, kv_len, cu_q, positions = t.split([B * M, B, B + 1, n])
        return PagedBatch(table.view(B, M), kv_len, None if all(c == 1 for c in counts) else cu_q,
                          positions, n, max(counts), max(self._rows[s] for s in seqs))
