"""The paged 4-bit KV cache and the rotary positions as timed cases.

Five operators, as a serving program calls them per layer: rope_apply (rotary
positions), paged_append (norm + rotation + quantisation into pages),
attn_decode_paged and attn_prefill_paged (attention over the pages) and
paged_read (rows back as f16).  `run` makes those calls where `own` is true and
computes the same values with elementary torch operations where it is false;
`exact` computes them in 64 bits from the definitions.

The cache: pages [num_pages, G, page_rows / 32, 9216] uint8.  A tile of 9216
bytes holds 32 rows of one KV head: K codes, V codes (4096 bytes each, eight
4-bit codes to a word), then the scales and offsets in f16 of K and of V
(512 bytes each), one pair per row and group of 64 columns.  A value is
f16((16 + code) * scale + offset).  Row r = 16 sub + m = 16 sub + 4 quad + i:
  K, column 64 g + 16 quad + 8 step + e: nibble e of word
      ((2 sub + g // 2) * 64 + 16 quad + m) * 4 + 2 (g % 2) + step
  V, column 64 g + 4 n + j: nibble i + 4 sub of word (64 g + 16 quad + n) * 4 + j
  K scale, offset: halves 2 (4 r + g) and the next, from byte 8192
  V scale: half (4 g + quad) * 16 + 2 i + sub from byte 8704, offset 8 halves on
"""
import math

import numpy as np
import torch

own = False

D = 256
TILE_ROWS, TILE_BYTES = 32, 9216
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_GOLDEN = 0.6180339887498949


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # the query of one decoded token, far into a long context
        _rope("rope, one token", 1, 16, "f16", "half", 64, "none", False),
        # the queries of a prompt chunk straight from the projection, scaled for a long context
        _rope("rope, 4099 tokens of projections", 4099, 16, "f32", "half", 64, "yarn", True),
        # a decode step of 64 sequences: one new row each
        _append("append, 64 sequences' tokens", 64, 16, 2, 1, 1, 1024, 32768, "f32", "half", 64, "none", True),
        # prompts of unequal length in one pass
        _append("append, five prompts", 5, 16, 2, 37, 2048, 0, 1000, "f16", "interleaved", 128, "linear", False),
        # a chat server's short contexts
        _decode("decode, 8 short sequences", 8, 16, 2, 0, 512, 32, True),
        # one user, long context
        _decode("decode, one of 32768 rows", 1, 16, 2, 32768, 32768, 64, True),
        # a full batch of unequal lengths
        _decode("decode, 64 of up to 32768 rows", 64, 16, 2, 1024, 32768, 128, True),
        # a prompt from an empty cache
        _prefill("prefill, 4096 tokens", 1, 16, 2, 4096, 4096, 0, 0, 64, True),
        # chunks of prompts behind cached rows, a single decoded token among them
        _prefill("prefill, six ragged chunks", 6, 16, 2, 1, 1000, 0, 16384, 64, True),
        # draft tokens of 16 sequences to be verified
        _prefill("verify, 16 sequences of 4 tokens", 16, 16, 2, 4, 4, 8192, 32768, 64, True),
        # the rows of one sequence to be saved
        _read("read, 777 rows", 1, 2, 777, 777, 64),
        # a batch's rows to be moved
        _read("read, 8 sequences", 8, 2, 1000, 16384, 128),
    ]


def _rope(name, n, heads, dtype, layout, rot, scaling, norm):
    return {"name": name, "op": "rope", "n": n, "heads": heads, "dtype": dtype, "layout": layout,
            "rot": rot, "scaling": scaling, "norm": norm}


def _append(name, batch, H, G, q0, q1, p0, p1, dtype, layout, rot, scaling, norm, page=64):
    """Sequences with q0 to q1 new tokens behind p0 to p1 cached rows."""
    return {"name": name, "op": "append", "batch": batch, "H": H, "G": G, "q0": q0, "q1": q1, "p0": p0,
            "p1": p1, "page": page, "dtype": dtype, "layout": layout, "rot": rot, "scaling": scaling,
            "norm": norm}


def _decode(name, batch, H, G, l0, l1, page, gate):
    return {"name": name, "op": "decode", "batch": batch, "H": H, "G": G, "l0": l0, "l1": l1, "page": page,
            "gate": gate}


def _prefill(name, batch, H, G, q0, q1, p0, p1, page, gate):
    return {"name": name, "op": "prefill", "batch": batch, "H": H, "G": G, "q0": q0, "q1": q1, "p0": p0,
            "p1": p1, "page": page, "gate": gate}


def _read(name, batch, G, l0, l1, page):
    return {"name": name, "op": "read", "batch": batch, "G": G, "l0": l0, "l1": l1, "page": page}


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(("rope", "append", "decode", "decode", "prefill", "prefill", "read"))
    H, G = rng.choice(((16, 2), (16, 2), (8, 1), (32, 4), (32, 8), (12, 3), (4, 4)))
    page = rng.choice((32, 64, 128, 256))
    gate = rng.random() < 0.6
    dtype = rng.choice(("f32", "f16", "bf16"))
    layout = rng.choice(("half", "interleaved"))
    rot = rng.choice((32, 64, 128, 192, 256))
    scaling = rng.choice(("none", "linear", "ntk", "yarn"))
    norm = rng.random() < 0.5
    if op == "rope":
        c = _rope("", _log(rng, 1, 8000), rng.randint(1, 24), dtype, layout, rot, scaling, norm)
    elif op == "append":
        batch, most = _log(rng, 1, 80), _log(rng, 1, 2000)
        c = _append("", batch, H, G, rng.randint(0, 1), max(1, min(most, 9000 // batch)), 0, _log(rng, 1, 3000),
                    dtype, layout, rot, scaling, norm, page)
    elif op == "decode":
        batch = _log(rng, 1, 64)
        c = _decode("", batch, H, G, rng.randint(0, 20), _log(rng, 40, min(32768, 700000 // (batch * G))), page, gate)
    elif op == "prefill":
        batch, q1 = _log(rng, 1, 12), _log(rng, 2, 2500)
        q1 = max(2, min(q1, 4000 // batch))
        c = _prefill("", batch, H, G, rng.randint(0, 1), q1, 0,
                     _log(rng, 1, max(2, min(16000, 5000000 // (batch * q1 * G)))), page, gate)
    else:
        batch = _log(rng, 1, 8)
        c = _read("", batch, G, 0, _log(rng, 20, 130000 // (batch * G)), page)
    del c["name"]
    return c


def _spread(a, b, count):
    """`count` lengths from a to b, the last b, in no order."""
    return [b if s == count - 1 else a + int((b - a + 1) * ((s + 1) * _GOLDEN % 1.0)) for s in range(count)]


def _sizes(case):
    """(new tokens, rows behind the call) of each sequence."""
    B = case["batch"]
    if case["op"] in ("append", "prefill"):
        new = _spread(case["q0"], case["q1"], B)
        past = _spread(case["p0"], case["p1"], B + 3)[1:B + 1]
        return new, [a + b for a, b in zip(new, past)]
    rows = _spread(case["l0"], case["l1"], B)
    return (rows if case["op"] == "read" else [1] * B), rows


# ----------------------------------------------------------------- inputs --

def _frequencies(rot, scaling):
    """The rotation frequencies of the pairs and the factor on the rotated columns."""
    theta, s, L0 = 1e7, 4.0, 8192
    if scaling == "ntk":
        theta *= s ** (rot / (rot - 2))
    f = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        f = [x / s for x in f]
    if scaling == "yarn":  # turns over the first context: from 1 (all scaled) to 32 (none)
        keep = [min(1.0, max(0.0, (L0 * x / (2 * math.pi) - 1.0) / 31.0)) for x in f]
        f = [x * g + x / s * (1 - g) for x, g in zip(f, keep)]
    return f, 0.1 * math.log(s) + 1.0 if scaling == "yarn" else 1.0


def _tables(gen, rows, page):
    """A pool of pages in no order: (pages in the pool, block table, unused entries -1)."""
    need = [-(-r // page) for r in rows]
    total, M = sum(need), max(1, max(need))
    pool = total + 3
    order = torch.randperm(pool, generator=gen)[:total].to(torch.int32)
    table = torch.full((len(rows), M), -1, dtype=torch.int32)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    return pool, table.cuda()


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed * 7919 + 1)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case, "kept": {}}
    if case["op"] == "rope":
        n, h, t = case["n"], case["heads"], _TYPES[case["dtype"]]
        # from a projection the queries stand beside their gates
        x = _normal(gen, (n, h, 2 * D if case["dtype"] == "f32" else D), t)
        s["x"] = x[..., :D]
        first = int(torch.randint(0, 120000, (1,), generator=host))
        s["positions"] = (first + torch.arange(n)).to(torch.int32).cuda()
    else:
        new, rows = _sizes(case)
        G, page = case["G"], case["page"]
        n = sum(new)
        pool, s["table"] = _tables(host, rows, page)
        s["kv_len"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
        s["cu_q"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
        s["n"], s["max_q"], s["max_len"] = n, max(new), max(rows)
        shape = (pool, G, page // TILE_ROWS, TILE_BYTES)
        if case["op"] == "append":
            s["pages"] = torch.zeros(shape, dtype=torch.uint8, device="cuda")
            t, H = _TYPES[case["dtype"]], case["H"]
            s["q"] = _normal(gen, (n, H, 2 * D if case["dtype"] == "f32" else D), t)[..., :D]
            # keys with a few strong channels, as trained models have them
            strong = torch.ones(D, device="cuda")
            strong[torch.randint(0, D, (6,), generator=host).cuda()] = 5.0
            s["k"] = (_normal(gen, (n, G, D), torch.float32) * strong).to(t)
            s["v"] = _normal(gen, (n, G, D), t)
        else:
            s["pages"] = _full_pages(gen, shape)
    if case.get("norm"):
        for w in ("q_w", "k_w"):
            s[w] = (1.0 + 0.1 * _normal(gen, (D,), torch.float32)).to(torch.bfloat16)
    if case["op"] in ("decode", "prefill"):
        H = case["H"]
        s["q"] = _normal(gen, (s["n"], H, D), torch.float16)
        s["gate"] = _normal(gen, (s["n"], H, D), torch.float16) if case["gate"] else None
    if "rot" in case:
        f, s["factor"] = _frequencies(case["rot"], case["scaling"])
        s["f"] = torch.tensor(f, dtype=torch.float64, device="cuda")
    return s


def _full_pages(gen, shape):
    """Pages of standard normal rows, as quantised: any codes, the range of 64 normal values."""
    pages = torch.randint(0, 256, shape, generator=gen, device="cuda", dtype=torch.uint8)
    halves = pages.view(torch.float16)
    for at, lay in ((4096, (32, 4, 2)), (4352, (16, 2, 8))):
        dim = 2 if at == 4096 else 1
        u = torch.rand(shape[:3] + lay, generator=gen, device="cuda")
        scale = (0.25 + 0.12 * u.select(3 + dim, 0)).half()
        low = -7.5 * scale.float() + 0.4 * (u.select(3 + dim, 1) - 0.5)
        both = torch.stack((scale, (low - 16 * scale.float()).half()), dim=3 + dim)
        halves[..., at:at + 256] = both.reshape(shape[:3] + (256,))
    return pages


# -------------------------------------------------------------- the calls --

def _keep(s, name, make):
    """What a program makes once and keeps: its rotation, its workspace."""
    if name not in s["kept"]:
        s["kept"][name] = make()
    return s["kept"][name]


def _own_rope(m, s):
    c = s["case"]
    if c["scaling"] == "yarn":  # the ramp is this file's, by turns, not what a type's name stands for
        f, factor = _frequencies(c["rot"], "yarn")
        return _keep(s, "rope", lambda: m.Rope(rotary_dim=c["rot"], layout=c["layout"], frequencies=f, factor=factor))
    scaling = None if c["scaling"] == "none" else {"type": c["scaling"], "factor": 4.0}
    return _keep(s, "rope", lambda: m.Rope(rotary_dim=c["rot"], theta=1e7, layout=c["layout"], scaling=scaling))


def _run_own(s):
    import moe_infer_amd as m

    c = s["case"]
    if c["op"] == "rope":
        return m.rope_apply(s["x"], s["positions"], _own_rope(m, s), norm_w=s.get("q_w"),
                            out_dtype=_TYPES["f16" if c["dtype"] == "f32" else c["dtype"]])
    if c["op"] == "append":
        cu = None if c["q0"] == c["q1"] == 1 else s["cu_q"]
        q = m.paged_append(s["pages"], s["table"], s["kv_len"], s["k"], s["v"], rope=_own_rope(m, s), cu_q=cu,
                           q=s["q"], q_norm_w=s.get("q_w"), k_norm_w=s.get("k_w"))
        k, v = m.paged_read(s["pages"], s["table"], s["kv_len"], cu_q=cu, n=s["n"])
        return {"q": q, "k": k, "v": v}
    if c["op"] == "read":
        k, v = m.paged_read(s["pages"], s["table"], s["kv_len"], cu_q=s["cu_q"], n=s["n"])
        return {"k": k, "v": v}
    ws = _keep(s, "ws", lambda: m.paged_workspace(c["batch"], s["n"], s["max_q"], s["max_len"], c["H"], c["G"]))
    if c["op"] == "decode":
        return m.attn_decode_paged(s["pages"], s["table"], s["kv_len"], s["q"], s["max_len"], gate=s["gate"],
                                   workspace=ws)
    return m.attn_prefill_paged(s["pages"], s["table"], s["kv_len"], s["cu_q"], s["q"], s["max_q"], s["max_len"],
                                gate=s["gate"], workspace=ws)


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["op"] == "rope":
        y = _rotated(state["x"], state.get("q_w"), state["positions"], state)
        return y.to(_TYPES["f16" if c["dtype"] == "f32" else c["dtype"]])
    if c["op"] == "append":
        _, at = _token_rows(state)
        q = _rotated(state["q"], state.get("q_w"), at, state)
        k = _rotated(state["k"], state.get("k_w"), at, state)
        return {"q": q.half(), "k": _quantised(k), "v": _quantised(state["v"].double())}
    if c["op"] == "read":
        return _read_rows(state)
    return _attend(state)


# ------------------------------------------------------------ plain forms --

def _rotated(x, w, positions, s):
    """Norm and rotation; 64 bits, for far angles and for values next to the border of two codes."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
    rot = s["case"]["rot"]
    angle = positions.double()[:, None, None] * s["f"]
    cos, sin = torch.cos(angle) * s["factor"], torch.sin(angle) * s["factor"]
    if s["case"]["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


def _to_half(x):
    """x (64 bits) rounded once to f16: a cast goes by way of 32 bits and rounds twice."""
    bits = 11 - torch.frexp(x).exponent.clamp(min=-13)
    return torch.ldexp(torch.round(torch.ldexp(x, bits)), -bits).half()


def _quantised(x):
    """The values that the 4-bit codes of x [n, G, D] (64 bits) stand for."""
    g = x.reshape(*x.shape[:-1], D // 64, 64)
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = _to_half((high - low) / 15).double()
    offset = _to_half(low - 16 * scale).double()
    code = torch.where(scale > 0, torch.round((g - offset) / scale) - 16, 0 * g).clamp(0, 15)
    return _to_half((16 + code) * scale + offset).reshape(x.shape)


def _token_rows(s):
    """The sequence and the row of every token of the call."""
    new = s["cu_q"][1:] - s["cu_q"][:-1]
    seq = torch.repeat_interleave(torch.arange(new.numel(), device="cuda"), new, output_size=s["n"])
    return seq, (s["kv_len"] - new)[seq] + torch.arange(s["n"], device="cuda") - s["cu_q"][:-1][seq]


def _cached(s):
    """K and V of the whole block tables, [B, G, rows, D] f32."""
    pages, table = s["pages"], s["table"].long().clamp(min=0)
    B, M = table.shape
    G, T = pages.shape[1], pages.shape[2]
    tiles = pages[table].permute(0, 2, 1, 3, 4).reshape(B, G, M * T, TILE_BYTES)
    nibble = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    kc = (tiles[..., :4096].contiguous().view(torch.int32).unsqueeze(-1) >> nibble) & 15
    kc = kc.reshape(B, G, M * T, 2, 2, 4, 16, 2, 2, 8).permute(0, 1, 2, 3, 6, 4, 7, 5, 8, 9)
    kc = kc.reshape(B, G, M * T * 32, 4, 64)
    vc = (tiles[..., 4096:8192].contiguous().view(torch.int32).unsqueeze(-1) >> nibble) & 15
    vc = vc.reshape(B, G, M * T, 4, 4, 16, 4, 2, 4).permute(0, 1, 2, 7, 4, 8, 3, 5, 6)
    vc = vc.reshape(B, G, M * T * 32, 4, 64)
    ks = tiles[..., 8192:8704].contiguous().view(torch.float16).float().reshape(B, G, M * T * 32, 4, 2)
    vs = tiles[..., 8704:].contiguous().view(torch.float16).float().reshape(B, G, M * T, 4, 4, 2, 4, 2)
    vs = vs.permute(0, 1, 2, 7, 4, 6, 3, 5).reshape(B, G, M * T * 32, 4, 2)
    value = lambda code, so: ((16 + code) * so[..., :1] + so[..., 1:]).half().float().flatten(-2)  # noqa: E731
    return value(kc, ks), value(vc, vs)


def _read_rows(s):
    seq, at = _token_rows(s)
    k, v = _cached(s)
    return {"k": k[seq, :, at].half(), "v": v[seq, :, at].half()}


def _attend(s):
    c = s["case"]
    B, H, G, n, Q = c["batch"], c["H"], c["G"], s["n"], s["max_q"]
    R = H // G
    k, v = _cached(s)
    L = k.shape[2]
    seq, at = _token_rows(s)
    slot = torch.arange(n, device="cuda") - s["cu_q"][:-1][seq]
    q = torch.zeros(B, Q, H, D, device="cuda")
    q[seq, slot] = s["q"].float()
    last = torch.full((B, Q), -1, device="cuda", dtype=torch.long)
    last[seq, slot] = at
    q = q.reshape(B, Q, G, R, D).permute(0, 2, 1, 3, 4).reshape(B * G, Q * R, D)
    kt = k.reshape(B * G, L, D).transpose(1, 2).contiguous()
    score = torch.bmm(q, kt).reshape(B, G, Q, R, L) / 16
    seen = (torch.arange(L, device="cuda") <= last[:, None, :, None, None])
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(score - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.reshape(B * G, Q * R, L), v.reshape(B * G, L, D)).reshape(B, G, Q, R, D)
    o = torch.where(total > 0, o / torch.where(total > 0, total, 1.0), 0.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, Q, H, D)[seq, slot]
    if s["gate"] is not None:
        o = o / (1 + torch.exp(-s["gate"].float()))
    return o.half()


# ----------------------------------------------------------- what is needed --

def work(case):
    size = {"f16": 2, "bf16": 2, "f32": 4}.get(case.get("dtype"), 2)
    if case["op"] == "rope":
        e = case["n"] * case["heads"] * D
        return {"bytes": e * (size + 2) + 4 * case["n"], "flops": 6 * e}
    new, rows = _sizes(case)
    G, row = case["G"], TILE_BYTES / TILE_ROWS
    if case["op"] == "append":
        e = sum(new) * D
        return {"bytes": e * (case["H"] * (size + 2) + 2 * G * size) + sum(new) * G * (row + 4 * D),
                "flops": e * 10 * (case["H"] + 2 * G)}
    if case["op"] == "read":
        return {"bytes": sum(rows) * G * (row + 4 * D), "flops": sum(rows) * G * 4 * D}
    H = case["H"]
    pairs = sum(a * r - a * (a - 1) // 2 for a, r in zip(new, rows))
    return {"bytes": sum(rows) * G * row + sum(new) * H * D * (6 if case["gate"] else 4),
            "flops": 4 * D * H * pairs}


# ----------------------------------------------------------------- 64 bits --

def _exact_turned(x, w, pos, case):
    """Norm and rotation of x [n, heads, D] at positions pos, pair by pair with complex numbers."""
    x = x.to(torch.float64)
    if w is not None:
        x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / D + 1e-6) * w.to(torch.float64)
    rot, scaling = case["rot"], case["scaling"]
    i = np.arange(rot // 2, dtype=np.float64)
    base = 1e7 * 4.0 ** (rot / (rot - 2.0)) if scaling == "ntk" else 1e7
    f = np.exp(-2.0 * i / rot * np.log(base))
    factor = 1.0
    if scaling == "linear":
        f = f * 0.25
    elif scaling == "yarn":
        turns = 8192 * f / (2 * np.pi)
        f = f * np.interp(turns, [1.0, 32.0], [0.25, 1.0])
        factor = 0.1 * np.log(4.0) + 1.0
    pairs = np.arange(rot).reshape(2, -1).T if case["layout"] == "half" else np.arange(rot).reshape(-1, 2)
    angle = pos.to(torch.float64)[:, None] * torch.from_numpy(f).cuda()
    turn = torch.polar(torch.full_like(angle, factor), angle)[:, None]
    out = x.clone()
    z = torch.complex(x[..., pairs[:, 0]], x[..., pairs[:, 1]]) * turn
    out[..., pairs[:, 0]], out[..., pairs[:, 1]] = z.real, z.imag
    return out


def _exact_stored(x):
    """What 4 bits keep of x [n, G, D] in 64 bits."""
    g = x.cpu().numpy().reshape(-1, 64)
    lo, hi = g.min(1), g.max(1)
    scale = ((hi - lo) / 15).astype(np.float16).astype(np.float64)
    offset = (lo - 16 * scale).astype(np.float16).astype(np.float64)
    with np.errstate(all="ignore"):
        code = np.rint((g - offset[:, None]) / scale[:, None]) - 16
    code = np.clip(np.where(scale[:, None] > 0, code, 0), 0, 15)
    return torch.from_numpy(((16 + code) * scale[:, None] + offset[:, None]).reshape(x.shape))


def _exact_rows(s, seq, head, rows):
    """K and V [rows, D] of one sequence and KV head, value by value from the layout."""
    page, G = s["case"]["page"], s["case"]["G"]
    T = page // TILE_ROWS
    r = torch.arange(rows, device="cuda")
    tile = (s["table"][seq].long()[r // page] * G + head) * T + r % page // TILE_ROWS
    words = s["pages"].view(torch.int32).reshape(-1)
    halves = s["pages"].view(torch.float16).reshape(-1)
    w, c = (r % TILE_ROWS)[:, None], torch.arange(D, device="cuda")[None]
    sub, m, g = w // 16, w % 16, c // 64
    start = tile[:, None] * TILE_BYTES
    k = words[start // 4 + ((2 * sub + g // 2) * 64 + 16 * (c // 16 % 4) + m) * 4 + 2 * (g % 2) + c // 8 % 2]
    k = (k >> (4 * (c % 8))) & 15
    at = start // 2 + 4096 + 2 * (4 * w + g)
    k = ((16 + k) * halves[at].double() + halves[at + 1].double()).half().double()
    v = words[start // 4 + 1024 + (64 * g + 16 * (m // 4) + c % 64 // 4) * 4 + c % 4]
    v = (v >> (4 * (m % 4 + 4 * sub))) & 15
    at = start // 2 + 4352 + (4 * g + m // 4) * 16 + 2 * (m % 4) + sub
    v = ((16 + v) * halves[at].double() + halves[at + 8].double()).half().double()
    return k, v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_turned(s["x"], s.get("q_w"), s["positions"], case)
    new, rows = _sizes(case)
    if case["op"] == "append":
        pos = torch.from_numpy(np.concatenate([np.arange(r - a, r) for a, r in zip(new, rows)])).cuda()
        return {"q": _exact_turned(s["q"], s.get("q_w"), pos, case),
                "k": _exact_stored(_exact_turned(s["k"], s.get("k_w"), pos, case)),
                "v": _exact_stored(s["v"].double())}
    G = case["G"]
    if case["op"] == "read":
        each = [[_exact_rows(s, b, h, r) for h in range(G)] for b, r in enumerate(rows)]
        return {name: torch.cat([torch.stack([kv[i] for kv in of], 1) for of in each]).half()
                for i, name in enumerate(("k", "v"))}
    H = case["H"]
    R = H // G
    out = torch.zeros(s["n"], H, D, dtype=torch.float64, device="cuda")
    at = 0
    for b, (a, r) in enumerate(zip(new, rows)):
        for h in range(G):
            if not a or not r:
                continue
            k, v = _exact_rows(s, b, h, r)
            q = s["q"][at:at + a, h * R:(h + 1) * R].double().reshape(a * R, D)
            dots = q @ k.T.contiguous() / math.sqrt(D)
            limit = (r - a + torch.arange(a, device="cuda")).repeat_interleave(R)
            dots.masked_fill_(torch.arange(r, device="cuda")[None] > limit[:, None], -math.inf)
            out[at:at + a, h * R:(h + 1) * R] = (torch.softmax(dots, -1) @ v).reshape(a, R, D)
        at += a
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return out
