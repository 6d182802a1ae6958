"""The operators of long contexts, as calls whose speed is tracked: attention with a sliding window and
first tokens that stay visible (forward, backward, and over the paged cache), rows into a paged cache of
4-bit floats and back, and attention over that cache.

A case is a dict of plain values. `listed()` are the fixed cases, `draw(rng)` gives one more of the same
ranges, `prepare` makes what a program holds before the call, `run` is one pass (`own` false: elementary
torch operations in 32 bits; true: the library's calls), `exact` the same outputs in 64 bits and `work`
the bytes and operations that a pass cannot do without.

Key j is seen from position i if j <= i and (i - j < window or j < sinks). A 4-bit row holds, for every 32
values of a head, a scale 2^e with the least e for which all of them are below 7 * 2^e, and the nearest
multiples (0, 0.5, 1, 1.5, 2, 3, 4, 6, and their negatives) of it, ties to the even code.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA = 10000.0
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # A short prompt of a small model, f32: latency.
        {"name": "window_small_f32", "kind": "forward", "dtype": "f32", "batch": 1, "q_heads": 2,
         "kv_heads": 2, "seq": 128, "dim": 64, "window": 32, "sinks": 4},
        # A long prompt: the largest.
        {"name": "window_prompt_bf16", "kind": "forward", "dtype": "bf16", "batch": 1, "q_heads": 32,
         "kv_heads": 8, "seq": 8192, "dim": 128, "window": 1024, "sinks": 4},
        # Two prompts of an odd length, heads of an odd width, a window off every tile.
        {"name": "window_odd_f16", "kind": "forward", "dtype": "f16", "batch": 2, "q_heads": 16,
         "kv_heads": 4, "seq": 1999, "dim": 80, "window": 500, "sinks": 3},
        # The gradients of a training step.
        {"name": "window_grad_bf16", "kind": "backward", "dtype": "bf16", "batch": 1, "q_heads": 32,
         "kv_heads": 8, "seq": 4096, "dim": 128, "window": 1024, "sinks": 4},
        # The same for a small model in f32.
        {"name": "window_grad_f32", "kind": "backward", "dtype": "f32", "batch": 2, "q_heads": 4,
         "kv_heads": 2, "seq": 300, "dim": 64, "window": 64, "sinks": 1},
        # One token each for a full batch of long contexts.
        {"name": "window_single_bf16", "kind": "paged", "dtype": "bf16", "seqs": 64, "tokens": 1,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "low": 512, "high": 8192, "page": 16,
         "window": 1024, "sinks": 4, "rope": True},
        # Chunks of a few prompts behind what is cached, pages that do not divide a tile.
        {"name": "window_chunk_f16", "kind": "paged", "dtype": "f16", "seqs": 6, "tokens": 64,
         "q_heads": 16, "kv_heads": 4, "dim": 64, "low": 300, "high": 5000, "page": 24,
         "window": 700, "sinks": 5, "rope": True},
        # The rows of one short draft into the 4-bit cache and back.
        {"name": "fp4_rows_f16", "kind": "rows", "dtype": "f16", "seqs": 2, "new": 3, "kv_heads": 4,
         "dim": 64, "low": 300, "high": 900, "page": 16},
        # Prompt chunks of a batch, ragged lengths.
        {"name": "fp4_rows_bf16", "kind": "rows", "dtype": "bf16", "seqs": 48, "new": 512,
         "kv_heads": 8, "dim": 128, "low": 0, "high": 1024, "page": 16},
        # One token each for a full batch of long contexts: the 4-bit cache is read once.
        {"name": "fp4_single_bf16", "kind": "fp4", "dtype": "bf16", "seqs": 64, "tokens": 1,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "low": 512, "high": 8192, "page": 16,
         "tree": False, "window": 0, "sinks": 0, "rope": True},
        # Drafted trees over it.
        {"name": "fp4_tree_f16", "kind": "fp4", "dtype": "f16", "seqs": 16, "tokens": 24,
         "q_heads": 32, "kv_heads": 8, "dim": 64, "low": 512, "high": 6000, "page": 32, "tree": True,
         "window": 0, "sinks": 0, "rope": True},
        # A chain for one request with a window, f32 queries: latency.
        {"name": "fp4_chain_f32", "kind": "fp4", "dtype": "f32", "seqs": 1, "tokens": 5,
         "q_heads": 16, "kv_heads": 4, "dim": 128, "low": 1000, "high": 1000, "page": 16,
         "tree": False, "window": 600, "sinks": 4, "rope": True},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["forward", "forward", "backward", "backward", "paged", "paged", "rows", "fp4", "fp4"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([g for g in (1, 2, 3, 4, 4, 8) if g * hkv <= 32])
    window, sinks = _log(rng, 1, 4096), rng.choice([0, 1, 4, 4, 16, 100])
    if kind in ("forward", "backward"):
        most = (8192 if kind == "forward" else 4096) // (4 if dtype == "f32" else 1)
        seq = _log(rng, 1, most)
        batch = rng.choice([b for b in (1, 1, 2, 3) if b * hkv * group <= 32])
        return {"kind": kind, "dtype": dtype, "batch": batch, "q_heads": hkv * group,
                "kv_heads": hkv, "seq": seq, "dim": rng.choice([32, 64, 80, 96, 128, 128]),
                "window": window, "sinks": sinks}
    page = rng.choice([8, 16, 16, 24, 32, 64])
    dim = rng.choice([32, 64, 96, 128, 128])
    if kind == "rows":
        return {"kind": kind, "dtype": dtype, "seqs": _log(rng, 1, 48),
                "new": _log(rng, 1, 256 if dtype == "f32" else 512), "kv_heads": hkv, "dim": dim,
                "low": 0, "high": _log(rng, 16, 1024), "page": page}
    seqs = _log(rng, 1, 24)
    high = _log(rng, 64, 2048 if dtype == "f32" else 8192)
    tokens = _log(rng, 1, 16 if dtype == "f32" else 64)
    tree = kind == "fp4" and rng.random() < 0.4
    if kind == "fp4" and (tree or rng.random() < 0.5):
        window = sinks = 0
    case = {"kind": kind, "dtype": dtype, "seqs": seqs, "tokens": tokens, "q_heads": hkv * group,
            "kv_heads": hkv, "dim": dim, "low": high // 16, "high": high, "page": page,
            "window": window, "sinks": sinks, "rope": rng.random() < 0.7}
    if kind == "fp4":
        case["tree"] = tree
    return case


# ------------------------------------------------------------------------------- sizes

def _lengths(case):
    """(live tokens, new tokens) of each sequence, the same for every seed; the first has the most."""
    n, most = case["seqs"], case.get("new", case.get("tokens"))
    r = np.random.default_rng([n, most, case["low"], case["high"]])
    lens = r.integers(case["low"], case["high"] + 1, n).astype(np.int32)
    new = r.integers((most + 1) // 2, most + 1, n).astype(np.int32)
    new[0] = most
    return lens, new


def _row_bytes(case):
    codes = case["kv_heads"] * case["dim"] // 2
    return (codes + codes // 16 + 15) // 16 * 16


# ------------------------------------------------------------------------------- state

class _State:
    pass


_context = None


def _library():
    """The library and this process's context."""
    global _context
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "flat-attention_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import flat_attention_amd as fa
    if _context is None:
        _context = fa.HipContext(0)
    return fa, _context


def _device(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


def _parents(case, r):
    """Random trees: each token hangs on one of the few before it, some on the root's side."""
    _lens, new = _lengths(case)
    n, most = case["seqs"], case["tokens"]
    at = np.arange(most)
    parents = np.maximum(at[None, :] - r.integers(1, 9, (n, most)), -1)
    parents[at[None, :] >= new[:, None]] = -1
    return parents.astype(np.int32)


def _inputs(case, seed):
    """Host tables and device tensors by name, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = TORCH[case["dtype"]]
    hkv, d = case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    if case["kind"] in ("forward", "backward"):
        b, s = case["batch"], case["seq"]
        t = {"q": normal(b, case["q_heads"], s, d), "k": normal(b, hkv, s, d),
             "v": normal(b, hkv, s, d)}
        if case["kind"] == "backward":
            out = _forward(t["q"], t["k"], t["v"], case["window"], case["sinks"])
            t.update(dout=normal(b, case["q_heads"], s, d), o=out["o"], lse=out["lse"])
        return {}, t
    r = np.random.default_rng(int(seed))
    lens, new = _lengths(case)
    page, n = case["page"], case["seqs"]
    need = -(-(lens.astype(np.int64) + new) // page)
    total = int(need.sum()) + 7
    order = r.permutation(total).astype(np.int32)
    table = np.zeros((n, int(need.max())), np.int32)
    ends = np.cumsum(need)
    for i, m in enumerate(need):
        table[i, :m] = order[ends[i] - m:ends[i]]
    h = {"lens": lens, "new": new, "table": table, "total": total}
    if case.get("tree"):
        h["parents"] = _parents(case, r)
    if case["kind"] == "rows":
        shape = (total, page, _row_bytes(case))
        t = {x: torch.zeros(shape, dtype=torch.uint8, device="cuda") for x in ("k_pool", "v_pool")}
        t["k"], t["v"] = (normal(n, case["new"], hkv, d) for _ in range(2))
        return h, t
    t = {x: normal(total, page, hkv, d) for x in ("k_pool", "v_pool")}
    if case["kind"] == "fp4":
        t = {x: _pack(y.flatten(0, 1), _row_bytes(case)).view(total, page, -1) for x, y in t.items()}
    t["q"] = normal(n, case["tokens"], case["q_heads"], d)
    return h, t


def prepare(case, seed):
    st = _State()
    st.case = case
    h, st.t = _inputs(case, seed)
    st.d = {k: _device(x) for k, x in h.items() if isinstance(x, np.ndarray)}
    st.total = h.get("total", 0)
    if case["kind"] == "rows":
        st.d["slots"] = _slots(st.d["table"], st.d["lens"], st.d["new"], case["new"], case["page"])
    if case.get("tree"):
        st.d["masks"], st.d["positions"] = _tree(st.d["parents"], st.d["new"], st.d["lens"])
    if own:
        _handles(st)
    torch.cuda.synchronize()
    return st


def _handles(st):
    """What a program that uses the library keeps: buffers around its tensors, the batch, the outputs."""
    fa, ctx = _library()
    case, t, d, kind = st.case, st.t, st.d, st.case["kind"]
    dt = TORCH[case["dtype"]]
    st.dtype = {"f32": fa.DTYPE_F32, "f16": fa.DTYPE_F16, "bf16": fa.DTYPE_BF16}[case["dtype"]]

    def buffer(x):
        return fa.DeviceBuffer(ctx, x.numel() * x.element_size(), x.data_ptr(), owned=False)

    st.buf = {k: buffer(x) for k, x in {**d, **t}.items()}
    st.config = fa.FlatAttentionConfig(True)
    if case.get("window"):
        st.window = fa.AttentionWindow(case["window"], case["sinks"])
    else:
        st.window = None
    if kind in ("forward", "backward"):
        st.shape = fa.GroupedAttentionShape(case["batch"], case["q_heads"], case["kv_heads"],
                                            case["seq"], case["dim"])
        if kind == "backward":
            st.op = fa.HipGroupedBackwardRecomputePipeline(ctx, st.dtype)
            st.out = {"dq": torch.empty_like(t["q"]), "dk": torch.empty_like(t["k"]),
                      "dv": torch.empty_like(t["v"])}
            st.out_buf = {k: buffer(x) for k, x in st.out.items()}
            return
        st.op = fa.HipRotaryGroupedAttention(ctx, st.dtype)
        lse_shape = (case["batch"], case["q_heads"], case["seq"])
    else:
        st.batch = fa.HipPagedBatch(ctx, st.buf["table"], st.buf["lens"], case["seqs"],
                                    d["table"].shape[1], case["page"], st.total)
        if kind == "rows":
            st.out = {"k": torch.empty_like(t["k"]), "v": torch.empty_like(t["v"])}
            st.out_buf = {k: buffer(x) for k, x in st.out.items()}
            return
        st.rotary = fa.RotaryEmbeddingConfig(THETA, 0) if case["rope"] else None
        lse_shape = (case["seqs"], case["q_heads"], case["tokens"])
    rows = t["q"].numel() // case["dim"]
    lay = fa.packed_layout(t["q"].numel(), rows, st.dtype)
    st.packed = torch.empty(lay.combined_bytes, dtype=torch.uint8, device="cuda")
    st.packed_buf = buffer(st.packed)
    at = lay.lse_byte_offset
    st.out = {"o": st.packed[:lay.output_bytes].view(dt).view(t["q"].shape),
              "lse": st.packed[at:at + 4 * rows].view(torch.float32).view(lse_shape)}


# ------------------------------------------------------------------------------- one pass

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    case, b, kind = st.case, st.buf, st.case["kind"]
    if kind == "forward":
        st.op.forward_window(b["q"], b["k"], b["v"], st.shape, st.config, st.window, None,
                             out=st.packed_buf)
    elif kind == "backward":
        g = st.out_buf
        st.op.encode_window(b["q"], b["k"], b["v"], b["dout"], b["o"], b["lse"].ptr, g["dq"],
                            g["dk"], g["dv"], st.shape, st.config, st.window)
    elif kind == "rows":
        g = st.out_buf
        st.batch.append_fp4(b["slots"], case["new"], b["k"], b["v"], b["k_pool"], b["v_pool"],
                            case["kv_heads"], case["dim"], None, st.dtype)
        st.batch.read_fp4(b["slots"], case["new"], b["k_pool"], b["v_pool"], g["k"], g["v"],
                          case["kv_heads"], case["dim"], st.dtype)
    elif kind == "paged":
        st.batch.window_attention(b["q"], b["k_pool"], b["v_pool"], st.packed_buf, b["new"],
                                  case["tokens"], case["q_heads"], case["kv_heads"], case["dim"],
                                  st.config, st.window, st.rotary, st.dtype)
    else:
        st.batch.attention_fp4(b["q"], b["k_pool"], b["v_pool"], st.packed_buf, b["new"],
                               case["tokens"], case["q_heads"], case["kv_heads"], case["dim"],
                               st.config, st.rotary, st.dtype, positions=b.get("positions"),
                               masks=b.get("masks"), window=st.window)
    return st.out


def _run_plain(st):
    case, d, t, kind = st.case, st.d, st.t, st.case["kind"]
    if kind == "forward":
        return _forward(t["q"], t["k"], t["v"], case["window"], case["sinks"])
    if kind == "backward":
        return _backward(t["q"], t["k"], t["v"], t["dout"], t["o"], t["lse"], case["window"],
                         case["sinks"])
    if kind == "rows":
        rows = d["slots"].flatten().long()
        live = rows >= 0
        out = {}
        for x in ("k", "v"):
            pool = t[x + "_pool"].view(-1, t[x + "_pool"].shape[-1])
            pool[rows[live]] = _pack(t[x].flatten(0, 1)[live], pool.shape[1])
            back = _unpack(pool[rows.clamp(min=0)], case["kv_heads"], case["dim"])
            out[x] = (back * live[:, None, None]).view(t[x].shape).to(t[x].dtype)
        return out
    page = case["page"]
    pages = d["table"].long()
    if kind == "fp4":
        k, v = (_unpack(t[x][pages].flatten(1, 2).flatten(0, 1), case["kv_heads"], case["dim"])
                for x in ("k_pool", "v_pool"))
    else:
        k, v = (t[x][pages].float().flatten(0, 2) for x in ("k_pool", "v_pool"))
    n, keys = pages.shape[0], pages.shape[1] * page
    k, v = (x.view(n, keys, case["kv_heads"], case["dim"]).transpose(1, 2).contiguous()
            for x in (k, v))
    return _attend(t["q"], k, v, d["lens"], d["new"], d.get("masks"), d.get("positions"),
                   case["window"], case["sinks"], case["rope"])


# Both files of tracked operators stand by themselves, so the slots, masks, positions and rotation that
# the device-resident batch has are written out here as well.

def _slots(table, lens, granted, most, page):
    """Pool row of each new token of each sequence, -1 past its granted ones."""
    at = torch.arange(most, device=table.device)[None, :]
    logical = lens[:, None].long() + at
    pages = table.long().gather(1, (logical // page).clamp(max=table.shape[1] - 1))
    return torch.where(at < granted[:, None], pages * page + logical % page, -1).to(torch.int32)


def _tree(parents, counts, lens):
    """Bit masks of each token's ancestors and itself, and its position lens + depth."""
    n, most = parents.shape
    at = torch.arange(most, device=parents.device)
    live = at[None, :] < counts[:, None]
    step = (parents[:, :, None] == at[None, None, :]).float() + torch.eye(most, device=parents.device)
    step *= (live[:, :, None] & live[:, None, :]).float()
    seen = torch.linalg.matrix_power(step, most) > 0
    words = (most + 63) // 64
    bits = torch.nn.functional.pad(seen.long(), (0, words * 64 - most)).view(n, most, words, 64)
    masks = (bits << torch.arange(64, device=parents.device)).sum(-1)
    depth = seen.sum(-1).to(torch.int32) - 1
    return masks, torch.where(live, lens[:, None] + depth, -1).to(torch.int32)


def _rotate(x, positions):
    """Interleaved rotation of x [n, tokens, heads, dim] f32 at `positions` [n, tokens]; frequencies and
    angles are f32 numbers by definition."""
    dim = x.shape[-1]
    theta, width = np.float32(THETA), np.float32(dim)
    freq = np.array([theta ** (np.float32(-2.0) * np.float32(j) / width)
                     for j in range(dim // 2)], np.float32)
    angle = (positions.float()[..., None] * _device(freq))[:, :, None, :].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack((even * cos - odd * sin, even * sin + odd * cos), -1).flatten(-2)


def _hidden(i, j, window, sinks):
    """Where key j is not seen from position i."""
    return (j > i) | ((i - j >= window) & (j >= sinks))


def _scores(q, k, window, sinks):
    """[B, Hkv, G * S, S] f32 scores of q [B, Hq, S, D] and k [B, Hkv, S, D], -inf where not seen."""
    b, hq, s, d = q.shape
    x = q.float().view(b, k.shape[1], -1, d)
    out = (x @ k.float().transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    at = torch.arange(s, device=q.device)
    hide = _hidden(at[:, None], at[None, :], window, sinks)
    return out.view(b, k.shape[1], -1, s, s).masked_fill_(hide, -math.inf).view(b, k.shape[1], -1, s)


def _forward(q, k, v, window, sinks):
    s = _scores(q, k, window, sinks)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ v.float()) / total
    return {"o": o.view(q.shape).to(q.dtype), "lse": (m + torch.log(total)).view(q.shape[:3])}


def _backward(q, k, v, dout, o, lse, window, sinks):
    b, hkv, s, d = k.shape
    x, g = (y.float().view(b, hkv, -1, d) for y in (q, dout))
    delta = (dout.float() * o.float()).sum(-1).view(b, hkv, -1, 1)
    p = _scores(q, k, window, sinks).sub_(lse.view(b, hkv, -1, 1)).exp_()
    dv = p.transpose(2, 3).contiguous() @ g
    ds = (g @ v.float().transpose(2, 3).contiguous()).sub_(delta).mul_(p)
    del p
    scale = 1.0 / math.sqrt(d)
    dq = (ds @ k.float()) * scale
    dk = (ds.transpose(2, 3).contiguous() @ x) * scale
    return {"dq": dq.view(q.shape).to(q.dtype), "dk": dk.to(k.dtype), "dv": dv.to(v.dtype)}


def _pack(x, row_bytes):
    """Rows [n, heads, dim] as 4-bit rows [n, row_bytes]: the codes of all heads (the even one of a pair
    low), their scales, zeros up to a multiple of 16 bytes."""
    y = x.float().reshape(x.shape[0], -1, 32)
    top = y.abs().amax(-1)
    e = ((top.view(torch.int32) + 0x200000) >> 23) - 129
    e = e.clamp(-127, 125)
    y = y * ((127 - e) << 23).view(torch.float32)[..., None]
    a = y.abs()
    code = (a > 0.25).to(torch.uint8)
    code += (a >= 0.75)
    code += (a > 1.25)
    code += (a >= 1.75)
    code += (a > 2.5)
    code += (a >= 3.5)
    code += (a > 5.0)
    code += torch.signbit(y) * 8
    code = code.view(x.shape[0], -1, 2)
    codes = code[..., 0] | (code[..., 1] << 4)
    scales = (e + 127).to(torch.uint8)
    row = torch.cat([codes, scales], 1)
    return torch.nn.functional.pad(row, (0, row_bytes - row.shape[1]))


def _unpack(rows, heads, dim):
    """4-bit rows [n, row_bytes] as f32 [n, heads, dim]."""
    n, size = heads * dim // 2, heads * dim // 32
    codes = rows[:, :n]
    code = torch.stack((codes & 15, codes >> 4), -1).view(rows.shape[0], -1, 32)
    level = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=rows.device)
    exponent = rows[:, n:n + size].int()
    scale = torch.where(exponent > 0, exponent << 23, 0x400000).view(torch.float32)
    value = level[code.int()] * scale[..., None]
    return value.view(rows.shape[0], heads, dim)


def _attend(q, k, v, lens, counts, masks, positions, window, sinks, rope):
    """Attention of q [n, tokens, hq, dim] over keys [n, hkv, keys, dim] of which lens + counts live."""
    n, tokens, hq, dim = q.shape
    hkv, keys = k.shape[1:3]
    at = torch.arange(tokens, device=q.device)
    if positions is None:
        positions = lens[:, None] + at[None, :]
    x = q.float()
    if rope:
        x = _rotate(x, positions)
    x = x.view(n, tokens, hkv, hq // hkv, dim).permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, dim)
    j = torch.arange(keys, device=q.device)[None, :] - lens[:, None]  # [n, keys], new ones from 0
    if masks is not None:
        word = (j >> 6).clamp(0, masks.shape[2] - 1).long()[:, None, :].expand(-1, tokens, -1)
        bit = (masks.gather(2, word) >> (j & 63).long()[:, None, :]) & 1
        seen = (j < 0)[:, None, :] | (bit > 0)
    elif window:
        key = torch.arange(keys, device=q.device)[None, None, :]
        seen = ~_hidden((lens[:, None] + at[None, :])[:, :, None], key, window, sinks)
    else:
        seen = j[:, None, :] <= at[None, :, None]
    seen = seen & (j < counts[:, None])[:, None, :] & (at[None, :] < counts[:, None])[:, :, None]
    seen = seen[:, None, :, None, :].expand(-1, -1, -1, hq // hkv, -1).reshape(n, 1, -1, keys)
    s = (x @ k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(dim))
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m.masked_fill(m == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, 1.0)
    lse = (m + torch.log(total)).view(n, hkv, tokens, hq // hkv).permute(0, 1, 3, 2)
    o = o.view(n, hkv, tokens, hq // hkv, dim).permute(0, 2, 1, 3, 4)
    return {"o": o.reshape(q.shape).to(q.dtype), "lse": lse.reshape(n, hq, tokens)}


# ------------------------------------------------------------------------------- 64 bits

def _turned(x, positions):
    """x [rows, heads, dim] float64, row i rotated at positions[i]."""
    dim = x.shape[-1]
    exponent = np.float32(-2.0) * np.arange(dim // 2, dtype=np.float32) / np.float32(dim)
    freq = np.array([np.float32(THETA) ** e for e in exponent], np.float32)
    angle = (np.asarray(positions, np.float32)[:, None] * freq[None, :]).astype(np.float64)
    turn = torch.polar(torch.ones(angle.shape, dtype=torch.float64),
                       torch.from_numpy(angle)).to(x.device)
    pairs = torch.view_as_complex(x.reshape(*x.shape[:-1], dim // 2, 2).contiguous())
    return torch.view_as_real(pairs * turn[:, None, :]).reshape(x.shape)


def _nearest(x):
    """What each value of x [rows, heads, dim] (float64, host) becomes in 4 bits: the nearest level times
    2^e, of two as near the one with the even code."""
    y = x.reshape(-1, 32)
    top = np.abs(y).max(1)
    with np.errstate(divide="ignore"):
        e = np.where(top > 0, np.floor(np.log2(np.where(top > 0, top, 1.0) / 7.0)) + 1, -127)
    e = np.where(top >= 7.0 * np.exp2(e), e + 1, np.where(top < 7.0 * np.exp2(e - 1), e - 1, e))
    e = np.clip(e, -127, 125)
    scaled = np.abs(y) / np.exp2(e)[:, None]
    best, gap = np.zeros_like(scaled), scaled.copy()
    for code, level in enumerate(LEVELS[1:], 1):
        off = np.abs(scaled - level)
        take = (off < gap) | ((off == gap) & (code % 2 == 0))
        best, gap = np.where(take, level, best), np.where(take, off, gap)
    return (np.sign(y) * best * np.exp2(e)[:, None]).reshape(x.shape)


def _values(rows, heads, dim):
    """What 4-bit rows (uint8, host) stand for, float64 [n, heads, dim]."""
    flat = rows.reshape(rows.shape[0], -1).astype(np.int64)
    n = heads * dim // 2
    out = np.empty((flat.shape[0], heads * dim))
    levels = np.array(LEVELS)
    for half in range(2):
        code = (flat[:, :n] >> (4 * half)) & 15
        out[:, half::2] = np.where(code & 8, -1.0, 1.0) * levels[code & 7]
    scale = np.exp2(flat[:, n:n + heads * dim // 32] - 127.0)
    return (out.reshape(flat.shape[0], -1, 32) * scale[:, :, None]).reshape(-1, heads, dim)


def _exact_dense(case, t):
    b, hq, s, d = t["q"].shape
    group = hq // case["kv_heads"]
    i = torch.arange(s, device="cuda")
    near = i[:, None] - i[None, :]
    sees = (near >= 0) & ((near < case["window"]) | (i[None, :] < case["sinks"]))
    names = ["o", "lse"] if case["kind"] == "forward" else ["dq", "dk", "dv"]
    like = {"o": "q", "dq": "q", "dk": "k", "dv": "v"}
    out = {x: torch.zeros(t[like[x]].shape if x in like else (b, hq, s), dtype=torch.float64,
                          device="cuda") for x in names}
    for n in range(b):
        for h in range(hq):
            g = h // group
            q, k, v = t["q"][n, h].double(), t["k"][n, g].double(), t["v"][n, g].double()
            z = (q @ k.t().contiguous()) / math.sqrt(d)
            z = torch.where(sees, z, -math.inf)
            if case["kind"] == "forward":
                ln = torch.logsumexp(z, 1)
                out["lse"][n, h] = ln
                out["o"][n, h] = torch.exp(z - ln[:, None]) @ v
                continue
            w = torch.exp(z - t["lse"][n, h].double()[:, None])
            up = t["dout"][n, h].double()
            out["dv"][n, g] += w.t().contiguous() @ up
            pull = up @ v.t().contiguous() - (up * t["o"][n, h].double()).sum(1)[:, None]
            pull = pull * w / math.sqrt(d)
            out["dq"][n, h] = pull @ k
            out["dk"][n, g] += pull.t().contiguous() @ q
    return out


def exact(case, seed):
    kind = case["kind"]
    h, t = _inputs(case, seed)
    if kind in ("forward", "backward"):
        return _exact_dense(case, t)
    lens, new, page, hkv, dim = h["lens"], h["new"], case["page"], case["kv_heads"], case["dim"]
    if kind == "rows":
        out = {}
        for x in ("k", "v"):
            near = _nearest(t[x].double().cpu().numpy())
            near[np.arange(case["new"])[None, :] >= new[:, None]] = 0.0
            out[x] = torch.from_numpy(near)
        return out
    n, tokens, hq = t["q"].shape[:3]
    group = hq // hkv
    o = torch.zeros((n, tokens, hq, dim), dtype=torch.float64, device="cuda")
    lse = torch.full((n, hq, tokens), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(n):
        length, count = int(lens[i]), int(new[i])
        at, key = length + np.arange(count), np.arange(length + count)
        depth = np.arange(count)
        if case.get("tree"):
            sees = np.ones((count, length + count), bool)
            sees[:, length:] = False
            for j in range(count):
                if h["parents"][i, j] >= 0:
                    sees[j, length:] = sees[h["parents"][i, j], length:]
                sees[j, length + j] = True
                depth[j] = sees[j, length:].sum() - 1
        else:
            sees = key[None, :] <= at[:, None]
            if case["window"]:
                sees &= (at[:, None] - key[None, :] < case["window"]) | (key < case["sinks"])[None, :]
        q = t["q"][i, :count].double()
        if case["rope"]:
            q = _turned(q, length + depth)
        rows = torch.from_numpy(h["table"][i, key // page].astype(np.int64) * page + key % page).cuda()
        k, v = (t[x].flatten(0, 1)[rows] for x in ("k_pool", "v_pool"))
        if kind == "fp4":
            k, v = (torch.from_numpy(_values(x.cpu().numpy(), hkv, dim)).cuda() for x in (k, v))
        hide = torch.from_numpy(~sees).cuda()[:, None, :]
        for g in range(hkv):
            mine = slice(g * group, (g + 1) * group)
            s = (q[:, mine].reshape(-1, dim) @ k[:, g].double().t().contiguous()) / math.sqrt(dim)
            s = s.view(count, group, -1).masked_fill(hide, -math.inf)
            ln = torch.logsumexp(s, -1)
            w = torch.exp(s - ln[..., None]).reshape(count * group, -1)
            o[i, :count, mine] = (w @ v[:, g].double().contiguous()).view(count, group, dim)
            lse[i, mine, :count] = ln.t()
    return {"o": o, "lse": lse}


# ------------------------------------------------------------------------------- work

def work(case):
    """Every input read once, every output written once; two operations per multiply-add over the
    (position, key) pairs that are seen (of a tree's drafted ones only the tokens themselves count)."""
    kind, dim, size = case["kind"], case["dim"], TORCH[case["dtype"]].itemsize
    hkv, window, sinks = case["kv_heads"], case.get("window", 0), case.get("sinks", 0)
    if kind in ("forward", "backward"):
        upto = np.arange(1, case["seq"] + 1)
        past = np.maximum(upto - window, 0)
        pairs = int((upto - past + np.minimum(past, sinks)).sum()) * case["batch"] * case["q_heads"]
        q = case["batch"] * case["q_heads"] * case["seq"] * dim * size
        kv = case["batch"] * hkv * case["seq"] * dim * size
        lse = q // (dim * size) * 4
        if kind == "forward":
            return {"bytes": 2 * q + 2 * kv + lse, "flops": 4 * pairs * dim}
        return {"bytes": 4 * q + 4 * kv + lse, "flops": 10 * pairs * dim}
    lens, new = (x.astype(np.int64) for x in _lengths(case))
    n, four = case["seqs"], hkv * dim // 2 + hkv * dim // 32
    if kind == "rows":
        row = hkv * dim * size
        return {"bytes": int(new.sum()) * 2 * (2 * four + row + 8) + n * case["new"] * 2 * row,
                "flops": int(new.sum()) * 4 * hkv * dim}
    hq, tokens = case["q_heads"], case["tokens"]
    row = four if kind == "fp4" else hkv * dim * size
    first = np.maximum(lens + 1 - window, 0) if window else np.zeros_like(lens)
    rows = int((lens + new - first + np.minimum(first, sinks)).sum())
    if case.get("tree"):
        pairs = int((new * (lens + 1)).sum())
    else:
        t = np.arange(tokens)[None, :]
        upto = np.where(t < new[:, None], lens[:, None] + t + 1, 0)
        past = np.maximum(upto - window, 0) if window else np.zeros_like(upto)
        pairs = int((upto - past + np.minimum(past, sinks)).sum())
    nbytes = 2 * rows * row + int(new.sum()) * hq * dim * size + n * tokens * hq * (dim * size + 4)
    if case.get("tree"):
        nbytes += int(new.sum()) * (8 * ((tokens + 63) // 64) + 4)
    return {"bytes": nbytes, "flops": 4 * pairs * hq * dim}
