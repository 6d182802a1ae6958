"""The operators of a speculative decoding step over the paged cache, as calls whose speed is tracked:
slots reserved from request lengths, the masks and positions of drafted trees, the append of their K/V
rows, attention of the drafted tokens over the cache, and the move of the accepted rows.

A case is a dict of plain values. `listed()` are the fixed cases, `draw(rng)` gives one more of the same
ranges, `prepare` makes what a program holds before the call, `run` is one pass (`own` false: elementary
torch operations in 32 bits; true: the library's calls), `exact` the same outputs in 64 bits and `work`
the bytes and operations that a pass cannot do without.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA = 10000.0


def listed():
    return [
        # One sequence takes its next token: the smallest call, all latency.
        {"name": "reserve_one", "kind": "reserve", "seqs": 1, "new": 1, "low": 500, "high": 500,
         "page": 16, "ended": 0},
        # A large batch of prompts and chunks comes in while some requests have ended.
        {"name": "reserve_prompts", "kind": "reserve", "seqs": 256, "new": 2048, "low": 0,
         "high": 4096, "page": 16, "ended": 24},
        # The drafts of a few requests.
        {"name": "masks_small", "kind": "masks", "seqs": 4, "tokens": 24, "low": 64, "high": 2048},
        # Wide trees for a full batch.
        {"name": "masks_large", "kind": "masks", "seqs": 192, "tokens": 256, "low": 64,
         "high": 8192},
        # The rows of one small draft, f32.
        {"name": "append_draft_f32", "kind": "append", "dtype": "f32", "seqs": 1, "new": 7,
         "kv_heads": 4, "dim": 64, "low": 900, "high": 900, "page": 16, "rope": True},
        # Prompt chunks of a batch, K rotated on the way, ragged lengths.
        {"name": "append_chunks_bf16", "kind": "append", "dtype": "bf16", "seqs": 48, "new": 512,
         "kv_heads": 8, "dim": 128, "low": 0, "high": 1024, "page": 16, "rope": True},
        # The verification of a short chain for one request: latency.
        {"name": "attend_chain_f16", "kind": "attend", "dtype": "f16", "seqs": 1, "tokens": 5,
         "q_heads": 16, "kv_heads": 4, "dim": 64, "low": 1000, "high": 1000, "page": 16,
         "tree": False, "rope": True},
        # One token each for a full batch from tables that stay on the GPU: the cache is read once.
        {"name": "attend_single_bf16", "kind": "attend", "dtype": "bf16", "seqs": 64, "tokens": 1,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "low": 512, "high": 8192, "page": 16,
         "tree": False, "rope": True},
        # Trees of 64 drafted tokens for a batch of long contexts: the largest.
        {"name": "attend_tree_bf16", "kind": "attend", "dtype": "bf16", "seqs": 24, "tokens": 64,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "low": 512, "high": 8192, "page": 16,
         "tree": True, "rope": True},
        # Small trees in an f32 cache with pages of an odd size.
        {"name": "attend_tree_f32", "kind": "attend", "dtype": "f32", "seqs": 6, "tokens": 13,
         "q_heads": 16, "kv_heads": 4, "dim": 64, "low": 200, "high": 3000, "page": 24,
         "tree": True, "rope": True},
        # The accepted rows of one short draft.
        {"name": "accept_small_f16", "kind": "accept", "dtype": "f16", "seqs": 2, "tokens": 16,
         "accept": 4, "kv_heads": 4, "dim": 64, "low": 300, "high": 900, "page": 16},
        # A full batch accepts long paths.
        {"name": "accept_large_bf16", "kind": "accept", "dtype": "bf16", "seqs": 128, "tokens": 64,
         "accept": 16, "kv_heads": 8, "dim": 128, "low": 64, "high": 1024, "page": 16},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["reserve", "masks", "append", "attend", "attend", "attend", "accept"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    page = rng.choice([8, 16, 16, 24, 32, 64])
    hkv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 80, 128, 128])
    if kind == "reserve":
        seqs = _log(rng, 1, 256)
        return {"kind": kind, "seqs": seqs, "new": _log(rng, 1, 2048), "low": 0,
                "high": _log(rng, 16, 4096), "page": page, "ended": rng.randint(0, seqs // 4)}
    if kind == "masks":
        return {"kind": kind, "seqs": _log(rng, 1, 192), "tokens": _log(rng, 1, 256), "low": 0,
                "high": _log(rng, 16, 8192)}
    if kind == "append":
        return {"kind": kind, "dtype": dtype, "seqs": _log(rng, 1, 48),
                "new": _log(rng, 1, 256 if dtype == "f32" else 512), "kv_heads": hkv, "dim": dim,
                "low": 0, "high": _log(rng, 16, 1024), "page": page, "rope": rng.random() < 0.8}
    if kind == "accept":
        accept = _log(rng, 1, 16)
        return {"kind": kind, "dtype": dtype, "seqs": _log(rng, 1, 64 if dtype == "f32" else 128),
                "tokens": 2 * accept + rng.randint(0, 32), "accept": accept, "kv_heads": hkv,
                "dim": dim, "low": 0, "high": _log(rng, 16, 1024), "page": page}
    group = rng.choice([1, 2, 4, 4, 8])
    seqs = _log(rng, 1, 24)
    high = _log(rng, 64, 2048 if dtype == "f32" else 8192)
    tokens = _log(rng, 1, 16 if dtype == "f32" else 64)
    if hkv * group > 32:
        group = 32 // hkv
    return {"kind": kind, "dtype": dtype, "seqs": seqs, "tokens": tokens, "q_heads": hkv * group,
            "kv_heads": hkv, "dim": dim, "low": high // 16, "high": high, "page": page,
            "tree": rng.random() < 0.75, "rope": rng.random() < 0.75}


# ------------------------------------------------------------------------------- sizes

def _lengths(case):
    """(live tokens, new tokens) of each sequence, the same for every seed. The first has the most new
    ones; in a reservation some have none and the last `ended` sequences give their pages back."""
    n, most = case["seqs"], case.get("new", case.get("tokens"))
    r = np.random.default_rng([n, most, case["low"], case["high"]])
    lens = r.integers(case["low"], case["high"] + 1, n).astype(np.int32)
    new = r.integers((most + 1) // 2 if case["kind"] in ("attend", "accept") else 1, most + 1, n)
    new[0] = most
    if case["kind"] == "reserve":
        new[1:][r.random(n - 1) < 0.1] = 0
        if case["ended"]:
            new[n - case["ended"]:] = -1
    return lens, new.astype(np.int32)


def _paged(case):
    """(live tokens, new tokens, mapped pages, pages a table row holds, physical pages)."""
    lens, new = _lengths(case)
    page = case["page"]
    need = -(-(lens.astype(np.int64) + np.maximum(new, 0)) // page)
    mapped = -(-lens.astype(np.int64) // page) if case["kind"] == "reserve" else need
    return lens, new, mapped, int(max(1, need.max())), int(max(need.sum(), 1)) + 7


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
    back = r.integers(1, 9, (n, most))
    parents = np.maximum(at[None, :] - back, -1)
    parents[at[None, :] >= new[:, None]] = -1
    return parents.astype(np.int32)


def _table(case, r):
    _lens, _new, mapped, width, total = _paged(case)
    order = r.permutation(total).astype(np.int32)
    table = np.zeros((case["seqs"], width), np.int32)
    at = 0
    for i, m in enumerate(mapped):
        table[i, :m] = order[at:at + m]
        at += int(m)
    return table, order[at:], total


def _inputs(case, seed):
    """Host tables and device tensors by name, from the seed alone."""
    r = np.random.default_rng(int(seed))
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    lens, new = _lengths(case)
    kind, n = case["kind"], case["seqs"]
    h = {"lens": lens, "new": new}
    if kind in ("masks", "accept") or case.get("tree"):
        h["parents"] = _parents(case, r)
    if kind == "masks":
        return h, {}
    _l, _n, mapped, _width, _total = _paged(case)
    h["table"], free, h["total"] = _table(case, r)
    if kind == "reserve":
        # room for the pages that come back
        h["free"] = np.concatenate([free, np.full(int(mapped.sum()) + 1, -1, np.int32)])
        h["count"] = np.array([free.size], np.int32)
        h["mapped"] = mapped.astype(np.int32)
        return h, {}
    if kind == "accept":
        # a path starts at token 0 and goes on at tokens behind the rows it is moved to
        a = case["accept"]
        h["accepted"] = np.minimum(r.integers(0, a + 1, n), new // 2).astype(np.int32)
        h["accepted"][0] = a
        paths = np.zeros((n, a), np.int32)
        for i in range(n):
            k = int(h["accepted"][i])
            if k > 1:
                paths[i, 1:k] = np.sort(r.permutation(np.arange(k, int(new[i])))[:k - 1])
        h["paths"] = paths
    hkv, d, dt = case["kv_heads"], case["dim"], TORCH[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    t = {"k_pool": normal(h["total"], case["page"], hkv, d),
         "v_pool": normal(h["total"], case["page"], hkv, d)}
    if kind == "append":
        t["k"], t["v"] = (normal(n, case["new"], hkv, d) for _ in range(2))
    if kind == "attend":
        t["q"] = normal(n, case["tokens"], case["q_heads"], d)
    return h, t


def prepare(case, seed):
    st = _State()
    st.case = case
    h, st.t = _inputs(case, seed)
    st.d = {k: _device(x) for k, x in h.items() if isinstance(x, np.ndarray)}
    st.total = h.get("total", 0)
    kind, n = case["kind"], case["seqs"]
    dev = torch.device("cuda")
    if kind == "reserve":
        st.out = {"slots": torch.empty((n, case["new"]), dtype=torch.int32, device=dev),
                  "granted": torch.empty(n, dtype=torch.int32, device=dev),
                  "mapped": torch.empty(n, dtype=torch.int32, device=dev),
                  "count": torch.empty(1, dtype=torch.int32, device=dev)}
    elif kind == "masks":
        words = (case["tokens"] + 63) // 64
        st.out = {"masks": torch.empty((n, case["tokens"], words), dtype=torch.int64, device=dev),
                  "positions": torch.empty((n, case["tokens"]), dtype=torch.int32, device=dev)}
    elif kind == "append":
        st.d["slots"] = _slots(st.d["table"], st.d["lens"], st.d["new"], case["new"], case["page"])
    elif kind == "accept":
        st.out = {"lens": torch.empty(n, dtype=torch.int32, device=dev)}
    elif case["tree"]:
        st.d["masks"], st.d["positions"] = _tree(st.d["parents"], st.d["new"], st.d["lens"])
    if own:
        _handles(st)
    torch.cuda.synchronize()
    return st


def _handles(st):
    """What a program that uses the library keeps: the batch, and a buffer around each tensor."""
    fa, ctx = _library()
    case, d = st.case, st.d
    st.fa, st.ctx = fa, ctx

    def buffer(t):
        return fa.DeviceBuffer(ctx, t.numel() * t.element_size(), t.data_ptr(), owned=False)

    kind, n = case["kind"], case["seqs"]
    st.buf = {k: buffer(x) for k, x in {**d, **st.t}.items()}
    st.out_buf = {k: buffer(x) for k, x in getattr(st, "out", {}).items()}
    page, table = case.get("page", 1), d.get("table")
    if table is None:  # trees alone: lengths without a table
        st.batch = fa.HipPagedBatch(ctx, None, st.buf["lens"], n, 1, 1, 1)
        return
    st.batch = fa.HipPagedBatch(ctx, st.buf["table"], st.buf["lens"], n, table.shape[1], page,
                                st.total)
    if kind == "reserve":
        return
    st.dtype = {"f32": fa.DTYPE_F32, "f16": fa.DTYPE_F16, "bf16": fa.DTYPE_BF16}[case["dtype"]]
    st.rotary = fa.RotaryEmbeddingConfig(THETA, 0) if case.get("rope") else None
    if kind == "attend":
        rows = n * case["tokens"] * case["q_heads"]
        lay = fa.packed_layout(rows * case["dim"], rows, st.dtype)
        st.packed = torch.empty(lay.combined_bytes, dtype=torch.uint8, device="cuda")
        st.packed_buf = buffer(st.packed)
        st.o = st.packed[:lay.output_bytes].view(TORCH[case["dtype"]]).view(st.t["q"].shape)
        at = lay.lse_byte_offset
        st.lse = st.packed[at:at + 4 * rows].view(torch.float32).view(n, case["q_heads"],
                                                                     case["tokens"])
        st.config = fa.FlatAttentionConfig(True)


# ------------------------------------------------------------------------------- one pass

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    case, b, kind = st.case, st.buf, st.case["kind"]
    if kind == "reserve":
        o = st.out_buf
        st.batch.reserve(b["new"], case["new"], b["mapped"], b["free"], b["count"], o["granted"],
                         o["slots"], mapped_out=o["mapped"], free_count_out=o["count"])
        return {"table": st.d["table"], "lens": st.d["lens"], "free": st.d["free"], **st.out}
    if kind == "masks":
        o = st.out_buf
        st.batch.tree_masks(b["parents"], b["new"], case["tokens"], o["masks"], o["positions"])
        return st.out
    if kind == "append":
        st.batch.append(b["slots"], case["new"], b["k"], b["v"], b["k_pool"], b["v_pool"],
                        case["kv_heads"], case["dim"], st.rotary, st.dtype)
        return {"k": st.t["k_pool"], "v": st.t["v_pool"]}
    if kind == "accept":
        st.batch.accept(b["paths"], case["accept"], b["accepted"], b["new"], b["k_pool"],
                        b["v_pool"], case["kv_heads"], case["dim"], st.dtype,
                        ctx_lens_out=st.out_buf["lens"])
        return {"k": st.t["k_pool"], "v": st.t["v_pool"], **st.out}
    st.batch.tree_attention(b["q"], b["k_pool"], b["v_pool"], st.packed_buf, b["new"],
                            case["tokens"], case["q_heads"], case["kv_heads"], case["dim"],
                            st.config, st.rotary, st.dtype, positions=b.get("positions"),
                            masks=b.get("masks"))
    return {"o": st.o, "lse": st.lse}


def _run_plain(st):
    case, d, t, kind = st.case, st.d, st.t, st.case["kind"]
    if kind == "reserve":
        return _reserve(d["table"], d["lens"], d["new"], d["mapped"], d["free"], d["count"],
                        case["new"], case["page"])
    if kind == "masks":
        masks, positions = _tree(d["parents"], d["new"], d["lens"])
        return {"masks": masks, "positions": positions}
    if kind == "append":
        return _append(t["k_pool"], t["v_pool"], t["k"], t["v"], d["slots"], d["lens"],
                       case["rope"])
    if kind == "accept":
        return _accept(t["k_pool"], t["v_pool"], d["table"], d["lens"], d["paths"], d["accepted"])
    return _attend(t["q"], t["k_pool"], t["v_pool"], d["table"], d["lens"], d["new"],
                   d.get("masks"), d.get("positions"), case["rope"])


def _slots(table, lens, granted, most, page):
    """Pool row of each new token of each sequence, -1 past its granted ones."""
    at = torch.arange(most, device=table.device)[None, :]
    logical = lens[:, None].long() + at
    pages = table.long().gather(1, (logical // page).clamp(max=table.shape[1] - 1))
    return torch.where(at < granted[:, None], pages * page + logical % page, -1).to(torch.int32)


def _reserve(table, lens, new, mapped, free, count, most, page):
    """Pages for lens + new tokens of each sequence from the top of the free stack, in sequence order;
    those of ended sequences (new < 0) go on the stack first."""
    width, cap = table.shape[1], free.numel()
    ended = new < 0
    back = torch.where(ended, mapped, 0).long()
    push_at = count.long() + torch.cumsum(back, 0) - back
    col = torch.arange(width, device=table.device)[None, :]
    pushed = ended[:, None] & (col < mapped[:, None])
    where = torch.where(pushed, push_at[:, None] + col, cap)
    stack = torch.cat([free, free.new_zeros(1)])
    stack.scatter_(0, where.flatten(), table.flatten())
    top = count.long() + back.sum()
    need = ((lens + new.clamp(min=0)).long() + page - 1) // page
    fits = need <= width
    need = torch.where(ended | (new == 0) | ~fits, 0, (need - mapped).clamp(min=0))
    upto = torch.cumsum(need, 0)
    ok = (new > 0) & fits & ((need == 0) | (upto <= top))
    granted = torch.where(ok, new, 0)
    take = torch.where(ok, need, 0)
    index = col - mapped[:, None]
    taken = (index >= 0) & (index < take[:, None])
    source = (top - 1 - (upto - need)[:, None] - index).clamp(0, cap)
    table.copy_(torch.where(taken, stack[source.flatten()].view_as(table), table))
    free.copy_(stack[:-1])
    lens.copy_(torch.where(ended, 0, lens))
    return {"table": table, "lens": lens, "free": free,
            "slots": _slots(table, lens, granted, most, page), "granted": granted,
            "mapped": torch.where(ended, 0, mapped + take).to(torch.int32),
            "count": (top - take.sum()).to(torch.int32).view(1)}


def _tree(parents, counts, lens):
    """Bit masks of each token's ancestors and itself, and its position lens + depth."""
    n, most = parents.shape
    at = torch.arange(most, device=parents.device)
    live = at[None, :] < counts[:, None]
    eye = torch.eye(most, device=parents.device)
    step = (parents[:, :, None] == at[None, None, :]).float() + eye
    step *= (live[:, :, None] & live[:, None, :]).float()
    for _ in range(max(1, (most - 1).bit_length())):
        step = ((step @ step) > 0).float()
    words = (most + 63) // 64
    bits = torch.nn.functional.pad(step, (0, words * 64 - most)).view(n, most, words, 64).long()
    masks = (bits << torch.arange(64, device=parents.device)).sum(-1)
    depth = step.sum(-1).to(torch.int32) - 1
    return masks, torch.where(live, lens[:, None] + depth, -1).to(torch.int32)


def _angles(positions, dim):
    """cos and sin [..., dim / 2]: frequencies and angles are f32 numbers by definition."""
    theta, width = np.float32(THETA), np.float32(dim)
    freq = np.array([theta ** (np.float32(-2.0) * np.float32(j) / width)
                     for j in range(dim // 2)], np.float32)
    angle = positions.float()[..., None] * _device(freq)
    return torch.cos(angle.double()).float(), torch.sin(angle.double()).float()


def _rotate(x, positions):
    """Interleaved rotation of x [n, tokens, heads, dim] f32 at `positions` [n, tokens]."""
    cos, sin = (a[:, :, None, :] for a in _angles(positions, x.shape[-1]))
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack((even * cos - odd * sin, even * sin + odd * cos), -1).flatten(-2)


def _append(k_pool, v_pool, k, v, slots, lens, rope):
    positions = lens[:, None] + torch.arange(k.shape[1], device=k.device)[None, :]
    if rope:
        k = _rotate(k.float(), positions).to(k_pool.dtype)
    live = slots.flatten() >= 0
    rows = slots.flatten()[live].long()
    k_pool.view(-1, *k.shape[2:])[rows] = k.flatten(0, 1)[live]
    v_pool.view(-1, *v.shape[2:])[rows] = v.flatten(0, 1)[live]
    return {"k": k_pool, "v": v_pool}


def _accept(k_pool, v_pool, table, lens, paths, accepted):
    page = k_pool.shape[1]
    at = torch.arange(paths.shape[1], device=paths.device)[None, :]
    live = (at < accepted[:, None]).flatten()

    def rows(logical):
        pages = table.long().gather(1, (logical // page).clamp(max=table.shape[1] - 1))
        return (pages * page + logical % page).flatten()[live]

    source, target = rows(lens[:, None].long() + paths), rows(lens[:, None].long() + at)
    k, v = k_pool.view(-1, *k_pool.shape[2:]), v_pool.view(-1, *v_pool.shape[2:])
    k[target], v[target] = k[source], v[source]
    return {"k": k_pool, "v": v_pool, "lens": lens + accepted}


def _attend(q, k_pool, v_pool, table, lens, counts, masks, positions, rope):
    n, tokens, hq, dim = q.shape
    page, hkv = k_pool.shape[1:3]
    keys = table.shape[1] * page
    at = torch.arange(tokens, device=q.device)
    if positions is None:
        positions = lens[:, None] + at[None, :]
    x = q.float()
    if rope:
        x = _rotate(x, positions)
    x = x.view(n, tokens, hkv, hq // hkv, dim).permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, dim)
    k, v = (p[table.long()].view(n, keys, hkv, dim).float().transpose(1, 2).contiguous()
            for p in (k_pool, v_pool))
    j = torch.arange(keys, device=q.device)[None, :] - lens[:, None]  # [n, keys], drafts from 0
    if masks is None:
        seen = j[:, None, :] <= at[None, :, None]
    else:
        word = (j >> 6).clamp(0, masks.shape[2] - 1).long()[:, None, :].expand(-1, tokens, -1)
        bit = (masks.gather(2, word) >> (j & 63).long()[:, None, :]) & 1
        seen = (j < 0)[:, None, :] | (bit > 0)
    seen &= (j < counts[:, None])[:, None, :] & (at[None, :] < counts[:, None])[:, :, None]
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


def exact(case, seed):
    kind = case["kind"]
    if kind in ("reserve", "masks"):
        return None  # whole numbers only
    h, t = _inputs(case, seed)
    page, table, lens, new = case["page"], h["table"], h["lens"], h["new"]

    def rows(i, first, count):
        logical = np.arange(first, first + count)
        return torch.from_numpy(table[i, logical // page].astype(np.int64) * page
                                + logical % page).cuda()

    k, v = (t[x].double().flatten(0, 1) for x in ("k_pool", "v_pool"))
    if kind == "append":
        for i in range(case["seqs"]):
            first, count = int(lens[i]), int(new[i])
            at = rows(i, first, count)
            fresh = t["k"][i, :count].double()
            k[at] = _turned(fresh, np.arange(first, first + count)) if case["rope"] else fresh
            v[at] = t["v"][i, :count].double()
        return {"k": k.view(t["k_pool"].shape), "v": v.view(t["v_pool"].shape)}
    if kind == "accept":
        for i in range(case["seqs"]):
            for j in range(int(h["accepted"][i])):
                to, of = rows(i, int(lens[i]) + j, 1), rows(i, int(lens[i]) + int(h["paths"][i, j]), 1)
                k[to], v[to] = k[of], v[of]
        return {"k": k.view(t["k_pool"].shape), "v": v.view(t["v_pool"].shape), "lens": None}
    n, tokens, hq, dim = t["q"].shape
    group = hq // case["kv_heads"]
    o = torch.zeros((n, tokens, hq, dim), dtype=torch.float64, device="cuda")
    lse = torch.full((n, hq, tokens), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(n):
        length, count = int(lens[i]), int(new[i])
        sees = np.ones((count, length + count), bool)
        depth = np.arange(count)
        sees[:, length:] = False
        for j in range(count):
            sees[j, length:] = sees[j - 1, length:] if j and not case["tree"] else False
            if case["tree"] and h["parents"][i, j] >= 0:
                sees[j, length:] = sees[h["parents"][i, j], length:]
            sees[j, length + j] = True
            depth[j] = sees[j, length:].sum() - 1
        q = t["q"][i, :count].double()
        if case["rope"]:
            q = _turned(q, length + depth)
        at = rows(i, 0, length + count)
        hide = torch.from_numpy(~sees).cuda()[:, None, :]
        for g in range(case["kv_heads"]):
            mine = slice(g * group, (g + 1) * group)
            s = (q[:, mine].reshape(-1, dim) @ k[at, g].t().contiguous()) / math.sqrt(dim)
            s = s.view(count, group, -1).masked_fill(hide, -math.inf)
            ln = torch.logsumexp(s, -1)
            w = torch.exp(s - ln[..., None]).reshape(count * group, -1)
            o[i, :count, mine] = (w @ v[at, g].contiguous()).view(count, group, dim)
            lse[i, mine, :count] = ln.t()
    return {"o": o, "lse": lse}


# ------------------------------------------------------------------------------- work

def work(case):
    """Every input read once, every output written once; two operations per multiply-add over the
    (token, key) pairs that are certain to be seen (a tree's tokens see the context and themselves)."""
    kind, n = case["kind"], case["seqs"]
    lens, new = (x.astype(np.int64) for x in _lengths(case))
    if kind == "masks":
        words = (case["tokens"] + 63) // 64
        return {"bytes": int(n * 8 + 4 * new.sum() + n * case["tokens"] * (8 * words + 4)),
                "flops": int(new.sum() * case["tokens"])}
    if kind == "reserve":
        _l, _n, mapped, _w, _t = _paged(case)
        fresh = np.where(new > 0, -(-(lens + np.maximum(new, 0)) // case["page"]) - mapped, 0).sum()
        back = mapped[new < 0].sum()
        return {"bytes": int(20 * n + 4 * n * case["new"] + 8 * (fresh + back)),
                "flops": int(2 * n * case["new"])}
    row = case["kv_heads"] * case["dim"] * TORCH[case["dtype"]].itemsize
    if kind == "append":
        return {"bytes": int(new.sum() * (4 * row + 4) + 4 * n), "flops": int(
            3 * new.sum() * case["kv_heads"] * case["dim"] if case["rope"] else 0)}
    if kind == "accept":
        moved = int(np.minimum(case["accept"] / 2, new / 2).sum())
        return {"bytes": int(4 * row * moved + 16 * n), "flops": 0}
    hq, dim, size = case["q_heads"], case["dim"], TORCH[case["dtype"]].itemsize
    pairs = int((new * lens + (new if case["tree"] else new * (new + 1) // 2)).sum())
    words = (case["tokens"] + 63) // 64
    nbytes = 2 * int((lens + new).sum()) * row + int(new.sum()) * hq * dim * size
    nbytes += n * case["tokens"] * hq * (dim * size + 4)
    nbytes += int(new.sum()) * (8 * words + 4) if case["tree"] else 0
    return {"bytes": nbytes, "flops": 4 * pairs * hq * dim}
