"""GPU parity of the device-resident batch (fa_paged_reserve_slots, fa_paged_tree_masks,
fa_paged_append_slots, fa_paged_tree_attention, fa_paged_accept) against plain models in integers and
float64, alone and as the steps of a decoding loop, eager and replayed from a graph.

Tolerances. h is half a rounding step of the storage type relative to the value (bf16 2^-8, f16 2^-11,
f32 2^-24). A rotated value comes from two products and a sum in f32 of factors that are off by a few
2^-24 themselves, then one rounding: h |x| + 2^-21 (|e| + |o|). A score is a sum of D products in f32 of
a query kept to h^2 (or f32): off by at most B ((D + 16) 2^-24 + h^2), B = scale * sum |q k|. LSE takes
that and the sum of n probabilities in f32 (each off by 2^-21): n 2^-24 + 2^-20, and the rounding of its
own value and of the running maximum. O adds the rounding of each probability and of itself:
h (|O| + sum p |v|).
"""
import numpy as np
import pytest

import _batch_model as model
import flat_attention_amd as fa

pytestmark = pytest.mark.gpu

F32, F16, BF16 = fa.DTYPE_F32, fa.DTYPE_F16, fa.DTYPE_BF16
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
THETA = 10000.0


def i32(hip, x):
    return fa.DeviceBuffer.from_array(hip, np.ascontiguousarray(x, np.int32))


def storage(x, dtype):
    """Values rounded to the storage type, as float64, and their stored form."""
    st = fa.host_storage(np.ascontiguousarray(x, np.float32), dtype)
    return fa.storage_to_f32(st.ravel(), dtype).reshape(x.shape).astype(np.float64), st


def load(buf, shape, dtype):
    raw = buf.download(fa.storage_np_dtype(dtype), int(np.prod(shape)))
    return fa.storage_to_f32(raw, dtype).reshape(shape).astype(np.float64)


def paged(rng, tokens, page, spare=3, width=None):
    """Tables over a shuffled pool for `tokens` rows of each sequence: (table, pages)."""
    need = [-(-int(t) // page) for t in tokens]
    total = sum(need) + spare
    ids = rng.permutation(total)
    table = np.full((len(need), width or max(1, max(need))), -1, np.int32)
    at = 0
    for s, m in enumerate(need):
        table[s, :m] = ids[at:at + m]
        at += m
    return table, total, ids[at:]


def drafts(rng, n, most, wide=8):
    """Random trees of at most `most` tokens: (parents, lengths), the first tree full."""
    lens = rng.integers(1, most + 1, n)
    lens[0] = most
    at = np.arange(most)
    return np.maximum(at - rng.integers(1, wide + 1, (n, most)), -1).astype(np.int32), lens


# ------------------------------------------------------------------------------- reservation

def _reserve(hip, table, ctx, new, mapped, free, count, max_new, page, pages, inplace):
    n, width = table.shape
    t, c, nl, m, f, k = (i32(hip, x) for x in (table, ctx, new, mapped, free, [count]))
    granted, slots = i32(hip, np.full(n, 77)), i32(hip, np.full((n, max_new), 77))
    out = {} if inplace else {"mapped_out": i32(hip, np.full(n, 77)), "free_count_out": i32(hip, [77])}
    batch = fa.HipPagedBatch(hip, t, c, n, width, page, pages)
    batch.reserve(nl, max_new, m, f, k, granted, slots, **out)
    mo, ko = out.get("mapped_out", m), out.get("free_count_out", k)
    if not inplace:
        assert np.array_equal(m.download(np.int32, n), mapped)
        assert k.download(np.int32, 1)[0] == count
    return {"table": t.download(np.int32, n * width).reshape(n, width),
            "ctx": c.download(np.int32, n), "mapped": mo.download(np.int32, n),
            "free": f.download(np.int32, len(free)), "count": ko.download(np.int32, 1)[0],
            "granted": granted.download(np.int32, n),
            "slots": slots.download(np.int32, n * max_new).reshape(n, max_new)}


def _compare(got, want):
    for k, w in want.items():
        assert np.array_equal(got[k], w), k


@pytest.mark.parametrize("inplace", [True, False])
@pytest.mark.parametrize("n,max_new,page,high,short,seed", [
    (1, 1, 16, 0, 1.0, 0), (1, 1, 16, 500, 1.0, 1), (3, 7, 5, 60, 1.0, 2), (64, 32, 16, 300, 0.5, 3),
    (65, 3, 1, 40, 0.3, 4), (300, 9, 16, 100, 0.7, 5), (1024, 8, 16, 64, 1.0, 6),
    (1030, 4, 16, 64, 0.6, 7), (2500, 20, 8, 50, 0.8, 8), (40, 2100, 16, 200, 0.6, 9),
    (2, 5000, 64, 100, 1.0, 10)])
def test_reserve_matches_the_model(hip, n, max_new, page, high, short, seed, inplace):
    """Some sequences end, some ask for nothing or too much, and the free pages cover `short` of what
    is asked."""
    rng = np.random.default_rng(seed)
    ctx = rng.integers(0, high + 1, n)
    mapped = -(-ctx // page) + rng.integers(0, 2, n)
    new = rng.integers(0, max_new + 1, n)
    width = int(max(mapped.max(), np.quantile(-(-(ctx + new) // page), 0.98), 1))
    table, pages, spare = paged(rng, mapped * page, page, spare=1 + n * (1 + max_new // page), width=width)
    if n > 2:
        new[rng.random(n) < 0.15] = -1
        new[rng.integers(0, n)] = max_new + 1
    wanted = int(np.maximum(-(-(ctx + np.maximum(new, 0)) // page) - mapped, 0).sum())
    count = min(spare.size, int(short * wanted) + 1)
    free = np.concatenate([spare[:count], np.full(int(mapped.sum()) + 1, -5)])
    want = model.reserve(table, ctx, new, mapped, free, count, max_new, page, pages)
    _compare(_reserve(hip, table, ctx, new, mapped, free, count, max_new, page, pages, inplace), want)


@pytest.mark.parametrize("n", [5, 1500])
def test_ended_sequences_with_many_pages(hip, n):
    """Rows of up to 700 pages go back on the stack, and the others take some of them at once."""
    rng = np.random.default_rng(n)
    mapped = np.where(rng.random(n) < 0.1, rng.integers(1, 701, n), 1)
    mapped[1] = 700
    new = np.where(mapped > 1, -1, 30)
    table, pages, spare = paged(rng, mapped, 1, width=702, spare=3)
    free = np.concatenate([spare, np.full(int(mapped.sum()), -5)])
    args = (table, np.minimum(mapped, 1), new, mapped, free, spare.size, 30, 1, pages)
    _compare(_reserve(hip, *args, True), model.reserve(*args))


def test_reserve_with_arrays_that_hold_nonsense(hip):
    """Negative lengths, mapped counts and free counts out of range, pages outside the pool, a stack too
    short for what comes back: those take no part, nothing else changes."""
    page, pages, width, max_new = 4, 20, 5, 6
    ctx = np.array([-3, 2147483647, 7, 3, 4, 0])
    new = np.array([2, 6, 2147483647, -2147483648, 3, 6])
    mapped = np.array([0, 3, -4, 99, 1, 0])
    table = np.arange(30).reshape(6, 5) - 3
    free = np.array([1, 2, 50, -9, 4, 5, 6, 7])
    for count in (6, -2, 1000):
        c = min(max(count, 0), free.size)
        want = model.reserve(table, ctx, new, mapped, free, c, max_new, page, pages)
        _compare(_reserve(hip, table, ctx, new, mapped, free, count, max_new, page, pages, False), want)


# ------------------------------------------------------------------------------- masks

@pytest.mark.parametrize("n,most,wide", [(1, 1, 1), (1, 64, 1), (3, 65, 4), (5, 7, 8), (2, 512, 1),
                                         (4, 512, 40), (200, 33, 3), (70, 256, 8)])
def test_tree_masks_match_a_walk(hip, n, most, wide):
    rng = np.random.default_rng(most)
    parents, lens = drafts(rng, n, most, wide)
    ctx = rng.integers(0, 100000, n)
    if n > 2:  # parents that are no earlier token, lengths out of range
        parents[1, rng.integers(0, most)] = most
        parents[2, most // 2] = -2
        if most > 3:
            parents[2, 3] = 3
    if n > 4:
        lens[3], lens[4], ctx[n - 1] = most + 1, 0, -1
    words = (most + 63) // 64
    masks, pos = fa.DeviceBuffer(hip, n * most * words * 8), i32(hip, np.full((n, most), 77))
    masks.fill_u32(0xffffffff)
    batch = fa.HipPagedBatch(hip, None, i32(hip, ctx), n, 1, 1, 1)
    batch.tree_masks(i32(hip, parents), i32(hip, lens), most, masks, pos)
    seen, want = model.tree(parents, lens, ctx, most)
    assert np.array_equal(pos.download(np.int32, n * most).reshape(n, most), want)
    assert np.array_equal(masks.download(np.uint64, n * most * words).reshape(n, most, words),
                          model.pack(seen))


# ------------------------------------------------------------------------------- append

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,most,page,hkv,D,rope,positions", [
    (1, 1, 16, 1, 8, True, False), (3, 7, 5, 2, 64, True, True), (2, 40, 16, 3, 80, True, False),
    (4, 33, 24, 8, 128, True, True), (5, 19, 16, 4, 40, False, False)])
def test_append_writes_the_slots_and_nothing_else(hip, dtype, n, most, page, hkv, D, rope, positions):
    rng = np.random.default_rng(most + D)
    ctx, new = rng.integers(0, 70, n), rng.integers(0, most + 1, n)
    table, pages, _ = paged(rng, ctx + most, page)
    rows = [(table[s, (c + np.arange(most)) // page].astype(np.int64) * page
             + (c + np.arange(most)) % page) for s, c in enumerate(ctx)]
    slots = np.where(np.arange(most) < new[:, None], np.array(rows), -1)
    if n > 2:
        slots[1, 0] = pages * page  # outside the pool
        slots[2, 0] = -2147483648
    pos = ctx[:, None] + rng.integers(0, 4, (n, most)) if positions else ctx[:, None] + np.arange(most)
    if positions:
        pos[0, 0] = -1  # no position: left out when rotating
        pos[0, 1] = table.shape[1] * page
    k, ks = storage(rng.standard_normal((n, most, hkv, D)), dtype)
    v, vs = storage(rng.standard_normal((n, most, hkv, D)), dtype)
    kp, kps = storage(rng.standard_normal((pages * page, hkv, D)), dtype)
    vp, vps = storage(rng.standard_normal((pages * page, hkv, D)), dtype)
    bufs = [fa.DeviceBuffer.from_array(hip, x) for x in (ks, vs, kps, vps)]
    batch = fa.HipPagedBatch(hip, None, i32(hip, ctx), n, table.shape[1], page, pages)
    off = 1000
    batch.append(i32(hip, slots), most, *bufs, hkv, D,
                 fa.RotaryEmbeddingConfig(THETA, off) if rope else None, dtype,
                 positions=i32(hip, pos) if positions else None)
    tol = np.zeros(kp.shape)
    for s in range(n):
        for t in range(most):
            r = int(slots[s, t])
            if not 0 <= r < pages * page or (rope and not 0 <= pos[s, t] < table.shape[1] * page):
                continue
            vp[r] = v[s, t]
            kp[r] = model.rotate(k[s, t][None], [pos[s, t] + off], THETA)[0] if rope else k[s, t]
            if rope:
                size = np.abs(k[s, t, :, 0::2]) + np.abs(k[s, t, :, 1::2])
                tol[r] = HALF_STEP[dtype] * np.abs(kp[r]) + 2.0 ** -21 * np.repeat(size, 2, -1)
                if dtype == F16:
                    tol[r] += 2.0 ** -25  # half a step of the smallest numbers
    assert np.array_equal(load(bufs[3], vp.shape, dtype), vp)
    assert (np.abs(load(bufs[2], kp.shape, dtype) - kp) <= tol).all()


# ------------------------------------------------------------------------------- attention

class Case:
    """Inputs of an attention call over a shuffled pool, its buffers and its float64 result."""

    def __init__(self, hip, dtype, ctx, lens, most, hq, hkv, D, page, seed, tree=True, rope=True,
                 scale=None, offset=0, magnitude=1.0, nan_outside=True, wide=5):
        self.hip, self.dtype, self.most, self.dims = hip, dtype, most, (hq, hkv, D)
        rng = np.random.default_rng(seed)
        self.ctx, self.lens, self.page = np.asarray(ctx), np.asarray(lens), page
        n = len(ctx)
        fit = [c + m if 0 <= c < 1 << 20 and 0 <= m <= most else 0 for c, m in zip(ctx, lens)]
        self.table, self.pages, _ = paged(rng, fit, page)
        self.q, qs = storage(magnitude * rng.standard_normal((n, most, hq, D)), dtype)
        rows = self.pages * page
        self.k, self.ks = storage(rng.standard_normal((rows, hkv, D)), dtype)
        self.v, self.vs = storage(rng.standard_normal((rows, hkv, D)), dtype)
        live = np.zeros(rows, bool)
        for s in range(n):
            live[self.rows(s, fit[s])] = True
        if nan_outside:  # rows that are nobody's: not a number
            nan = fa.host_storage(np.array([np.nan], np.float32), dtype)[0]
            self.ks[~live] = nan
            self.vs[~live] = nan
        self.seen, self.pos, self.masks = None, None, None
        at = np.arange(most)
        self.sees = np.broadcast_to(np.tril(np.ones((most, most), bool)), (n, most, most))
        self.where = self.ctx[:, None] + at
        if tree:
            parents, _ = drafts(rng, n, most, wide)
            self.sees, self.where = model.tree(parents, self.lens, self.ctx, most)
            self.masks, self.pos = model.pack(self.sees), self.where
        self.scale, self.offset, self.rope = scale, offset, rope
        self.bufs = [fa.DeviceBuffer.from_array(hip, x) for x in (qs, self.ks, self.vs)]
        self.batch = fa.HipPagedBatch(hip, i32(hip, self.table), i32(hip, self.ctx), n,
                                      self.table.shape[1], page, self.pages)
        self.len_buf = i32(hip, self.lens)
        self.lay = self.batch.layout(most, hq, D, dtype)
        self.out = fa.DeviceBuffer(hip, self.lay.combined_bytes)

    def rows(self, s, count):
        at = np.arange(count)
        return self.table[s, at // self.page].astype(np.int64) * self.page + at % self.page

    def upload(self):
        for buf, x in zip(self.bufs[1:], (self.ks, self.vs)):
            buf.upload(x)

    def call(self, upload=True):
        hq, hkv, D = self.dims
        if upload:
            self.keep = (None if self.masks is None else fa.DeviceBuffer.from_array(self.hip, self.masks),
                         None if self.pos is None else i32(self.hip, self.pos))
        m, p = self.keep
        self.batch.tree_attention(
            *self.bufs, self.out, self.len_buf, self.most, hq, hkv, D,
            fa.FlatAttentionConfig(True, self.scale),
            fa.RotaryEmbeddingConfig(THETA, self.offset) if self.rope else None, self.dtype,
            positions=p, masks=m)

    def get(self):
        hq, hkv, D = self.dims
        n = len(self.ctx)
        r = fa.download_attention(self.out, self.lay, self.dtype)
        o = fa.storage_to_f32(r.output, self.dtype).reshape(n, self.most, hq, D)
        return o, r.lse.reshape(n, hq, self.most)

    def run(self):
        self.out.fill_u32(0x7fc07fc0)
        self.call()
        return self.get()

    def check(self, only=None):
        """Every row (or those of sequences `only`) against float64."""
        o, lse = self.run()
        hq, hkv, D = self.dims
        scale = self.scale if self.scale is not None else float(np.float32(1) / np.sqrt(np.float32(D)))
        h = HALF_STEP[self.dtype]
        for s in range(len(self.ctx)) if only is None else only:
            c, m = int(self.ctx[s]), int(self.lens[s])
            ok = c >= 0 and 0 <= m <= self.most and c + m <= self.table.shape[1] * self.page
            m = m if ok else 0
            sees = np.ones((m, c + m if ok else 0), bool)
            if ok:
                sees[:, c:] = self.sees[s, :m, :m]
            at = self.rows(s, c + m if ok else 0)
            q = self.q[s, :m]
            if self.rope:
                q = model.rotate(q, self.where[s, :m] + self.offset, THETA)
                sees = sees & (self.where[s, :m] >= 0)[:, None]
            eo, el, av, size = model.attend(q, self.k[at], self.v[at], sees, scale)
            n = sees.shape[1]
            assert (o[s, m:] == 0).all() and (lse[s, :, m:] == -np.inf).all()
            ds = size * ((D + 16) * 2.0 ** -24 + (h * h if self.dtype != F32 and self.rope else 0))
            empty = el == -np.inf
            assert np.array_equal(np.isneginf(lse[s, :, :m]), empty), s
            assert (o[s, :m][empty.T] == 0).all()
            tl = ds + n * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * (np.abs(np.where(empty, 0, el)) + size)
            err = np.abs(np.where(empty, 0, lse[s, :, :m] - np.where(empty, 0, el)))
            assert (err <= tl).all(), (s, (err / tl).max())
            to = h * (np.abs(eo) + av) + (2 * ds.T[..., None] + n * 2.0 ** -23 + 2.0 ** -19) * av
            if self.dtype == F16:
                to = to + 2.0 ** -25
            err = np.abs(o[s, :m] - eo)
            assert (err <= to).all(), (s, (err / np.maximum(to, 1e-30)).max())
        return o, lse


SHAPES = [  # context lengths, tree lengths, most, q heads, kv heads, head dim, page
    ([0], [1], 1, 1, 1, 64, 16),
    ([1], [1], 1, 4, 1, 128, 16),
    ([63, 0, 5], [3, 5, 0], 5, 4, 2, 64, 16),
    ([200, 17, 64], [7, 16, 1], 16, 8, 2, 128, 16),
    ([31, 32, 33, 96], [33, 31, 1, 32], 33, 4, 4, 64, 5),
    ([1000, 3, 257], [13, 2, 9], 13, 6, 2, 128, 24),
    ([513, 90], [64, 40], 64, 16, 2, 128, 16),
    ([129], [70], 70, 3, 1, 40, 1),
    ([700, 129], [130, 65], 130, 2, 1, 96, 32),
    ([40], [512], 512, 2, 2, 32, 16),
    ([2500, 11], [4, 4], 4, 12, 12, 80, 64),
    ([300, 150, 1], [3, 2, 3], 3, 40, 1, 64, 8),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("tree,rope", [(True, True), (False, True), (True, False)])
def test_tree_attention_matches_float64(hip, dtype, shape, tree, rope):
    ctx, lens, most, hq, hkv, D, page = SHAPES[shape]
    Case(hip, dtype, ctx, lens, most, hq, hkv, D, page, 100 + shape, tree, rope,
         offset=37 if shape % 2 else 0, scale=0.2 if shape % 3 == 0 else None).check()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("page,ctx,hq,hkv,most", [(1, 5000, 4, 2, 9), (2, 2600, 2, 2, 65),
                                                  (16, 20000, 2, 1, 3)])
def test_more_table_entries_than_are_held_at_a_time(hip, dtype, page, ctx, hq, hkv, most):
    Case(hip, dtype, [ctx, 3, ctx // 2], [most, 1, most - 1], most, hq, hkv, 64, page, 7).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,most", [(70, 3), (300, 2), (700, 1)])
def test_many_sequences(hip, dtype, n, most):
    """More sequences than a workgroup has threads; some without drafted tokens."""
    rng = np.random.default_rng(n)
    lens = rng.integers(0, most + 1, n)
    case = Case(hip, dtype, rng.integers(0, 90, n), lens, most, 4, 2, 32, 16, 8)
    case.check()


@pytest.mark.parametrize("dtype,most,hq,hkv", [(BF16, 1, 8, 8), (F32, 1, 8, 8), (F16, 9, 8, 4), (BF16, 40, 8, 4),
                                               (F32, 20, 8, 4), (BF16, 65, 8, 2)])
def test_long_and_short_sequences_share_the_ranges(hip, dtype, most, hq, hkv):
    """Enough keys that a range holds several steps: ranges that cover short sequences whole, end in
    their start, and cut long ones in parts."""
    rng = np.random.default_rng(most)
    ctx = np.where(rng.random(40) < 0.5, rng.integers(0, 60, 40), rng.integers(1000, 3200, 40))
    Case(hip, dtype, ctx, rng.integers(0, most + 1, 40), most, hq, hkv, 64, 16, 12).check()


@pytest.mark.parametrize("dtype,ctx,lens,most,hq,hkv,D,page", [
    (BF16, [70, 9], [5, 2], 5, 8, 8, 8, 16), (F16, [70, 9], [40, 2], 40, 8, 4, 8, 3),
    (F32, [70, 9], [5, 2], 5, 4, 4, 4, 16), (F32, [140, 9], [40, 1], 40, 4, 2, 4, 1),
    (BF16, [600], [512], 512, 16, 2, 64, 16), (F32, [100], [300], 300, 8, 2, 64, 16),
    (BF16, [5000], [512], 512, 1, 1, 128, 1 << 13), (F16, [40, 0], [3, 1], 3, 96, 1, 64, 16)])
def test_narrow_heads_and_many_rows(hip, dtype, ctx, lens, most, hq, hkv, D, page):
    Case(hip, dtype, ctx, lens, most, hq, hkv, D, page, 13).check()


def test_two_contexts_at_once(hip):
    """Two contexts of one GPU, their calls in turn and neither waited for: each has its own stream and
    workspaces, and gets what it gets alone."""
    other = fa.HipContext(0)
    try:
        cases = [Case(c, BF16, [2500, 3, 700], [9, 4, 6], 9, 8, 4, 64, 16, 14 + i)
                 for i, c in enumerate((hip, other))]
        alone = [c.check() for c in cases]
        for _ in range(5):
            for c in cases:
                c.out.fill_u32(0x7fc07fc0)
            for _ in range(4):
                for c in cases:
                    c.call(upload=False)
            for c, (o, lse) in zip(cases, alone):
                o1, l1 = c.get()
                assert np.array_equal(o, o1) and np.array_equal(lse, l1)
    finally:
        other.close()


def test_large_scores_and_empty_rows(hip):
    """Scores of hundreds (the running maximum moves), and a mask that leaves rows nothing."""
    for dtype in (BF16, F16, F32):
        Case(hip, dtype, [700, 33], [20, 12], 20, 8, 2, 128, 16, 9, magnitude=60.0).check()
        case = Case(hip, dtype, [0, 64, 0], [20, 18, 1], 20, 4, 2, 64, 16, 10)
        case.masks = np.zeros_like(case.masks)  # no token sees a drafted one
        case.sees = np.zeros_like(case.sees)
        o, lse = case.check()
        assert np.isneginf(lse[0]).all() and np.isfinite(lse[1, :, :18]).all()


def test_sequences_and_tokens_that_do_not_fit(hip):
    """Lengths out of range, positions outside the table: O = 0 and LSE = -inf there, the others as
    without them."""
    for dtype in (BF16, F32):
        ctx, lens = [40, -1, 2147483647, 40, 17, 60], [6, 3, 2, -2, 9, 8]
        case = Case(hip, dtype, ctx, lens, 8, 4, 2, 64, 16, 11)
        case.pos = case.pos.copy()
        case.pos[5, :3] = [-1, 5 * 16, 2147483647]  # (the table row holds 5 pages)
        case.where = np.where(case.pos < 5 * 16, case.pos, -1)
        assert case.table.shape[1] == 5
        o, lse = case.check()
        assert (o[1:5] == 0).all() and np.isneginf(lse[1:5]).all()
        assert (o[5, :3] == 0).all() and np.isneginf(lse[5, :, :3]).all()
        assert np.isfinite(lse[5, :, 3:]).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq,most", [(2, 6), (8, 30), (8, 70)])
def test_pages_outside_the_pool_are_as_if_masked(hip, dtype, hq, most):
    case = Case(hip, dtype, [300, 90], [most, most - 1], most, hq, 2, 64, 16, 12)
    for s, lp, page in ((0, 2, -1), (0, 11, case.pages), (1, 0, 2147483647), (1, 3, -2147483648)):
        case.table[s, lp] = page
    case.batch.block_tables.upload(case.table.astype(np.int32))
    o, lse = case.run()
    for s in range(2):
        c, m = int(case.ctx[s]), int(case.lens[s])
        keys = np.arange(c + m)
        there = (case.table[s, keys // 16] >= 0) & (case.table[s, keys // 16] < case.pages)
        sees = np.ones((m, c + m), bool)
        sees[:, c:] = case.sees[s, :m, :m]
        q = model.rotate(case.q[s, :m], case.where[s, :m], THETA)
        at = np.where(there, case.table[s, keys // 16], 0).astype(np.int64) * 16 + keys % 16
        eo, el, av, size = model.attend(q, case.k[at], case.v[at], sees & there, 64.0 ** -0.5)
        h = HALF_STEP[dtype]
        ds = size * (80 * 2.0 ** -24 + (h * h if dtype != F32 else 0)) + 2.0 ** -15
        assert (np.abs(lse[s, :, :m] - el) <= ds).all()
        assert (np.abs(o[s, :m] - eo) <= h * (np.abs(eo) + av) + 3 * ds.T[..., None] * av + 2.0 ** -25).all()


@pytest.mark.filterwarnings("ignore:invalid value")
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq,most,ctx", [(2, 6, 40), (8, 40, 500), (4, 64, 31), (16, 33, 2000)])
def test_special_values_reach_the_rows_that_see_them(hip, dtype, hq, most, ctx):
    """NaN and infinities in K and V of drafted rows and of the last live rows: rows that do not see the
    key are bitwise what they are without it; in those that do, a V value brings its own kind to its
    column, a K that is NaN all columns."""
    clean = Case(hip, dtype, [ctx, 5], [most, 2], most, hq, 2, 64, 16, 13)
    o0, l0 = clean.run()
    case = Case(hip, dtype, [ctx, 5], [most, 2], most, hq, 2, 64, 16, 13)
    group = hq // 2
    rows = case.rows(0, ctx + most)
    sees = np.ones((most, ctx + most), bool)
    sees[:, ctx:] = case.sees[0]
    vs = case.vs.reshape(case.v.shape)
    put = {x: fa.host_storage(np.array([x], np.float32), dtype)[0] for x in (np.nan, np.inf, -np.inf)}
    spots = [(ctx + most - 1, 0, 3, np.nan), (ctx + most // 2, 0, 3, np.inf), (ctx, 1, 9, np.inf),
             (ctx + most // 3, 1, 9, -np.inf), (ctx - 1, 1, 60, -np.inf), (ctx + 1, 0, 17, -np.inf)]
    want = np.zeros((most, hq, 64))
    for key, head, d, x in spots:
        vs[rows[key], head, d] = put[x]
        add = np.where(sees[:, key], x, 0.0)
        want[:, head * group:(head + 1) * group, d] += add[:, None]
    case.upload()
    o1, l1 = case.run()
    assert np.array_equal(l1.view(np.uint32), l0.view(np.uint32))
    hit = want != 0
    assert np.array_equal(o1[0][~hit].view(np.uint32), o0[0][~hit].view(np.uint32))
    assert np.array_equal(o1[1].view(np.uint32), o0[1].view(np.uint32))
    assert np.array_equal(o1[0][hit], want[hit], equal_nan=True)
    # K: a drafted token that not every row sees
    ks = case.ks.reshape(case.k.shape)
    case.vs[:] = clean.vs
    key = ctx + most // 2
    ks[rows[key], 1, 7] = put[np.nan]
    case.upload()
    o2, l2 = case.run()
    hit = np.zeros((most, hq), bool)
    hit[:, group:] = sees[:, key][:, None]
    assert np.isnan(o2[0][hit]).all() and np.isnan(l2[0].T[hit]).all()
    assert np.array_equal(o2[0][~hit].view(np.uint32), o0[0][~hit].view(np.uint32))
    assert np.array_equal(l2[0].T[~hit].view(np.uint32), l0[0].T[~hit].view(np.uint32))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_results_do_not_depend_on_page_order_or_repetition(hip, dtype):
    a = Case(hip, dtype, [900, 31, 400], [16, 9, 3], 16, 8, 2, 128, 16, 14)
    o0, l0 = a.run()
    for _ in range(3):
        o1, l1 = a.run()
        assert np.array_equal(o0, o1) and np.array_equal(l0, l1)
    # the same rows on other pages
    rng = np.random.default_rng(99)
    order = rng.permutation(a.pages)
    inv = np.argsort(order)
    ks, vs = (x.reshape(a.pages, -1)[order].reshape(x.shape) for x in (a.ks, a.vs))
    a.ks, a.vs = ks, vs
    a.upload()
    moved = np.where(a.table >= 0, inv[np.maximum(a.table, 0)], -1)
    a.batch.block_tables.upload(moved.astype(np.int32))
    o1, l1 = a.run()
    assert np.array_equal(o0, o1) and np.array_equal(l0, l1)


def test_single_tokens_match_the_paged_decode(hip):
    """One token a sequence without masks is the decode step of fa_paged_decode_*."""
    for dtype in (BF16, F16, F32):
        case = Case(hip, dtype, [511, 0, 2047, 76], [1] * 4, 1, 16, 4, 128, 16, 15, tree=False)
        o, lse = case.check()
        plan = fa.PagedDecodePlan(hip, case.table.clip(0), case.ctx + 1, 16, case.pages, 16, 4, 128,
                                  fa.FlatAttentionConfig(True), THETA, dtype)
        out = fa.DeviceBuffer(hip, plan.layout().combined_bytes)
        plan.launch(*case.bufs, out)
        r = fa.download_attention(out, plan.layout(), dtype)
        ref = fa.storage_to_f32(r.output, dtype).reshape(o.shape)
        assert np.abs(lse.reshape(-1) - r.lse).max() < 2e-5
        assert np.abs(o - ref).max() <= (4 * HALF_STEP[dtype] + 2e-6) * np.abs(ref).max()


# ------------------------------------------------------------------------------- accept

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("inplace", [True, False])
@pytest.mark.parametrize("n,most,width,page,hkv,D", [(1, 1, 1, 16, 1, 8), (6, 20, 9, 5, 2, 64),
                                                     (40, 64, 64, 16, 8, 128), (5, 512, 200, 24, 3, 40)])
def test_accept_moves_rows_like_the_model(hip, dtype, inplace, n, most, width, page, hkv, D):
    rng = np.random.default_rng(most)
    ctx, lens = rng.integers(0, 60, n), rng.integers(1, most + 1, n)
    table, pages, _ = paged(rng, ctx + lens, page)
    accepted = np.array([rng.integers(0, min(l, width) + 1) for l in lens])
    paths = np.full((n, width), -7)
    for s in range(n):
        paths[s, :accepted[s]] = np.sort(rng.permutation(lens[s])[:accepted[s]])
    if n > 4:  # what is no path, no length, no page
        k = 2
        accepted[0], lens[0] = k, max(lens[0], 3)
        paths[0, :k] = [1, 1]
        accepted[1] = lens[1] + 1 if lens[1] < width else -1
        accepted[2], paths[2, 0] = 1, lens[2]
        lens[3] = 600
        accepted[4], paths[4, 0] = 1, lens[4] - 1
        table[4, (ctx[4] + lens[4] - 1) // page] = pages
    rows = pages * page
    k, ks = storage(rng.standard_normal((rows, hkv * D)), dtype)
    v, vs = storage(rng.standard_normal((rows, hkv * D)), dtype)
    kb, vb = fa.DeviceBuffer.from_array(hip, ks), fa.DeviceBuffer.from_array(hip, vs)
    c = i32(hip, ctx)
    out = None if inplace else i32(hip, np.full(n, 77))
    batch = fa.HipPagedBatch(hip, i32(hip, table), c, n, table.shape[1], page, pages)
    batch.accept(i32(hip, paths), width, i32(hip, accepted), i32(hip, lens), kb, vb, hkv, D, dtype,
                 ctx_lens_out=out)
    ek, ev, ec = model.accept(k, v, table, ctx, paths, accepted, lens, page, pages, 512)
    assert np.array_equal((out or c).download(np.int32, n), ec)
    assert np.array_equal(load(kb, k.shape, dtype), ek)
    assert np.array_equal(load(vb, v.shape, dtype), ev)
    if out is not None:
        assert np.array_equal(c.download(np.int32, n), ctx)


# ------------------------------------------------------------------------------- the loop

class Loop:
    """A speculative decoding loop on the GPU beside its float64 model: requests come and go, every
    step drafts a tree, appends it, attends, and accepts a path."""

    def __init__(self, hip, dtype, seed):
        self.hip, self.dtype, self.n, self.most, self.page = hip, dtype, 3, 12, 8
        self.hq, self.hkv, self.D, self.width, self.pages, self.accept = 8, 2, 64, 12, 24, 5
        self.rng = np.random.default_rng(seed)
        n, most = self.n, self.most
        self.state = {"table": np.zeros((n, self.width), np.int64), "ctx": np.zeros(n, np.int64),
                      "mapped": np.zeros(n, np.int64), "count": self.pages,
                      "free": self.rng.permutation(self.pages)}
        s = self.state
        self.b = {k: i32(hip, np.atleast_1d(s[k])) for k in s}
        for name, shape in (("new", (n,)), ("granted", (n,)), ("slots", (n, most)),
                            ("parents", (n, most)), ("pos", (n, most)), ("paths", (n, self.accept)),
                            ("accepted", (n,))):
            self.b[name] = i32(hip, np.zeros(shape))
        self.b["masks"] = fa.DeviceBuffer(hip, n * most * 8)
        eb = 4 if dtype == F32 else 2
        self.k, self.v = (np.zeros((self.pages * self.page, self.hkv, self.D)) for _ in range(2))
        self.kp, self.vp = (fa.DeviceBuffer.from_array(hip, fa.host_storage(
            np.zeros(self.k.size, np.float32), dtype)) for _ in range(2))
        self.q, self.ks, self.vs = (fa.DeviceBuffer(hip, n * most * h * self.D * eb)
                                    for h in (self.hq, self.hkv, self.hkv))
        self.batch = fa.HipPagedBatch(hip, self.b["table"], self.b["ctx"], n, self.width, self.page,
                                      self.pages)
        self.lay = self.batch.layout(most, self.hq, self.D, dtype)
        self.out = fa.DeviceBuffer(hip, self.lay.combined_bytes)

    def enqueue(self):
        b, rot = self.b, fa.RotaryEmbeddingConfig(THETA, 0)
        self.batch.reserve(b["new"], self.most, b["mapped"], b["free"], b["count"], b["granted"],
                           b["slots"])
        self.batch.tree_masks(b["parents"], b["granted"], self.most, b["masks"], b["pos"])
        self.batch.append(b["slots"], self.most, self.ks, self.vs, self.kp, self.vp, self.hkv, self.D,
                          rot, self.dtype, positions=b["pos"])
        self.batch.tree_attention(self.q, self.kp, self.vp, self.out, b["granted"], self.most, self.hq,
                                  self.hkv, self.D, fa.FlatAttentionConfig(), rot, self.dtype,
                                  positions=b["pos"], masks=b["masks"])
        self.batch.accept(b["paths"], self.accept, b["accepted"], b["granted"], self.kp, self.vp,
                          self.hkv, self.D, self.dtype)

    def step(self, launch):
        n, most, rng, b, s = self.n, self.most, self.rng, self.b, self.state
        new = rng.integers(1, most + 1, n)
        new[rng.random(n) < 0.2] = -1
        parents, _ = drafts(rng, n, most, 4)
        q, qs = storage(rng.standard_normal((n, most, self.hq, self.D)), self.dtype)
        k, ks = storage(rng.standard_normal((n, most, self.hkv, self.D)), self.dtype)
        v, vs = storage(rng.standard_normal((n, most, self.hkv, self.D)), self.dtype)
        want = model.reserve(s["table"], s["ctx"], new, s["mapped"], s["free"], s["count"], most,
                             self.page, self.pages)
        granted, ctx = want["granted"], want["ctx"]
        seen, pos = model.tree(parents, granted, ctx, most)
        paths, accepted = np.zeros((n, self.accept), np.int64), np.zeros(n, np.int64)
        for i in range(n):
            if granted[i]:
                leaf = int(rng.integers(0, granted[i]))
                path = np.flatnonzero(seen[i, leaf])[:self.accept]
                accepted[i] = path.size
                paths[i, :path.size] = path
        for name, x in (("new", new), ("parents", parents), ("paths", paths), ("accepted", accepted)):
            b[name].upload(x.astype(np.int32))
        for buf, x in ((self.q, qs), (self.ks, ks), (self.vs, vs)):
            buf.upload(x)
        self.out.fill_u32(0x7fc07fc0)
        launch()
        # the model's step; K as the GPU rotated and rounded it is read back below
        assert np.array_equal(b["slots"].download(np.int32, n * most).reshape(n, most), want["slots"])
        assert np.array_equal(b["granted"].download(np.int32, n), granted)
        assert np.array_equal(b["pos"].download(np.int32, n * most).reshape(n, most), pos)
        r = fa.download_attention(self.out, self.lay, self.dtype)
        o = fa.storage_to_f32(r.output, self.dtype).reshape(n, most, self.hq, self.D)
        lse = r.lse.reshape(n, self.hq, most)
        for i in range(n):
            for t in range(int(granted[i])):
                row = want["slots"][i, t]
                x, _ = storage(model.rotate(k[i, t][None], [pos[i, t]], THETA)[0], self.dtype)
                self.k[row], self.v[row] = x, v[i, t]
        h = HALF_STEP[self.dtype]
        for i in range(n):
            c, m = int(ctx[i]), int(granted[i])
            at = np.arange(c + m)
            at = want["table"][i, at // self.page] * self.page + at % self.page
            sees = np.ones((m, c + m), bool)
            sees[:, c:] = seen[i, :m, :m]
            eo, el, av, size = model.attend(model.rotate(q[i, :m], pos[i, :m], THETA), self.k[at],
                                            self.v[at], sees, self.D ** -0.5)
            # (the model's K may be rounded to the other neighbour: another h of every score)
            ds = size * (80 * 2.0 ** -24 + 2 * h + 2.0 ** -20) + 2.0 ** -15
            assert (np.abs(lse[i, :, :m] - el) <= ds).all()
            assert (np.abs(o[i, :m] - eo) <= h * (np.abs(eo) + av) + 3 * ds.T[..., None] * av).all()
            assert (o[i, m:] == 0).all() and np.isneginf(lse[i, :, m:]).all()
        width = self.hkv * self.D
        k2, v2, ctx2 = model.accept(self.k.reshape(-1, width), self.v.reshape(-1, width), want["table"],
                                    ctx, paths, accepted, granted, self.page, self.pages, 512)
        self.k, self.v = k2.reshape(self.k.shape), v2.reshape(self.v.shape)
        want["ctx"] = ctx2
        assert np.array_equal(b["ctx"].download(np.int32, n), ctx2)
        assert b["count"].download(np.int32, 1)[0] == want["count"]
        assert np.array_equal(b["mapped"].download(np.int32, n), want["mapped"])
        got = load(self.kp, self.k.shape, self.dtype)
        size = np.abs(self.k[..., 0::2]) + np.abs(self.k[..., 1::2])
        assert (np.abs(got - self.k) <= 2 * h * np.abs(self.k) + 2.0 ** -20 * np.repeat(size, 2, -1)
                + 2.0 ** -24).all()
        assert np.array_equal(load(self.vp, self.v.shape, self.dtype), self.v)
        self.state = {x: want[x] for x in self.state}
        return ctx2


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decoding_loop_on_the_gpu(hip, dtype):
    loop = Loop(hip, dtype, 21)
    longest = 0
    for _ in range(25):
        longest = max(longest, int(loop.step(loop.enqueue).max()))
    assert longest > 2 * loop.page


def test_decoding_loop_replayed_from_a_graph(hip):
    """The five calls captured once: every replay reads the lengths that the one before it left. Eager
    calls of another shape, which use the same workspaces, run between the replays."""
    loop = Loop(hip, BF16, 22)
    loop.step(loop.enqueue)  # (sizes the context's workspaces and tables)
    other = Case(hip, BF16, [300, 20], [7, 3], 7, 8, 2, 64, 16, 16)
    o0, l0 = other.run()
    with hip.capture() as cap:
        loop.enqueue()
    with hip.capture() as cap2:
        other.call(upload=False)
    for i in range(8):
        loop.step(cap.graph.launch)
        other.out.fill_u32(0x7fc07fc0)
        if i % 2:
            other.call(upload=False)  # (the graph reads the same masks and positions)
        else:
            cap2.graph.launch()
        o1, l1 = other.get()
        assert np.array_equal(o0, o1) and np.array_equal(l0, l1)


def test_capture_refuses_calls_that_would_allocate(hip):
    ctx = fa.HipContext(0)
    try:
        case = Case(ctx, BF16, [300], [7], 7, 8, 2, 64, 16, 17)
        m, p = fa.DeviceBuffer.from_array(ctx, case.masks), i32(ctx, case.pos)
        with ctx.capture():
            with pytest.raises(fa.FlatHipError) as e:
                case.batch.tree_attention(*case.bufs, case.out, case.len_buf, 7, 8, 2, 64,
                                          fa.FlatAttentionConfig(), fa.RotaryEmbeddingConfig(THETA), BF16,
                                          positions=p, masks=m)
            assert e.value.variant == "GraphCapture"
        case.check()
    finally:
        ctx.close()


def test_telemetry_and_kernel_timing(hip):
    case = Case(hip, BF16, [300, 20], [7, 3], 7, 8, 2, 64, 16, 18)
    hip.set_kernel_timing(True)
    case.run()
    t = hip.last_telemetry()
    assert t.kernel_id == "TreeAttention" and t.query_rows == 32 and t.dispatch_count == 2
    for name in ("TreeAttention", "TreeCombine"):
        ms, launches = hip.kernel_timing(name)
        assert launches == 1 and 0 < ms < 10
    hip.set_kernel_timing(False)
