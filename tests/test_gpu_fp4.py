"""GPU parity of the 4-bit paged cache: rows in and out (fa_paged_append_slots_fp4, fa_paged_read_slots_fp4)
exactly, attention over it (fa_paged_attention_fp4) against float64, and both as steps of a decoding loop.

Tolerances of the attention. The 4-bit values are exact operands. A score is a sum in f32 of D products with
the parts of a query: two bf16 parts hold 2^-18 of a value (half a step of the second, 2^-8 of the first's
2^-8, is 2^-16 for the worst value, h_q), three all of an f32. LSE as in test_gpu_batch. A probability is
carried to e_p: one bf16 part 2^-8 (half a step is 2^-9 of the value; the bound counts a whole one as the others
do), two 2^-16, three 2^-24; O adds that and its own rounding, h |O| + e_p sum p |v|.
"""
import numpy as np
import pytest

import _batch_model as batch_model
import _window_model as model
import flat_attention_amd as fa
from test_gpu_batch import BF16, F16, F32, HALF_STEP, THETA, drafts, i32, load, paged, storage

pytestmark = pytest.mark.gpu

PARTS = {BF16: 2.0 ** -8, F16: 2.0 ** -16, F32: 2.0 ** -24}


def buf(hip, x):
    return fa.DeviceBuffer.from_array(hip, x)


# ------------------------------------------------------------------------------- rows

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,most,page,hkv,D", [(1, 1, 16, 1, 32), (3, 7, 5, 2, 64), (2, 40, 16, 3, 96),
                                               (4, 33, 24, 8, 128), (5, 19, 1, 5, 32)])
def test_rows_go_in_and_out_exactly(hip, dtype, n, most, page, hkv, D):
    rng = np.random.default_rng(most + D)
    pages = n * most + 3
    slots = rng.permutation(pages * page)[:n * most].reshape(n, most).astype(np.int64)
    if n > 2:
        slots[1, 0], slots[2, 0], slots[2, 1] = pages * page, -2147483648, -1
    x = rng.standard_normal((2, n, most, hkv, D)) * np.exp2(rng.integers(-20, 14, (2, n, most, hkv, 1)))
    levels = np.array([0, .25, .5, .75, 1.25, 1.5, 1.75, 2.5, 3.5, 5, 5.5, 6, 6.5, 3, 4, 2])
    x[0, 0, 0, 0, :32] = np.r_[levels, -levels]  # the borders between codes
    x[1, 0, 0, 0, :32] = 0.0
    x[1, 0, 0, 0, 1:32] = -0.0
    if n > 2:
        x[0, 2, 2, 0, 31], x[1, 0, 1, 1, 0] = np.inf, np.nan
        x[1, 2, 2, 0, :32] = np.linspace(-7, 7, 32)
        if dtype != F16:
            x[0, 1, 1, 0, :32] *= 2.0 ** -130 / np.abs(x[0, 1, 1, 0, :32]).max()
            x[0, 1, 2, 0, :32] = 3.3e38
    with np.errstate(over="ignore"):
        (k, ks), (v, vs) = (storage(y, dtype) for y in x)
    rb = fa.fp4_row_bytes(hkv, D)
    assert rb % 16 == 0 and rb >= hkv * D * 17 // 32
    pools = [buf(hip, rng.integers(0, 256, (pages * page, rb), np.uint8)) for _ in range(2)]
    want = [p.download(np.uint8, pages * page * rb).reshape(-1, rb) for p in pools]
    batch = fa.HipPagedBatch(hip, None, i32(hip, np.zeros(n)), n, max(1, most), page, pages)
    slot_buf = i32(hip, np.clip(slots, -2147483648, 2147483647))
    batch.append_fp4(slot_buf, most, buf(hip, ks), buf(hip, vs), *pools, hkv, D, None, dtype)
    ok = (slots >= 0) & (slots < pages * page)
    for p, w, y in zip(pools, want, (k, v)):
        w[slots[ok]] = model.to_rows(y[ok])
        assert np.array_equal(p.download(np.uint8, w.size).reshape(w.shape), w)
    out = [fa.DeviceBuffer(hip, x.nbytes) for x in (ks, vs)]
    for o in out:
        o.fill_u32(0x7fc07fc0)
    batch.read_fp4(slot_buf, most, *pools, *out, hkv, D, dtype)
    for o, w in zip(out, want):
        values = np.zeros((n, most, hkv, D))
        values[ok] = model.from_rows(w[slots[ok]], hkv, D)
        with np.errstate(over="ignore", invalid="ignore"):
            values = storage(values, dtype)[0]
        assert np.array_equal(load(o, values.shape, dtype), values, equal_nan=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rotated_rows_are_a_neighbouring_code_away_at_most(hip, dtype):
    """K is rotated in f32 (off by 2^-21 (|e| + |o|)): where that crosses no border the bytes are the model's;
    where it may, the value is at most a code from it."""
    rng = np.random.default_rng(3)
    n, most, page, hkv, D = 3, 50, 16, 4, 128
    ctx = rng.integers(0, 70, n)
    pages = 40
    slots = rng.permutation(pages * page)[:n * most].reshape(n, most)
    pos = ctx[:, None] + np.arange(most)
    pos[1, 3], pos[2, 0] = -1, 128 * page
    k, ks = storage(rng.standard_normal((n, most, hkv, D)), dtype)
    v, vs = storage(rng.standard_normal((n, most, hkv, D)), dtype)
    rb = fa.fp4_row_bytes(hkv, D)
    pools = [fa.DeviceBuffer(hip, pages * page * rb) for _ in range(2)]
    for p in pools:
        p.fill_u32(0)
    batch = fa.HipPagedBatch(hip, None, i32(hip, ctx), n, 128, page, pages)
    batch.append_fp4(i32(hip, slots), most, buf(hip, ks), buf(hip, vs), *pools, hkv, D,
                     fa.RotaryEmbeddingConfig(THETA, 9), dtype, positions=i32(hip, pos))
    got = [p.download(np.uint8, pages * page * rb).reshape(-1, rb) for p in pools]
    left = (pos >= 0) & (pos < 128 * page)
    assert not got[0][slots[~left]].any() and not got[1][slots[~left]].any()
    assert np.array_equal(got[1][slots[left]], model.to_rows(v[left]))
    turned = batch_model.rotate(k[left], pos[left] + 9, THETA)
    pair = np.repeat(np.abs(k[left]).reshape(*turned.shape[:-1], -1, 2).sum(-1), 2, -1)
    off = 2.0 ** -21 * pair
    bounds = [model.from_rows(model.to_rows(turned + s * off), hkv, D) for s in (-1, 1)]
    low, high = np.minimum(*bounds), np.maximum(*bounds)
    value = model.from_rows(got[0][slots[left]], hkv, D)
    # (a scale that changes with the largest value moves its group: those few groups are left to the bound)
    step = np.maximum(np.abs(bounds[0] - bounds[1]), 0)
    assert ((value >= low - step) & (value <= high + step)).mean() > 0.9999
    assert np.abs(value - turned).max() <= np.abs(turned).max()
    assert (value == bounds[0]).mean() > 0.9999


# ------------------------------------------------------------------------------- attention

class Case:
    def __init__(self, hip, dtype, ctx, lens, most, hq, hkv, D, page, seed=0, kind="tree", rope=True, window=None,
                 magnitude=1.0, scale=None, offset=0):
        rng = np.random.default_rng([seed, most, D])
        self.hip, self.dtype, self.most, self.dims = hip, dtype, most, (hq, hkv, D)
        self.ctx, self.lens, self.page = np.asarray(ctx), np.asarray(lens), page
        self.window = fa.AttentionWindow(*window) if window else None
        self.scale, self.rope, self.offset = scale, rope, offset
        n = len(ctx)
        fit = [c + m if 0 <= c < 1 << 20 and 0 <= m <= most else 0 for c, m in zip(ctx, lens)]
        self.table, self.pages, _ = paged(rng, fit, page)
        self.q, qs = storage(magnitude * rng.standard_normal((n, most, hq, D)), dtype)
        rows = self.pages * page
        self.kr, self.vr = (model.to_rows(np.float32(rng.standard_normal((rows, hkv, D))).astype(np.float64)
                                          * np.exp2(rng.integers(-2, 2, (rows, hkv, 1)))) for _ in range(2))
        live = np.zeros(rows, bool)
        for s in range(n):
            live[self.rows(s, fit[s])] = True
        self.kr[~live] = 255  # rows that are nobody's: NaN
        self.vr[~live] = 255
        self.values()
        at = np.arange(most)
        self.masks = None
        self.sees = np.broadcast_to(np.tril(np.ones((most, most), bool)), (n, most, most))
        self.where = self.ctx[:, None] + at
        if kind == "tree":
            parents, _ = drafts(rng, n, most, 5)
            self.sees, self.where = batch_model.tree(parents, self.lens, self.ctx, most)
            self.masks = buf(hip, batch_model.pack(self.sees))
        self.pos = i32(hip, self.where) if kind == "tree" else None
        self.bufs = [buf(hip, x) for x in (qs, self.kr, self.vr)]
        self.table_buf = i32(hip, self.table)
        self.batch = fa.HipPagedBatch(hip, self.table_buf, i32(hip, self.ctx), n, self.table.shape[1], page,
                                      self.pages)
        self.len_buf = i32(hip, self.lens)
        self.lay = self.batch.layout(most, hq, D, dtype)
        self.out = fa.DeviceBuffer(hip, self.lay.combined_bytes)

    def values(self):
        _, hkv, D = self.dims
        self.k, self.v = (model.from_rows(x, hkv, D) for x in (self.kr, self.vr))

    def rows(self, s, count):
        at = np.arange(count)
        return self.table[s, at // self.page].astype(np.int64) * self.page + at % self.page

    def call(self):
        hq, hkv, D = self.dims
        self.batch.attention_fp4(*self.bufs, self.out, self.len_buf, self.most, hq, hkv, D,
                                 fa.FlatAttentionConfig(True, self.scale),
                                 fa.RotaryEmbeddingConfig(THETA, self.offset) if self.rope else None,
                                 self.dtype, positions=self.pos, masks=self.masks, window=self.window)

    def get(self):
        hq, _, D = self.dims
        n = len(self.ctx)
        r = fa.download_attention(self.out, self.lay, self.dtype)
        o = fa.storage_to_f32(r.output, self.dtype).reshape(n, self.most, hq, D)
        return o, r.lse.reshape(n, hq, self.most)

    def seen(self, s):
        """(new tokens, [m, c + m] bool) of sequence s."""
        c, m = int(self.ctx[s]), int(self.lens[s])
        if c < 0 or not 0 <= m <= self.most or c + m > self.table.shape[1] * self.page:
            return 0, None
        if self.window:
            return m, model.sees(c + np.arange(m), c + m, self.window.window, self.window.sinks)
        see = np.ones((m, c + m), bool)
        see[:, c:] = self.sees[s, :m, :m]
        return m, see

    def check(self, skip_keys=None):
        self.out.fill_u32(0x7fc07fc0)
        self.call()
        o, lse = self.get()
        hq, hkv, D = self.dims
        h, ep = HALF_STEP[self.dtype], PARTS[self.dtype]
        scale = self.scale if self.scale is not None else model.resolved(D)
        for s in range(len(self.ctx)):
            m, see = self.seen(s)
            assert (o[s, m:] == 0).all() and (lse[s, :, m:] == -np.inf).all()
            if not m:
                continue
            c = int(self.ctx[s])
            at = self.rows(s, c + m)
            if skip_keys is not None:
                see = see & ~skip_keys(s, c + m)[None, :]
                at = np.where(skip_keys(s, c + m), 0, at)
            q = self.q[s, :m]
            if self.rope:
                q = batch_model.rotate(q, self.where[s, :m] + self.offset, THETA)
                see = see & (self.where[s, :m] >= 0)[:, None]
            k, v = (np.nan_to_num(x[at]) for x in (self.k, self.v))
            eo, el, av, size = batch_model.attend(q, k, v, see, scale)
            empty = el == -np.inf
            assert np.array_equal(np.isneginf(lse[s, :, :m]), empty), s
            assert (o[s, :m][empty.T] == 0).all()
            n = see.shape[1]
            ds = size * ((D + 16) * 2.0 ** -24 + (2.0 ** -16 if self.dtype != F32 else 0))
            tl = ds + n * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * (np.abs(np.where(empty, 0, el)) + size)
            err = np.abs(np.where(empty, 0, lse[s, :, :m] - np.where(empty, 0, el)))
            assert (err <= tl).all(), (s, (err / tl).max())
            to = h * np.abs(eo) + (ep + 2 * ds.T[..., None] + n * 2.0 ** -23 + 2.0 ** -19) * av
            if self.dtype == F16:
                to = to + 2.0 ** -25
            # n probabilities below 2^-126, the smallest normal f32, may be zero
            to = to + n * 2.0 ** -126 * np.abs(v).max()
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
    ([129], [70], 70, 3, 1, 32, 1),
    ([700, 129], [130, 65], 130, 2, 1, 96, 32),
    ([40], [512], 512, 2, 2, 32, 16),
    ([2500, 11], [4, 4], 4, 12, 12, 96, 64),
    ([300, 150, 1], [3, 2, 3], 3, 40, 1, 64, 8),
    ([260, 70], [3, 2], 3, 16, 8, 64, 16),
    ([515, 9], [5, 20], 20, 8, 8, 96, 24),
    ([1030, 31], [1, 1], 1, 12, 12, 32, 16),
    ([90, 333], [1, 1], 1, 16, 4, 96, 16),
    ([600, 5], [33, 7], 33, 8, 8, 128, 32),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("kind,rope", [("tree", True), ("chain", True), ("tree", False), ("window", True)])
def test_attention_matches_float64(hip, dtype, shape, kind, rope):
    Case(hip, dtype, *SHAPES[shape], seed=shape, kind=kind, rope=rope, offset=37 if shape % 2 else 0,
         scale=0.2 if shape % 3 == 0 else None,
         window=(1 + 37 * shape, [0, 4, 70][shape % 3]) if kind == "window" else None).check()


@pytest.mark.parametrize("dtype,most,hq,hkv", [(BF16, 1, 8, 8), (F32, 1, 8, 8), (F16, 9, 8, 4), (BF16, 40, 8, 4),
                                               (F32, 20, 6, 3), (BF16, 1, 14, 7)])
def test_long_and_short_sequences_share_the_ranges(hip, dtype, most, hq, hkv):
    rng = np.random.default_rng(most)
    ctx = np.where(rng.random(40) < 0.5, rng.integers(0, 60, 40), rng.integers(1000, 3200, 40))
    Case(hip, dtype, ctx, rng.integers(0, most + 1, 40), most, hq, hkv, 64, 16, 12).check()
    Case(hip, dtype, ctx, rng.integers(0, most + 1, 40), most, hq, hkv, 64, 16, 12, kind="window",
         window=(500, 4)).check()


@pytest.mark.parametrize("n,most", [(70, 3), (300, 2), (700, 1)])
def test_many_sequences(hip, n, most):
    rng = np.random.default_rng(n)
    Case(hip, BF16, rng.integers(0, 90, n), rng.integers(0, most + 1, n), most, 4, 2, 32, 16, 8).check()


def test_large_scores(hip):
    for dtype in (BF16, F16, F32):
        Case(hip, dtype, [700, 33], [20, 12], 20, 8, 2, 128, 16, 9, magnitude=60.0).check()


def test_sequences_that_do_not_fit_and_pages_outside_the_pool(hip):
    for dtype in (BF16, F32):
        Case(hip, dtype, [40, -1, 2147483647, 40, 17], [6, 3, 2, -2, 9], 8, 4, 2, 64, 16, 11).check()
        case = Case(hip, dtype, [100, 70], [5, 3], 5, 4, 2, 64, 16, 12)
        table = case.table.copy()
        gone = {(0, 2): -1, (0, 4): case.pages, (1, 0): 2147483647}
        for (s, p), x in gone.items():
            table[s, p] = x
        case.table_buf.upload(table)
        case.check(skip_keys=lambda s, n: np.isin(np.arange(n) // 16, [p for (t, p) in gone if t == s]))


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("kind", ["chain", "window"])
def test_nan_rows_reach_those_who_see_them_and_nobody_else(hip, which, kind):
    for dtype in (BF16, F16, F32):
        case = Case(hip, dtype, [300, 40], [40, 3], 40, 4, 2, 128, 16, 13, kind=kind,
                    window=(50, 2) if kind == "window" else None)
        base, lse0 = case.check()
        for row in (1, 280, 310):
            rows = (case.kr if which == "k" else case.vr).copy()
            rows[case.rows(0, 340)[row], 128 + 1 * 4 + 2] = 255  # a group of head 1
            case.bufs[1 if which == "k" else 2].upload(rows)
            case.call()
            o, lse = case.get()
            _, see = case.seen(0)
            hit = np.zeros(o.shape[:3], bool)
            hit[0, :40, 2:] = see[:, row][:, None]
            assert np.isnan(o[hit]).all()
            assert np.array_equal(o[~hit], base[~hit])
            assert np.array_equal(lse.transpose(0, 2, 1)[~hit], lse0.transpose(0, 2, 1)[~hit])


def test_scales_from_the_smallest_to_the_largest(hip):
    """V's scales range over what a sum holds: the largest key's value dominates, the others round away."""
    case = Case(hip, F32, [60], [1], 1, 2, 1, 64, 16, 14, rope=False)
    case.vr[:, 32:34] = np.random.default_rng(0).integers(60, 180, (case.vr.shape[0], 2))
    case.bufs[2].upload(case.vr)
    case.values()
    case.check()


@pytest.mark.parametrize("dtype,most,hq,hkv,D", [(BF16, 1, 16, 8, 128), (F16, 9, 8, 8, 64), (F32, 9, 8, 4, 128),
                                                 (F16, 3, 6, 3, 96)])
def test_two_contexts_at_once_give_the_same_bits_each_time(hip, dtype, most, hq, hkv, D):
    other = fa.HipContext(0)
    try:
        cases = [Case(c, dtype, [900, 3, 77, 2100], [most, 1, most, most], most, hq, hkv, D, 16, seed=5)
                 for c in (hip, other)]
        bits = []
        for _ in range(3):
            for c in cases:
                c.out.fill_u32(0x7fc07fc0)
            for _ in range(2):
                for c in cases:
                    c.call()
            for c in cases:
                bits.append(c.out.download(np.uint8, c.lay.combined_bytes))
        assert all(np.array_equal(b, bits[0]) for b in bits)
        for c in cases:
            c.check()
    finally:
        del cases
        other.close()


@pytest.mark.parametrize("hkv,D,most", [(8, 128, 1), (4, 96, 6), (3, 64, 6)])
def test_rows_past_four_gigabytes_of_a_pool(hip, hkv, D, most):
    """The same rows at the end of pools that 32 bits do not address, and in small ones: the same bits."""
    rng = np.random.default_rng(hkv)
    rb, page, n, width, dtype = fa.fp4_row_bytes(hkv, D), 16, 2, 5, BF16
    hq = 2 * hkv
    keys = [storage(rng.standard_normal((n, width * page, hkv, D)), dtype)[1] for _ in range(2)]
    q = storage(rng.standard_normal((n, most, hq, D)), dtype)[1]
    order = rng.permutation(n * width).reshape(n, width)
    results = []
    for pages in (n * width, (1 << 32) // (rb * page) + 2 * n * width):
        table = (pages - n * width + order).astype(np.int32)
        pools = [fa.DeviceBuffer(hip, pages * page * rb) for _ in range(2)]
        batch = fa.HipPagedBatch(hip, i32(hip, table), i32(hip, [width * page - most, 33]), n, width, page, pages)
        at = np.arange(width * page)
        slots = i32(hip, table[:, at // page] * page + at % page)
        batch.append_fp4(slots, width * page, *(buf(hip, x) for x in keys), *pools, hkv, D, None, dtype)
        out = [fa.DeviceBuffer(hip, x.nbytes) for x in keys]
        batch.read_fp4(slots, width * page, *pools, *out, hkv, D, dtype)
        lay = batch.layout(most, hq, D, dtype)
        o = fa.DeviceBuffer(hip, lay.combined_bytes)
        batch.attention_fp4(buf(hip, q), *pools, o, i32(hip, [most, most]), most, hq, hkv, D,
                            fa.FlatAttentionConfig(True), None, dtype)
        results.append([x.download(np.uint8, x_bytes) for x, x_bytes in
                        ((out[0], keys[0].nbytes), (out[1], keys[1].nbytes), (o, lay.combined_bytes))])
    assert all(np.array_equal(a, b) for a, b in zip(*results))
    assert np.isfinite(fa.storage_to_f32(results[0][0].view(np.uint16), dtype)).all()


# ------------------------------------------------------------------------------- together

@pytest.mark.parametrize("windowed", [False, True])
def test_a_decoding_loop_eager_and_replayed(hip, windowed):
    """Slots reserved, drafts appended in 4 bits, attended over (with masks, or with a window), accepted:
    four steps, eagerly and from one captured graph, against the model over the rows that were written."""
    rng = np.random.default_rng(21)
    n, most, hq, hkv, D, page, pages, width, dtype = 3, 6, 4, 2, 64, 8, 64, 20, BF16
    rb = fa.fp4_row_bytes(hkv, D)
    steps = []
    for _ in range(4):
        parents, lens = drafts(rng, n, most, 3)
        if windowed:
            parents = np.broadcast_to(np.arange(most) - 1, parents.shape)
        accepted = np.minimum(rng.integers(1, 4, n), lens)
        paths = np.zeros((n, most), np.int64)
        for s in range(n):
            paths[s, :accepted[s]] = (np.arange(accepted[s]) if windowed else
                                      np.sort(rng.permutation(lens[s])[:accepted[s]]))
        steps.append((parents, lens, accepted, paths,
                      *(storage(rng.standard_normal(s), dtype)[1] for s in
                        ((n, most, hq, D), (n, most, hkv, D), (n, most, hkv, D)))))

    def session(replay):
        rngp = np.random.default_rng(22)
        table = np.full((n, width), -1, np.int32)
        b = {"table": i32(hip, table), "ctx": i32(hip, [0, 5, 17]), "mapped": i32(hip, [0, 0, 0]),
             "free": i32(hip, rngp.permutation(pages)), "count": i32(hip, [pages]), "lens": i32(hip, [0] * n),
             "granted": i32(hip, [0] * n), "slots": i32(hip, np.zeros((n, most))),
             "parents": i32(hip, np.zeros((n, most))), "masks": fa.DeviceBuffer(hip, n * most * 8),
             "pos": i32(hip, np.zeros((n, most))), "paths": i32(hip, np.zeros((n, most))),
             "accepted": i32(hip, [0] * n)}
        pools = [fa.DeviceBuffer(hip, pages * page * rb) for _ in range(2)]
        for p in pools:
            p.fill_u32(0)
        q, k, v = (fa.DeviceBuffer(hip, x.nbytes) for x in steps[0][4:])
        batch = fa.HipPagedBatch(hip, b["table"], b["ctx"], n, width, page, pages)
        lay = batch.layout(most, hq, D, dtype)
        out = fa.DeviceBuffer(hip, lay.combined_bytes)
        rot = fa.RotaryEmbeddingConfig(THETA, 0)

        def step():
            batch.reserve(b["lens"], most, b["mapped"], b["free"], b["count"], b["granted"], b["slots"])
            batch.tree_masks(b["parents"], b["granted"], most, b["masks"], b["pos"])
            batch.append_fp4(b["slots"], most, k, v, *pools, hkv, D, rot, dtype, positions=b["pos"])
            batch.attention_fp4(q, *pools, out, b["granted"], most, hq, hkv, D, fa.FlatAttentionConfig(True), rot,
                                dtype, positions=None if windowed else b["pos"],
                                masks=None if windowed else b["masks"],
                                window=fa.AttentionWindow(9, 2) if windowed else None)
            batch.accept_fp4(b["paths"], most, b["accepted"], b["granted"], *pools, hkv, D)

        graph = None
        seen = []
        for i, (parents, lens, accepted, paths, qs, ks, vs) in enumerate(steps):
            for name, x in (("parents", parents), ("lens", lens), ("accepted", accepted), ("paths", paths)):
                b[name].upload(np.ascontiguousarray(x, np.int32))
            for dst, x in ((q, qs), (k, ks), (v, vs)):
                dst.upload(x)
            before = b["ctx"].download(np.int32, n)
            if replay and i:
                if graph is None:
                    hip.capture_begin()
                    step()
                    graph = hip.capture_end()
                graph.launch()
            else:
                step()
            r = fa.download_attention(out, lay, dtype)
            seen.append((before, b["ctx"].download(np.int32, n), b["table"].download(np.int32, n * width),
                         [p.download(np.uint8, pages * page * rb) for p in pools], r.output, r.lse))
        if graph is not None:
            graph.release()
        return seen

    eager, replayed = session(False), session(True)
    for i, (x, y) in enumerate(zip(eager, replayed)):
        assert all(np.array_equal(np.asarray(a), np.asarray(c)) for a, c in zip(x, y)), i
    for (parents, lens, accepted, paths, qs, ks, vs), (before, after, table, pools, o, lse) in zip(steps, eager):
        assert np.array_equal(after, before + accepted)
        # the accepted rows lie in place: the model's rows of what was given, V's exactly
        v = storage(fa.storage_to_f32(vs, dtype).reshape(n, most, hkv, D), dtype)[0]
        pool = pools[1].reshape(-1, rb)
        for s in range(n):
            at = before[s] + np.arange(accepted[s])
            rows = table.reshape(n, width)[s, at // page] * page + at % page
            assert np.array_equal(pool[rows], model.to_rows(v[s, paths[s, :accepted[s]]]))
        assert np.isfinite(fa.storage_to_f32(o, dtype)).all()
