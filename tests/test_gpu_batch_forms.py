"""The device-resident batch where its kernels differ: ranges of several steps and units at every padded
head width, kv heads side by side or alone, non-finite values and pages outside the pool in each of
those. Models, inputs and tolerances are those of test_gpu_batch.py.
"""
import numpy as np
import pytest

import _batch_model as model
import flat_attention_amd as fa
from test_gpu_batch import BF16, F16, F32, HALF_STEP, THETA, Case, i32, load, paged, storage

pytestmark = pytest.mark.gpu


# (storage, tokens, q heads, kv heads): one, two, four and eight row blocks, heads alone, in pairs and in
# fours, one, two and four key groups
KERNELS = [(BF16, 1, 8, 8), (F16, 3, 9, 3), (BF16, 12, 16, 4), (F16, 14, 9, 3), (BF16, 40, 8, 4), (F16, 65, 8, 2),
           (F32, 1, 8, 8), (F32, 5, 6, 2), (F32, 3, 9, 3), (F32, 20, 8, 4), (F32, 65, 8, 2)]


@pytest.mark.parametrize("D", [80, 128])
@pytest.mark.parametrize("dtype,most,hq,hkv", KERNELS)
@pytest.mark.parametrize("rope", [True, False])
def test_several_steps_and_units_a_range_at_wide_heads(hip, dtype, most, hq, hkv, D, rope):
    """More steps than there are ranges, several times over, of short and long sequences."""
    rng = np.random.default_rng(most + D)
    n = 60
    ctx = np.where(rng.random(n) < 0.5, rng.integers(0, 60, n), rng.integers(1000, 3200, n))
    ctx[:4] = [3001, 5, 0, 1999]
    lens = rng.integers(0, most + 1, n)
    lens[:4] = [most, most, 1, most]
    Case(hip, dtype, ctx, lens, most, hq, hkv, D, 16, 31, rope=rope).check(only=[0, 1, 2, 3, 17, 29, 58, 59])


def attend_by_head(q, k, v, sees, scale):
    """model.attend with the rows of a head in one product (every row sees some key)."""
    T, hq, D = q.shape
    group, hide = hq // k.shape[1], np.where(sees, 0.0, -np.inf)
    o, av, lse, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros((hq, T)), np.zeros((hq, T))
    for h in range(hq):
        kk, vv = k[:, h // group], v[:, h // group]
        s = scale * (q[:, h] @ kk.T) + hide
        m = s.max(1)
        p = np.exp(s - m[:, None])
        l = p.sum(1)
        o[:, h], av[:, h] = p @ vv / l[:, None], p @ np.abs(vv) / l[:, None]
        lse[h] = m + np.log(l)
        size[h] = np.where(sees, scale * (np.abs(q[:, h]) @ np.abs(kk).T), 0).max(1)
    return o, lse, av, size


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [8, 80, 128])
@pytest.mark.parametrize("page", [1, 2])
def test_a_range_takes_its_table_entries_in_parts(hip, monkeypatch, dtype, D, page):
    """So many rows that two ranges have all 3012 keys, more than a thousand pages each."""
    monkeypatch.setattr(model, "attend", attend_by_head)
    Case(hip, dtype, [2500 * page], [512], 512, 64, 1, D, page, 33).check()


@pytest.mark.parametrize("dtype,most,hq,hkv,D", [
    (BF16, 6, 8, 2, 128), (F16, 30, 8, 4, 80), (BF16, 70, 8, 2, 128), (F16, 5, 9, 3, 128), (F32, 1, 8, 8, 64),
    (F32, 6, 4, 4, 128), (F32, 30, 4, 2, 80), (F32, 70, 8, 2, 128)])
def test_pages_outside_the_pool_in_every_form(hip, dtype, most, hq, hkv, D):
    case = Case(hip, dtype, [300, 90], [most, max(1, most - 1)], most, hq, hkv, D, 16, 34)
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
        at = np.where(there, case.table[s, keys // 16], 0).astype(np.int64) * 16 + keys % 16
        eo, el, av, size = model.attend(model.rotate(case.q[s, :m], case.where[s, :m], THETA), case.k[at],
                                        case.v[at], sees & there, float(np.float32(1) / np.sqrt(np.float32(D))))
        h = HALF_STEP[dtype]
        n = c + m
        ds = size * ((D + 16) * 2.0 ** -24 + (h * h if dtype != F32 else 0))
        tl = ds + n * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * (np.abs(el) + size)
        to = h * (np.abs(eo) + av) + (2 * ds.T[..., None] + n * 2.0 ** -23 + 2.0 ** -19) * av + 2.0 ** -25
        assert (np.abs(lse[s, :, :m] - el) <= tl).all()
        assert (np.abs(o[s, :m] - eo) <= to).all()


@pytest.mark.filterwarnings("ignore:invalid value")
@pytest.mark.parametrize("dtype,most,hq,hkv,D,ctx", [
    (BF16, 6, 4, 2, 128, 40), (F16, 40, 8, 2, 128, 500), (BF16, 64, 8, 2, 80, 31), (F16, 33, 16, 2, 128, 2000),
    (F16, 9, 6, 3, 80, 700), (F32, 6, 4, 4, 64, 900), (F32, 1, 8, 8, 128, 300), (F32, 12, 4, 4, 80, 70),
    (F32, 20, 4, 2, 128, 333), (F32, 64, 8, 2, 128, 1000)])
def test_special_values_reach_the_rows_that_see_them_in_every_form(hip, dtype, most, hq, hkv, D, ctx):
    """NaN and infinities in V of drafted rows and of the last live rows, NaN in K of a drafted one."""
    args = ([ctx, 5], [most, min(2, most)], most, hq, hkv, D, 16, 35)
    clean = Case(hip, dtype, *args)
    o0, l0 = clean.run()
    case = Case(hip, dtype, *args)
    group, rows = hq // hkv, case.rows(0, ctx + most)
    sees = np.ones((most, ctx + most), bool)
    sees[:, ctx:] = case.sees[0]
    put = {x: fa.host_storage(np.array([x], np.float32), dtype)[0] for x in (np.nan, np.inf, -np.inf)}
    spots = {(ctx + most - 1, 0, 3): np.nan, (ctx + most // 2, 0, 3): np.inf, (ctx, 1, D - 1): np.inf,
             (ctx + most // 3, 1, D - 1): -np.inf, (ctx - 1, hkv - 1, 60): -np.inf, (ctx, 0, 17): -np.inf}
    vs, want = case.vs.reshape(case.v.shape), np.zeros((most, hq, D))
    for (key, head, d), x in spots.items():
        vs[rows[key], head, d] = put[x]
        want[:, head * group:(head + 1) * group, d] += np.where(sees[:, key], x, 0.0)[:, None]
    case.upload()
    o1, l1 = case.run()
    assert np.array_equal(l1.view(np.uint32), l0.view(np.uint32))
    hit = want != 0
    assert hit.any()
    assert np.array_equal(o1[0][~hit].view(np.uint32), o0[0][~hit].view(np.uint32))
    assert np.array_equal(o1[1].view(np.uint32), o0[1].view(np.uint32))
    assert np.array_equal(o1[0][hit], want[hit], equal_nan=True)
    case.vs[:] = clean.vs
    key = ctx + most // 2
    case.ks.reshape(case.k.shape)[rows[key], hkv - 1, D - 2] = put[np.nan]
    case.upload()
    o2, l2 = case.run()
    hit = np.zeros((most, hq), bool)
    hit[:, (hkv - 1) * group:] = sees[:, key][:, None]
    assert np.isnan(o2[0][hit]).all() and np.isnan(l2[0].T[hit]).all()
    assert np.array_equal(o2[0][~hit].view(np.uint32), o0[0][~hit].view(np.uint32))
    assert np.array_equal(l2[0].T[~hit].view(np.uint32), l0[0].T[~hit].view(np.uint32))


@pytest.mark.parametrize("n,most,width,page,hkv,D", [(6, 20, 9, 5, 2, 64), (40, 64, 16, 16, 8, 128),
                                                     (3, 30, 30, 24, 3, 8)])
def test_accept_moves_f16_rows_like_the_model(hip, n, most, width, page, hkv, D):
    rng = np.random.default_rng(most)
    ctx, lens = rng.integers(0, 60, n), rng.integers(1, most + 1, n)
    table, pages, _ = paged(rng, ctx + lens, page)
    accepted = np.array([rng.integers(0, min(l, width) + 1) for l in lens])
    paths = np.zeros((n, width), np.int64)
    for s in range(n):
        paths[s, :accepted[s]] = np.sort(rng.permutation(lens[s])[:accepted[s]])
    (k, ks), (v, vs) = (storage(rng.standard_normal((pages * page, hkv * D)), F16) for _ in range(2))
    kb, vb, c = fa.DeviceBuffer.from_array(hip, ks), fa.DeviceBuffer.from_array(hip, vs), i32(hip, ctx)
    batch = fa.HipPagedBatch(hip, i32(hip, table), c, n, table.shape[1], page, pages)
    batch.accept(i32(hip, paths), width, i32(hip, accepted), i32(hip, lens), kb, vb, hkv, D, F16)
    ek, ev, ec = model.accept(k, v, table, ctx, paths, accepted, lens, page, pages, 512)
    assert np.array_equal(c.download(np.int32, n), ec)
    assert np.array_equal(load(kb, k.shape, F16), ek) and np.array_equal(load(vb, v.shape, F16), ev)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("ctx,lens,last,bad,live,drafted", [
    ([1500], [512], 0, 1000, 1001, 2000), ([100, 100, 40, 40], [512, 512, 500, 490], 1, 20, 5, 400)])
def test_infinity_beside_a_page_outside_the_pool(hip, dtype, ctx, lens, last, bad, live, drafted):
    """An infinity that all rows see, among table entries with one outside the pool; behind them in the same range
    (entries of the same sequence that follow, or another sequence) a drafted row that holds one too."""
    case = Case(hip, dtype, ctx, lens, 512, 64, 1, 64, 1, 41)
    vs = case.vs.reshape(case.v.shape)
    for s, key, d in ((0, live, 3), (last, drafted, 9)):
        vs[case.rows(s, key + 1)[key], 0, d] = fa.host_storage(np.array([np.inf], np.float32), dtype)[0]
    case.upload()
    case.table[0, bad] = case.pages
    case.batch.block_tables.upload(case.table.astype(np.int32))
    o, lse = case.run()
    want = np.zeros(o.shape, bool)
    want[0, :lens[0], :, 3] = True
    want[last, case.sees[last, :, drafted - ctx[last]], :, 9] = True
    assert np.isposinf(o[want]).all() and np.isfinite(o[~want]).all()


@pytest.mark.parametrize("first,then", [
    ((F16, 64, 4, 1, 64), (F16, 32, 4, 1, 64)), ((BF16, 192, 4, 1, 128), (BF16, 128, 4, 1, 128)),
    ((F32, 40, 4, 4, 128), (F32, 8, 4, 4, 128)), ((BF16, 9, 8, 4, 128), (F16, 9, 8, 4, 128))])
def test_an_earlier_larger_call_sizes_the_workspaces(first, then):
    """A call captured before its shape has run eagerly, after one larger call on a new context."""
    ctx = fa.HipContext(0)
    try:
        for k, (dtype, most, hq, hkv, D) in enumerate((first, then)):
            case = Case(ctx, dtype, [300, 20, 7][k:], [most, 3, 5][k:], most, hq, hkv, D, 16, 44)
            if k == 0:
                case.check()
        # (held here: the graph reads them, and an eager run makes others)
        held = case.keep = fa.DeviceBuffer.from_array(ctx, case.masks), i32(ctx, case.pos)
        with ctx.capture() as cap:
            case.call(upload=False)
        for _ in range(3):
            case.out.fill_u32(0x7fc07fc0)
            cap.graph.launch()
            o0, l0 = case.get()
            o1, l1 = case.check()
            assert np.array_equal(o0, o1) and np.array_equal(l0, l1)
        del held
    finally:
        ctx.close()


def test_an_earlier_reservation_sizes_the_plan():
    """One of more sequences and slots in one launch, then a captured one that takes two."""
    ctx = fa.HipContext(0)
    try:
        for n, max_new in ((100, 40), (7, 570)):
            page, width, pages = 16, 40, 300
            table, lens, new = np.full((n, width), -1), np.zeros(n, np.int64), np.full(n, max_new)
            free = np.arange(pages)
            state = [i32(ctx, x) for x in (table, lens, new, lens, free, [pages])]
            t, c, nl, m, f, k = state
            granted, slots = i32(ctx, np.full(n, 77)), i32(ctx, np.full((n, max_new), 77))
            batch = fa.HipPagedBatch(ctx, t, c, n, width, page, pages)
            if n == 100:
                batch.reserve(nl, max_new, m, f, k, granted, slots)
        with ctx.capture() as cap:
            batch.reserve(nl, max_new, m, f, k, granted, slots)
        cap.graph.launch()
        want = model.reserve(table, lens, new, lens, free, pages, max_new, page, pages)
        assert np.array_equal(granted.download(np.int32, n), want["granted"])
        assert np.array_equal(slots.download(np.int32, n * max_new).reshape(n, max_new), want["slots"])
        assert k.download(np.int32, 1)[0] == want["count"]
    finally:
        ctx.close()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("most,hq,hkv", [(1, 4, 1), (1, 4, 2), (20, 2, 1), (20, 4, 1), (40, 4, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_many_small_probabilities_beside_large_ones(hip, dtype, most, hq, hkv, D):
    """One score in 32 is 17.625 (25.4 powers of two) above the others, and its V is 0, so O is what the small ones
    add up to. f16: besides its relative rounding each of them may lose half a step of the smallest numbers, 2^-25
    of the 2^7-fold of the largest probability; their sum is at least that of the large ones, one a run of 32."""
    n = 1500 + most
    case = Case(hip, dtype, [1500], [most], most, hq, hkv, D, 16, 43, tree=False, rope=False, scale=1.0)
    at = case.rows(0, n)
    q, k, v = np.zeros(case.q.shape), np.zeros(case.k.shape), np.zeros(case.v.shape)
    q[..., 0] = 1.0
    k[at[7::32], :, 0] = 17.625
    v[at] = 1024.0
    v[at[7::32]] = 0.0
    (q, qs), (k, case.ks), (v, case.vs) = (storage(x, dtype) for x in (q, k, v))
    case.bufs[0].upload(qs)
    case.upload()
    o, lse = case.run()
    sees = np.ones((most, n), bool)
    sees[:, 1500:] = np.tril(np.ones((most, most), bool))
    eo, el, av, size = model.attend(q[0], k[at], v[at], sees, 1.0)
    ds = size * (D + 16) * 2.0 ** -24
    tl = ds + n * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * (np.abs(el) + size)
    to = HALF_STEP[dtype] * (eo + av) + (2 * ds.T[..., None] + n * 2.0 ** -23 + 2.0 ** -19) * av
    if dtype == F16:
        to += 2.0 ** -25 + n * 2.0 ** -32 * 1024 / (1500 // 32)
    assert (np.abs(lse[0] - el) <= tl).all()
    assert (np.abs(o[0] - eo) <= to).all()


@pytest.mark.parametrize("dtype,page", [(BF16, 16), (F32, 24)])
def test_pools_of_more_than_four_gib(hip, dtype, page):
    """The same rows in the first pages of a pool of 5 GiB and in its last: appended, attended and moved alike."""
    n, most, hq, hkv, D, ctx = 2, 9, 8, 4, 128, 70
    row = hkv * D * (4 if dtype == F32 else 2)
    pages = (5 << 30) // (page * row)
    rng = np.random.default_rng(45)
    new = {x: rng.standard_normal((n, most, h, D)).astype(np.float32) for x, h in (("q", hq), ("k", hkv), ("v", hkv))}
    old = [rng.standard_normal((n, ctx, hkv, D)).astype(np.float32) for _ in range(2)]
    width = -(-(ctx + most) // page)
    pools = [fa.DeviceBuffer(hip, pages * page * row) for _ in range(2)]

    def put(x):
        return fa.DeviceBuffer.from_array(hip, fa.host_storage(np.ascontiguousarray(x).ravel(), dtype))

    def through(first):
        table = first + np.arange(n * width).reshape(width, n).T
        at = np.arange(ctx + most)
        rows = table[:, at // page] * page + at % page
        lens = i32(hip, [ctx] * n)
        batch = fa.HipPagedBatch(hip, i32(hip, table), lens, n, width, page, pages)
        batch.append(i32(hip, rows[:, :ctx]), ctx, put(old[0]), put(old[1]), *pools, hkv, D, None, dtype)
        batch.append(i32(hip, rows[:, ctx:]), most, put(new["k"]), put(new["v"]), *pools, hkv, D, None, dtype)
        lay = batch.layout(most, hq, D, dtype)
        out, q = fa.DeviceBuffer(hip, lay.combined_bytes), put(new["q"])
        results = []
        for tokens in (most, 3):
            batch.tree_attention(q, *pools, out, i32(hip, [tokens] * n), most, hq, hkv, D, fa.FlatAttentionConfig(),
                                 fa.RotaryEmbeddingConfig(THETA), dtype)
            r = fa.download_attention(out, lay, dtype)
            results += [r.output, r.lse]
            if tokens == most:
                batch.accept(i32(hip, [[0, 4, 8]] * n), 3, i32(hip, [3] * n), i32(hip, [most] * n), *pools, hkv, D,
                             dtype)
                results.append(lens.download(np.int32, n))
        for pool in pools:
            results.append(np.stack([pool.download(np.uint8, row, int(r) * row) for r in rows[:, ctx:ctx + 3].ravel()]))
        return results

    low, high = through(0), through(pages - n * width)
    assert np.isfinite(low[1]).all()
    for a, b in zip(low, high):
        assert np.array_equal(a, b)


def test_the_most_sequences(hip):
    """2^20 sequences of one token each: the largest batch."""
    n, page, D = 1 << 20, 16, 8
    rng = np.random.default_rng(46)
    q, k, v = (storage(rng.standard_normal((n, 1, D)).astype(np.float32), BF16) for _ in range(3))
    pool = [fa.DeviceBuffer(hip, n * page * D * 2) for _ in range(2)]
    t, c, m, new = (i32(hip, np.full(n, x)) for x in (-1, 0, 0, 1))
    free, count = i32(hip, np.arange(n)), i32(hip, [n - 5])
    granted, slots = i32(hip, np.full(n, 77)), i32(hip, np.full(n, 77))
    batch = fa.HipPagedBatch(hip, t, c, n, 1, page, n)
    batch.reserve(new, 1, m, free, count, granted, slots)
    got = np.arange(n) < n - 5
    assert np.array_equal(granted.download(np.int32, n), got)
    assert np.array_equal(t.download(np.int32, n), np.where(got, n - 6 - np.arange(n), -1))
    assert np.array_equal(slots.download(np.int32, n), np.where(got, (n - 6 - np.arange(n)) * page, -1))
    assert count.download(np.int32, 1)[0] == 0 and np.array_equal(m.download(np.int32, n), got)
    parents, masks, pos = i32(hip, np.full(n, -1)), fa.DeviceBuffer(hip, n * 8), i32(hip, np.full(n, 77))
    batch.tree_masks(parents, granted, 1, masks, pos)
    assert np.array_equal(masks.download(np.uint64, n), got) and np.array_equal(pos.download(np.int32, n), got - 1)
    qb, kb, vb = (fa.DeviceBuffer.from_array(hip, x[1]) for x in (q, k, v))
    batch.append(slots, 1, kb, vb, *pool, 1, D, None, BF16)
    lay = batch.layout(1, 1, D, BF16)
    out = fa.DeviceBuffer(hip, lay.combined_bytes)
    batch.tree_attention(qb, *pool, out, granted, 1, 1, 1, D, fa.FlatAttentionConfig(softmax_scale=0.5), None, BF16,
                         positions=pos, masks=masks)
    r = fa.download_attention(out, lay, BF16)
    o = fa.storage_to_f32(r.output, BF16).reshape(n, 1, D)
    assert np.array_equal(o[got], v[0][got]) and (o[~got] == 0).all() and np.isneginf(r.lse[~got]).all()
    want = 0.5 * (q[0] * k[0]).sum((1, 2))
    size = 0.5 * np.abs(q[0] * k[0]).sum((1, 2))
    assert (np.abs(r.lse - want)[got] <= (size * (D + 16) * 2.0 ** -24 + 2.0 ** -22 * (np.abs(want) + size))[got]).all()
    batch.accept(i32(hip, np.zeros(n)), 1, granted, granted, *pool, 1, D, BF16)
    assert np.array_equal(c.download(np.int32, n), got)
