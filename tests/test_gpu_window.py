"""GPU parity of attention with a sliding window and sinks: fa_forward_gqa_window, fa_backward_gqa_window and
fa_paged_window_attention against float64.

Tolerances. h is half a rounding step of the storage type relative to the value (bf16 2^-8, f16 2^-11, f32
2^-24). A score is a sum in f32 of D exact products, off by B (D + 16) 2^-24 of B = scale * sum |q k|; with
rotary and 16-bit storage Q and K are rounded once before, each product off by 2 h + h^2, and the rotation
itself is off by 2^-21 of (|e| + |o|) for each factor. LSE takes that and the sum of n probabilities (each off
by 2^-21): n 2^-24 + 2^-20, and the rounding of its own value and of the running maximum. O adds the rounding
of each probability and of itself, h (|O| + sum p |v|). The gradients' bounds are in the model.
"""
import numpy as np
import pytest

import _batch_model as batch_model
import _window_model as model
import flat_attention_amd as fa
from test_gpu_batch import BF16, F16, F32, HALF_STEP, THETA, i32, load, paged, storage

pytestmark = pytest.mark.gpu


def buf(hip, x):
    return fa.DeviceBuffer.from_array(hip, x)


class Dense:
    def __init__(self, hip, dtype, B, hq, hkv, S, D, window, sinks, seed=0, magnitude=1.0, scale=None):
        rng = np.random.default_rng([seed, S, D])
        self.hip, self.dtype, self.window = hip, dtype, fa.AttentionWindow(window, sinks)
        self.shape = fa.GroupedAttentionShape(B, hq, hkv, S, D)
        self.config = fa.FlatAttentionConfig(True, scale)
        self.scale = model.resolved(D) if scale is None else scale
        self.q, self.qs = storage(magnitude * rng.standard_normal((B, hq, S, D)), dtype)
        self.k, self.ks = storage(rng.standard_normal((B, hkv, S, D)), dtype)
        self.v, self.vs = storage(rng.standard_normal((B, hkv, S, D)), dtype)
        self.dout, self.douts = storage(rng.standard_normal((B, hq, S, D)), dtype)
        self.bufs = [buf(hip, x) for x in (self.qs, self.ks, self.vs)]
        self.op = fa.HipRotaryGroupedAttention(hip, dtype)
        self.out = fa.DeviceBuffer(hip, self.op.layout(self.shape).combined_bytes)

    def call(self, rotary=None):
        self.op.forward_window(*self.bufs, self.shape, self.config, self.window, rotary, out=self.out)

    def get(self):
        s = self.shape
        r = fa.download_attention(self.out, self.op.layout(s), self.dtype)
        o = fa.storage_to_f32(r.output, self.dtype).reshape(self.q.shape)
        return o.astype(np.float64), r.lse.reshape(s.batch, s.q_heads, s.seq_len).astype(np.float64)

    def check_forward(self, rotary=None):
        self.out.fill_u32(0x7fc07fc0)
        self.call(rotary)
        o, lse = self.get()
        h, S, D = HALF_STEP[self.dtype], self.shape.seq_len, self.shape.head_dim
        for b in range(self.shape.batch):
            q, k = self.q[b], self.k[b]
            turned = 0.0
            if rotary is not None:
                at = np.arange(S) + rotary.position_offset
                q, k = (batch_model.rotate(x.transpose(1, 0, 2), at, rotary.theta).transpose(1, 0, 2)
                        for x in (q, k))
                pair = [np.abs(x).reshape(*x.shape[:-1], -1, 2).sum(-1).max() for x in (q, k)]
                turned = 2.0 ** -19 * self.scale * D * pair[0] * pair[1]
            eo, el, av, size = model.forward(q, k, self.v[b], self.window.window, self.window.sinks, self.scale)
            n = min(S, self.window.window + self.window.sinks)
            ds = size * ((D + 16) * 2.0 ** -24 + (2 * h + h * h if rotary is not None and self.dtype != F32 else 0))
            ds = ds + turned
            tl = ds + n * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * (np.abs(el) + size)
            err = np.abs(lse[b] - el)
            assert (err <= tl).all(), (b, (err / tl).max())
            to = h * (np.abs(eo) + av) + (2 * ds[..., None] + n * 2.0 ** -23 + 2.0 ** -19) * av
            if self.dtype == F16:
                to = to + 2.0 ** -25
            err = np.abs(o[b] - eo)
            assert (err <= to).all(), (b, (err / to).max())
        return o, lse

    def check_backward(self):
        s = self.shape
        w, h = self.window, HALF_STEP[self.dtype]
        os_, lses = np.empty_like(self.qs.reshape(self.q.shape)), np.empty(self.q.shape[:3], np.float32)
        o = np.empty(self.q.shape)
        for b in range(s.batch):
            eo, el, _, _ = model.forward(self.q[b], self.k[b], self.v[b], w.window, w.sinks, self.scale)
            o[b], st = storage(eo, self.dtype)
            os_[b], lses[b] = st.reshape(eo.shape), el
        grads = [fa.DeviceBuffer(self.hip, x.nbytes) for x in (self.qs, self.ks, self.vs)]
        for g in grads:
            g.fill_u32(0x7fc07fc0)
        keep = [buf(self.hip, x) for x in (self.douts, os_, lses)]
        fa.HipGroupedBackwardRecomputePipeline(self.hip, self.dtype).encode_window(
            *self.bufs, keep[0], keep[1], keep[2].ptr, *grads, s, self.config, w)
        got = [load(g, x.shape, self.dtype) for g, x in zip(grads, (self.q, self.k, self.v))]
        for b in range(s.batch):
            want, tol = model.backward(self.q[b], self.k[b], self.v[b], self.dout[b], o[b],
                                       lses[b].astype(np.float64), w.window, w.sinks, self.scale, h)
            for name, x, e, t in zip(("dq", "dk", "dv"), got, want, tol):
                if self.dtype == F16:
                    t = t + 2.0 ** -25
                err = np.abs(x[b] - e)
                # (not > : a NaN fails)
                assert (err <= t).all(), (name, b, (err / np.maximum(t, 1e-30)).max())
        return got


DENSE = [  # batch, q heads, kv heads, length, head dim, window, sinks
    (1, 1, 1, 1, 64, 1, 0),
    (1, 2, 1, 5, 8, 1, 0),
    (2, 2, 2, 65, 64, 1, 3),
    (1, 4, 2, 128, 128, 32, 4),
    (1, 3, 1, 200, 40, 64, 0),
    (1, 4, 1, 333, 128, 100, 70),
    (2, 2, 1, 257, 32, 257, 2),
    (1, 2, 2, 300, 96, 5000, 9000),
    (1, 8, 2, 700, 64, 63, 1),
    (1, 2, 1, 1100, 80, 130, 129),
    (1, 1, 1, 640, 16, 64, 64),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", range(len(DENSE)))
@pytest.mark.parametrize("rope", [False, True])
def test_forward_matches_float64(hip, dtype, case, rope):
    Dense(hip, dtype, *DENSE[case], scale=0.2 if case % 3 == 0 else None).check_forward(
        fa.RotaryEmbeddingConfig(THETA, 11 if case % 2 else 0) if rope else None)


@pytest.mark.parametrize("dtype,shape", [
    (BF16, (2, 64, 32, 520, 64, 100, 4)), (F16, (4, 32, 16, 500, 128, 150, 5)),
    (F32, (3, 32, 32, 400, 32, 90, 2)), (BF16, (1, 16, 4, 1500, 128, 300, 4)),
    (F32, (1, 16, 16, 1200, 128, 200, 40)), (F32, (1, 32, 32, 1100, 64, 500, 3))])
def test_forward_with_rows_for_every_workgroup_layout(hip, dtype, shape):
    """Enough rows that each rule of the launch's choice (rows a workgroup, key groups) comes up."""
    Dense(hip, dtype, *shape).check_forward()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", range(len(DENSE)))
def test_backward_matches_float64(hip, dtype, case):
    Dense(hip, dtype, *DENSE[case], seed=1, scale=0.2 if case % 3 == 0 else None).check_backward()


@pytest.mark.parametrize("dtype,shape", [(BF16, (2, 16, 4, 1000, 128, 200, 4)), (F32, (1, 8, 2, 900, 64, 130, 300)),
                                         (F16, (1, 32, 8, 700, 64, 40, 1)), (BF16, (1, 4, 1, 3000, 128, 50, 2))])
def test_backward_with_key_blocks_in_parts(hip, dtype, shape):
    """Key blocks with sinks, and few key blocks without, dealt to several workgroups."""
    Dense(hip, dtype, *shape, seed=2).check_backward()


def test_a_window_as_long_as_the_sequence_is_causal_attention(hip):
    for dtype, tol in ((F32, 1e-5), (BF16, 2e-2)):
        d = Dense(hip, dtype, 1, 4, 2, 300, 64, 300, 0)
        o, lse = d.check_forward()
        plain = d.op.forward_resident(*d.bufs, d.shape, d.config, None)
        r = fa.download_attention(plain, d.op.layout(d.shape), dtype)
        assert np.abs(fa.storage_to_f32(r.output, dtype).reshape(o.shape) - o).max() <= tol
        assert np.abs(r.lse.reshape(lse.shape) - lse).max() <= tol


def test_large_scores(hip):
    for dtype in (BF16, F16, F32):
        Dense(hip, dtype, 1, 4, 2, 400, 128, 90, 6, magnitude=60.0).check_forward()


def test_infinities_and_nan_outside_what_a_row_sees(hip):
    """Keys behind the window change nothing in the rows that do not see them: NaN in K is replaced before
    the maximum, and V of those keys lies in tiles that such rows' blocks skip, or weighs zero with finite V."""
    for dtype in (BF16, F16, F32):
        d = Dense(hip, dtype, 1, 2, 1, 1000, 64, 64, 4)
        base, lse0 = d.check_forward()
        ks = d.ks.reshape(d.k.shape).copy()
        ks[:, :, 300] = fa.host_storage(np.array([np.nan], np.float32), dtype)[0]
        d.bufs[1].upload(ks)
        d.call()
        o, lse = d.get()
        far = np.r_[0:300, 364:1000]
        assert np.array_equal(o[:, :, far], base[:, :, far]) and np.array_equal(lse[:, :, far], lse0[:, :, far])
        assert np.isnan(o[:, :, 300:364]).all()


# ------------------------------------------------------------------------------- over the paged cache

class Paged:
    def __init__(self, hip, dtype, ctx, lens, most, hq, hkv, D, page, window, sinks, seed=0, rope=True,
                 positions=False, offset=0, drop=False):
        rng = np.random.default_rng([seed, most, D])
        self.hip, self.dtype, self.most, self.dims = hip, dtype, most, (hq, hkv, D)
        self.ctx, self.lens, self.page = np.asarray(ctx), np.asarray(lens), page
        self.window = fa.AttentionWindow(window, sinks)
        n = len(ctx)
        fit = [c + m if 0 <= c < 1 << 20 and 0 <= m <= most else 0 for c, m in zip(ctx, lens)]
        self.table, self.pages, _ = paged(rng, fit, page)
        self.q, qs = storage(rng.standard_normal((n, most, hq, D)), dtype)
        rows = self.pages * page
        self.k, self.ks = storage(rng.standard_normal((rows, hkv, D)), dtype)
        self.v, self.vs = storage(rng.standard_normal((rows, hkv, D)), dtype)
        self.rope, self.offset = rope, offset
        self.where = self.ctx[:, None] + np.arange(most)
        if positions:
            self.where = self.where + 5
        if drop:  # what no token sees is not a number, and pages that hold nothing else are gone
            nan = fa.host_storage(np.array([np.nan], np.float32), dtype)[0]
            used = np.zeros(rows, bool)
            for s in range(n):
                see = model.sees(ctx[s] + np.arange(lens[s]), fit[s], window, sinks).any(0)
                at = self.rows(s, fit[s])
                used[at[see]] = True
                for p in range(-(-fit[s] // page)):
                    if not see[p * page:(p + 1) * page].any():
                        self.table[s, p] = [-1, self.pages, 2147483647][p % 3]
            self.ks[~used] = nan
            self.vs[~used] = nan
        self.bufs = [buf(hip, x) for x in (qs, self.ks, self.vs)]
        self.batch = fa.HipPagedBatch(hip, i32(hip, self.table), i32(hip, self.ctx), n, self.table.shape[1],
                                      page, self.pages)
        self.len_buf = i32(hip, self.lens)
        self.pos = i32(hip, self.where) if positions else None
        self.lay = self.batch.layout(most, hq, D, dtype)
        self.out = fa.DeviceBuffer(hip, self.lay.combined_bytes)

    def rows(self, s, count):
        at = np.arange(count)
        return self.table[s, at // self.page].astype(np.int64) * self.page + at % self.page

    def call(self):
        hq, hkv, D = self.dims
        self.batch.window_attention(*self.bufs, self.out, self.len_buf, self.most, hq, hkv, D,
                                    fa.FlatAttentionConfig(True), self.window,
                                    fa.RotaryEmbeddingConfig(THETA, self.offset) if self.rope else None,
                                    self.dtype, positions=self.pos)

    def get(self):
        hq, _, D = self.dims
        n = len(self.ctx)
        r = fa.download_attention(self.out, self.lay, self.dtype)
        o = fa.storage_to_f32(r.output, self.dtype).reshape(n, self.most, hq, D)
        return o, r.lse.reshape(n, hq, self.most)

    def check(self):
        self.out.fill_u32(0x7fc07fc0)
        self.call()
        o, lse = self.get()
        hq, hkv, D = self.dims
        h = HALF_STEP[self.dtype]
        for s in range(len(self.ctx)):
            c, m = int(self.ctx[s]), int(self.lens[s])
            ok = c >= 0 and 0 <= m <= self.most and c + m <= self.table.shape[1] * self.page
            m = m if ok else 0
            assert (o[s, m:] == 0).all() and (lse[s, :, m:] == -np.inf).all()
            if not m:
                continue
            see = model.sees(c + np.arange(m), c + m, self.window.window, self.window.sinks)
            at = self.rows(s, c + m)
            at = np.where(see.any(0), at, 0)
            q = self.q[s, :m]
            if self.rope:  # (a token without a position in the table: as if it saw nothing)
                q = batch_model.rotate(q, self.where[s, :m] + self.offset, THETA)
                see = see & (self.where[s, :m] < self.table.shape[1] * self.page)[:, None]
            eo, el, av, size = batch_model.attend(q, self.k[at], self.v[at], see, model.resolved(D))
            empty = el == -np.inf
            assert np.array_equal(np.isneginf(lse[s, :, :m]), empty), s
            assert (o[s, :m][empty.T] == 0).all()
            el = np.where(empty, 0, el)
            ds = size * ((D + 16) * 2.0 ** -24 + (h * h if self.dtype != F32 and self.rope else 0))
            n = see.shape[1]
            tl = ds + n * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * (np.abs(el) + size)
            err = np.abs(np.where(empty, 0, lse[s, :, :m]) - el)
            assert (err <= tl).all(), (s, (err / tl).max())
            to = h * (np.abs(eo) + av) + (2 * ds.T[..., None] + n * 2.0 ** -23 + 2.0 ** -19) * av
            if self.dtype == F16:
                to = to + 2.0 ** -25
            err = np.abs(o[s, :m] - eo)
            assert (err <= to).all(), (s, (err / np.maximum(to, 1e-30)).max())
        return o, lse


PAGED = [  # context lengths, new lengths, most, q heads, kv heads, head dim, page, window, sinks
    ([0], [1], 1, 1, 1, 64, 16, 1, 0),
    ([500, 3], [1, 1], 1, 4, 1, 128, 16, 100, 4),
    ([63, 0, 5], [3, 5, 0], 5, 4, 2, 64, 16, 7, 2),
    ([1000, 17, 640], [7, 16, 1], 16, 8, 2, 128, 16, 200, 40),
    ([310, 32, 33, 960], [33, 31, 1, 32], 33, 4, 4, 64, 5, 64, 64),
    ([1000, 3, 257], [13, 2, 9], 13, 6, 2, 96, 24, 129, 1),
    ([2513, 90], [64, 40], 64, 16, 2, 128, 16, 300, 4),
    ([700], [70], 70, 3, 1, 32, 1, 1, 0),
    ([700, 129], [130, 65], 130, 2, 1, 96, 32, 30, 500),
    ([40], [512], 512, 2, 2, 32, 16, 100, 3),
    ([2500, 11], [4, 4], 4, 12, 12, 64, 64, 4000, 9000),
    ([20000], [3], 3, 2, 1, 64, 1, 1100, 1050),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", range(len(PAGED)))
@pytest.mark.parametrize("rope", [True, False])
def test_paged_matches_float64(hip, dtype, case, rope):
    Paged(hip, dtype, *PAGED[case], rope=rope, positions=case % 2 == 1, offset=37 if case % 3 else 0).check()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", [1, 3, 5, 6, 11])
def test_rows_that_no_token_sees_may_be_gone(hip, dtype, case):
    Paged(hip, dtype, *PAGED[case], drop=True).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_infinities_behind_the_window_of_some_tokens(hip, dtype):
    """V is infinite at a row that the first tokens see and the last do not, or the other way around."""
    p = Paged(hip, dtype, [400], [40], 40, 4, 2, 64, 16, 50, 2)
    base, _ = p.check()
    for row in (370, 1, 420):
        vs = p.vs.reshape(p.v.shape).copy()
        vs[p.rows(0, 440)[row], :, 5] = fa.host_storage(np.array([np.inf], np.float32), dtype)[0]
        p.bufs[2].upload(vs)
        p.call()
        o, _ = p.get()
        see = model.sees(400 + np.arange(40), 440, 50, 2)[:, row]
        assert np.array_equal(o[0, ~see], base[0, ~see])
        assert (o[0, see][..., 5] == np.inf).all()
        other = np.arange(64) != 5
        assert np.array_equal(o[0, see][..., other], base[0, see][..., other])


def test_sequences_that_do_not_fit(hip):
    Paged(hip, BF16, [40, -1, 2147483647, 40, 17], [6, 3, 2, -2, 9], 8, 4, 2, 64, 16, 10, 1).check()


def test_many_sequences_of_mixed_lengths(hip):
    rng = np.random.default_rng(5)
    ctx = np.where(rng.random(200) < 0.5, rng.integers(0, 60, 200), rng.integers(500, 3200, 200))
    for dtype, most in ((BF16, 1), (F16, 9), (F32, 2)):
        Paged(hip, dtype, ctx, rng.integers(0, most + 1, 200), most, 8, 4, 64, 16, 256, 4).check()


def test_the_same_call_again_gives_the_same_bits(hip):
    d = Dense(hip, BF16, 1, 8, 2, 700, 64, 63, 1)
    first, again = d.check_backward(), d.check_backward()
    assert all(np.array_equal(x, y) for x, y in zip(first, again))
    p = Paged(hip, BF16, *PAGED[6])
    (o, l), (o2, l2) = p.check(), p.check()
    assert np.array_equal(o, o2) and np.array_equal(l, l2)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_captured_calls_replay(hip, dtype):
    """Forward, backward and paged calls captured together and replayed over new inputs, with eager calls
    and synchronizations in between. (One head_dim: a context holds the angles of one.)"""
    d = Dense(hip, dtype, 1, 8, 2, 700, 128, 63, 1)
    p = Paged(hip, dtype, *PAGED[3])
    back = fa.HipGroupedBackwardRecomputePipeline(hip, dtype)
    grads = [fa.DeviceBuffer(hip, x.nbytes) for x in (d.qs, d.ks, d.vs)]
    dout = buf(hip, d.douts)
    lse = d.out.ptr + d.op.layout(d.shape).lse_byte_offset
    rot = fa.RotaryEmbeddingConfig(THETA, 0)

    def calls():
        d.call(rot)
        d.call()
        back.encode_window(*d.bufs, dout, d.out, lse, *grads, d.shape, d.config, d.window)
        p.call()

    def results():
        return [d.get(), p.get(), [load(g, (g.nbytes // (4 if dtype == F32 else 2),), dtype) for g in grads]]

    calls()
    hip.capture_begin()
    calls()
    graph = hip.capture_end()
    rng = np.random.default_rng(1)
    for _ in range(4):
        for b, x in zip(d.bufs, (d.q, d.k, d.v)):
            b.upload(storage(rng.standard_normal(x.shape), dtype)[1])
        calls()
        want = results()
        for b in [d.out, p.out] + grads:
            b.fill_u32(0x7fc07fc0)
        graph.launch()
        got = results()
        for x, y in zip(want, got):
            assert all(np.array_equal(a, b) for a, b in zip(x, y))
    graph.release()
