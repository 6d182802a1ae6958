"""Refusals of the sliding-window and 4-bit calls, all before any device work (as in test_batch_host: pointers
that nothing may follow and no context), and the models of their GPU tests against differences and plain
arithmetic."""
import numpy as np
import pytest

import _window_model as model
import flat_attention_amd as fa
from flat_attention_amd import _lib as L

P = 0x10000
BIG = 1 << 40


def batch(n=4, max_pages=8, page=16, pages=64, tables=P, tables_bytes=BIG, ctx=P, ctx_bytes=BIG):
    return L.PagedBatchC(tables, tables_bytes, ctx, ctx_bytes, n, max_pages, page, pages)


def _call(name, defaults, kw, first=None):
    assert set(kw) <= set(defaults)
    a = {**defaults, **kw}
    args = list(a.values())
    rc = getattr(L.lib(), name)(None, *([first] if first is not None else []), *args)
    return L.STATUS[rc]


CAUSAL = L.ConfigC(1, 0, 0.0)


def forward(**kw):
    shape = kw.pop("shape", (2, 4, 2, 100, 64))
    return _call("fa_forward_gqa_window", dict(
        q=P, q_bytes=BIG, k=P, v=P, kv_bytes=BIG, out=P, out_bytes=BIG, shape=L.GroupedShapeC(*shape),
        config=CAUSAL, window=L.WindowC(10, 1), rotary=None, dtype=fa.DTYPE_BF16), kw)


def backward(**kw):
    shape = kw.pop("shape", (2, 4, 2, 100, 64))
    return _call("fa_backward_gqa_window", dict(
        q=P, k=P, v=P, d_out=P, out=P, lse=P, dq=P, dk=P, dv=P, shape=L.GroupedShapeC(*shape), config=CAUSAL,
        window=L.WindowC(10, 1), dtype=fa.DTYPE_BF16), kw)


def paged(b=None, **kw):
    return _call("fa_paged_window_attention", dict(
        q=P, q_bytes=BIG, k_pool=P, v_pool=P, pool_bytes=BIG, out=P, out_bytes=BIG, lens=P, lens_bytes=BIG,
        positions=None, positions_bytes=0, tokens=8, q_heads=4, kv_heads=2, head_dim=64, config=CAUSAL,
        window=L.WindowC(10, 1), rotary=None, dtype=fa.DTYPE_BF16), kw, b if b is not None else batch())


def attend(b=None, **kw):
    return _call("fa_paged_attention_fp4", dict(
        q=P, q_bytes=BIG, k_pool=P, v_pool=P, pool_bytes=BIG, out=P, out_bytes=BIG, lens=P, lens_bytes=BIG,
        positions=None, positions_bytes=0, masks=None, masks_bytes=0, tokens=8, q_heads=4, kv_heads=2,
        head_dim=64, config=CAUSAL, window=None, rotary=None, dtype=fa.DTYPE_BF16), kw,
        b if b is not None else batch())


def append(b=None, **kw):
    return _call("fa_paged_append_slots_fp4", dict(
        slots=P, slots_bytes=BIG, positions=None, positions_bytes=0, max_new=8, k=P, v=P, src_bytes=BIG,
        k_pool=P, v_pool=P, pool_bytes=BIG, kv_heads=2, head_dim=64, rotary=None, dtype=fa.DTYPE_BF16), kw,
        b if b is not None else batch())


def read(b=None, **kw):
    return _call("fa_paged_read_slots_fp4", dict(
        slots=P, slots_bytes=BIG, max_new=8, k_pool=P, v_pool=P, pool_bytes=BIG, k=P, v=P, src_bytes=BIG,
        kv_heads=2, head_dim=64, dtype=fa.DTYPE_BF16), kw, b if b is not None else batch())


def accept(b=None, **kw):
    return _call("fa_paged_accept_fp4", dict(
        paths=P, paths_bytes=BIG, max_accept=4, accepted=P, accepted_bytes=BIG, lens=P, lens_bytes=BIG, out=P,
        out_bytes=BIG, k_pool=P, v_pool=P, pool_bytes=BIG, kv_heads=2, head_dim=64), kw,
        b if b is not None else batch())


def context_is_null(status):
    return status == "NullArgument" and "context is null" in L.lib().fa_last_error_message().decode()


def test_complete_calls_reach_the_context():
    for call in (forward, backward, paged, attend, append, read, accept):
        assert context_is_null(call()), call.__name__


@pytest.mark.parametrize("call", [forward, backward])
def test_contiguous_windows(call):
    assert call(window=None) == "NullArgument"
    assert call(window=L.WindowC(0, 4)) == "ZeroDimension"
    for window, sinks in ((1, 0), (1 << 63, 0), (5, 1 << 63), ((1 << 64) - 1, (1 << 64) - 1)):
        assert context_is_null(call(window=L.WindowC(window, sinks)))
    assert call(config=L.ConfigC(0, 0, 0.0)) == call(config=None) == "CausalVisibilityMismatch"
    assert call(config=L.ConfigC(1, 1, float("nan"))) == "InvalidScale"
    assert call(dtype=7) == "UnsupportedDtype"
    for i in range(5):
        shape = [2, 4, 2, 100, 64]
        shape[i] = 0
        assert call(shape=shape) == "ZeroDimension"
    assert call(shape=(2, 3, 2, 100, 64)) == "InvalidHeadGrouping"
    assert call(shape=(2, 4, 2, 100, 136)) == "UnsupportedHeadDim"
    for dtype in (fa.DTYPE_F32, fa.DTYPE_F16):
        assert call(shape=(2, 4, 2, 100, 36), dtype=dtype) == "UnsupportedHeadDim"
        assert context_is_null(call(shape=(2, 4, 2, 100, 40), dtype=dtype))
    big = {} if call is backward else dict(q_bytes=1 << 62, kv_bytes=1 << 62, out_bytes=1 << 62)
    assert call(shape=(1, 1, 1, 1 << 24, 64), **big) == "IndexSpaceExceeded"  # a slice of 2 GiB
    assert context_is_null(call(shape=(1, 1, 1, (1 << 24) - 1, 64), **big))
    assert call(shape=(1 << 10, 32, 32, 1 << 13, 64), **big) == "IndexSpaceExceeded"  # query rows
    assert call(shape=(1 << 62, 1 << 62, 1, 1, 64), **big) == "ShapeOverflow"
    assert call(q=None) == call(k=None) == call(v=None) == call(out=None) == "NullArgument"
    assert not context_is_null(call(q=None))
    assert call(q=P + 8) == call(k=P + 2) == call(v=P + 4) == call(out=P + 8) == "Misaligned"


def test_forward_buffers_and_rotation():
    q, kv = 2 * 4 * 100 * 64 * 2, 2 * 2 * 100 * 64 * 2
    assert forward(q_bytes=q - 1) == forward(kv_bytes=kv - 1) == "BufferTooSmall"
    assert forward(out_bytes=q + 2 * 4 * 100 * 4 - 1) == "BufferTooSmall"
    assert context_is_null(forward(q_bytes=q, kv_bytes=kv, out_bytes=q + 2 * 4 * 100 * 4))
    assert forward(rotary=L.RotaryC(0.0, 0)) == "InvalidRotaryTheta"
    assert forward(rotary=L.RotaryC(1e4, (1 << 31) - 50)) == "PositionOverflow"


def test_backward_tensors():
    for name in ("d_out", "lse", "dq", "dk", "dv"):
        assert backward(**{name: None}) == "NullArgument" and not context_is_null(backward(**{name: None}))
        assert (backward(**{name: P + 4}) == "Misaligned") == (name != "lse")


def test_paged_windows():
    assert paged(window=None) == "NullArgument" and not context_is_null(paged(window=None))
    for call in (paged, attend):
        assert call(window=L.WindowC(0, 1)) == "ZeroDimension"
        assert context_is_null(call(window=L.WindowC((1 << 64) - 1, (1 << 64) - 1)))
        assert call(batch(ctx=None)) == call(batch(tables=None)) == call(lens=None) == "NullArgument"
        assert call(tokens=513) == call(q_heads=1 << 28) == "IndexSpaceExceeded"
        assert call(q_heads=3) == "InvalidHeadGrouping"
        assert call(q=P + 4) == call(out=P + 8) == "Misaligned"
        assert call(positions=P, positions_bytes=127) == call(lens_bytes=15) == "BufferTooSmall"
        assert call(rotary=L.RotaryC(float("inf"), 0)) == "InvalidRotaryTheta"
    assert attend(window=L.WindowC(5, 1), masks=P, masks_bytes=BIG) == "CausalVisibilityMismatch"
    assert attend(tokens=65, masks=P, masks_bytes=4 * 65 * 2 * 8 - 1) == "BufferTooSmall"
    assert paged(pool_bytes=64 * 16 * 2 * 64 * 2 - 1) == "BufferTooSmall"
    # a combine of 4 * 2^22 workgroups of 256 threads, and one less
    for heads in (4, 3):
        rc = attend(batch(n=1 << 20, max_pages=1), tokens=1, q_heads=heads, kv_heads=heads, head_dim=32,
                    q_bytes=1 << 62, out_bytes=1 << 62)
        assert rc == ("IndexSpaceExceeded" if heads == 4 else "NullArgument")


@pytest.mark.parametrize("call", [attend, append, read, accept])
def test_fp4_pools(call):
    need = 64 * 16 * fa.fp4_row_bytes(2, 64)
    assert call(pool_bytes=need - 1) == "BufferTooSmall"
    assert context_is_null(call(pool_bytes=need))
    for name in ("k_pool", "v_pool"):
        assert call(**{name: None}) == "NullArgument"
        assert call(**{name: P + 8}) == "Misaligned"
    assert call(kv_heads=0) == call(head_dim=0) == "ZeroDimension"
    assert call(head_dim=48) == call(head_dim=160) == "UnsupportedHeadDim"
    assert call(kv_heads=1 << 40) == "ShapeOverflow"
    if call is not accept:
        assert call(dtype=3) == "UnsupportedDtype"
    assert call(batch(n=0)) == "ZeroDimension" and call(batch(page=0)) == "PagedZeroDimension"


def test_fp4_rows():
    assert [fa.fp4_row_bytes(*x) for x in ((1, 32), (8, 128), (2, 64), (3, 96))] == [32, 544, 80, 160]
    for heads, dim, name in ((0, 64, "ZeroDimension"), (2, 16, "UnsupportedHeadDim"), (1 << 40, 32, "ShapeOverflow")):
        with pytest.raises(fa.FlatHipError) as e:
            fa.fp4_row_bytes(heads, dim)
        assert e.value.variant == name
    assert L.STATUS[L.lib().fa_fp4_row_bytes(2, 64, None)] == "NullArgument"
    for call in (append, read):
        assert call(max_new=0) == "ZeroDimension"
        assert call(k=None) == call(v=None) == call(slots=None) == "NullArgument"
        assert call(k=P + 8) == call(v=P + 2) == "Misaligned"
        assert call(src_bytes=4 * 8 * 2 * 64 * 2 - 1) == call(slots_bytes=127) == "BufferTooSmall"
        assert call(batch(n=1 << 15), max_new=1 << 15, kv_heads=8, head_dim=128) == "IndexSpaceExceeded"
    assert append(positions=P, positions_bytes=127) == "BufferTooSmall"
    assert append(rotary=L.RotaryC(1e4, 1 << 31)) == "PositionOverflow"
    assert accept(max_accept=513) == "IndexSpaceExceeded"
    assert accept(paths=None) == "NullArgument"


# ------------------------------------------------------------------------------- the models

@pytest.mark.parametrize("S,window,sinks,hq,hkv", [(9, 3, 1, 2, 1), (12, 1, 4, 2, 2), (10, 40, 0, 3, 1),
                                                   (11, 4, 6, 1, 1)])
def test_model_gradient_matches_differences(S, window, sinks, hq, hkv):
    """Central differences of sum dO * O over every element, in float64: off by eps^2 of a third derivative
    (bounded by the inputs' sizes) and 2^-52 / eps."""
    rng = np.random.default_rng(S)
    q, dout = rng.standard_normal((2, hq, S, 4))
    k, v = rng.standard_normal((2, hkv, S, 4))
    o, lse, _, _ = model.forward(q, k, v, window, sinks, 0.5)
    grads, _ = model.backward(q, k, v, dout, o, lse, window, sinks, 0.5, 0.0)

    def value(*x):
        return (dout * model.forward(*x, window, sinks, 0.5)[0]).sum()

    eps = 2.0 ** -13
    for n, x in enumerate((q, k, v)):
        for at in np.ndindex(x.shape):
            moved = []
            for step in (eps, -eps):
                y = x.copy()
                y[at] += step
                moved.append(value(*[y if i == n else z for i, z in enumerate((q, k, v))]))
            assert abs((moved[0] - moved[1]) / (2 * eps) - grads[n][at]) < 1e-5


@pytest.mark.parametrize("window,sinks", [(-1, 0), (4, -1)])
def test_negative_windows_are_refused(window, sinks):
    with pytest.raises(ValueError, match="negative"):
        fa.AttentionWindow(window, sinks).c()


def test_model_forward_is_the_definition():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((3, 1, 7, 4))
    o, lse, _, _ = model.forward(q, k, v, 2, 1, 0.5)
    for i in range(7):
        keys = sorted({0, max(0, i - 1), i} if i else {0})
        s = np.array([0.5 * (q[0, i] @ k[0, j]) for j in keys])
        assert np.isclose(lse[0, i], np.log(np.exp(s).sum()))
        assert np.allclose(o[0, i], np.exp(s - lse[0, i]) @ v[0, keys])


def test_model_rows_take_the_nearest_value():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 1, 32)) * np.exp2(rng.integers(-30, 30, (40, 1, 1)))
    rows = model.to_rows(x)
    got = model.from_rows(rows, 1, 32)
    scale = np.exp2(rows[:, 16].astype(float) - 127)[:, None, None]
    grid = np.concatenate([-model.LEVELS, model.LEVELS]) * scale[..., None]
    assert np.array_equal(np.abs(got - x), np.abs(grid - x[..., None]).min(-1))
    top = np.abs(x).max(-1)[:, 0] / scale[:, 0, 0]
    assert (top < 7).all() and (top >= 3.5).all()
    assert np.array_equal(model.to_rows(got), rows)
    odd = np.zeros((3, 1, 32))
    odd[0, 0, 3], odd[1, 0, 4] = np.nan, -np.inf
    assert np.array_equal(model.to_rows(odd)[:, 16], [255, 255, 0])
