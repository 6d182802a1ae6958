"""Refusals of the device-resident batch's calls, which all come before any device work: they are made
here without a GPU, with pointers that nothing may follow and no context, so that a call that passes
every other check fails with NullArgument for the context."""
import ctypes

import pytest

import flat_attention_amd as fa
from flat_attention_amd import _lib as L

P = 0x10000  # an address, a multiple of 16
BIG = 1 << 40


def batch(n=4, max_pages=8, page=16, pages=64, tables=P, tables_bytes=BIG, ctx=P, ctx_bytes=BIG):
    return L.PagedBatchC(tables, tables_bytes, ctx, ctx_bytes, n, max_pages, page, pages)


def refused(rc):
    return L.STATUS[rc]


def reserve(b=None, **kw):
    a = dict(new=P, new_bytes=BIG, max_new=8, mapped=P, mapped_out=P, mapped_bytes=BIG, free=P,
             free_bytes=BIG, count=P, count_out=P, count_bytes=BIG, granted=P, granted_bytes=BIG,
             slots=P, slots_bytes=BIG)
    assert set(kw) <= set(a)
    a.update(kw)
    return refused(L.lib().fa_paged_reserve_slots(None, b if b is not None else batch(), *a.values()))


def masks(b=None, **kw):
    a = dict(parents=P, parents_bytes=BIG, lens=P, lens_bytes=BIG, tokens=8, masks=P, masks_bytes=BIG,
             positions=P, positions_bytes=BIG)
    assert set(kw) <= set(a)
    a.update(kw)
    return refused(L.lib().fa_paged_tree_masks(None, b if b is not None else batch(), *a.values()))


def append(b=None, **kw):
    a = dict(slots=P, slots_bytes=BIG, positions=None, positions_bytes=0, max_new=8, k=P, v=P,
             src_bytes=BIG, k_pool=P, v_pool=P, pool_bytes=BIG, kv_heads=2, head_dim=64, rotary=None,
             dtype=fa.DTYPE_BF16)
    assert set(kw) <= set(a)
    a.update(kw)
    return refused(L.lib().fa_paged_append_slots(None, b if b is not None else batch(), *a.values()))


def attend(b=None, **kw):
    a = dict(q=P, q_bytes=BIG, k_pool=P, v_pool=P, pool_bytes=BIG, out=P, out_bytes=BIG, lens=P,
             lens_bytes=BIG, positions=None, positions_bytes=0, masks=None, masks_bytes=0, tokens=8,
             q_heads=4, kv_heads=2, head_dim=64, config=L.ConfigC(0, 0, 0.0), rotary=None,
             dtype=fa.DTYPE_BF16)
    assert set(kw) <= set(a)
    a.update(kw)
    return refused(L.lib().fa_paged_tree_attention(None, b if b is not None else batch(), *a.values()))


def accept(b=None, **kw):
    a = dict(paths=P, paths_bytes=BIG, max_accept=4, accepted=P, accepted_bytes=BIG, lens=P,
             lens_bytes=BIG, out=P, out_bytes=BIG, k_pool=P, v_pool=P, pool_bytes=BIG, kv_heads=2,
             head_dim=64, dtype=fa.DTYPE_BF16)
    assert set(kw) <= set(a)
    a.update(kw)
    return refused(L.lib().fa_paged_accept(None, b if b is not None else batch(), *a.values()))


CALLS = [reserve, masks, append, attend, accept]


@pytest.mark.parametrize("call", CALLS)
def test_batch_geometry(call):
    assert call() == "NullArgument"
    assert "context is null" in L.lib().fa_last_error_message().decode()
    assert call(batch(n=0)) == "ZeroDimension"
    assert call(batch(max_pages=0)) == "ZeroDimension"
    assert call(batch(page=0)) == "PagedZeroDimension"
    assert call(batch(pages=0)) == "PagedZeroDimension"
    assert call(batch(page=1 << 16, pages=1 << 15)) == "IndexSpaceExceeded"
    assert call(batch(page=1 << 16, max_pages=1 << 15)) == "IndexSpaceExceeded"
    assert call(batch(n=1 << 29)) == "IndexSpaceExceeded"
    assert call(batch(n=1 << 63, max_pages=2)) == "IndexSpaceExceeded"
    assert call(batch(page=1 << 63, pages=2)) == "IndexSpaceExceeded"
    assert call(batch(ctx=None)) == "NullArgument"
    assert call(batch(ctx_bytes=15)) == "BufferTooSmall"
    tables = call in (reserve, attend, accept)
    assert call(batch(tables=None)) == "NullArgument"
    assert ("block tables" in L.lib().fa_last_error_message().decode()) == tables
    assert (call(batch(tables_bytes=4 * 4 * 8 - 1)) == "BufferTooSmall") == tables


@pytest.mark.parametrize("call,name,need", [
    (reserve, "new", 16), (reserve, "mapped", 16), (reserve, "free", 4), (reserve, "count", 4),
    (reserve, "granted", 16), (reserve, "slots", 4 * 4 * 8),
    (masks, "parents", 4 * 4 * 8), (masks, "lens", 16), (masks, "masks", 8 * 4 * 8),
    (masks, "positions", 4 * 4 * 8),
    (append, "slots", 4 * 4 * 8), (attend, "q", 4 * 8 * 4 * 64 * 2),
    (attend, "out", 4 * 8 * 4 * (64 * 2 + 4)), (attend, "lens", 16),
    (accept, "paths", 4 * 4 * 4), (accept, "accepted", 16), (accept, "lens", 16), (accept, "out", 16)])
def test_buffers_are_there_and_large_enough(call, name, need):
    assert call(**{name: None}) == "NullArgument"
    assert "context is null" not in L.lib().fa_last_error_message().decode()
    assert call(**{name + "_bytes": need - 1}) == "BufferTooSmall"
    assert call(**{name + "_bytes": need}) == "NullArgument"
    assert "context is null" in L.lib().fa_last_error_message().decode()


@pytest.mark.parametrize("call", [append, attend, accept])
def test_pools(call):
    need = 64 * 16 * 2 * 64 * 2
    assert call(pool_bytes=need - 1) == "BufferTooSmall"
    for name in ("k_pool", "v_pool"):
        assert call(**{name: None}) == "NullArgument"
        assert call(**{name: P + 8}) == "Misaligned"
    assert call(dtype=3) == "UnsupportedDtype"
    assert call(kv_heads=0) == call(head_dim=0) == "ZeroDimension"
    assert call(head_dim=36) == "UnsupportedHeadDim"
    assert call(head_dim=34, dtype=fa.DTYPE_F32) == "UnsupportedHeadDim"
    assert call(head_dim=36, dtype=fa.DTYPE_F32) == "NullArgument"
    assert call(kv_heads=1 << 62) == "ShapeOverflow"


def test_other_arguments():
    assert reserve(max_new=0) == "ZeroDimension"
    assert reserve(max_new=1 << 30) == reserve(max_new=1 << 62) == "IndexSpaceExceeded"
    assert reserve(mapped_out=None) == reserve(count_out=None) == "NullArgument"
    for call in (masks, attend):
        assert call(tokens=0) == "ZeroDimension"
        assert call(tokens=513) == "IndexSpaceExceeded"
        assert call(tokens=512) == "NullArgument"
    assert masks(batch(n=1 << 22, max_pages=1), tokens=512) == "IndexSpaceExceeded"
    assert accept(max_accept=0) == "ZeroDimension"
    assert accept(max_accept=513) == "IndexSpaceExceeded"
    assert append(max_new=0) == "ZeroDimension"
    assert append(batch(n=1 << 20), max_new=1 << 20) == "IndexSpaceExceeded"
    assert append(batch(n=1 << 15), max_new=1 << 15, kv_heads=8, head_dim=128) == "IndexSpaceExceeded"
    assert append(k=P + 8) == append(v=P + 2) == "Misaligned"
    assert append(k=None) == append(v=None) == "NullArgument"
    assert append(src_bytes=4 * 8 * 256 - 1) == "BufferTooSmall"
    assert append(positions=P, positions_bytes=127) == "BufferTooSmall"
    assert append(rotary=L.RotaryC(0.0, 0)) == "InvalidRotaryTheta"
    assert append(rotary=L.RotaryC(1e4, (1 << 31) - 8 * 16)) == "NullArgument"
    assert append(rotary=L.RotaryC(1e4, (1 << 31) - 8 * 16 + 1)) == "PositionOverflow"
    assert append(head_dim=136) == "NullArgument"  # (rows of any width without rotation)
    assert append(head_dim=136, rotary=L.RotaryC(1e4, 0)) == "UnsupportedHeadDim"
    assert attend(q_heads=0) == "ZeroDimension"
    assert attend(q_heads=3) == "InvalidHeadGrouping"
    assert attend(head_dim=136) == "UnsupportedHeadDim"
    assert attend(q=P + 4) == attend(out=P + 8) == "Misaligned"
    assert attend(q_heads=1 << 28) == "IndexSpaceExceeded"
    assert attend(q_heads=1 << 62) == "IndexSpaceExceeded"
    assert attend(config=L.ConfigC(0, 1, float("nan"))) == "InvalidScale"
    assert attend(config=L.ConfigC(0, 1, -1.0)) == "InvalidScale"
    assert attend(config=None) == "NullArgument"  # (no config: the default scale)
    assert "context is null" in L.lib().fa_last_error_message().decode()
    assert attend(rotary=L.RotaryC(float("inf"), 0)) == "InvalidRotaryTheta"
    assert attend(rotary=L.RotaryC(1e4, 1 << 31)) == "PositionOverflow"
    assert attend(positions=P, positions_bytes=127) == "BufferTooSmall"
    assert attend(tokens=65, masks=P, masks_bytes=4 * 65 * 2 * 8 - 1) == "BufferTooSmall"


def test_launches_stay_within_the_grid():
    for call in CALLS:
        assert call(batch(n=(1 << 20) + 1, max_pages=1)) == "IndexSpaceExceeded"
        assert call(batch(n=1 << 20, max_pages=1)) in ("NullArgument", "BufferTooSmall")
    # a combine of 2^24 workgroups of 256 threads, and one less
    for heads in (16, 15):
        rc = attend(batch(n=1 << 20, max_pages=1), tokens=1, q_heads=heads, kv_heads=heads, head_dim=8,
                    q_bytes=1 << 62, out_bytes=1 << 62)
        assert rc == ("IndexSpaceExceeded" if heads == 16 else "NullArgument")
    # rows of 16 bytes: 2^32 - 256 pieces are the most that an append moves
    one = dict(kv_heads=2, head_dim=8, src_bytes=1 << 62, slots_bytes=1 << 62)
    assert append(batch(n=1 << 20, max_pages=1), max_new=2047, **one) == "NullArgument"
    assert append(batch(n=(1 << 20) - 1, max_pages=1), max_new=2048, **dict(one, kv_heads=3)) \
        == "IndexSpaceExceeded"


def test_python_mirror_names_the_error():
    class Ctx:  # a context that was closed
        handle = None

    buf = ctypes.create_string_buffer(64)

    class Buf:
        ptr, nbytes = ctypes.addressof(buf) // 16 * 16 + 16, 8

    b = fa.HipPagedBatch(Ctx, None, Buf, 2, 1, 1, 1)
    with pytest.raises(fa.FlatHipError) as e:
        b.tree_masks(Buf, Buf, 1, Buf, Buf)
    assert e.value.variant == "BufferTooSmall"
    assert b.layout(3, 4, 8, fa.DTYPE_BF16).lse_elements == 24


def test_lengths_leave_room_for_whole_steps():
    """The kernels round a length up to whole steps, and step past its end, in 32 bits."""
    most = (1 << 31) - 1024
    for call in CALLS:
        assert call(batch(n=1, max_pages=most, page=1, pages=1)) == "NullArgument"
        assert "context is null" in L.lib().fa_last_error_message().decode()
        assert call(batch(n=1, max_pages=most + 1, page=1, pages=1)) == "IndexSpaceExceeded"
        assert call(batch(n=1, max_pages=1, page=most + 1, pages=1)) == "IndexSpaceExceeded"
    one = batch(n=1)
    assert reserve(one, max_new=most) == "NullArgument"
    assert "context is null" in L.lib().fa_last_error_message().decode()
    assert reserve(one, max_new=most + 1) == reserve(one, max_new=(1 << 31) - 1) == "IndexSpaceExceeded"
