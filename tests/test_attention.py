"""What the attention entry points refuse, and with which message: checked before any pointer is read
and before any HIP call, so it runs without a GPU."""
import ctypes

import pytest


def _rows(bk, batch_stride=1 << 20, head_stride=1 << 10, row_stride=64, data=1 << 20):
    return bk.Rows(data, batch_stride, head_stride, row_stride)


def _shape(bk, **kw):
    values = dict(type=bk.BF16, dim=64, batch=2, query_heads=4, state_heads=2, queries=3, states=16, scale=0.125)
    values.update(kw)
    return bk.AttentionShape(*values.values())


def _attend(bk, shape=None, queries=None, keys=None, values=None, out=None, mask=None, mask_stride=0, workspace=None):
    L = bk.lib()
    one = _rows(bk)
    status = L.bitsknn_cross_attention(shape or _shape(bk), queries or one, keys or one, values or one, None, mask,
                                       mask_stride, out or one, None, workspace, 0, None)
    return status, L.bitsknn_last_error().decode()


SHAPES = [
    (dict(type=2), "UNSUPPORTED", "unknown type 2"),
    (dict(dim=0), "UNSUPPORTED", "Unsupported dim: 0"),
    (dict(dim=60), "UNSUPPORTED", "Unsupported dim: 60"),
    (dict(dim=264), "UNSUPPORTED", "Unsupported dim: 264"),
    (dict(batch=-1), "INVALID", "negative size"),
    (dict(queries=-1), "INVALID", "negative size"),
    (dict(states=-7), "INVALID", "negative size"),
    (dict(state_heads=0), "INVALID", "do not share"),
    (dict(query_heads=3), "INVALID", "3 query heads do not share 2 state heads"),
    (dict(query_heads=0), "INVALID", "do not share"),
    (dict(scale=0.0), "INVALID", "not positive and finite"),
    (dict(scale=-1.0), "INVALID", "not positive and finite"),
    (dict(scale=float("inf")), "INVALID", "not positive and finite"),
    (dict(scale=float("nan")), "INVALID", "not positive and finite"),
    (dict(scale=3e38), "INVALID", "not positive and finite"),
    (dict(queries=1 << 30, query_heads=8), "UNSUPPORTED", "too many rows"),
    (dict(states=0x7FFFFFFF), "UNSUPPORTED", "too many rows"),
]


@pytest.mark.parametrize("change,code,message", SHAPES)
def test_shapes_that_are_refused(bk, change, code, message):
    status, text = _attend(bk, _shape(bk, **change))
    assert status == getattr(bk, "ERR_" + code) and message in text, text
    assert bk.lib().bitsknn_cross_attention_workspace_bytes(_shape(bk, **change)) == 0


ROWS = [
    (dict(data=0), "null pointer"),
    (dict(data=(1 << 20) + 8), "16-byte boundaries"),
    (dict(row_stride=68), "16-byte boundaries"),
    (dict(head_stride=-64), "16-byte boundaries"),
    (dict(batch_stride=4), "16-byte boundaries"),
    (dict(batch_stride=1 << 44), "stride"),
    (dict(row_stride=1 << 24), "row stride"),
]


@pytest.mark.parametrize("which", ["queries", "keys", "values", "out"])
@pytest.mark.parametrize("change,message", ROWS)
def test_vectors_that_are_refused(bk, which, change, message):
    status, text = _attend(bk, **{which: _rows(bk, **change)})
    assert status in (bk.ERR_INVALID, bk.ERR_UNSUPPORTED) and message in text and which in text, text


@pytest.mark.parametrize("change", [dict(row_stride=0), dict(head_stride=0), dict(batch_stride=0), dict(row_stride=56),
                                    dict(head_stride=128), dict(row_stride=1 << 10), dict(batch_stride=1 << 10)])
def test_outputs_that_overlap_are_refused(bk, change):
    status, text = _attend(bk, out=_rows(bk, **change))
    assert status == bk.ERR_INVALID and "out: vectors overlap" in text, text


def test_other_refusals(bk):
    L = bk.lib()
    one = _rows(bk)
    assert L.bitsknn_cross_attention(None, one, one, one, None, None, 0, one, None, None, 0, None) == bk.ERR_INVALID
    assert L.bitsknn_cross_attention(_shape(bk), one, None, one, None, None, 0, one, None, None, 0, None) == bk.ERR_INVALID
    status, text = _attend(bk, workspace=ctypes.c_void_p(8))
    assert status == bk.ERR_INVALID and "workspace" in text
    status, text = _attend(bk, mask=ctypes.c_void_p(64), mask_stride=1 << 60)
    assert status == bk.ERR_INVALID and "mask stride" in text
    # nothing to do: no launch, whatever the pointers
    empty = bk.Rows(None, 0, 0, 0)
    assert _attend(bk, _shape(bk, batch=0), empty, empty, empty, empty)[0] == bk.OK
    assert _attend(bk, _shape(bk, queries=0), empty, one, one, empty)[0] == bk.OK


def test_workspace_sizes(bk):
    """Ranges only where the rows leave most of the GPU idle, each at least four tiles of 64 states."""
    size = bk.lib().bitsknn_cross_attention_workspace_bytes
    assert size(_shape(bk, states=255)) == 0
    assert size(_shape(bk, batch=64, query_heads=64, state_heads=64, states=1 << 20)) == 0
    few = size(_shape(bk, states=4096))
    assert 0 < few <= 64 * 2 * 4 * 3 * (64 * 4 + 8)
    assert size(_shape(bk, states=1 << 20)) >= few


# ---- the cache ------------------------------------------------------------------------------------


def _cache(bk, **kw):
    values = dict(key_codes=1 << 20, value_codes=1 << 21, key_scales=1 << 22, value_scales=1 << 23,
                  block_counts=1 << 24, blocks=8, state_heads=2, block=16, dim=64)
    values.update(kw)
    return bk.Cache(*values.values())


def _store(bk, cache=None, type=0, batch=2, states=20, keys=None, values=None, table=64, table_stride=2):
    L = bk.lib()
    one = _rows(bk)
    status = L.bitsknn_cache_store(cache or _cache(bk), type, batch, states, keys or one, values or one, None,
                                   ctypes.c_void_p(table), table_stride, None)
    return status, L.bitsknn_last_error().decode()


def _read(bk, cache=None, shape=None, queries=None, out=None, table=64, table_stride=2, workspace=None):
    L = bk.lib()
    one = _rows(bk)
    status = L.bitsknn_cached_attention(shape or _shape(bk), queries or one, cache or _cache(bk), ctypes.c_void_p(table),
                                        table_stride, None, out or one, None, workspace, 0, None)
    return status, L.bitsknn_last_error().decode()


CACHES = [
    (dict(block=0), "UNSUPPORTED", "Unsupported block: 0"),
    (dict(block=24), "UNSUPPORTED", "Unsupported block: 24"),
    (dict(block=512), "UNSUPPORTED", "Unsupported block: 512"),
    (dict(dim=0), "UNSUPPORTED", "Unsupported dim: 0"),
    (dict(dim=65), "UNSUPPORTED", "Unsupported dim: 65"),
    (dict(dim=264), "UNSUPPORTED", "Unsupported dim: 264"),
    (dict(blocks=-1), "INVALID", "a cache of -1 blocks"),
    (dict(state_heads=0), "INVALID", "0 heads"),
    (dict(key_codes=0), "INVALID", "cache: null pointer"),
    (dict(value_scales=0), "INVALID", "cache: null pointer"),
    (dict(block_counts=0), "INVALID", "cache: null pointer"),
    (dict(key_codes=(1 << 20) + 8), "INVALID", "16-byte boundaries"),
    (dict(value_codes=(1 << 20) + 4), "INVALID", "16-byte boundaries"),
]


@pytest.mark.parametrize("change,code,message", CACHES)
@pytest.mark.parametrize("entry", [_store, _read])
def test_caches_that_are_refused(bk, entry, change, code, message):
    status, text = entry(bk, _cache(bk, **change))
    assert status == getattr(bk, "ERR_" + code) and message in text, text


def test_store_refusals(bk):
    assert _store(bk, type=3) == (bk.ERR_UNSUPPORTED, "bitsknn_cache_store: unknown type 3")
    assert _store(bk, batch=-1)[0] == bk.ERR_INVALID
    assert _store(bk, states=-1)[0] == bk.ERR_INVALID
    status, text = _store(bk, table=None)
    assert status == bk.ERR_INVALID and "table: null pointer" in text
    status, text = _store(bk, table_stride=1 << 40)
    assert status == bk.ERR_INVALID and "table stride" in text
    for change, message in ROWS:
        for which in ("keys", "values"):
            status, text = _store(bk, **{which: _rows(bk, **change)})
            assert status != bk.OK and message in text and which in text
    # nothing to do
    assert _store(bk, batch=0)[0] == bk.OK and _store(bk, states=0)[0] == bk.OK
    assert _store(bk, _cache(bk, blocks=0))[0] == bk.OK


def test_cached_attention_refusals(bk):
    for change, code, message in SHAPES:
        status, text = _read(bk, shape=_shape(bk, **change))
        assert status == getattr(bk, "ERR_" + code) and message in text, text
    assert _read(bk, shape=_shape(bk, dim=128))[0] == bk.ERR_INVALID
    assert _read(bk, shape=_shape(bk, query_heads=3, state_heads=1))[0] == bk.ERR_INVALID
    status, text = _read(bk, table=None)
    assert status == bk.ERR_INVALID and "table: null pointer" in text
    assert _read(bk, table_stride=1 << 40)[0] == bk.ERR_INVALID
    assert _read(bk, workspace=ctypes.c_void_p(4))[0] == bk.ERR_INVALID
    status, text = _read(bk, out=_rows(bk, row_stride=0))
    assert status == bk.ERR_INVALID and "out: vectors overlap" in text
    assert _read(bk, shape=_shape(bk, queries=0), queries=bk.Rows(), out=bk.Rows())[0] == bk.OK


# ---- launches that a grid cannot hold -----------------------------------------------------------------


def _backward(bk, shape, lse=64, workspace=64, workspace_bytes=1 << 60):
    L = bk.lib()
    one = _rows(bk, batch_stride=1 << 20, head_stride=1 << 16, row_stride=256)
    status = L.bitsknn_cross_attention_backward(shape, one, one, one, one, one, ctypes.c_void_p(lse), None, None, 0, one,
                                                one, one, ctypes.c_void_p(workspace), workspace_bytes, None)
    return status, L.bitsknn_last_error().decode()


# A grid has fewer than 2^32 threads.  Workgroups of the walk by states: 512 threads from 72 to 128
# dimensions, 256 else; of the walk by rows 256; of the rows' deltas 8, 16 or 32 threads per row.
@pytest.mark.parametrize("change", [
    dict(dim=128, batch=1 << 23, query_heads=1, state_heads=1, queries=1, states=1),
    dict(dim=72, batch=1 << 22, query_heads=1, state_heads=1, queries=1, states=257),
    dict(dim=128, batch=1 << 23, query_heads=1, state_heads=1, queries=0, states=1),
    dict(dim=64, batch=1 << 24, query_heads=1, state_heads=1, queries=1, states=1),
    dict(dim=256, batch=1 << 24, query_heads=1, state_heads=1, queries=1, states=1),
    dict(dim=64, batch=1 << 20, query_heads=2, state_heads=1, queries=256, states=1),
    dict(dim=128, batch=1 << 20, query_heads=2, state_heads=1, queries=128, states=1),
    dict(dim=256, batch=1 << 20, query_heads=2, state_heads=1, queries=64, states=1),
    dict(dim=64, batch=1 << 20, query_heads=16, state_heads=16, queries=129, states=1),
])
def test_backward_grids_that_are_refused_before_any_launch(bk, change):
    status, text = _backward(bk, _shape(bk, **change))
    assert status == bk.ERR_UNSUPPORTED and "too many rows" in text, text


# Workgroups of up to 64 rows: 256 threads per 32 of them; of more rows: 512 threads per 256 of them, 256
# per 128 above 128 dimensions.
@pytest.mark.parametrize("change", [
    dict(dim=64, batch=1 << 24, query_heads=1, state_heads=1, queries=1),
    dict(dim=128, batch=1 << 23, query_heads=1, state_heads=1, queries=33),
    dict(dim=64, batch=1 << 23, query_heads=1, state_heads=1, queries=65),
    dict(dim=128, batch=1 << 22, query_heads=1, state_heads=1, queries=257),
    dict(dim=256, batch=1 << 23, query_heads=1, state_heads=1, queries=129),
])
def test_forward_grids_that_are_refused_before_any_launch(bk, change):
    shape = _shape(bk, **change)
    one = _rows(bk, batch_stride=1 << 17, head_stride=1 << 17, row_stride=256)
    status, text = _attend(bk, shape, one, one, one, one)
    assert status == bk.ERR_UNSUPPORTED and "too many rows" in text, text
    status, text = _read(bk, _cache(bk, dim=shape.dim, state_heads=shape.state_heads), shape, one, one)
    assert status == bk.ERR_UNSUPPORTED and "too many rows" in text, text


def test_store_boundaries_by_type(bk):
    """16-byte boundaries are strides of whole eights for the 16-bit types, of whole fours for float32."""
    odd = _rows(bk, row_stride=68)
    for kind in (bk.BF16, bk.FP16):
        status, text = _store(bk, type=kind, keys=odd)
        assert status == bk.ERR_INVALID and "keys: vectors must start on 16-byte boundaries" in text
    for change in (dict(row_stride=66), dict(head_stride=1022), dict(batch_stride=(1 << 20) + 2)):
        status, text = _store(bk, type=bk.F32, values=_rows(bk, **change))
        assert status == bk.ERR_INVALID and "values: vectors must start on 16-byte boundaries" in text
    # behind these boundaries, the next check speaks
    status, text = _store(bk, type=bk.F32, keys=odd, values=odd, table=None)
    assert status == bk.ERR_INVALID and "table: null pointer" in text


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_ranges_of_states(bk, dim):
    """Ranges of at least 512 states up to 64 rows per state head, of at least 256 with more rows, no more
    than give the GPU 512 or 256 workgroups, and no more than 64."""
    size = bk.lib().bitsknn_cross_attention_workspace_bytes
    padded = 64 * -(-dim // 64) if dim <= 128 else 256

    def ranges(**kw):
        shape = _shape(bk, dim=dim, **kw)
        per = shape.batch * shape.query_heads * shape.queries * (4 * padded + 8)
        assert size(shape) % per == 0
        return size(shape) // per

    few = dict(batch=1, query_heads=4, state_heads=2, queries=32)
    assert ranges(states=1023, **few) == 0 and ranges(states=1024, **few) == 2
    assert ranges(states=1 << 20, **few) == 64
    many = dict(batch=1, query_heads=4, state_heads=2, queries=33)
    assert ranges(states=511, **many) == 0 and ranges(states=512, **many) == 2
    assert ranges(states=1 << 20, **many) == 64
    # 256 and 128 workgroups already: one more each makes 512 and 256
    assert ranges(states=1 << 20, batch=64, query_heads=8, state_heads=4, queries=1) == 2
    assert ranges(states=1 << 20, batch=128, query_heads=8, state_heads=4, queries=1) == 0
    assert ranges(states=1 << 20, batch=32, query_heads=8, state_heads=4, queries=33) == 2
    assert ranges(states=1 << 20, batch=64, query_heads=8, state_heads=4, queries=33) == 0
