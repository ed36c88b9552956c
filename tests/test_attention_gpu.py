"""Attention over states of another length (bitsknn_cross_attention) against the definition in 64 bits;
the bounds are derived in attention_ref.py."""
import math

import pytest

import attention_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]
# batch, query heads, state heads, queries, states, dim
SHAPES = [
    (1, 1, 1, 1, 1, 8),
    (2, 4, 2, 3, 63, 64),
    (1, 2, 1, 33, 64, 72),
    (2, 2, 2, 129, 65, 128),
    (1, 8, 2, 1, 1000, 128),
    (3, 16, 16, 1, 333, 64),
    (1, 3, 3, 5, 300, 256),
    (2, 6, 2, 31, 257, 80),
    (1, 1, 1, 200, 5, 200),
    (1, 10, 2, 7, 2049, 40),
    (4, 5, 1, 64, 128, 16),
    (2, 4, 4, 300, 700, 128),
]


def _inputs(dev, shape, dtype, seed=1):
    b, h, hs, q, n, d = shape
    return (ref.made(seed, (b, h, q, d), dtype, 1.5).to(dev), ref.made(seed + 1, (b, hs, n, d), dtype).to(dev),
            ref.made(seed + 2, (b, hs, n, d), dtype).to(dev))


def _check(bk, queries, keys, values, counts=None, mask=None, scale=None, **kw):
    keep = ref.taking_part(keys.shape[0], keys.shape[2], counts, mask)
    used = queries.shape[3] ** -0.5 if scale is None else scale
    out, lse, out_bound, lse_bound = ref.attention(queries, keys, values, used, keep)
    got, got_lse = bk.cross_attention(queries, keys, values, counts=counts, mask=mask, scale=scale, **kw)
    torch.cuda.synchronize()
    ref.check(got, out, out_bound, "out")
    ref.check(got_lse, lse, lse_bound, "lse")
    return got, got_lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_all_states(bk, dev, shape, dtype):
    _check(bk, *_inputs(dev, shape, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["counts", "mask", "both"])
def test_states_that_take_no_part_hold_anything(bk, dev, shape, dtype, kind):
    b, _, _, _, n, _ = shape
    queries, keys, values = _inputs(dev, shape, dtype, 7)
    counts = mask = None
    gen = torch.Generator()
    gen.manual_seed(3)
    if kind != "mask":
        counts = torch.randint(0, n + 1, (b,), generator=gen, dtype=torch.int32)
        counts[0] = (n + 1) // 2
        counts = counts.to(dev)
    if kind != "counts":
        mask = torch.rand((b, n), generator=gen) < 0.6
        mask[b - 1] = False
        mask = mask.to(dev)
    gone = ~ref.taking_part(b, n, counts, mask).to(dev)[:, None, :, None]
    keys = keys.masked_fill(gone, math.nan)
    values = values.masked_fill(gone, math.inf)
    got, lse = _check(bk, queries, keys, values, counts=counts, mask=mask)
    empty = ~ref.taking_part(b, n, counts, mask).any(1)
    assert (got[empty.to(dev)] == 0).all() and (lse[empty.to(dev)] == -math.inf).all()


def test_counts_outside_the_range(bk, dev):
    queries, keys, values = _inputs(dev, (4, 2, 2, 3, 100, 64), torch.bfloat16)
    counts = torch.tensor([-5, 0, 1, 1000], dtype=torch.int32, device=dev)
    got, lse = bk.cross_attention(queries, keys, values, counts=counts)
    plain, plain_lse = bk.cross_attention(queries, keys, values,
                                          counts=torch.tensor([0, 0, 1, 100], dtype=torch.int32, device=dev))
    assert torch.equal(got, plain) and torch.equal(lse, plain_lse)
    assert (got[:2] == 0).all() and torch.equal(got[2], values[2, :, :1].expand(2, 3, 64))


@pytest.mark.parametrize("dtype", TYPES)
def test_masks_of_bytes_and_with_a_row_stride(bk, dev, dtype):
    queries, keys, values = _inputs(dev, (2, 4, 2, 9, 200, 64), dtype)
    wide = torch.randint(0, 3, (2, 333), generator=torch.Generator().manual_seed(0), dtype=torch.uint8).to(dev)
    _check(bk, queries, keys, values, mask=wide[:, 100:300])
    _check(bk, queries, keys, values, mask=wide[:1, 7:207].expand(2, 200))


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts_and_strides(bk, dev, dtype):
    b, h, hs, q, n, d = 2, 6, 3, 50, 130, 72
    queries, keys, values = _inputs(dev, (b, h, hs, q, n, d), dtype, 20)
    want, want_lse = _check(bk, queries, keys, values)
    # batch x rows x heads x dim, queries, keys and values side by side in wider rows
    rows = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    wide = torch.full((b, n, hs, 2 * d + 8), math.nan, dtype=dtype, device=dev)
    wide[..., :d] = keys.transpose(1, 2)
    wide[..., d + 8:] = values.transpose(1, 2)
    out = torch.full((b, q, h, 96), 3.0, dtype=dtype, device=dev)
    got, lse = bk.cross_attention(rows(queries), wide[..., :d].transpose(1, 2), wide[..., d + 8:].transpose(1, 2),
                                  out=out[..., 8:80].transpose(1, 2))
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    assert (out[..., :8] == 3).all() and (out[..., 80:] == 3).all()
    # one sequence's states read by the whole batch, and one query row by every head
    shared = bk.cross_attention(queries, keys[:1].expand(b, -1, -1, -1), values[:1].expand(b, -1, -1, -1))
    again = bk.cross_attention(queries, keys[:1].repeat(b, 1, 1, 1), values[:1].repeat(b, 1, 1, 1))
    assert torch.equal(shared[0], again[0]) and torch.equal(shared[1], again[1])
    one = queries[:, :1, :1].expand(b, h, q, d)
    _check(bk, one, keys, values)


@pytest.mark.parametrize("shape", [(2, 2, 2, 0, 5, 64), (0, 2, 2, 3, 5, 64), (2, 2, 1, 3, 0, 64)])
def test_sizes_of_zero(bk, dev, shape):
    queries, keys, values = _inputs(dev, shape, torch.bfloat16)
    out, lse = bk.cross_attention(queries, keys, values)
    torch.cuda.synchronize()
    assert out.shape == queries.shape and (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread", [1e-3, 8.0, 60.0])
def test_flat_and_peaked_weights(bk, dev, dtype, spread):
    queries, keys, values = _inputs(dev, (1, 4, 2, 17, 500, 128), dtype, 5)
    _check(bk, queries, keys, values, scale=spread * 128 ** -0.5)


@pytest.mark.parametrize("order", ["rising", "falling"])
def test_scores_in_order(bk, dev, order):
    """The maximum moves with every tile, or never after the first."""
    n, d = 1100, 64
    keys = torch.zeros((1, 1, n, d))
    ramp = torch.arange(n, dtype=torch.float32) / 8
    keys[0, 0, :, 0] = ramp if order == "rising" else ramp.flip(0)
    queries = torch.zeros((1, 1, 40, d))
    queries[..., 0] = torch.linspace(-4, 4, 40)[None, None]
    values = ref.made(4, (1, 1, n, d), torch.bfloat16)
    _check(bk, queries.bfloat16().to(dev), keys.bfloat16().to(dev), values.to(dev), scale=1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_workspaces(bk, dev, dtype):
    """Few rows over many states: with the ranges that the call wants, with room for fewer, with none."""
    queries, keys, values = _inputs(dev, (1, 4, 2, 3, 4100, 128), dtype, 9)
    counts = torch.tensor([2500], dtype=torch.int32, device=dev)
    need = bk.cross_attention_workspace_bytes(queries, keys)
    assert need > 0
    for size in (need, need // 2, need // 5, 16, 0):
        room = torch.full((size + 64,), 0xAB, dtype=torch.uint8, device=dev)
        _check(bk, queries, keys, values, counts=counts, workspace=room[:size])
        assert (room[size:] == 0xAB).all()


def test_offsets_beyond_32_bits(bk, dev):
    """Keys and values whose rows lie 2^16 elements apart: the last ones begin behind 2^32 elements."""
    n, d, stride = 70000, 64, 1 << 16
    store = torch.empty(n * stride, dtype=torch.bfloat16, device=dev)
    keys = store.as_strided((1, 1, n, d), (0, 0, stride, 1))
    values = store.as_strided((1, 1, n, d), (0, 0, stride, 1), 128)
    dense = ref.made(1, (1, 1, n, d), torch.bfloat16).to(dev), ref.made(2, (1, 1, n, d), torch.bfloat16).to(dev)
    keys.copy_(dense[0])
    values.copy_(dense[1])
    for q in (1, 150):
        queries = ref.made(3, (1, 1, q, d), torch.bfloat16, 2.0).to(dev)
        got = bk.cross_attention(queries, keys, values)
        want = bk.cross_attention(queries, *dense)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_another_stream_and_repeated_calls(bk, dev):
    queries, keys, values = _inputs(dev, (2, 8, 2, 1, 3000, 128), torch.float16, 11)
    want = bk.cross_attention(queries, keys, values)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [bk.cross_attention(queries, keys, values) for _ in range(3)]
    side.synchronize()
    for out, lse in got:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_replayed_from_a_graph(bk, dev):
    """Counts and mask change between the replays; eager calls run in between."""
    queries, keys, values = _inputs(dev, (3, 8, 2, 2, 2000, 64), torch.bfloat16, 13)
    counts = torch.tensor([2000, 7, 0], dtype=torch.int32, device=dev)
    mask = torch.ones((3, 2000), dtype=torch.bool, device=dev)
    out = torch.empty_like(queries)
    lse = torch.empty(queries.shape[:3], device=dev)
    room = torch.empty(bk.cross_attention_workspace_bytes(queries, keys), dtype=torch.uint8, device=dev)
    bk.cross_attention(queries, keys, values, counts, mask, out=out, lse=lse, workspace=room)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bk.cross_attention(queries, keys, values, counts, mask, out=out, lse=lse, workspace=room)
    for replay in range(4):
        counts.copy_(torch.tensor([2000 - 300 * replay, 100 * replay, 999], dtype=torch.int32))
        mask[:, replay::5] = False
        want = bk.cross_attention(queries, keys, values, counts, mask)
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), replay


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [3, 64, 65, 200])
@pytest.mark.parametrize("kind", ["counts", "mask"])
def test_rows_without_states_whatever_the_queries_hold(bk, dev, dtype, dim, rows, kind):
    """A padded batch: sequence 1 has no state, its queries hold NaN and infinities.  Also with enough
    states for several ranges."""
    for n in (70, 1100):
        queries, keys, values = _inputs(dev, (3, 1, 1, rows, n, dim), dtype, 15)
        queries[1, :, 0::3] = math.nan
        queries[1, :, 1::3, 0] = math.inf
        queries[1, :, 2::3, -1] = -math.inf
        counts = torch.tensor([n, 0, n // 2 + 1], dtype=torch.int32, device=dev)
        mask = torch.arange(n, device=dev)[None] < counts[:, None]
        gone = ~mask[:, None, :, None]
        keys, values = keys.masked_fill(gone, math.nan), values.masked_fill(gone, math.inf)
        out, lse = bk.cross_attention(queries, keys, values, **({"counts": counts} if kind == "counts" else {"mask": mask}))
        assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
        for b in (0, 2):
            want = ref.attention(queries[b:b + 1], keys[b:b + 1], values[b:b + 1], dim ** -0.5, mask[b:b + 1].cpu())
            ref.check(out[b:b + 1], want[0], want[2], "out")
            ref.check(lse[b:b + 1], want[1], want[3], "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [64, 65])
def test_scores_of_minus_infinity(bk, dev, dtype, rows):
    """Rows all of whose scores are minus infinity count as rows without states, whatever is masked; one
    finite score decides a row."""
    queries, keys, values = _inputs(dev, (1, 1, 1, rows, 150, 64), dtype, 16)
    keys[..., 0] = keys[..., 0].abs() + 1
    keys[0, 0, 77, 0] = 0.0
    queries[..., 0] = -math.inf
    mask = torch.rand((1, 150), generator=torch.Generator().manual_seed(5)) < 0.7
    mask[0, 77] = False
    out, lse = bk.cross_attention(queries, keys, values, mask=mask.to(dev))
    assert (out == 0).all() and (lse == -math.inf).all()
    queries[..., 0] = 1.0
    keys[..., 0] = -math.inf
    mask[0, 77] = True
    keys[0, 0, 77, 0] = 0.0
    out, lse = bk.cross_attention(queries, keys, values, mask=mask.to(dev))
    assert torch.equal(out, values[:, :, 77:78].expand_as(out)) and lse.isfinite().all()


def test_more_rows_than_a_join_could_hold(bk, dev):
    """2^26 rows and some: more than one launch of the kernel that joins ranges could take, which a call with
    enough rows does not launch.  Against a call with the last rows only."""
    rows = (1 << 26) + 5
    queries = torch.empty((1, 1, rows, 8), dtype=torch.bfloat16, device=dev)
    queries[:] = ref.made(31, (1, 1, 1, 8), torch.bfloat16).to(dev)
    last = ref.made(32, (1, 1, 517, 8), torch.bfloat16).to(dev)
    queries[:, :, -517:] = last
    keys, values = (ref.made(s, (1, 1, 5, 8), torch.bfloat16).to(dev) for s in (33, 34))
    out, lse = bk.cross_attention(queries, keys, values)
    want, want_lse = bk.cross_attention(last, keys, values)
    assert torch.equal(out[:, :, -517:], want) and torch.equal(lse[:, :, -517:], want_lse)
    assert torch.equal(out[:, :, 1 << 25], out[:, :, 0]) and torch.equal(lse[:, :, 1 << 25], lse[:, :, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 70])
@pytest.mark.parametrize("scale", [1e-44, 1e-38, 1e-20])
def test_scales_near_zero(bk, dev, dtype, rows, scale):
    """Below fp32's least normal number too: all states that take part count the same, the others nothing."""
    queries, keys, values = _inputs(dev, (2, 2, 1, rows, 200, 64), dtype, 18)
    mask = torch.rand((2, 200), generator=torch.Generator().manual_seed(6)) < 0.5
    _check(bk, queries, keys, values, mask=mask.to(dev), scale=scale)


def test_autograd_does_not_see_the_call(bk, dev):
    """As documented: inputs that require gradients are taken, the result has no history."""
    queries, keys, values = (x.requires_grad_() for x in _inputs(dev, (1, 2, 2, 3, 40, 64), torch.bfloat16))
    out, lse = bk.cross_attention(queries, keys, values)
    assert not out.requires_grad and not lse.requires_grad
    grads = bk.cross_attention_backward(torch.ones_like(out), queries, keys, values, out, lse)
    assert not any(x.requires_grad for x in grads)
    assert "autograd does not see" in bk.cross_attention.__doc__
