"""Gradients of attention over states of another length (bitsknn_cross_attention_backward) against the
formula in 64 bits and against differences; the bounds are derived in attention_ref.py."""
import math

import pytest

import attention_ref as ref
from test_attention_gpu import SHAPES, TYPES

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

MORE = [(2, 8, 2, 65, 257, 64), (1, 2, 2, 1, 600, 128), (1, 8, 1, 90, 33, 96), (2, 1, 1, 700, 31, 128),
        (1, 2, 1, 40, 140, 256), (9, 3, 3, 2, 2, 24)]


def _inputs(dev, shape, dtype, seed=1):
    b, h, hs, q, n, d = shape
    return [ref.made(seed, (b, h, q, d), dtype).to(dev), ref.made(seed + 1, (b, h, q, d), dtype, 1.5).to(dev),
            ref.made(seed + 2, (b, hs, n, d), dtype).to(dev), ref.made(seed + 3, (b, hs, n, d), dtype).to(dev)]


def _check(bk, grad_out, queries, keys, values, counts=None, mask=None, scale=None, out=None, lse=None, **kw):
    used = queries.shape[3] ** -0.5 if scale is None else scale
    if out is None:
        out, lse = bk.cross_attention(queries, keys, values, counts, mask, scale)
    keep = ref.taking_part(keys.shape[0], keys.shape[2], counts, mask)
    got = bk.cross_attention_backward(grad_out, queries, keys, values, out, lse, counts, mask, scale, **kw)
    torch.cuda.synchronize()
    wants = ref.gradients(grad_out, queries, keys, values, out, lse, used, keep)
    for name, one, (want, bound) in zip(("queries", "keys", "values"), got, wants):
        ref.check(one, want, bound, name)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES + MORE)
def test_all_states(bk, dev, shape, dtype):
    _check(bk, *_inputs(dev, shape, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES + MORE)
@pytest.mark.parametrize("kind", ["counts", "mask", "both"])
def test_states_that_take_no_part(bk, dev, shape, dtype, kind):
    """They hold NaN and infinities; their gradients are zero, and so are those of rows without states."""
    b, _, _, _, n, _ = shape
    grad_out, queries, keys, values = _inputs(dev, shape, dtype, 7)
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
    keep = ref.taking_part(b, n, counts, mask).to(dev)
    gone = ~keep[:, None, :, None]
    keys = keys.masked_fill(gone, math.inf)
    values = values.masked_fill(gone, math.nan)
    grads = _check(bk, grad_out, queries, keys, values, counts=counts, mask=mask)
    assert (grads[0][~keep.any(1)] == 0).all()
    for x in grads[1:]:
        assert (x.masked_fill(keep[:, None, :, None], 0.0) == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_very_low_and_high_log_sums(bk, dev, dtype):
    """All scores far below or above zero, some states masked: their weights from zeros are out of range."""
    shape = (2, 2, 1, 40, 100, 64)
    grad_out, queries, keys, values = _inputs(dev, shape, dtype, 11)
    mask = torch.ones((2, 100), dtype=torch.bool)
    mask[:, ::3] = False
    for sign in (-1, 1):
        q = queries.clone()
        q[..., 0] = 16 * sign
        k = keys.clone()
        k[..., 0] = 12
        _check(bk, grad_out, q, k, values, mask=mask.to(dev), scale=1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts_and_strides(bk, dev, dtype):
    b, h, hs, q, n, d = shape = (2, 6, 3, 50, 130, 72)
    tensors = _inputs(dev, shape, dtype, 20)
    want = _check(bk, *tensors)
    rows = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in tensors]
    out, lse = bk.cross_attention(*rows[1:])
    wide = [torch.full((b, m, g, 96), 3.0, dtype=dtype, device=dev) for m, g in ((q, h), (n, hs), (n, hs))]
    got = bk.cross_attention_backward(*rows, out, lse, grad_queries=wide[0][..., 8:80].transpose(1, 2),
                                      grad_keys=wide[1][..., 8:80].transpose(1, 2),
                                      grad_values=wide[2][..., 16:88].transpose(1, 2))
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    for x, first in zip(wide, (8, 8, 16)):
        assert (x[..., :first] == 3).all() and (x[..., first + 72:] == 3).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_broadcast_inputs(bk, dev, dtype):
    """States that the batch shares and a gradient that all rows share come in with strides of zero; a
    state's gradients come out per sequence."""
    b, h, hs, q, n, d = shape = (3, 4, 2, 30, 70, 64)
    grad_out, queries, keys, values = _inputs(dev, shape, dtype, 30)
    keys, values = (x[:1].expand(b, -1, -1, -1) for x in (keys, values))
    grad_out = grad_out[:1, :1, :1].expand(b, h, q, d)
    grads = _check(bk, grad_out, queries, keys, values)
    again = _check(bk, grad_out.contiguous(), queries, keys.contiguous(), values.contiguous())
    for x, y in zip(grads, again):
        assert x.shape == y.shape and torch.equal(x, y)


@pytest.mark.parametrize("shape", [(2, 2, 2, 0, 5, 64), (0, 2, 2, 3, 5, 64), (2, 2, 1, 3, 0, 64)])
def test_sizes_of_zero(bk, dev, shape):
    for x in _check(bk, *_inputs(dev, shape, torch.bfloat16)):
        assert (x == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 4, 2, 9, 40, 64), (2, 2, 1, 70, 150, 128)])
def test_against_differences(bk, dev, shape, dtype):
    """The slope of sum(grad_out * out) along a direction, from the definition of out in 64 bits at two
    points, against the gradients' product with the direction.  What the gradients may be off by: their
    bounds times the direction, and what the rounding of out adds through delta (u |out| per value, times
    P |k| and the like); the difference itself is off by far less (h^2 of the third derivative)."""
    grad_out, queries, keys, values = _inputs(dev, shape, dtype, 40)
    scale = shape[-1] ** -0.5
    keep = ref.taking_part(shape[0], shape[4])
    out, lse = bk.cross_attention(queries, keys, values)
    got = bk.cross_attention_backward(grad_out, queries, keys, values, out, lse)
    torch.cuda.synchronize()
    exact = ref.attention(queries, keys, values, scale, keep)
    g = grad_out.cpu().double()
    points = [x.cpu().double() for x in (queries, keys, values)]
    names = ("queries", "keys", "values")

    class As64:  # a float64 tensor that the reference takes as one of the 16-bit type
        def __init__(self, x):
            self.x, self.dtype, self.shape = x, dtype, x.shape

        def detach(self):
            return self

        def cpu(self):
            return self

        def double(self):
            return self.x

    wants = ref.gradients(grad_out, queries, keys, values, As64(exact[0]), As64(exact[1]), scale, keep)
    share = shape[1] // shape[2]
    k = points[1].repeat_interleave(share, 1)
    weights = torch.exp(points[0] @ k.mT * scale - exact[1][..., None])
    off = ((g.abs() * exact[2]).sum(-1, keepdim=True) + (exact[3][..., None] + 1e-6) * (g * exact[0]).abs().sum(-1, keepdim=True)) * weights
    lse_off = (exact[3][..., None] * 2) * weights * (g @ points[2].repeat_interleave(share, 1).mT).abs()
    extra = [scale * (off + lse_off) @ k.abs(),
             scale * ((off + lse_off).mT @ points[0].abs()).view(shape[0], shape[2], share, shape[4], -1).sum(2),
             ((exact[3][..., None] * 2 * weights).mT @ g.abs()).view(shape[0], shape[2], share, shape[4], -1).sum(2)]
    h = 1e-4
    for i, name in enumerate(names):
        along = ref.made(60 + i, points[i].shape, torch.float64)
        ends = []
        for sign in (1, -1):
            moved = [As64(x + sign * h * along if j == i else x) for j, x in enumerate(points)]
            ends.append((g * ref.attention(*moved, scale, keep)[0]).sum())
        slope = float((ends[0] - ends[1]) / (2 * h))
        product = float((got[i].cpu().double() * along).sum())
        room = float(((wants[i][1] + extra[i]) * along.abs()).sum()) + 1e-5 * abs(slope)
        assert abs(product - slope) <= room, (name, product, slope, room)
        assert abs(float((wants[i][0] * along).sum()) - slope) <= 1e-5 * (1 + abs(slope)), name


def test_workspaces(bk, dev):
    grad_out, queries, keys, values = _inputs(dev, (1, 4, 2, 33, 700, 64), torch.bfloat16, 50)
    need = bk.cross_attention_backward_workspace_bytes(queries, keys)
    room = torch.full((need + 64,), 0xAB, dtype=torch.uint8, device=dev)
    _check(bk, grad_out, queries, keys, values, workspace=room[:need])
    assert (room[need:] == 0xAB).all()
    out, lse = bk.cross_attention(queries, keys, values)
    with pytest.raises(bk.BitsKnnError, match="a workspace of 16 bytes"):
        bk.cross_attention_backward(grad_out, queries, keys, values, out, lse, workspace=room[:16])


def test_the_same_bits_every_time(bk, dev):
    grad_out, queries, keys, values = _inputs(dev, (2, 8, 2, 300, 900, 128), torch.bfloat16, 52)
    out, lse = bk.cross_attention(queries, keys, values)
    first = bk.cross_attention_backward(grad_out, queries, keys, values, out, lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [bk.cross_attention_backward(grad_out, queries, keys, values, out, lse) for _ in range(3)]
    side.synchronize()
    for grads in again:
        for x, y in zip(grads, first):
            assert torch.equal(x, y)


def test_offsets_beyond_32_bits(bk, dev):
    n, d, stride = 70000, 64, 1 << 16
    store = torch.empty(n * stride, dtype=torch.bfloat16, device=dev)
    views = [store.as_strided((1, 1, n, d), (0, 0, stride, 1), 128 * i) for i in range(4)]
    dense = [ref.made(i, (1, 1, n, d), torch.bfloat16).to(dev) for i in (1, 2)]
    views[0].copy_(dense[0])
    views[1].copy_(dense[1])
    queries, grad_out = (ref.made(i, (1, 1, 40, d), torch.bfloat16).to(dev) for i in (3, 4))
    out, lse = bk.cross_attention(queries, *dense)
    want = bk.cross_attention_backward(grad_out, queries, *dense, out, lse)
    got = bk.cross_attention_backward(grad_out, queries, views[0], views[1], out, lse, grad_keys=views[2],
                                      grad_values=views[3])
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_step_replayed_from_a_graph(bk, dev):
    """Forward and backward captured together; inputs, counts and mask change between the replays while
    eager steps on the same tensors run in between."""
    shape = (3, 4, 2, 70, 500, 64)
    grad_out, queries, keys, values = _inputs(dev, shape, torch.float16, 54)
    counts = torch.tensor([500, 7, 0], dtype=torch.int32, device=dev)
    mask = torch.ones((3, 500), dtype=torch.bool, device=dev)
    out, lse = torch.empty_like(queries), torch.empty(queries.shape[:3], device=dev)
    grads = [torch.empty_like(x) for x in (queries, keys, values)]
    rooms = [torch.empty(f(queries, keys), dtype=torch.uint8, device=dev)
             for f in (bk.cross_attention_workspace_bytes, bk.cross_attention_backward_workspace_bytes)]

    def step():
        bk.cross_attention(queries, keys, values, counts, mask, out=out, lse=lse, workspace=rooms[0])
        bk.cross_attention_backward(grad_out, queries, keys, values, out, lse, counts, mask, None, *grads, rooms[1])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for replay in range(4):
        keys.mul_(1.1)
        values.neg_()
        counts.copy_(torch.tensor([500 - 60 * replay, 30 * replay, 99], dtype=torch.int32))
        mask[:, replay::5] = False
        eager_out, eager_lse = bk.cross_attention(queries, keys, values, counts, mask)
        want = bk.cross_attention_backward(grad_out, queries, keys, values, eager_out, eager_lse, counts, mask)
        for x in grads:
            x.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip([out, lse] + grads, [eager_out, eager_lse] + list(want)):
            assert torch.equal(x, y), replay


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [3, 64, 65, 200])
@pytest.mark.parametrize("kind", ["counts", "mask"])
def test_rows_without_states_whatever_they_hold(bk, dev, dtype, dim, rows, kind):
    """Sequence 1 has no state; its queries and its incoming gradients hold NaN and infinities."""
    n = 100
    grad_out, queries, keys, values = _inputs(dev, (3, 1, 1, rows, n, dim), dtype, 60)
    for x, shift in ((queries, 0), (grad_out, 1)):
        x[1, :, shift::3] = math.nan
        x[1, :, (shift + 1) % 3::3, 0] = math.inf
        x[1, :, (shift + 2) % 3::5, -1] = -math.inf
    counts = torch.tensor([n, 0, n // 2 + 1], dtype=torch.int32, device=dev)
    mask = torch.arange(n, device=dev)[None] < counts[:, None]
    part = {"counts": counts} if kind == "counts" else {"mask": mask}
    out = torch.zeros_like(queries)
    lse = torch.full(queries.shape[:3], -math.inf, device=dev)
    for b in (0, 2):
        one, one_lse = bk.cross_attention(queries[b:b + 1], keys[b:b + 1], values[b:b + 1], mask=mask[b:b + 1])
        out[b], lse[b] = one[0], one_lse[0]
    got = bk.cross_attention_backward(grad_out, queries, keys, values, out, lse, **part)
    for x in got:
        assert (x[1] == 0).all()
    for b in (0, 2):
        s = slice(b, b + 1)
        wants = ref.gradients(grad_out[s], queries[s], keys[s], values[s], out[s], lse[s], dim ** -0.5, mask[s].cpu())
        for name, one, (want, bound) in zip(("queries", "keys", "values"), got, wants):
            ref.check(one[s], want, bound, name)


def _check_large(bk, grad_out, queries, keys, values, scale, mask=None):
    """fp16 gradients where derivatives of the scores are beyond fp16's largest number.  A derivative then
    enters the products times a power of two of its row (queries) or state (keys) that brings the largest
    to at least 2^14, so what vanishes below fp16's least number, 2^-25, is at most 2^-25 times
    (largest / 2^14): added to the bound, for all rows and states."""
    out, lse = bk.cross_attention(queries, keys, values, mask=mask, scale=scale)
    keep = ref.taking_part(keys.shape[0], keys.shape[2], None, mask)
    got = bk.cross_attention_backward(grad_out, queries, keys, values, out, lse, mask=mask, scale=scale)
    torch.cuda.synchronize()
    wants = ref.gradients(grad_out, queries, keys, values, out, lse, scale, keep)
    b, hs, n, dim = keys.shape
    share = queries.shape[1] // hs
    q, g, o, l = (x.cpu().double() for x in (queries, grad_out, out, lse))
    gone = ~keep[:, None, :, None]
    k, v = (x.cpu().double().masked_fill(gone, 0.0).repeat_interleave(share, 1) for x in (keys, values))
    weights = torch.exp(q @ k.mT * scale - l[..., None]).masked_fill(~keep[:, None, None, :], 0.0)
    slope = (weights * (g @ v.mT - (g * o).sum(-1, keepdim=True))).abs()
    by_row = slope.amax(-1, keepdim=True)
    by_state = slope.amax(2).view(b, hs, share, n).amax(2).repeat_interleave(share, 1)[:, :, None]
    assert float(by_row.max()) > 65504 and float(by_state.max()) > 65504  # what this is about
    lost = [1.1 * 2.0 ** -25 * x / 2.0 ** 14 for x in (by_row, by_state)]
    extra = [scale * lost[0] * k.abs().sum(2, keepdim=True),
             scale * (lost[1].mT * q.abs().sum(2, keepdim=True)).view(b, hs, share, n, dim).sum(2), 0.0]
    finite = [float((want.abs() < 60000).double().mean()) for want, _ in wants]
    assert min(finite) > 0.5, finite
    for name, one, (want, bound), more in zip(("queries", "keys", "values"), got, wants, extra):
        ref.check(one, want, bound + more, name)


@pytest.mark.parametrize("shape", [(2, 4, 2, 70, 150, 128), (1, 2, 1, 40, 140, 256), (2, 2, 1, 90, 300, 64), (1, 8, 1, 33, 40, 72)])
@pytest.mark.parametrize("power", [12, 13])
def test_large_derivatives_in_fp16(bk, dev, shape, power):
    grad_out, queries, keys, values = _inputs(dev, shape, torch.float16, 70)
    _check_large(bk, grad_out * 2.0 ** power, queries, keys, values * 8, shape[-1] ** -0.5)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_derivatives_that_grow_in_fp16(bk, dev, dim):
    """They leave fp16's range late in both walks, for some rows and states only; peaked weights."""
    b, h, hs, q, n, d = shape = (2, 2, 1, 150, 260, dim)
    grad_out, queries, keys, values = _inputs(dev, shape, torch.float16, 80)
    grad_out = grad_out * torch.exp2(torch.linspace(-4, 12, q, device=dev))[:, None].half()
    values = values * torch.exp2(torch.linspace(-4, 5, n, device=dev))[:, None].half()
    grad_out[:, :, 5::7] = grad_out[:, :, 5::7] * 2.0 ** -14
    mask = torch.rand((b, n), generator=torch.Generator().manual_seed(1)) < 0.8
    _check_large(bk, grad_out, queries, keys, values, 2.0 * d ** -0.5, mask.to(dev))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_that_hold_no_numbers_spoil_their_own_gradients_only(bk, dev, dtype, dim):
    """A NaN in a row's incoming gradient: NaN in its query's gradient and in those of the states that it
    reads; the rows beside it and the other sequence as without it, large ones too."""
    grad_out, queries, keys, values = _inputs(dev, (2, 2, 1, 70, 90, dim), dtype, 90)
    grad_out = grad_out * 2.0 ** 11
    grad_out[1, :, 5::9] = 0.0
    out, lse = bk.cross_attention(queries, keys, values)
    want = bk.cross_attention_backward(grad_out, queries, keys, values, out, lse)
    grad_out[1, :, 5::9] = math.nan
    got = bk.cross_attention_backward(grad_out, queries, keys, values, out, lse)
    spoilt = torch.zeros(70, dtype=torch.bool, device=dev)
    spoilt[5::9] = True
    for x, y in zip(got, want):
        assert torch.equal(x[0], y[0])
    assert torch.equal(got[0][1, :, ~spoilt], want[0][1, :, ~spoilt])
    assert got[0][1, :, spoilt].isnan().all() and got[1][1].isnan().all() and got[2][1].isnan().all()
