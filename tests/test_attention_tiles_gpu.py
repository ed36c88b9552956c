"""More rows per state head than the stream kernel takes (64): the kernels that share tiles of states among
waves, for states of the caller and of the cache, at the contents and sizes where a tile's hand-over, the
moving reference of the exponents, ranges and part blocks can go wrong.  Bounds as in attention_ref.py."""
import math

import pytest

import attention_ref as ref
import test_attention_gpu as plain
import test_state_cache_gpu as cached

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = plain.TYPES
DIMS = [40, 64, 72, 128, 200, 256]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("rows,states", [(65, 700), (290, 513), (100, 64), (257, 97), (66, 1)])
def test_all_states(bk, dev, dtype, dim, rows, states):
    plain._check(bk, *plain._inputs(dev, (2, 2, 1, rows // 2 + 1, states, dim), dtype, 3))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("order", ["rising", "falling", "late"])
@pytest.mark.parametrize("ranges", [True, False])
def test_scores_in_order(bk, dev, dim, order, ranges):
    """The maximum moves with every tile, never after the first, or only at the last states."""
    n, rows = 1100, 150
    ramp = torch.arange(n, dtype=torch.float32) / 8
    if order == "falling":
        ramp = ramp.flip(0)
    if order == "late":
        ramp = torch.where(torch.arange(n) >= n - 3, ramp, ramp / 64)
    keys = torch.zeros((1, 1, n, dim))
    keys[0, 0, :, 0] = ramp
    queries = torch.zeros((1, 1, rows, dim))
    queries[..., 0] = torch.linspace(-4, 4, rows)[None, None]
    values = ref.made(4, (1, 1, n, dim), torch.bfloat16)
    room = None if ranges else torch.empty(0, dtype=torch.uint8, device=dev)
    plain._check(bk, queries.bfloat16().to(dev), keys.bfloat16().to(dev), values.to(dev), scale=1.0, workspace=room)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 200])
@pytest.mark.parametrize("spread", [1e-3, 8.0, 60.0])
def test_flat_and_peaked_weights(bk, dev, dtype, dim, spread):
    plain._check(bk, *plain._inputs(dev, (1, 4, 2, 50, 900, dim), dtype, 5), scale=spread * dim ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_workspaces(bk, dev, dtype, dim):
    """With the ranges that the call wants, with room for fewer, with none."""
    queries, keys, values = plain._inputs(dev, (2, 4, 2, 70, 2100, dim), dtype, 9)
    counts = torch.tensor([2100, 777], dtype=torch.int32, device=dev)
    need = bk.cross_attention_workspace_bytes(queries, keys)
    assert need > 0
    for size in (need, need // 2, need // 5, 16, 0):
        room = torch.full((size + 64,), 0xAB, dtype=torch.uint8, device=dev)
        plain._check(bk, queries, keys, values, counts=counts, workspace=room[:size])
        assert (room[size:] == 0xAB).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_masks(bk, dev, dtype, dim):
    """Bytes of any value, rows of a wider array, tiles without any state at either end and in the middle."""
    n = 600
    queries, keys, values = plain._inputs(dev, (2, 4, 2, 45, n, dim), dtype)
    wide = torch.randint(0, 3, (2, 2 * n), generator=torch.Generator().manual_seed(0), dtype=torch.uint8)
    wide[0, 100:300] = 0
    wide[1, 100 + 64:100 + 192] = 0
    wide[1, 100 + n - 130:] = 0
    wide = wide.to(dev)
    gone = (wide[:, 100:100 + n] == 0)[:, None, :, None]
    plain._check(bk, queries, keys.masked_fill(gone, math.nan), values.masked_fill(gone, math.inf),
                 mask=wide[:, 100:100 + n])
    plain._check(bk, queries, keys, values, mask=wide[:1, 7:7 + n].expand(2, n))


def test_replayed_from_a_graph(bk, dev):
    """Counts and mask change between the replays; eager calls run in between."""
    queries, keys, values = plain._inputs(dev, (3, 8, 2, 40, 2000, 64), torch.bfloat16, 13)
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


@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 64, 64), (4, 16, 16, 1, 1500, 64), (3, 12, 4, 333, 1001, 80),
                                   (2, 16, 4, 512, 2048, 128), (2, 2, 1, 130, 700, 256)])
def test_the_same_bits_every_time(bk, dev, shape):
    """Few rows and many, with ranges and without."""
    inputs = plain._inputs(dev, shape, torch.bfloat16, 17)
    first = bk.cross_attention(*inputs)
    for _ in range(5):
        again = bk.cross_attention(*inputs)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


# ---- states of the cache --------------------------------------------------------------------------

# batch, query heads, state heads, queries, entries, dim, block
CACHED = [
    (2, 4, 2, 40, 9, 40, 16),
    (1, 2, 1, 150, 21, 64, 16),
    (2, 3, 3, 66, 5, 64, 64),
    (1, 8, 2, 20, 3, 64, 256),
    (2, 2, 1, 50, 7, 128, 32),
    (1, 2, 2, 140, 12, 200, 16),
    (2, 4, 1, 33, 3, 256, 128),
    (1, 1, 1, 129, 9, 256, 32),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", CACHED)
@pytest.mark.parametrize("powers", [True, False])
def test_cached_whole_blocks(bk, dev, shape, dtype, powers):
    cache, table = cached._cache(bk, dev, shape, 1, powers)
    cached._check(bk, dev, cached._queries(shape, dtype), cache, table)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", CACHED)
def test_cached_part_and_missing_blocks(bk, dev, shape, dtype):
    """What takes no part holds NaN codes and scales that are NaN or infinite."""
    b, _, _, _, slots, _, block = shape
    cache, table = cached._cache(bk, dev, shape, 2)
    gen = torch.Generator().manual_seed(3)
    held = torch.randint(0, block + 1, cache.block_counts.shape, generator=gen, dtype=torch.int32)
    cache.block_counts.copy_(held)
    behind = (torch.arange(block)[None] >= held[:, None])[:, None, :, None].to(dev)
    cache.key_codes.masked_fill_(behind, 0x7F)
    cache.value_codes.masked_fill_(behind, 0xFF)
    empty = (held == 0)[:, None].to(dev)
    cache.key_scales.masked_fill_(empty, math.nan)
    cache.value_scales.masked_fill_(empty, math.inf)
    counts = torch.randint(0, slots * block + 1, (b,), generator=gen, dtype=torch.int32)
    for i, wrong in enumerate((2 ** 31 - 1, -1, -2 ** 31, int(cache.block_counts.numel()))):
        if slots > 2:
            table[i % b, (2 * i + 1) % slots] = wrong
    cached._check(bk, dev, cached._queries(shape, dtype), cache, table, counts)
    cached._check(bk, dev, cached._queries(shape, dtype), cache, table)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_cached_scales_far_apart(bk, dev, dtype, dim):
    """Values' scales from 2^-40 to 2^20, by sixteen states; then one block that decides every row."""
    shape = (1, 2, 1, 45, 12, dim, 16)
    cache, table = cached._cache(bk, dev, shape, 5)
    cache.value_scales.copy_(torch.exp2(torch.linspace(-40, 20, 16)).view(16, 1))
    cache.key_scales.copy_(torch.exp2(torch.arange(16) % 5 - 7.0).view(16, 1))
    cached._check(bk, dev, cached._queries(shape, dtype), cache, table)
    cache.key_scales.fill_(2.0 ** -20)
    chosen = int(table[0, 7])
    cache.key_scales[chosen] = 2.0 ** -4
    for name, power in ((chosen, -30.0), (int(table[0, 2]), 1.0)):
        cache.value_scales[name] = 2.0 ** power
    cached._check(bk, dev, cached._queries(shape, dtype), cache, table, scale=1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_cached_block_named_twice_counts_twice(bk, dev, dtype):
    shape = (2, 4, 2, 40, 6, 64, 32)
    cache, table = cached._cache(bk, dev, shape, 4)
    table[0, 3] = table[0, 1]
    table[1, :] = table[0, 0]
    cached._check(bk, dev, cached._queries(shape, dtype), cache, table)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_cached_workspaces(bk, dev, dtype, dim):
    shape = (2, 8, 2, 20, 50, dim, 32)
    cache, table = cached._cache(bk, dev, shape, 6)
    queries = cached._queries(shape, dtype)
    counts = torch.tensor([1500, 634], dtype=torch.int32)
    need = bk.cached_attention_workspace_bytes(queries.to(dev), cache, 50)
    assert need > 0
    for size in (need, need // 3, 0):
        room = torch.full((size + 64,), 0xAB, dtype=torch.uint8, device=dev)
        cached._check(bk, dev, queries, cache, table, counts, workspace=room[:size])
        assert (room[size:] == 0xAB).all()
