"""The 8-bit state cache: what bitsknn_cache_store writes (bit for bit against the definition on the
CPU) and attention over it (bitsknn_cached_attention) against the definition in 64 bits."""
import math

import pytest

import attention_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def _stored(x, block, count):
    """(codes, scales by block) of one head's states x (n x dim), the first `count` of them."""
    n, dim = x.shape
    codes, scales = [], []
    for first in range(0, count, block):
        part = x[first:min(count, first + block)].double()
        finite = part.masked_fill(~part.isfinite(), 0.0)
        top = float(finite.abs().max())
        exponent = -126
        if top > 0:
            mantissa, exponent = math.frexp(top / 448)
            exponent = max(-126, exponent - (mantissa == 0.5))
        part = part.masked_fill(~part.isfinite(), math.nan) / 2.0 ** exponent
        codes.append(part.float().to(torch.float8_e4m3fn))
        scales.append(2.0 ** exponent)
    return codes, scales


def _inputs(seed, shape, dtype):
    x = ref.made(seed, shape, torch.float32)
    b, h, n, d = shape
    x *= torch.exp2(torch.randint(-9, 9, (b, h, n // 16 + 1, 1), generator=torch.Generator().manual_seed(seed))
                    .float()).repeat_interleave(16, 2)[:, :, :n]
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES + [torch.float32])
@pytest.mark.parametrize("batch,heads,states,dim,block", [
    (1, 1, 1, 8, 16), (2, 3, 100, 64, 16), (2, 2, 130, 72, 32), (1, 2, 257, 128, 64), (3, 1, 300, 200, 128),
    (1, 2, 600, 256, 256), (2, 4, 64, 128, 64),
])
def test_codes_scales_and_counts(bk, dev, dtype, batch, heads, states, dim, block):
    slots = -(-states // block)
    blocks = batch * slots + 3
    keys, values = (_inputs(s, (batch, heads, states, dim), dtype) for s in (1, 2))
    keys[0, 0, 0, 0] = math.nan
    values[batch - 1, heads - 1, states // 2, dim // 2] = -math.inf
    values[0, 0, :16] = 0.0
    counts = torch.tensor([states - 7 * i for i in range(batch)], dtype=torch.int32).clamp_min(0)
    table = torch.randperm(blocks, generator=torch.Generator().manual_seed(9))[: batch * slots].to(torch.int32)
    table = table.view(batch, slots)
    if slots > 1:
        table[0, 0] = blocks  # names no block
        table[-1, 1] = -1
    cache = bk.state_cache(blocks, heads, block, dim, dev)
    for t, v in zip(cache, (0x55, 0x55, 3.0, 3.0, -4)):
        t.fill_(v)
    want = [t.cpu().clone() for t in cache]
    for b in range(batch):
        for h in range(heads):
            for kind, x in enumerate((keys, values)):
                codes, scales = _stored(x[b, h], block, int(counts[b]))
                for slot, (code, scale) in enumerate(zip(codes, scales)):
                    name = int(table[b, slot])
                    if 0 <= name < blocks:
                        want[kind][name, h, : len(code)] = code.view(torch.uint8)
                        want[2 + kind][name, h] = scale
                        want[4][name] = len(code)
    bk.cache_store(cache, keys.to(dev), values.to(dev), table.to(dev), counts.to(dev))
    torch.cuda.synchronize()
    for kind in range(2):
        got = cache[kind].cpu()
        nan = (want[kind] & 0x7F) == 0x7F
        assert torch.equal((got & 0x7F) == 0x7F, nan)
        assert torch.equal(got.masked_fill(nan, 0), want[kind].masked_fill(nan, 0))
        assert torch.equal(cache[2 + kind].cpu(), want[2 + kind])
    assert torch.equal(cache.block_counts.cpu(), want[4])


def test_store_from_views_and_broadcasts(bk, dev):
    batch, heads, states, dim, block = 2, 3, 90, 64, 32
    x = ref.made(4, (1, states, heads, 2, dim), torch.bfloat16).to(dev)
    keys, values = (x[:, :, :, i].transpose(1, 2).expand(batch, -1, -1, -1) for i in range(2))
    table = torch.arange(6, dtype=torch.int32, device=dev).view(batch, 3)
    one = bk.cache_store(bk.state_cache(6, heads, block, dim, dev), keys, values, table)
    two = bk.cache_store(bk.state_cache(6, heads, block, dim, dev), keys.contiguous(), values.contiguous(), table)
    for a, b in zip(one, two):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES + [torch.float32])
def test_extreme_magnitudes(bk, dev, dtype):
    """Each block's largest magnitude at the ends of the type, at the border of two scales, and zero."""
    info = torch.finfo(dtype)
    tops = [0.0, info.tiny, info.smallest_normal, 448.0, 449.0, 450.0, 1.75, 1.7578125, 2.0, info.max]
    x = torch.zeros((1, 1, 16 * len(tops), 8), dtype=dtype)
    for i, top in enumerate(tops):
        x[0, 0, 16 * i:16 * i + 16] = (ref.made(i, (16, 8), torch.float32).clamp(-2, 2) / 2 * min(top, 1e38)).to(dtype)
        x[0, 0, 16 * i, 0] = top
    table = torch.arange(len(tops), dtype=torch.int32)[None]
    cache = bk.cache_store(bk.state_cache(len(tops), 1, 16, 8, dev), x.to(dev), x.to(dev), table.to(dev))
    codes, scales = _stored(x[0, 0], 16, x.shape[2])
    assert cache.key_scales.cpu().flatten().tolist() == scales
    assert torch.equal(cache.key_codes.cpu(), torch.stack(codes)[:, None].view(torch.uint8))
    assert torch.equal(cache.value_codes, cache.key_codes)


# ---- attention over the cache --------------------------------------------------------------------

# batch, query heads, state heads, queries, entries, dim, block
SHAPES = [
    (1, 1, 1, 1, 1, 8, 16),
    (2, 4, 2, 3, 5, 64, 16),
    (1, 8, 2, 1, 63, 128, 16),
    (2, 2, 1, 40, 4, 72, 32),
    (3, 16, 2, 1, 9, 128, 64),
    (2, 6, 3, 130, 3, 80, 128),
    (1, 3, 3, 5, 2, 256, 256),
    (5, 5, 1, 2, 7, 200, 32),
    (1, 16, 1, 2, 33, 64, 64),
    (2, 8, 8, 300, 6, 128, 64),
    (1, 64, 1, 1, 40, 128, 128),
]


def _cache(bk, dev, shape, seed=1, powers=True):
    b, h, hs, q, slots, d, block = shape
    blocks = b * slots + 4
    cache = bk.state_cache(blocks, hs, block, d, dev)
    gen = torch.Generator().manual_seed(seed)
    for t in cache[:2]:
        codes = torch.randn(t.shape, generator=gen) * 60
        t.copy_(codes.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    for t in cache[2:4]:
        scales = torch.exp2(torch.randint(-7, -4, t.shape, generator=gen).float())
        t.copy_(scales if powers else scales * (1 + torch.rand(t.shape, generator=gen)))
    cache.block_counts.fill_(block)
    table = torch.randperm(blocks, generator=gen)[: b * slots].to(torch.int32).view(b, slots)
    return cache, table


def _states(cache, table):
    """(keys, values, taking part) of the places that the table names, in 64 bits on the CPU."""
    blocks, hs, block, d = cache.key_codes.shape
    b, slots = table.shape
    there = (table >= 0) & (table < blocks)
    names = table.clamp(0, blocks - 1).long()
    found = []
    for codes, scales in ((cache.key_codes, cache.key_scales), (cache.value_codes, cache.value_scales)):
        x = codes.cpu().view(torch.float8_e4m3fn).float().double() * scales.cpu().double()[..., None, None]
        found.append(x[names].transpose(1, 2).reshape(b, hs, slots * block, d))
    held = cache.block_counts.cpu()[names].masked_fill(~there, 0)
    keep = (torch.arange(block)[None, None] < held[:, :, None]).view(b, slots * block)
    return found[0], found[1], keep


def _check(bk, dev, queries, cache, table, counts=None, scale=None, **kw):
    keys, values, keep = _states(cache, table)
    if counts is not None:
        keep = keep & (torch.arange(keep.shape[1])[None] < counts.long()[:, None])
    used = queries.shape[3] ** -0.5 if scale is None else scale
    # bf16 queries: a weight times its value's scale is rounded to bf16; fp16 queries: to two bf16 pieces
    step = 2.0 ** -16 if queries.dtype == torch.float16 else None
    out, lse, out_bound, lse_bound = ref.attention(queries, keys, values, used, keep, step)
    got, got_lse = bk.cached_attention(queries.to(dev), cache, table.to(dev),
                                       None if counts is None else counts.to(dev), scale, **kw)
    torch.cuda.synchronize()
    ref.check(got, out, out_bound, "out")
    ref.check(got_lse, lse, lse_bound, "lse")
    return got, got_lse


def _queries(shape, dtype, seed=50):
    b, h, _, q, _, d, _ = shape
    return ref.made(seed, (b, h, q, d), dtype, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("powers", [True, False])
def test_whole_blocks(bk, dev, shape, dtype, powers):
    cache, table = _cache(bk, dev, shape, 1, powers)
    _check(bk, dev, _queries(shape, dtype), cache, table)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_counts_part_blocks_and_missing_blocks(bk, dev, shape, dtype):
    """What takes no part holds NaN codes and NaN scales; entries name no block at both ends of int32."""
    b, _, _, _, slots, _, block = shape
    cache, table = _cache(bk, dev, shape, 2)
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
    _check(bk, dev, _queries(shape, dtype), cache, table, counts)
    _check(bk, dev, _queries(shape, dtype), cache, table)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_block_named_twice_counts_twice(bk, dev, dtype):
    shape = (2, 4, 2, 3, 6, 64, 32)
    cache, table = _cache(bk, dev, shape, 4)
    table[0, 3] = table[0, 1]
    table[1, :] = table[0, 0]
    _check(bk, dev, _queries(shape, dtype), cache, table)


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_far_apart(bk, dev, dtype):
    """Values' scales from 2^-40 to 2^20: the blocks with small ones win the softmax for some rows."""
    shape = (1, 2, 1, 9, 12, 64, 16)
    cache, table = _cache(bk, dev, shape, 5)
    cache.value_scales.copy_(torch.exp2(torch.linspace(-40, 20, 16)).view(16, 1))
    cache.key_scales.copy_(torch.exp2(torch.arange(16) % 5 - 7.0).view(16, 1))
    _check(bk, dev, _queries(shape, dtype), cache, table)
    # one block decides every row
    cache.key_scales.fill_(2.0 ** -20)
    chosen = int(table[0, 7])
    cache.key_scales[chosen] = 2.0 ** -4
    for name, power in ((chosen, -30.0), (int(table[0, 2]), 1.0)):
        cache.value_scales[name] = 2.0 ** power
    _check(bk, dev, _queries(shape, dtype), cache, table, scale=1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_workspaces_strides_and_wide_tables(bk, dev, dtype):
    shape = (2, 8, 2, 1, 100, 128, 32)
    cache, table = _cache(bk, dev, shape, 6)
    queries = _queries(shape, dtype)
    counts = torch.tensor([3100, 1234], dtype=torch.int32)
    wide = torch.full((2, 117), -9, dtype=torch.int32)
    wide[:, 9:109] = table
    wide = wide.to(dev)
    need = bk.cached_attention_workspace_bytes(queries.to(dev), cache, 100)
    assert need > 0
    for size in (need, need // 3, 0):
        room = torch.full((size + 64,), 0xAB, dtype=torch.uint8, device=dev)
        got, lse = _check(bk, dev, queries, cache, table, counts, workspace=room[:size])
        assert (room[size:] == 0xAB).all()
        same, same_lse = bk.cached_attention(queries.to(dev).transpose(1, 2).contiguous().transpose(1, 2), cache,
                                             wide[:, 9:109], counts.to(dev), workspace=room[:size])
        assert torch.equal(got, same) and torch.equal(lse, same_lse)


def test_codes_beyond_32_bits(bk, dev):
    """More than 2^32 bytes of codes: the blocks at the end against the same blocks in a small cache."""
    hs, block, d = 8, 256, 256
    blocks = (1 << 32) // (hs * block * d) + 5
    small, table = _cache(bk, dev, (1, 8, hs, 1, 8, d, block), 7)
    big = bk.StateCache(*(torch.zeros((blocks, hs, block, d), dtype=torch.uint8, device=dev) for _ in range(2)),
                        *(torch.ones((blocks, hs), device=dev) for _ in range(2)),
                        torch.zeros(blocks, dtype=torch.int32, device=dev))
    count = small.block_counts.numel()
    for a, b in zip(big, small):
        a[blocks - count:] = b
    for q in (1, 150):
        queries = ref.made(8, (1, 8, q, d), torch.bfloat16).to(dev)
        want = bk.cached_attention(queries, small, table.to(dev))
        got = bk.cached_attention(queries, big, (table + blocks - count).to(dev))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    states = ref.made(9, (1, hs, 2 * block, d), torch.bfloat16).to(dev)
    names = torch.tensor([[blocks - 1, blocks - 2]], dtype=torch.int32, device=dev)
    bk.cache_store(big, states, states, names)
    bk.cache_store(small, states, states, names - (blocks - count))
    for a, b in zip(big, small):
        assert torch.equal(a[blocks - 2:], b[count - 2:])


def test_store_and_read_replayed_from_a_graph(bk, dev):
    """A step that stores new states and reads them, captured once: contents, counts and tables change."""
    shape = (2, 8, 2, 1, 20, 64, 32)
    cache, table = _cache(bk, dev, shape, 8)
    table = table.to(dev)
    counts = torch.tensor([640, 33], dtype=torch.int32, device=dev)
    fresh = torch.tensor([32, 16], dtype=torch.int32, device=dev)
    keys, values = (ref.made(s, (2, 2, 32, 64), torch.bfloat16).to(dev) for s in (1, 2))
    queries = _queries(shape, torch.bfloat16).to(dev)
    last = table[:, :1].contiguous()
    out, lse = torch.empty_like(queries), torch.empty(queries.shape[:3], device=dev)
    room = torch.empty(bk.cached_attention_workspace_bytes(queries, cache, 20), dtype=torch.uint8, device=dev)

    def step(o, l, w):
        bk.cache_store(cache, keys, values, last, fresh)
        return bk.cached_attention(queries, cache, table, counts, out=o, lse=l, workspace=w)

    step(out, lse, room)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, lse, room)
    for replay in range(4):
        keys.mul_(1.5)
        values.neg_()
        counts.copy_(torch.tensor([640 - 100 * replay, 33 * replay], dtype=torch.int32))
        table[:, 1:] = table[:, 1:].roll(1, 1)
        fresh.fill_(8 * replay)
        out.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), lse.clone()
        want = step(None, None, None)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), replay


def test_search_store_and_read_together(bk, dev):
    """As they are used: states enter the cache; a search over the blocks' mean keys finds each query's
    nearest blocks; its labels are the table that the attention reads, and labels of no block (a list
    longer than the candidates) name none.  Against the same steps on the CPU in 64 bits."""
    heads, block, blocks, dim, k = 2, 16, 11, 32, 16
    keys, values = (ref.made(s, (1, heads, blocks * block - 5, dim), torch.bfloat16) for s in (1, 2))
    names = torch.arange(blocks, dtype=torch.int32)[None]
    cache = bk.cache_store(bk.state_cache(blocks, heads, block, dim, dev), keys.to(dev), values.to(dev), names.to(dev))
    means = torch.nn.functional.pad(keys[0, 0].float(), (0, 0, 0, 5)).view(blocks, block, dim).mean(1)
    queries = ref.made(3, (40, heads, 1, dim), torch.bfloat16)
    dist, labels = bk.fused_l2_topk(queries[:, 0, 0].float().t().contiguous().to(dev), means.t().contiguous().to(dev), k)
    torch.cuda.synchronize()
    found = labels.cpu()
    assert (found[:, blocks:] == 2 ** 31 - 1).all() and (found[:, :blocks] < blocks).all()
    _check(bk, dev, queries, cache, found)
    near = labels[:, :4].contiguous()
    got, _ = bk.cached_attention(queries.to(dev), cache, near)
    _check(bk, dev, queries, cache, near.cpu())
    whole, _ = bk.cached_attention(queries.to(dev), cache, names.to(dev).expand(40, -1))
    assert not torch.equal(got, whole)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [3, 64, 65, 200])
def test_sequences_without_states_whatever_the_queries_hold(bk, dev, dtype, dim, rows):
    """No entry names a block, all blocks are empty, or the count is 0; the queries hold NaN and infinities."""
    shape = (4, 1, 1, rows, 40, dim, 32)
    cache, table = _cache(bk, dev, shape, 9)
    queries = _queries(shape, dtype)
    queries[1:, :, 0::3] = math.nan
    queries[1:, :, 1::3, 0] = math.inf
    queries[1:, :, 2::3, -1] = -math.inf
    table[1] = torch.tensor([-1, 2 ** 31 - 1]).repeat(20)
    cache.block_counts[table[2].long()] = 0
    counts = torch.tensor([1280, 1280, 1280, 0], dtype=torch.int32)
    out, lse = bk.cached_attention(queries.to(dev), cache, table.to(dev), counts.to(dev))
    assert (out[1:] == 0).all() and (lse[1:] == -math.inf).all()
    _check(bk, dev, queries[:1], cache, table[:1])


@pytest.mark.parametrize("rows", [3, 65])
def test_key_scales_that_overflow_with_the_scale(bk, dev, rows):
    """A key's scale times the call's is beyond fp32: scores of zero stay zero."""
    shape = (1, 1, 1, rows, 3, 64, 16)
    cache, table = _cache(bk, dev, shape, 10)
    cache.key_scales.fill_(2.0 ** 127)
    _check(bk, dev, torch.zeros_like(_queries(shape, torch.bfloat16)), cache, table, scale=64.0)


def test_float32_vectors_on_16_byte_boundaries(bk, dev):
    """Strides of whole fours: 16 bytes, though not whole eights as the 16-bit types want them."""
    wide = ref.made(20, (2, 3, 50, 24), torch.float32).to(dev)
    odd = ref.made(21, (2, 3, 50, 12), torch.float32).to(dev)
    table = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)
    for k, v in ((wide[..., :8], wide[..., 12:20]), (odd[..., :8], odd[..., 4:])):
        one = bk.cache_store(bk.state_cache(8, 3, 16, 8, dev), k, v, table)
        two = bk.cache_store(bk.state_cache(8, 3, 16, 8, dev), k.contiguous(), v.contiguous(), table)
        for a, b in zip(one, two):
            assert torch.equal(a, b)
