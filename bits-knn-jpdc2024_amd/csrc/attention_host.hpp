// Checks of the attention entry points' arguments: everything is refused before any launch.
#ifndef BITSKNN_CSRC_ATTENTION_HOST_HPP_
#define BITSKNN_CSRC_ATTENTION_HOST_HPP_

#include "attention.hpp"

namespace bitsknn
{
namespace
{

// Whether a launch can hold so many workgroups of so many threads: a grid has fewer than 2^32 threads.
inline bool fits_grid(u64 groups, u64 threads) { return groups <= 0xFFFFFFFFULL / threads; }

inline int check_shape(const char* name, const bitsknn_attention_shape& s)
{
    if (s.type != BITSKNN_BF16 && s.type != BITSKNN_FP16)
    {
        return fail(BITSKNN_ERR_UNSUPPORTED, "%s: unknown type %d", name, s.type);
    }
    if (s.dim < 1 || s.dim > 256 || s.dim % 8 != 0)
    {
        return fail(BITSKNN_ERR_UNSUPPORTED, "%s: Unsupported dim: %d (a multiple of 8 up to 256)", name, s.dim);
    }
    if (s.batch < 0 || s.queries < 0 || s.states < 0)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: negative size (batch %d, queries %d, states %d)", name, s.batch,
                    s.queries, s.states);
    }
    if (s.state_heads < 1 || s.query_heads < 1 || s.query_heads % s.state_heads != 0)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: %d query heads do not share %d state heads", name, s.query_heads,
                    s.state_heads);
    }
    // the kernels use it times log2(e)
    if (!(s.scale > 0.0F) || !(s.scale * LOG2E <= 3.402823466e38F))
    {
        return fail(BITSKNN_ERR_INVALID, "%s: scale %g is not positive and finite", name, static_cast<double>(s.scale));
    }
    // 32-bit row numbers in the kernels, with room for a tile behind the last row
    if (static_cast<u64>(s.query_heads / s.state_heads) * static_cast<u64>(s.queries) > 0x7FFF0000ULL ||
        s.states > 0x7FFF0000 || static_cast<u64>(s.batch) * static_cast<u64>(s.query_heads) > 0x7FFFFFFFULL)
    {
        return fail(BITSKNN_ERR_UNSUPPORTED, "%s: too many rows", name);
    }
    return BITSKNN_OK;
}

inline int fill_shape(attention_args& a, const bitsknn_attention_shape& s)
{
    a.dim = s.dim;
    a.state_heads = s.state_heads;
    a.group = s.query_heads / s.state_heads;
    a.queries_per_head = static_cast<u32>(s.queries);
    a.rows = static_cast<u32>(a.group) * a.queries_per_head;
    a.states = static_cast<u32>(s.states);
    a.scale = s.scale;
    a.exponent_scale = s.scale * LOG2E;
    return BITSKNN_OK;
}

// Whether vectors of `dim` values at these strides (extents above 1 only) never overlap: every stride
// reaches past all that the smaller ones span.
inline bool apart(std::int64_t dim, std::int64_t (&stride)[3], const std::int64_t (&extent)[3])
{
    std::int64_t s[3];
    std::int64_t e[3];
    int n = 0;
    for (int i = 0; i < 3; ++i)
    {
        if (extent[i] > 1)
        {
            int at = n++;
            for (; at > 0 && s[at - 1] > stride[i]; --at)
            {
                s[at] = s[at - 1];
                e[at] = e[at - 1];
            }
            s[at] = stride[i];
            e[at] = extent[i];
        }
    }
    std::int64_t span = dim;
    for (int i = 0; i < n; ++i)
    {
        if (s[i] < span)
        {
            return false;
        }
        span += s[i] * (e[i] - 1);
    }
    return true;
}

// Strides are looked at where their extent is above 1; the view gets 0 elsewhere.  value_bytes: of a
// vector's value.
inline int check_rows(const char* name, const char* what, const bitsknn_rows& r, const bitsknn_attention_shape& s,
                      int heads, int rows, bool written, rows_view& view, int value_bytes = 2)
{
    const std::int64_t extent[3] = {s.batch, heads, rows};
    std::int64_t stride[3] = {r.batch_stride, r.head_stride, r.row_stride};
    if (s.batch == 0 || rows == 0)
    {
        view = rows_view{nullptr, 0, 0, 0};
        return BITSKNN_OK;
    }
    if (r.data == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: %s: null pointer", name, what);
    }
    if (reinterpret_cast<std::uintptr_t>(r.data) % 16 != 0)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: %s: vectors must start on 16-byte boundaries", name, what);
    }
    for (int i = 0; i < 3; ++i)
    {
        stride[i] = extent[i] > 1 ? stride[i] : 0;
        if (stride[i] < 0 || stride[i] % (16 / value_bytes) != 0)
        {
            return fail(BITSKNN_ERR_INVALID, "%s: %s: vectors must start on 16-byte boundaries (strides %lld, %lld, %lld)",
                        name, what, static_cast<long long>(r.batch_stride), static_cast<long long>(r.head_stride),
                        static_cast<long long>(r.row_stride));
        }
        if (stride[i] > (1LL << 44) / extent[i])
        {
            return fail(BITSKNN_ERR_INVALID, "%s: %s: stride %lld", name, what, static_cast<long long>(stride[i]));
        }
    }
    if (stride[2] >= 1LL << 24)
    {
        // the rows of a tile are addressed in 32 bits
        return fail(BITSKNN_ERR_UNSUPPORTED, "%s: %s: row stride %lld (below 2^24)", name, what,
                    static_cast<long long>(stride[2]));
    }
    if (written && !apart(s.dim, stride, extent))
    {
        return fail(BITSKNN_ERR_INVALID, "%s: %s: vectors overlap (strides %lld, %lld, %lld)", name, what,
                    static_cast<long long>(r.batch_stride), static_cast<long long>(r.head_stride),
                    static_cast<long long>(r.row_stride));
    }
    view = rows_view{static_cast<char*>(r.data), stride[0], stride[1], stride[2]};
    return BITSKNN_OK;
}

inline int check_mask(const char* name, const bitsknn_attention_shape& s, const void* mask, size_t mask_stride)
{
    if (mask != nullptr && s.batch > 1 && mask_stride > (1ULL << 44))
    {
        return fail(BITSKNN_ERR_INVALID, "%s: mask stride %zu", name, mask_stride);
    }
    return BITSKNN_OK;
}

inline int check_cache(const char* name, const bitsknn_state_cache* c, cache_view& view)
{
    if (c == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: null pointer", name);
    }
    if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128 && c->block != 256)
    {
        return fail(BITSKNN_ERR_UNSUPPORTED, "Unsupported block: %d (16, 32, 64, 128 or 256 states)", c->block);
    }
    if (c->dim < 1 || c->dim > 256 || c->dim % 8 != 0)
    {
        return fail(BITSKNN_ERR_UNSUPPORTED, "%s: Unsupported dim: %d (a multiple of 8 up to 256)", name, c->dim);
    }
    if (c->blocks < 0 || c->state_heads < 1)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: a cache of %d blocks, %d heads", name, c->blocks, c->state_heads);
    }
    if (c->blocks > 0 && (c->key_codes == nullptr || c->value_codes == nullptr || c->key_scales == nullptr ||
                          c->value_scales == nullptr || c->block_counts == nullptr))
    {
        return fail(BITSKNN_ERR_INVALID, "%s: cache: null pointer", name);
    }
    if (reinterpret_cast<std::uintptr_t>(c->key_codes) % 16 != 0 || reinterpret_cast<std::uintptr_t>(c->value_codes) % 16 != 0)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: cache: codes must start on 16-byte boundaries", name);
    }
    view.key_codes = c->key_codes;
    view.value_codes = c->value_codes;
    view.key_scales = c->key_scales;
    view.value_scales = c->value_scales;
    view.block_counts = c->block_counts;
    view.blocks = static_cast<u32>(c->blocks);
    view.block_shift = 4;
    while ((1 << view.block_shift) < c->block)
    {
        ++view.block_shift;
    }
    return BITSKNN_OK;
}

inline int check_table(const char* name, const std::int32_t* table, size_t table_stride, std::int32_t batch,
                       std::int32_t states, cache_view& view)
{
    if (table == nullptr && batch > 0 && states > 0)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: table: null pointer", name);
    }
    if (batch > 1 && table_stride > (1ULL << 32))
    {
        return fail(BITSKNN_ERR_INVALID, "%s: table stride %zu", name, table_stride);
    }
    view.table = table;
    view.table_stride = batch > 1 ? static_cast<std::int64_t>(table_stride) : 0;
    return BITSKNN_OK;
}

inline int check_workspace(const char* name, const void* workspace)
{
    if (reinterpret_cast<std::uintptr_t>(workspace) % 16 != 0)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: the workspace must start on a 16-byte boundary", name);
    }
    return BITSKNN_OK;
}

} // namespace
} // namespace bitsknn

#endif // BITSKNN_CSRC_ATTENTION_HOST_HPP_
