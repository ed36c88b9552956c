// Attention over states of another length and over the 8-bit state cache: kernels, split rule and
// entry points.
#include "attention.hpp"

#include "attention_host.hpp"
#include "attention_loader.hpp"
#include "attention_stream.hpp"

namespace bitsknn
{
namespace
{

constexpr u32 TILE_KEYS = 64; // states per tile: the width of a wave's ballot
constexpr u32 WAVE_ROWS = 32; // rows per wave: the columns of a matrix product

#ifndef TW
#define TW 8
#endif
// Waves that share a tile.  In 256 dimensions a wave needs all the registers of its quarter of the unit.
constexpr u32 tile_waves(int padded_dim) { return padded_dim <= 128 ? TW : 4; }
constexpr u32 tile_rows(int padded_dim) { return WAVE_ROWS * tile_waves(padded_dim); }

// What a wave keeps of its 32 rows: lane 32 h + c holds of row c the columns 32 block + 8 (i / 4) +
// 4 h + i % 4 of the sum.
template <int DP>
struct row_state
{
    vfloat16 sum[DP / 32];
    float top;    // the reference of the exponents, in base-2 exponents; both halves hold the same
    float weight; // this half's part of the sum of weights
};

template <int DP>
__device__ __forceinline__ void store_rows(const attention_args& a, const row_state<DP>& s, u32 b, u32 head, u32 row,
                                           u32 split)
{
    const u32 half = (threadIdx.x & 63) / 32;
    const float weight = s.weight + other_half(s.weight);
    if (row >= a.rows)
    {
        return;
    }
    const size_t flat = (static_cast<size_t>(b) * static_cast<u32>(a.state_heads) + head) * a.rows + row;
    if (a.splits > 1)
    {
        const size_t at = flat * a.splits + split;
        if (half == 0)
        {
            a.part_ml[at] = float2{s.top, weight};
        }
#pragma unroll
        for (int n = 0; n < DP / 32; ++n)
        {
#pragma unroll
            for (int g = 0; g < 4; ++g)
            {
                *reinterpret_cast<vfloat4*>(a.part + at * DP + 32 * n + 8 * g + 4 * half) =
                    vfloat4{s.sum[n][4 * g], s.sum[n][4 * g + 1], s.sum[n][4 * g + 2], s.sum[n][4 * g + 3]};
            }
        }
        return;
    }
    if (half == 0 && a.lse != nullptr)
    {
        // without a state: weight 0, log2 of it -inf
        a.lse[flat] = weight == 0.0F ? -__builtin_inff() : (s.top + __builtin_log2f(weight)) * LN2;
    }
}

template <typename T, int DP>
__device__ __forceinline__ void store_out(const attention_args& a, const row_state<DP>& s, u32 b, u32 head, u32 row)
{
    const u32 half = (threadIdx.x & 63) / 32;
    const float weight = s.weight + other_half(s.weight);
    if (row >= a.rows)
    {
        return;
    }
    const float inverse = weight == 0.0F ? 0.0F : 1.0F / weight;
    char* out = a.out.data + 2 * row_offset(a.out, a, b, head, row);
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
    {
#pragma unroll
        for (int g = 0; g < 4; ++g)
        {
            const u32 column = 32 * n + 8 * g + 4 * half;
            if (column < static_cast<u32>(a.dim))
            {
                *reinterpret_cast<vuint2*>(out + 2 * column) =
                    vuint2{pack2<T>(s.sum[n][4 * g] * inverse, s.sum[n][4 * g + 1] * inverse),
                           pack2<T>(s.sum[n][4 * g + 2] * inverse, s.sum[n][4 * g + 3] * inverse)};
            }
        }
    }
}

// Bound by the matrix instructions and the LDS reads that feed them.  A workgroup's waves hold 32 rows
// each and share tiles of 64 states in LDS, two of them: while one is multiplied, the next is on its
// way into registers and then into the other, so that a step has one barrier.
template <typename T, int DP, bool CACHE>
__global__ void __launch_bounds__(64 * tile_waves(DP), DP <= 128 ? 2 : 1) attention_tile_kernel(const attention_args a)
{
    constexpr u32 THREADS = 64 * tile_waves(DP);
    using loader = state_loader<T, DP, CACHE, TILE_KEYS, THREADS>;
    using V = typename loader::V;
    constexpr u32 TILE_BYTES = TILE_KEYS * DP * 2;
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE_BYTES];
    const u32 lane = threadIdx.x & 63;
    const u32 half = lane / 32;
    const u32 id = die_order(blockIdx.x, gridDim.x);
    const u32 row_tile = id % a.row_tiles;
    const u32 split = id / a.row_tiles % a.splits;
    const u32 head = id / a.row_tiles / a.splits % static_cast<u32>(a.state_heads);
    const u32 b = id / a.row_tiles / a.splits / static_cast<u32>(a.state_heads);
    const u32 row = row_tile * tile_rows(DP) + threadIdx.x / 64 * WAVE_ROWS + lane % 32;

    vuint4 query[DP / 16];
    load_operand<DP>(query, a.queries.data + 2 * row_offset(a.queries, a, b, head, row < a.rows ? row : 0),
                     row < a.rows, static_cast<u32>(a.dim));
    row_state<DP> st;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
    {
        st.sum[n] = vfloat16{};
    }
    st.top = -__builtin_inff();
    st.weight = 0.0F;

    const u32 count = state_count(a, b);
    const u32 tiles = (count + TILE_KEYS - 1) / TILE_KEYS;
    const u32 begin = static_cast<u32>(static_cast<u64>(tiles) * split / a.splits);
    const u32 end = static_cast<u32>(static_cast<u64>(tiles) * (split + 1) / a.splits);
    const loader w{a, b, head, count};
    vuint4 next_keys[loader::LOADS];
    vuint4 next_values[loader::LOADS];
    typename loader::place now;   // of the tile in LDS
    typename loader::place next;  // of the tile in the registers
    typename loader::place after; // of the tile after it; its table entry is one further ahead
    u64 in = 0;                   // of the tile in LDS
    u64 next_in = 0;
    if (begin < end)
    {
        w.look_up_block(now, begin);
        w.look_up_block(next, begin + 1);
        w.look_up_block(after, begin + 2);
        w.look_up_state(now, begin);
        w.look_up_state(next, begin + 1);
        in = w.taking_part(now, begin);
        w.template load<true>(next_keys, now, begin, in);
        w.template load<false>(next_values, now, begin, in);
        w.template put<T>(lds, next_keys);
        w.template put<V>(lds + TILE_BYTES, next_values);
        __syncthreads();
    }
    for (u32 tile = begin; tile < end; ++tile)
    {
        const char* const keys = lds + ((tile - begin) % 2) * 2 * TILE_BYTES;
        const char* const values = keys + TILE_BYTES;
        const bool more = tile + 1 < end;
        const typename loader::place current = now;
        if (more)
        {
            now = next;
            next.block = after.block;
            next_in = w.taking_part(now, tile + 1);
            w.look_up_block(after, tile + 3);
            w.look_up_state(next, tile + 2);
            w.template load<true>(next_keys, now, tile + 1, next_in);
            w.template load<false>(next_values, now, tile + 1, next_in);
        }
        if (in != 0) // the same in every wave
        {
            vfloat16 score[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
            {
                score[u] = vfloat16{};
#pragma unroll
                for (int s = 0; s < DP / 16; ++s)
                {
                    score[u] = mfma<T>::run(tile_row<DP>(keys, 32 * u + lane % 32, s), query[s], score[u]);
                }
            }
            if constexpr (CACHE)
            {
#pragma unroll
                for (int g = 0; g < 4; ++g)
                {
                    const float scale = w.of_sixteen(current.key_scale, g);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                    {
                        score[g / 2][8 * (g % 2) + i] *= scale;
                    }
                }
            }
            if (in != ~0ULL)
            {
#pragma unroll
                for (int u = 0; u < 2; ++u)
                {
                    const u32 bits = static_cast<u32>(in >> (32 * u)) >> (4 * half);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                    {
                        score[u][i] = ((bits >> (8 * (i / 4) + i % 4)) & 1) != 0 ? score[u][i] : -__builtin_inff();
                    }
                }
            }
            float most = score[0][0];
#pragma unroll
            for (int i = 1; i < 32; ++i)
            {
                most = fmaxf(most, score[i / 16][i % 16]);
            }
            most = fmaxf(most, other_half(most)) * a.exponent_scale;
            // The reference of the exponents follows the maximum only where that has grown by more than
            // 8: weights stay below 2^8, and the sums are seldom rescaled.
            if (__any(most > st.top + 8.0F))
            {
                const float top = fmaxf(most, st.top);
                const float shrink = __builtin_amdgcn_exp2f(st.top - (top == -__builtin_inff() ? 0.0F : top));
                st.weight *= shrink;
#pragma unroll
                for (int n = 0; n < DP / 32; ++n)
                {
                    st.sum[n] *= shrink;
                }
                st.top = top;
            }
            const float base = st.top == -__builtin_inff() ? 0.0F : st.top;
            float weight = 0.0F;
#pragma unroll
            for (int i = 0; i < 32; ++i)
            {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(score[i / 16][i % 16], a.exponent_scale, -base));
                score[i / 16][i % 16] = x;
                weight += x;
            }
            st.weight += weight;
            if constexpr (CACHE)
            {
#pragma unroll
                for (int g = 0; g < 4; ++g)
                {
                    // a sixteen without a state that takes part: its weights are zero, its scale may be anything
                    const float scale = ((in >> (16 * g)) & 0xFFFFU) != 0 ? w.of_sixteen(current.value_scale, g) : 0.0F;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                    {
                        score[g / 2][8 * (g % 2) + i] *= scale;
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
            {
                const vuint4 p = operand<V>(score[s / 2], s % 2);
                vuint4 rest;
                if constexpr (loader::PIECES)
                {
                    rest = operand_rest(score[s / 2], s % 2, p);
                }
#pragma unroll
                for (int n = 0; n < DP / 32; ++n)
                {
                    const vuint4 v = tile_column<DP>(values, s, n);
                    st.sum[n] = mfma<V>::run(v, p, st.sum[n]);
                    if constexpr (loader::PIECES)
                    {
                        st.sum[n] = mfma<V>::run(v, rest, st.sum[n]);
                    }
                }
            }
        }
        in = next_in;
        if (more)
        {
            char* const other = lds + ((tile + 1 - begin) % 2) * 2 * TILE_BYTES;
            w.template put<T>(other, next_keys);
            w.template put<V>(other + TILE_BYTES, next_values);
        }
        __syncthreads();
    }
    store_rows<DP>(a, st, b, head, row, split);
    if (a.splits == 1)
    {
        store_out<T, DP>(a, st, b, head, row);
    }
}

// Joins the splits of a row: one wave per row.
template <typename T, int DP>
__global__ void __launch_bounds__(256) attention_join_kernel(const attention_args a, size_t rows)
{
    const size_t flat = static_cast<size_t>(blockIdx.x) * 4 + threadIdx.x / 64;
    const u32 lane = threadIdx.x & 63;
    if (flat >= rows)
    {
        return;
    }
    float2 ml = {-__builtin_inff(), 0.0F};
    if (lane < a.splits)
    {
        ml = a.part_ml[flat * a.splits + lane];
    }
    float top = ml.x;
#pragma unroll
    for (int o = 32; o > 0; o /= 2)
    {
        top = fmaxf(top, __shfl_xor(top, o));
    }
    const float base = top == -__builtin_inff() ? 0.0F : top;
    const float factor = __builtin_amdgcn_exp2f(ml.x - base);
    float weight = ml.y * factor;
#pragma unroll
    for (int o = 32; o > 0; o /= 2)
    {
        weight += __shfl_xor(weight, o);
    }
    constexpr int PER = DP / 64;
    float sum[PER] = {};
    for (u32 s = 0; s < a.splits; ++s)
    {
        const float f = __shfl(factor, static_cast<int>(s));
        const float l = __shfl(ml.y, static_cast<int>(s));
        if (l == 0.0F)
        {
            continue; // a split without a state
        }
#pragma unroll
        for (int i = 0; i < PER; ++i)
        {
            sum[i] += f * a.part[(flat * a.splits + s) * DP + PER * lane + i];
        }
    }
    const u32 b = static_cast<u32>(flat / a.rows / static_cast<u32>(a.state_heads));
    const u32 head = static_cast<u32>(flat / a.rows % static_cast<u32>(a.state_heads));
    const u32 row = static_cast<u32>(flat % a.rows);
    const float inverse = weight == 0.0F ? 0.0F : 1.0F / weight;
    if (lane == 0 && a.lse != nullptr)
    {
        a.lse[flat] = weight == 0.0F ? -__builtin_inff() : (top + __builtin_log2f(weight)) * LN2;
    }
    T* out = reinterpret_cast<T*>(a.out.data) + row_offset(a.out, a, b, head, row);
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        const u32 column = PER * lane + i;
        if (column < static_cast<u32>(a.dim))
        {
            out[column] = static_cast<T>(sum[i] * inverse);
        }
    }
}

int padded_dim(int dim) { return dim <= 64 ? 64 : (dim <= 128 ? 128 : 256); }

// Few rows stream past 32 at a time, more of them share tiles of 128 rows.
constexpr u32 MOST_STREAM_ROWS = 64;

// two per compute unit (1024 and 2048: 3 and 6 us longer for 64 sequences of 32 heads over 8192 states)
constexpr size_t WANTED_WORKGROUPS = 512;

bool streams(size_t rows) { return rows <= MOST_STREAM_ROWS; }

u32 row_tiles_of(size_t rows, int dim)
{
    const size_t per = streams(rows) ? STREAM_ROWS : tile_rows(padded_dim(dim));
    return static_cast<u32>((rows + per - 1) / per);
}

// How many ranges the states are cut into: as many as give the GPU enough workgroups, at least 512
// states each (a join of ranges costs a launch: 12.1 us for three of 333 states, 12.6 us for one of 1000).
u32 wanted_splits(const bitsknn_attention_shape& s)
{
    const size_t rows = static_cast<size_t>(s.queries) * static_cast<u32>(s.query_heads / s.state_heads);
    const size_t groups = static_cast<size_t>(s.batch) * static_cast<u32>(s.state_heads) * row_tiles_of(rows, s.dim);
    const size_t most = static_cast<size_t>(s.states) / 512;
    if (groups == 0 || groups >= WANTED_WORKGROUPS)
    {
        return 1;
    }
    size_t splits = (WANTED_WORKGROUPS + groups - 1) / groups;
    splits = splits < most ? splits : most;
    splits = splits < 64 ? splits : 64;
    return splits < 1 ? 1 : static_cast<u32>(splits);
}

size_t bytes_per_split(const bitsknn_attention_shape& s)
{
    return static_cast<size_t>(s.batch) * static_cast<u32>(s.query_heads) * static_cast<u32>(s.queries) *
           (static_cast<size_t>(padded_dim(s.dim)) * sizeof(float) + sizeof(float2));
}

size_t workspace_bytes_of(const bitsknn_attention_shape& s)
{
    const u32 splits = wanted_splits(s);
    return splits > 1 ? splits * bytes_per_split(s) : 0;
}

template <typename T, int DP, bool CACHE>
int launch(attention_args& a, size_t rows, u32 batch, hipStream_t stream)
{
    const u64 blocks = static_cast<u64>(batch) * static_cast<u32>(a.state_heads) * a.splits * a.row_tiles;
    if (blocks > MOST_WORKGROUPS || (rows + 3) / 4 > MOST_WORKGROUPS)
    {
        return fail(BITSKNN_ERR_UNSUPPORTED, "attention: too many rows (%zu)", rows);
    }
    if (streams(a.rows))
    {
        hipLaunchKernelGGL((attention_stream_kernel<T, DP, CACHE>), dim3(static_cast<u32>(blocks)),
                           dim3(64 * STREAM_WAVES), 0, stream, a);
    }
    else
    {
        hipLaunchKernelGGL((attention_tile_kernel<T, DP, CACHE>), dim3(static_cast<u32>(blocks)), dim3(64 * tile_waves(DP)), 0,
                           stream, a);
    }
    BITSKNN_HIP_CHECK(hipGetLastError());
    if (a.splits > 1)
    {
        hipLaunchKernelGGL((attention_join_kernel<T, DP>), dim3(static_cast<u32>((rows + 3) / 4)), dim3(256), 0, stream,
                           a, rows);
        BITSKNN_HIP_CHECK(hipGetLastError());
    }
    return BITSKNN_OK;
}

template <bool CACHE>
int run(attention_args& a, const bitsknn_attention_shape& s, void* workspace, size_t workspace_bytes, void* stream)
{
    const size_t rows = static_cast<size_t>(s.batch) * static_cast<u32>(s.query_heads) * static_cast<u32>(s.queries);
    a.row_tiles = row_tiles_of(a.rows, s.dim);
    a.splits = wanted_splits(s);
    const size_t fit = workspace == nullptr ? 0 : workspace_bytes / bytes_per_split(s);
    if (a.splits > fit)
    {
        a.splits = fit > 1 ? static_cast<u32>(fit) : 1;
    }
    const int padded = padded_dim(s.dim);
    a.part = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part + rows * a.splits * static_cast<u32>(padded));
    const auto st = static_cast<hipStream_t>(stream);
    const u32 batch = static_cast<u32>(s.batch);
    if (s.type == BITSKNN_BF16)
    {
        return padded == 64    ? launch<__bf16, 64, CACHE>(a, rows, batch, st)
               : padded == 128 ? launch<__bf16, 128, CACHE>(a, rows, batch, st)
                               : launch<__bf16, 256, CACHE>(a, rows, batch, st);
    }
    return padded == 64    ? launch<_Float16, 64, CACHE>(a, rows, batch, st)
           : padded == 128 ? launch<_Float16, 128, CACHE>(a, rows, batch, st)
                           : launch<_Float16, 256, CACHE>(a, rows, batch, st);
}

} // namespace
} // namespace bitsknn

extern "C" size_t bitsknn_cross_attention_workspace_bytes(const bitsknn_attention_shape* shape)
{
    using namespace bitsknn;
    clear_error();
    if (shape == nullptr || check_shape("bitsknn_cross_attention_workspace_bytes", *shape) != BITSKNN_OK)
    {
        return 0;
    }
    return workspace_bytes_of(*shape);
}

extern "C" int bitsknn_cross_attention(const bitsknn_attention_shape* shape, const bitsknn_rows* queries,
                                       const bitsknn_rows* keys, const bitsknn_rows* values, const int32_t* counts,
                                       const uint8_t* mask, size_t mask_stride, const bitsknn_rows* out, float* lse,
                                       void* workspace, size_t workspace_bytes, void* stream)
{
    using namespace bitsknn;
    clear_error();
    const char* name = "bitsknn_cross_attention";
    if (shape == nullptr || queries == nullptr || keys == nullptr || values == nullptr || out == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: null pointer", name);
    }
    const bitsknn_attention_shape& s = *shape;
    attention_args a = {};
    int status = check_shape(name, s);
    status = status != BITSKNN_OK ? status : fill_shape(a, s);
    status = status != BITSKNN_OK ? status : check_rows(name, "queries", *queries, s, s.query_heads, s.queries, false, a.queries);
    status = status != BITSKNN_OK ? status : check_rows(name, "keys", *keys, s, s.state_heads, s.states, false, a.keys);
    status = status != BITSKNN_OK ? status : check_rows(name, "values", *values, s, s.state_heads, s.states, false, a.values);
    status = status != BITSKNN_OK ? status : check_rows(name, "out", *out, s, s.query_heads, s.queries, true, a.out);
    status = status != BITSKNN_OK ? status : check_mask(name, s, mask, mask_stride);
    status = status != BITSKNN_OK ? status : check_workspace(name, workspace);
    if (status != BITSKNN_OK || s.batch == 0 || s.queries == 0)
    {
        return status;
    }
    a.counts = counts;
    a.mask = mask;
    a.mask_stride = static_cast<std::int64_t>(mask_stride);
    a.lse = lse;
    return run<false>(a, s, workspace, workspace_bytes, stream);
}

extern "C" size_t bitsknn_cached_attention_workspace_bytes(const bitsknn_attention_shape* shape)
{
    return bitsknn_cross_attention_workspace_bytes(shape);
}

extern "C" int bitsknn_cached_attention(const bitsknn_attention_shape* shape, const bitsknn_rows* queries,
                                        const bitsknn_state_cache* cache, const int32_t* table, size_t table_stride,
                                        const int32_t* counts, const bitsknn_rows* out, float* lse, void* workspace,
                                        size_t workspace_bytes, void* stream)
{
    using namespace bitsknn;
    clear_error();
    const char* name = "bitsknn_cached_attention";
    if (shape == nullptr || queries == nullptr || cache == nullptr || out == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: null pointer", name);
    }
    const bitsknn_attention_shape& s = *shape;
    attention_args a = {};
    int status = check_shape(name, s);
    status = status != BITSKNN_OK ? status : fill_shape(a, s);
    status = status != BITSKNN_OK ? status : check_rows(name, "queries", *queries, s, s.query_heads, s.queries, false, a.queries);
    status = status != BITSKNN_OK ? status : check_rows(name, "out", *out, s, s.query_heads, s.queries, true, a.out);
    status = status != BITSKNN_OK ? status : check_cache(name, cache, a.cache);
    status = status != BITSKNN_OK ? status : check_table(name, table, table_stride, s.batch, s.states, a.cache);
    status = status != BITSKNN_OK ? status : check_workspace(name, workspace);
    if (status == BITSKNN_OK && (cache->dim != s.dim || cache->state_heads != s.state_heads))
    {
        return fail(BITSKNN_ERR_INVALID, "%s: a cache of %d heads x %d, queries for %d x %d", name, cache->state_heads,
                    cache->dim, s.state_heads, s.dim);
    }
    if (status != BITSKNN_OK || s.batch == 0 || s.queries == 0)
    {
        return status;
    }
    a.counts = counts;
    a.lse = lse;
    return run<true>(a, s, workspace, workspace_bytes, stream);
}
