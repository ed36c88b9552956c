// Attention over states of another length and over the 8-bit state cache: kernels, split rule and
// entry points.
#include "attention.hpp"

#include "attention_host.hpp"

namespace bitsknn
{
namespace
{

constexpr u32 TILE_KEYS = 64; // states per tile: the width of a wave's ballot
constexpr u32 WAVE_ROWS = 32; // rows per wave: the columns of a matrix product
constexpr u32 WAVES = 4;

// What is known of a tile's states: which take part, and in the cache their scales by sixteens.
struct tile_states
{
    u64 in;
    float key_scale[4];
    float value_scale[4];
};

__device__ __forceinline__ std::int32_t block_of(const attention_args& a, u32 b, u32 j)
{
    return a.cache.table[static_cast<std::int64_t>(b) * a.cache.table_stride + (j >> a.cache.block_shift)];
}

template <bool CACHE>
__device__ __forceinline__ tile_states look_up(const attention_args& a, u32 b, u32 head, u32 count, u32 first)
{
    tile_states t;
    if constexpr (!CACHE)
    {
        t.in = states_taking_part(a, b, count, first);
    }
    else
    {
        const u32 j = first + (threadIdx.x & 63);
        bool in = j < count;
        float ks = 1.0F;
        float vs = 1.0F;
        if (in)
        {
            const u32 id = static_cast<u32>(block_of(a, b, j));
            in = id < a.cache.blocks &&
                 static_cast<std::int32_t>(j & ((1U << a.cache.block_shift) - 1)) < a.cache.block_counts[id];
            if (in)
            {
                const size_t at = static_cast<size_t>(id) * static_cast<u32>(a.state_heads) + head;
                ks = a.cache.key_scales[at];
                vs = a.cache.value_scales[at];
            }
        }
        t.in = __ballot(in);
        // the states of a block that take part are its first ones, so the first of sixteen has the
        // scale of all that do; where none does, the scale stays 1
#pragma unroll
        for (int g = 0; g < 4; ++g)
        {
            t.key_scale[g] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks), 16 * g));
            t.value_scale[g] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vs), 16 * g));
        }
    }
    return t;
}

// One tile of keys or values into LDS; what takes no part becomes zero.
template <int DP, typename T, bool CACHE, bool KEYS>
__device__ __forceinline__ void stage(char* tile, const attention_args& a, u32 b, u32 head, u32 first, u64 in)
{
    constexpr u32 CHUNKS = DP / 8;
    const rows_view& v = KEYS ? a.keys : a.values;
    const char* base = nullptr;
    if constexpr (!CACHE)
    {
        base = v.data + 2 * (b * v.batch_stride + head * v.head_stride + first * v.row_stride);
    }
#pragma unroll
    for (u32 c = threadIdx.x; c < TILE_KEYS * CHUNKS; c += 64 * WAVES)
    {
        const u32 row = c / CHUNKS;
        const u32 chunk = c % CHUNKS;
        vuint4 x = {0, 0, 0, 0};
        if (((in >> row) & 1) != 0 && chunk * 8 < static_cast<u32>(a.dim))
        {
            if constexpr (!CACHE)
            {
                x = *reinterpret_cast<const vuint4*>(base + 2 * (row * v.row_stride + chunk * 8));
            }
            else
            {
                const u32 j = first + row;
                const size_t id = static_cast<u32>(block_of(a, b, j));
                const size_t at =
                    (((id * static_cast<u32>(a.state_heads) + head) << a.cache.block_shift) +
                     (j & ((1U << a.cache.block_shift) - 1))) * static_cast<u32>(a.dim) + chunk * 8;
                x = decode8<T>(*reinterpret_cast<const vuint2*>((KEYS ? a.cache.key_codes : a.cache.value_codes) + at));
            }
        }
        *reinterpret_cast<vuint4*>(tile + tile_chunk<DP>(row, chunk)) = x;
    }
}

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

// Scores of 32 states (rows of the product) and the wave's 32 rows (columns), weights, and the sum.
template <typename T, int DP, bool CACHE>
__global__ void __launch_bounds__(64 * WAVES) attention_tile_kernel(const attention_args a)
{
    // the cache's codes are exact in either type; the weights times the values' scale need the range
    // of bf16, so its second product is taken in bf16 (fp16 queries: the weight as two bf16 pieces,
    // sixteen bits, so that an fp16 result loses nothing)
    using V = std::conditional_t<CACHE, __bf16, T>;
    constexpr bool PIECES = CACHE && std::is_same_v<T, _Float16>;
    __shared__ __attribute__((aligned(16))) char keys[TILE_KEYS * DP * 2];
    __shared__ __attribute__((aligned(16))) char values[TILE_KEYS * DP * 2];
    const u32 lane = threadIdx.x & 63;
    const u32 half = lane / 32;
    const u32 id = die_order(blockIdx.x, gridDim.x);
    const u32 row_tile = id % a.row_tiles;
    const u32 split = id / a.row_tiles % a.splits;
    const u32 head = id / a.row_tiles / a.splits % static_cast<u32>(a.state_heads);
    const u32 b = id / a.row_tiles / a.splits / static_cast<u32>(a.state_heads);
    const u32 row = row_tile * (WAVE_ROWS * WAVES) + threadIdx.x / 64 * WAVE_ROWS + lane % 32;

    vuint4 query[DP / 16];
    {
        const u32 r = row < a.rows ? row : 0;
        const char* q = a.queries.data + 2 * row_offset(a.queries, a, b, head, r);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
        {
            const u32 at = 16 * s + 8 * half;
            query[s] = vuint4{0, 0, 0, 0};
            if (row < a.rows && at < static_cast<u32>(a.dim))
            {
                query[s] = *reinterpret_cast<const vuint4*>(q + 2 * at);
            }
        }
    }
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
    for (u32 tile = begin; tile < end; ++tile)
    {
        const u32 first = tile * TILE_KEYS;
        const tile_states t = look_up<CACHE>(a, b, head, count, first);
        if (t.in == 0)
        {
            continue; // the same in every wave: the workgroup's barriers stay together
        }
        __syncthreads();
        stage<DP, T, CACHE, true>(keys, a, b, head, first, t.in);
        stage<DP, V, CACHE, false>(values, a, b, head, first, t.in);
        __syncthreads();
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
            for (int u = 0; u < 2; ++u)
            {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    score[u][i] *= t.key_scale[2 * u + i / 8];
                }
            }
        }
        if (t.in != ~0ULL)
        {
#pragma unroll
            for (int u = 0; u < 2; ++u)
            {
                const u32 bits = static_cast<u32>(t.in >> (32 * u)) >> (4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    score[u][i] = ((bits >> (8 * (i / 4) + i % 4)) & 1) != 0 ? score[u][i] : -__builtin_inff();
                }
            }
        }
        float top = score[0][0];
#pragma unroll
        for (int i = 1; i < 32; ++i)
        {
            top = fmaxf(top, score[i / 16][i % 16]);
        }
        top = fmaxf(top, other_half(top)) * a.exponent_scale;
        top = fmaxf(top, st.top);
        const float base = top == -__builtin_inff() ? 0.0F : top;
        const float shrink = __builtin_amdgcn_exp2f(st.top - base);
        st.top = top;
        float weight = 0.0F;
#pragma unroll
        for (int i = 0; i < 32; ++i)
        {
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(score[i / 16][i % 16], a.exponent_scale, -base));
            score[i / 16][i % 16] = x;
            weight += x;
        }
        st.weight = st.weight * shrink + weight;
#pragma unroll
        for (int n = 0; n < DP / 32; ++n)
        {
            st.sum[n] *= shrink;
        }
        if constexpr (CACHE)
        {
#pragma unroll
            for (int i = 0; i < 32; ++i)
            {
                score[i / 16][i % 16] *= t.value_scale[i / 8];
            }
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
        {
            vuint4 p;
            vuint4 rest;
#pragma unroll
            for (int w = 0; w < 4; ++w)
            {
                const float x = score[s / 2][8 * (s % 2) + 2 * w];
                const float y = score[s / 2][8 * (s % 2) + 2 * w + 1];
                p[w] = pack2<V>(x, y);
                if constexpr (PIECES)
                {
                    rest[w] = pack2<V>(x - __builtin_bit_cast(float, p[w] << 16),
                                       y - __builtin_bit_cast(float, p[w] & 0xFFFF0000U));
                }
            }
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
            {
                const vuint4 v = tile_column<DP>(values, s, n);
                st.sum[n] = mfma<V>::run(v, p, st.sum[n]);
                if constexpr (PIECES)
                {
                    st.sum[n] = mfma<V>::run(v, rest, st.sum[n]);
                }
            }
        }
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

u32 row_tiles_of(size_t rows) { return static_cast<u32>((rows + WAVE_ROWS * WAVES - 1) / (WAVE_ROWS * WAVES)); }

// How many ranges the states are cut into: as many as give the GPU two workgroups per compute unit, at
// least four tiles each.
u32 wanted_splits(const bitsknn_attention_shape& s)
{
    const size_t rows = static_cast<size_t>(s.queries) * static_cast<u32>(s.query_heads / s.state_heads);
    const size_t groups = static_cast<size_t>(s.batch) * static_cast<u32>(s.state_heads) * row_tiles_of(rows);
    const size_t tiles = (static_cast<size_t>(s.states) + TILE_KEYS - 1) / TILE_KEYS;
    if (groups == 0 || groups >= 512)
    {
        return 1;
    }
    size_t splits = (512 + groups - 1) / groups;
    splits = splits < tiles / 4 ? splits : tiles / 4;
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
    hipLaunchKernelGGL((attention_tile_kernel<T, DP, CACHE>), dim3(static_cast<u32>(blocks)), dim3(64 * WAVES), 0, stream, a);
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
    a.row_tiles = row_tiles_of(a.rows);
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
