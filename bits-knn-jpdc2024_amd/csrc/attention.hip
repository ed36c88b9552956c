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

constexpr u32 WAVE_ROWS = 32; // rows per wave: the columns of a matrix product

// Waves that share a tile.  In 256 dimensions a wave needs all the registers of its quarter of the unit.
constexpr u32 tile_waves(int padded_dim) { return padded_dim <= 128 ? 8 : 4; }
// States per tile: five tiles have to fit LDS.
constexpr u32 tile_keys(int padded_dim) { return padded_dim <= 128 ? 64 : 32; }
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

// Sequences of one length: neighbours, which read the same states, on one die.  Of different lengths: the
// tiles of each dealt out to all dies, so that they end together (101 against 109 us for 4 x 16/4 heads,
// 512 rows over up to 4096 states of the cache; with one length 568 against 551 us for 4 x 16/4 heads, 2048 x
// 8192).
template <bool CACHE>
__device__ __forceinline__ u32 tile_order(const attention_args& a)
{
    return CACHE || a.counts != nullptr ? blockIdx.x : die_order(blockIdx.x, gridDim.x);
}

// Bound by the matrix instructions.  A workgroup's waves hold 32 rows each and share tiles of states in
// LDS.  A wave goes through the states by 32: one step takes the scores of the next 32 on the matrix
// path, turns those of the present 32 into weights on the vector unit meanwhile, multiplies them with
// the values, and looks for the next scores' maximum.  The next tile's vectors are on their way into
// registers while a tile is worked on; they are put into LDS (two tiles of keys, three of values, since
// the slowest wave may still read the last values of the tile before) ahead of a tile's last step, which
// already reads the next keys: one barrier per tile.  Weights are rounded to 16 bits for the second product, as
// the matrix instructions want them; their sum is taken before that.
template <typename T, int DP, bool CACHE>
__global__ void __launch_bounds__(64 * tile_waves(DP), DP <= 64 ? 4 : (DP <= 128 ? 2 : 1)) attention_tile_kernel(const attention_args a)
{
    constexpr u32 THREADS = 64 * tile_waves(DP);
    constexpr u32 KEYS = tile_keys(DP);
    constexpr u32 STEPS = KEYS / 32;
    using loader = state_loader<T, DP, CACHE, KEYS, THREADS>;
    using V = typename loader::V;
    constexpr u32 TILE_BYTES = KEYS * DP * 2;
    // what a tile's scores need: the cache's scales by sixteens
    struct tile_info
    {
        float factor[KEYS / 16];
        float mantissa_log[KEYS / 16];
        float mantissa_inverse[KEYS / 16];
    };
    __shared__ __attribute__((aligned(512))) char lds[5 * TILE_BYTES];
    __shared__ tile_info infos[3];
    const u32 lane = threadIdx.x & 63;
    const u32 half = lane / 32;
    const u32 id = tile_order<CACHE>(a);
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
    float base = 0.0F; // top, or 0 while there is none

    const u32 count = state_count(a, b);
    const u32 tiles = (count + KEYS - 1) / KEYS;
    const u32 begin = uniform(static_cast<u32>(static_cast<u64>(tiles) * split / a.splits));
    const u32 end = uniform(static_cast<u32>(static_cast<u64>(tiles) * (split + 1) / a.splits));
    const loader w{a, b, head, count};
    vuint4 next_keys[loader::LOADS];
    vuint4 next_values[loader::LOADS];
    typename loader::place now;   // of the tile in the registers
    typename loader::place next;  // of the tile after it
    typename loader::place after; // its table entry only, one further ahead
    typename loader::bits in = 0;     // of the tile in the registers
    typename loader::bits taking = 0; // of the tile that is worked on

    // the tile in the registers into LDS: keys to place k of two, the rest to place v of three
    const auto put = [&](u32 k, u32 v) {
        const bool mine = ((in >> (lane % KEYS)) & 1) != 0;
        const typename loader::scales scales = w.ready(now, mine);
        w.template put<true>(lds + k * TILE_BYTES, next_keys, 1.0F);
        w.template put<false>(lds + (2 + v) * TILE_BYTES, next_values, scales.value_scale);
        if (CACHE && threadIdx.x < KEYS && threadIdx.x % 16 == 0)
        {
            tile_info& t = infos[v];
            t.factor[threadIdx.x / 16] = scales.key_factor;
            t.mantissa_log[threadIdx.x / 16] = scales.mantissa_log;
            t.mantissa_inverse[threadIdx.x / 16] = scales.mantissa_inverse;
        }
    };
    // the vectors of tile t on their way into the registers
    const auto fetch = [&](u32 t) {
        now = next;
        next.block = after.block;
        in = t < end ? w.taking_part(now, t) : 0;
        w.look_up_block(after, t + 2);
        w.look_up_state(next, t + 1);
        w.template load<true>(next_keys, now, t, in);
        w.template load<false>(next_values, now, t, in);
    };
    // a lane's places in a tile, in one register each
    const u32 row_at = row_address<DP>(lds, lane % 32);
    const u32 first_at = column_address<DP>(lds, 0);
    const u32 second_at = column_address<DP>(lds, 8);
    // scores of the 32 states u of a tile
    const auto scores_of = [&](u32 k, u32 u) {
        const u32 key_row = row_at + k * TILE_BYTES + u * 32 * DP * 2;
        vfloat16 score = {};
#pragma unroll
        for (u32 s = 0; s < DP / 16; ++s)
        {
            score = mfma<T>::run(lds_read<vuint4>(key_row ^ (32 * s)), query[s], score);
        }
        return score;
    };
    // A score of a state that takes no part is -inf, whatever its query holds: the product of a zero key
    // with an infinity or a NaN is none.  Tiles that are whole pass by (start values of 0 and -inf for all
    // tiles instead: 557 against 540 us for 4 x 16/4 heads, 2048 x 8192; 30.5 against 31.0 us where a mask
    // leaves no tile whole, 3 x 12/4 heads, 333 x 1001 x 80).
    const auto leave_out = [&](vfloat16& score, typename loader::bits part, u32 u) {
        const u32 bits = static_cast<u32>(part >> (32 * u));
        if (bits != ~0U)
        {
            asm volatile(""); // stays a branch
            const u32 mine = bits >> (4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                // all ones where the state takes part
                const u32 keep = static_cast<u32>(static_cast<std::int32_t>(mine << (31 - (8 * (i / 4) + i % 4))) >> 31);
                const float x = score[i];
                score[i] = __builtin_bit_cast(float, (__builtin_bit_cast(u32, x) & keep) | (0xFF800000U & ~keep));
            }
        }
    };
    // The reference of the exponents follows the maximum only where that has grown by more than 8:
    // weights stay below 2^8, and the sums are seldom rescaled.
    const auto follow = [&](const vfloat16& score, vfloat2 factor) {
        float largest[2] = {score[0], score[8]};
#pragma unroll
        for (int i = 1; i < 8; ++i)
        {
            largest[0] = fmaxf(largest[0], score[i]);
            largest[1] = fmaxf(largest[1], score[8 + i]);
        }
        float most = CACHE ? fmaxf(largest[0] * factor.x, largest[1] * factor.y)
                           : fmaxf(largest[0], largest[1]) * a.exponent_scale;
        most = fmaxf(most, other_half(most));
        if (__any(most > st.top + 8.0F))
        {
            asm volatile(""); // stays a branch: multiplied every time, the sums cost half the vector work
            const float from = st.top; // -inf at first: the sums are zero and stay it
            st.top = fmaxf(most, st.top);
            base = st.top == -__builtin_inff() ? 0.0F : st.top;
            const float shrink = __builtin_amdgcn_exp2f(from - base);
            st.weight *= shrink;
#pragma unroll
            for (int n2 = 0; n2 < DP / 32; ++n2)
            {
                st.sum[n2] *= shrink;
            }
        }
    };

    // the factors from scores to exponents of the two sixteens of the 32 states u (read ahead of the branch
    // that leaves states out)
    const auto factors_of = [&](u32 v, u32 u) {
        return CACHE ? vfloat2{infos[v].factor[2 * u], infos[v].factor[2 * u + 1]} : vfloat2{a.exponent_scale, a.exponent_scale};
    };

    vfloat16 score = {};
    if (begin < end)
    {
        w.look_up_block(next, begin);
        w.look_up_block(after, begin + 1);
        w.look_up_state(next, begin);
        fetch(begin);
        put(0, 0);
        taking = in;
        fetch(begin + 1);
        __syncthreads();
        score = scores_of(0, 0);
        leave_out(score, taking, 0);
        follow(score, factors_of(0, 0));
    }
    u32 key_place = 0;
    u32 value_place = 0;
    for (u32 tile = begin; tile < end; ++tile)
    {
        const u32 next_key_place = 1 - key_place;
        const u32 next_value_place = value_place == 2 ? 0 : value_place + 1;
#pragma unroll
        for (u32 u = 0; u < STEPS; ++u)
        {
            const bool last = u == STEPS - 1;
            if (last)
            {
                put(next_key_place, next_value_place);
                taking = in;
                fetch(tile + 2);
                __syncthreads();
            }
            const tile_info& t = infos[value_place];
            const u32 first = first_at + (2 + value_place) * TILE_BYTES + u * 32 * DP * 2;
            const u32 second = second_at + (2 + value_place) * TILE_BYTES + u * 32 * DP * 2;
            if constexpr (!CACHE)
            {
                // the wave at the matrix path goes first (537 against 551 us for 4 x 16/4 heads, 2048 x
                // 8192; the cache's, with more of its time on the vector unit: 115 against 109 us)
                __builtin_amdgcn_s_setprio(1);
            }
            vfloat16 next_score = last ? scores_of(next_key_place, 0) : scores_of(key_place, u + 1);
#pragma unroll
            for (u32 g = 0; g < 2; ++g)
            {
                const float factor = CACHE ? t.factor[2 * u + g] : a.exponent_scale;
                const float from = CACHE ? t.mantissa_log[2 * u + g] - base : -base;
                float weight = 0.0F;
#pragma unroll
                for (u32 i = 8 * g; i < 8 * g + 8; ++i)
                {
                    score[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[i], factor, from));
                    weight += score[i];
                }
                st.weight = CACHE ? __builtin_fmaf(weight, t.mantissa_inverse[2 * u + g], st.weight) : st.weight + weight;
            }
#pragma unroll
            for (u32 s = 0; s < 2; ++s)
            {
                const vuint4 p = operand<V>(score, static_cast<int>(s));
                vuint4 rest;
                if constexpr (loader::PIECES)
                {
                    rest = operand_rest<V>(score, static_cast<int>(s), p);
                }
#pragma unroll
                for (u32 m = 0; m < DP / 32; ++m)
                {
                    const u32 rows_on = 16 * s * DP * 2;
                    const vuint4 v = read_column((first ^ (64 * m)) + rows_on, (second ^ (64 * m)) + rows_on);
                    st.sum[m] = mfma<V>::run(v, p, st.sum[m]);
                    if constexpr (loader::PIECES)
                    {
                        st.sum[m] = mfma<V>::run(v, rest, st.sum[m]);
                    }
                }
            }
            if constexpr (!CACHE)
            {
                __builtin_amdgcn_s_setprio(0);
            }
            const vfloat2 next_factors = factors_of(last ? next_value_place : value_place, last ? 0 : u + 1);
            leave_out(next_score, taking, last ? 0 : u + 1);
            follow(next_score, next_factors);
            score = next_score;
        }
        key_place = next_key_place;
        value_place = next_value_place;
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

// Up to two tiles of 32 rows stream the states past, more rows share tiles of states (48 rows, streamed:
// 22 us; 80 rows in tiles: 23 us; 4 x 4 heads over 4096 states x 64).
constexpr u32 MOST_STREAM_ROWS = 64;

// Two workgroups per compute unit stream (1024 and 2048 in all: 3 and 6 us longer than 512 for 64
// sequences of 32 heads over 8192 states); of those that share tiles one fills a unit (512 in all: 122
// against 109 us for 4 x 16/4 heads, 512 rows over 4096 states of the cache).
constexpr size_t WANTED_STREAMS = 512;
constexpr size_t WANTED_TILES = 256;

bool streams(size_t rows) { return rows <= MOST_STREAM_ROWS; }

u32 row_tiles_of(size_t rows, int dim)
{
    const size_t per = streams(rows) ? STREAM_ROWS : tile_rows(padded_dim(dim));
    return static_cast<u32>((rows + per - 1) / per);
}

// How many ranges the states are cut into: as many as give the GPU enough workgroups, at least 512
// states each where they stream (a join of ranges costs a launch: 12.1 us for three of 333 states, 12.6 us
// for one of 1000), 256 where rows share tiles (128: 39 against 31 us for 3 x 12/4 heads, 333 x 1001).
u32 wanted_splits(const bitsknn_attention_shape& s)
{
    const size_t rows = static_cast<size_t>(s.queries) * static_cast<u32>(s.query_heads / s.state_heads);
    const size_t groups = static_cast<size_t>(s.batch) * static_cast<u32>(s.state_heads) * row_tiles_of(rows, s.dim);
    const size_t wanted = streams(rows) ? WANTED_STREAMS : WANTED_TILES;
    const size_t most = static_cast<size_t>(s.states) / (streams(rows) ? 512 : 256);
    if (groups == 0 || groups >= wanted)
    {
        return 1;
    }
    size_t splits = (wanted + groups - 1) / groups;
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
    const u32 threads = 64 * (streams(a.rows) ? STREAM_WAVES : tile_waves(DP));
    if (!fits_grid(blocks, threads) || (a.splits > 1 && !fits_grid((rows + 3) / 4, 256)))
    {
        return fail(BITSKNN_ERR_UNSUPPORTED, "attention: too many rows (%zu)", rows);
    }
    if (streams(a.rows))
    {
        hipLaunchKernelGGL((attention_stream_kernel<T, DP, CACHE>), dim3(static_cast<u32>(blocks)), dim3(threads), 0,
                           stream, a);
    }
    else
    {
        hipLaunchKernelGGL((attention_tile_kernel<T, DP, CACHE>), dim3(static_cast<u32>(blocks)), dim3(threads), 0,
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
