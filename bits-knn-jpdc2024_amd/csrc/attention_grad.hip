// Gradients of attention over states of another length.
//
//   P = exp(scale q k - lse)      delta_i = sum(grad_out_i out_i)
//   grad_v = P^T grad_out         dS = P (grad_out v^T - delta)
//   grad_q = scale dS k           grad_k = scale dS^T q
//
// The scores are formed again from the log-sum-exps, nothing of their size is kept.  Two kernels walk
// the same score matrix, one by tiles of states with the sums of their gradients in registers, one by
// tiles of rows with those of the queries' gradients: eight products (four each, in the second one of them
// in two pieces) instead of the five of a single walk, and in return no sum is shared between workgroups:
// every result has one order of addition.  Neither walk is cut into ranges: a workgroup walks all rows, or
// all states, of its sequence and head, so few workgroups take long (1 x 8/1 heads, 2048 x 256 x 128: one
// workgroup walks by states, 800 us in all; 1 x 1 heads, 16 x 8192 x 64: one by rows, 196 us).
#include "attention_host.hpp"
#include "attention_loader.hpp"

namespace bitsknn
{
namespace
{

// The walk by rows: four waves of 32 rows each share tiles of states, in 128 dimensions of 32 states (64:
// 26 registers spilled, 1243 against 957 us for 2 x 16/4 heads, 2048 x 8192).
constexpr u32 ROW_WAVES = 4;
constexpr u32 ROW_THREADS = 64 * ROW_WAVES;
constexpr u32 GRAD_ROWS = 32 * ROW_WAVES;
constexpr u32 step_keys(int padded_dim) { return padded_dim <= 64 ? 64 : 32; }

// The walk by states: waves of 32 states each share steps of 32 rows.  In 128 dimensions a wave keeps its
// values in LDS instead of in registers, so that two waves per quarter of the unit have room (74
// registers spilled otherwise), and eight waves share the steps (four: 847 against 791 us).
constexpr u32 STEP_ROWS = 32;
constexpr bool values_in_lds(int padded_dim) { return padded_dim == 128; }
constexpr u32 state_waves(int padded_dim) { return padded_dim == 128 ? 8 : 4; }
constexpr u32 states_per_group(int padded_dim) { return 32 * state_waves(padded_dim); }

// Both walks take workgroups in the order of their numbers, which deals the tiles of a sequence and head
// out to all dies: sequences of different lengths then end together (one die per sequence and head: 4 %
// longer).

// Eight values per lane, DP / 8 lanes per row.
template <typename T, int DP>
__global__ void __launch_bounds__(256) attention_delta_kernel(const attention_grad_args g, size_t rows)
{
    const attention_args& a = g.f;
    constexpr u32 LANES = DP / 8;
    const size_t flat = static_cast<size_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    const u32 lane = threadIdx.x % LANES;
    float sum = 0.0F;
    if (flat < rows && 8 * lane < static_cast<u32>(a.dim))
    {
        const u32 row = static_cast<u32>(flat % a.rows);
        const u32 group = static_cast<u32>(flat / a.rows);
        const u32 head = group % static_cast<u32>(a.state_heads);
        const u32 b = group / static_cast<u32>(a.state_heads);
        using v8 = typename mfma<T>::v8;
        const v8 x = *reinterpret_cast<const v8*>(a.out.data + 2 * row_offset(a.out, a, b, head, row) + 16 * lane);
        const v8 y = *reinterpret_cast<const v8*>(g.grad_out.data + 2 * row_offset(g.grad_out, a, b, head, row) + 16 * lane);
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            sum = __builtin_fmaf(static_cast<float>(x[i]), static_cast<float>(y[i]), sum);
        }
    }
#pragma unroll
    for (u32 o = LANES / 2; o > 0; o /= 2)
    {
        sum += __shfl_xor(sum, static_cast<int>(o));
    }
    if (lane == 0 && flat < rows)
    {
        g.delta[flat] = sum;
    }
}

// The log-sum-exp of a row in base-2 exponents; a row without any state has weights of zero.
__device__ __forceinline__ float exponent_base(float lse)
{
    return lse == -__builtin_inff() ? __builtin_inff() : lse * LOG2E;
}

// Derivatives enter the products in the vectors' type.  fp16 ends at 65504, which P (dP - delta) passes
// where the gradient, smaller by the scale, need not.  One infinite derivative leaves no number in its row's
// or state's sums, so a walk is taken as it comes and its sums are looked at; where a workgroup finds such a
// sum, it walks again in range: a lane's derivatives, all of one row or all of one state, are multiplied by a
// power of two (1 as long as they fit) that brings the largest so far below 2^15, exactly in fp32, and the
// sums follow it.  What falls below fp16's least number then is below 2^-39 of the largest, and a row or
// state whose derivatives fit gets the same bits in either walk.  (All walks in
// range: 30.3 against 26.0 us for 2 x 8/2 heads, 65 x 257 x 64, 440 against 370 us for 2 x 16/4 heads, 2048 x
// 4096 x 64; bf16 has the exponents of fp32 and needs none of this.)
template <typename T>
constexpr bool RANGE = std::is_same_v<T, _Float16>;

// the sums times a power of two
template <int DP>
__device__ __forceinline__ void scale_sums(vfloat16 (&sum)[DP / 32], float power)
{
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
    {
        if constexpr (DP == 256)
        {
            // they stay in the accumulation registers before and after (194 registers spilled otherwise)
            asm volatile("" : "+a"(sum[n]));
        }
        sum[n] *= power;
        if constexpr (DP == 256)
        {
            asm volatile("" : "+a"(sum[n]));
        }
    }
}

// derivatives weight * slope: the power goes into the slopes
template <int DP>
__device__ __forceinline__ void keep_in_range(const vfloat16& weight, vfloat16& slope, float& power, vfloat16 (&sum)[DP / 32])
{
    float most = 0.0F;
#pragma unroll
    for (int i = 0; i < 16; ++i)
    {
        most = fmaxf(most, __builtin_fabsf(weight[i] * slope[i]));
    }
    most = fmaxf(most, other_half(most));
    if (most * power > 65504.0F)
    {
        // most is in [2^e, 2^(e + 1)), e >= 15: times 2^(14 - e)
        const u32 exponent = __builtin_bit_cast(u32, most) >> 23;
        const float next = __builtin_bit_cast(float, (2 * 127 + 14 - exponent) << 23);
        scale_sums<DP>(sum, next / power);
        power = next;
    }
    slope *= power;
}

__device__ __forceinline__ bool finite(float x)
{
    return (__builtin_bit_cast(u32, x) & 0x7F800000U) != 0x7F800000U;
}

// Steps of 32 rows of queries and incoming gradients into LDS, and what a row's scores need: the base of
// its exponents and its delta.  Rows behind the last one are zero with weights of zero.
template <int DP>
struct row_loader
{
    static constexpr u32 THREADS = 64 * state_waves(DP);
    static constexpr u32 CHUNKS = DP / 8;
    static constexpr int LOADS = STEP_ROWS * CHUNKS / THREADS;
    static_assert(LOADS >= 1 && STEP_ROWS * CHUNKS % THREADS == 0);

    const attention_grad_args& g;
    const u32 b;
    const u32 head;
    // where the step's first row stands: the same in all lanes, moved on by 32 rows per step
    u32 first = 0;
    u32 first_in_group = 0;
    u32 first_position = 0;
    vuint4 queries[LOADS];
    vuint4 grads[LOADS];
    float lse;
    float delta;

    __device__ __forceinline__ void fetch()
    {
        const attention_args& a = g.f;
        const u32 chunk = threadIdx.x % CHUNKS;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
        {
            const u32 row = (static_cast<u32>(i) * THREADS + threadIdx.x) / CHUNKS;
            u32 in_group = first_in_group;
            u32 position = first_position + row;
            while (position >= a.queries_per_head)
            {
                position -= a.queries_per_head;
                ++in_group;
            }
            queries[i] = vuint4{0, 0, 0, 0};
            grads[i] = vuint4{0, 0, 0, 0};
            if (first + row < a.rows && chunk * 8 < static_cast<u32>(a.dim))
            {
                const u32 h = head * static_cast<u32>(a.group) + in_group;
                queries[i] = *reinterpret_cast<const vuint4*>(
                    a.queries.data + 2 * (b * a.queries.batch_stride + h * a.queries.head_stride + position * a.queries.row_stride) + 16 * chunk);
                grads[i] = *reinterpret_cast<const vuint4*>(
                    g.grad_out.data + 2 * (b * g.grad_out.batch_stride + h * g.grad_out.head_stride + position * g.grad_out.row_stride) + 16 * chunk);
            }
        }
        lse = __builtin_inff();
        delta = 0.0F;
        if (threadIdx.x < STEP_ROWS && first + threadIdx.x < a.rows)
        {
            const size_t flat = (static_cast<size_t>(b) * static_cast<u32>(a.state_heads) + head) * a.rows + first + threadIdx.x;
            lse = a.lse[flat];
            delta = g.delta[flat];
        }
        first += STEP_ROWS;
        first_position += STEP_ROWS;
        while (first_position >= a.queries_per_head)
        {
            first_position -= a.queries_per_head;
            ++first_in_group;
        }
    }

    __device__ __forceinline__ void put(char* query_tile, char* grad_tile, float* bases, float* deltas) const
    {
        const u32 chunk = threadIdx.x % CHUNKS;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
        {
            const u32 at = tile_chunk<DP>((static_cast<u32>(i) * THREADS + threadIdx.x) / CHUNKS, chunk);
            *reinterpret_cast<vuint4*>(query_tile + at) = queries[i];
            *reinterpret_cast<vuint4*>(grad_tile + at) = grads[i];
        }
        if (threadIdx.x < STEP_ROWS)
        {
            bases[threadIdx.x] = exponent_base(lse);
            deltas[threadIdx.x] = delta;
        }
    }
};

// a lane's column of a transposed sum (dim x 32), times a factor
template <typename T, int DP>
__device__ __forceinline__ void store_vector(char* at, const vfloat16 (&x)[DP / 32], float factor, u32 dim)
{
    const u32 half = (threadIdx.x & 63) / 32;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
    {
#pragma unroll
        for (int g = 0; g < 4; ++g)
        {
            const u32 column = 32 * n + 8 * g + 4 * half;
            if (column < dim)
            {
                *reinterpret_cast<vuint2*>(at + 2 * column) =
                    vuint2{pack2<T>(x[n][4 * g] * factor, x[n][4 * g + 1] * factor),
                           pack2<T>(x[n][4 * g + 2] * factor, x[n][4 * g + 3] * factor)};
            }
        }
    }
}

// By states: a wave keeps 32 keys and values as operands and their gradients' sums, and walks over the
// rows that read them, those of all heads that share them.  While 32 rows are multiplied, the next are on
// their way into registers and then into the other half of LDS: one barrier per step.
template <typename T, int DP>
__global__ void __launch_bounds__(64 * state_waves(DP), DP <= 128 ? 2 : 1) attention_grad_states_kernel(const attention_grad_args g)
{
    const attention_args& a = g.f;
    constexpr u32 TILE_BYTES = STEP_ROWS * DP * 2;
    constexpr bool KEEP = !values_in_lds(DP);
    __shared__ __attribute__((aligned(512))) char lds[4 * TILE_BYTES];
    __shared__ __attribute__((aligned(512))) char kept[KEEP ? 16 : states_per_group(DP) * DP * 2];
    __shared__ __attribute__((aligned(16))) float bases[2][STEP_ROWS];
    __shared__ __attribute__((aligned(16))) float deltas[2][STEP_ROWS];
    const u32 lane = threadIdx.x & 63;
    const u32 half = lane / 32;
    const u32 id = blockIdx.x;
    const u32 key_tile = id % g.key_tiles;
    const u32 head = id / g.key_tiles % static_cast<u32>(a.state_heads);
    const u32 b = id / g.key_tiles / static_cast<u32>(a.state_heads);
    const u32 state = key_tile * states_per_group(DP) + threadIdx.x / 64 * 32 + lane % 32;
    const u32 count = state_count(a, b);
    bool in = state < count;
    if (a.mask != nullptr && in)
    {
        in = a.mask[static_cast<std::int64_t>(b) * a.mask_stride + state] != 0;
    }
    vuint4 key[DP / 16];
    vuint4 value[DP / 16];
    load_operand<DP>(key, a.keys.data + 2 * (b * a.keys.batch_stride + head * a.keys.head_stride + state * a.keys.row_stride),
                     in, static_cast<u32>(a.dim));
    load_operand<DP>(value, a.values.data + 2 * (b * a.values.batch_stride + head * a.values.head_stride + state * a.values.row_stride),
                     in, static_cast<u32>(a.dim));
    char* const my_values = kept + (KEEP ? 0 : threadIdx.x / 64 * 32 * DP * 2);
    if constexpr (!KEEP)
    {
        // a wave's own part: no barrier
#pragma unroll
        for (u32 s = 0; s < DP / 16; ++s)
        {
            *reinterpret_cast<vuint4*>(my_values + tile_chunk<DP>(lane % 32, 2 * s + half)) = value[s];
        }
    }
    vfloat16 key_sum[DP / 32];
    vfloat16 value_sum[DP / 32];
    const u32 steps = __syncthreads_or(in) != 0 ? (a.rows + STEP_ROWS - 1) / STEP_ROWS : 0;
    const auto walk = [&](auto in_range) {
        float power = 1.0F; // of the lane's state: times key_sum
#pragma unroll
        for (int n = 0; n < DP / 32; ++n)
        {
            key_sum[n] = vfloat16{};
            value_sum[n] = vfloat16{};
        }
        if (steps == 0)
        {
            return;
        }
        row_loader<DP> rows{g, b, head};
        rows.fetch();
        rows.put(lds, lds + TILE_BYTES, bases[0], deltas[0]);
        __syncthreads();
        const u32 row_at = row_address<DP>(lds, lane % 32);
        const u32 value_at = row_address<DP>(my_values, lane % 32);
        const u32 first_at = column_address<DP>(lds, 0);
        const u32 second_at = column_address<DP>(lds, 8);
        for (u32 step = 0; step < steps; ++step)
        {
            const u32 place = step % 2;
            // hidden from the compiler, which would keep the addresses of every step and block in
            // registers that the sums need
            u32 row = row_at + place * 2 * TILE_BYTES;
            u32 own = value_at;
            u32 first = first_at + place * 2 * TILE_BYTES;
            u32 second = second_at + place * 2 * TILE_BYTES;
            asm volatile("" : "+v"(row), "+v"(own), "+v"(first), "+v"(second));
            rows.fetch();
            vfloat16 p = {};
            vfloat16 slope = {};
#pragma unroll
            for (u32 s = 0; s < DP / 16; ++s)
            {
                p = mfma<T>::run(lds_read<vuint4>(row ^ (32 * s)), key[s], p);
            }
#pragma unroll
            for (u32 s = 0; s < DP / 16; ++s)
            {
                const vuint4 v = KEEP ? value[s] : lds_read<vuint4>(own ^ (32 * s));
                slope = mfma<T>::run(lds_read<vuint4>((row ^ (32 * s)) + TILE_BYTES), v, slope);
            }
#pragma unroll
            for (int i = 0; i < 16; i += 4)
            {
                const vfloat4 top = *reinterpret_cast<const vfloat4*>(bases[place] + 2 * i + 4 * half);
                const vfloat4 d = *reinterpret_cast<const vfloat4*>(deltas[place] + 2 * i + 4 * half);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    p[i + j] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i + j], a.exponent_scale, -top[j]));
                    slope[i + j] -= d[j];
                }
            }
            if constexpr (in_range())
            {
                keep_in_range<DP>(p, slope, power, key_sum);
            }
            slope *= p;
            const vuint4 weight[2] = {operand<T>(p, 0), operand<T>(p, 1)};
            const vuint4 change[2] = {operand<T>(slope, 0), operand<T>(slope, 1)};
#pragma unroll
            for (u32 n = 0; n < DP / 32; ++n)
            {
#pragma unroll
                for (u32 s = 0; s < 2; ++s)
                {
                    const u32 x = (first ^ (64 * n)) + 16 * s * DP * 2;
                    const u32 y = (second ^ (64 * n)) + 16 * s * DP * 2;
                    value_sum[n] = mfma<T>::run(read_column(x + TILE_BYTES, y + TILE_BYTES), weight[s], value_sum[n]);
                    key_sum[n] = mfma<T>::run(read_column(x, y), change[s], key_sum[n]);
                }
            }
            char* const other = lds + (1 - place) * 2 * TILE_BYTES;
            rows.put(other, other + TILE_BYTES, bases[1 - place], deltas[1 - place]);
            __syncthreads();
        }
        if constexpr (in_range())
        {
            scale_sums<DP>(key_sum, 1.0F / power);
        }
    };
    walk(std::false_type{});
    if constexpr (RANGE<T>)
    {
        if (__syncthreads_or(in && !finite(key_sum[0][0])) != 0)
        {
            walk(std::true_type{});
        }
    }
    if (state >= a.states)
    {
        return;
    }
    if (!in)
    {
        // no part, no gradient: the sums may hold anything, its vectors were taken as zero
#pragma unroll
        for (int n = 0; n < DP / 32; ++n)
        {
            key_sum[n] = vfloat16{};
            value_sum[n] = vfloat16{};
        }
    }
    store_vector<T, DP>(g.grad_keys.data + 2 * (b * g.grad_keys.batch_stride + head * g.grad_keys.head_stride + state * g.grad_keys.row_stride),
                        key_sum, a.scale, static_cast<u32>(a.dim));
    store_vector<T, DP>(g.grad_values.data + 2 * (b * g.grad_values.batch_stride + head * g.grad_values.head_stride + state * g.grad_values.row_stride),
                        value_sum, 1.0F, static_cast<u32>(a.dim));
}

// By rows: a wave keeps 32 rows of queries and incoming gradients as operands and the sums of the
// queries' gradients, and walks over the states, staged as above.  A score starts from 0, or from -inf
// where the state takes no part: its weight is then 0.
// The derivatives of a row's scores sum to zero, so what the keys have in common cancels in their
// product, but not in the rounding errors of the derivatives: they enter in two pieces (3 % more time for
// 2 x 16/4 heads, 2048 x 8192 x 128; the gradient's error 2.6e-3 -> 1.7e-3, which is its own rounding).
template <typename T, int DP>
__global__ void __launch_bounds__(ROW_THREADS, DP <= 128 ? 2 : 1) attention_grad_rows_kernel(const attention_grad_args g)
{
    const attention_args& a = g.f;
    constexpr u32 KEYS = step_keys(DP);
    using loader = state_loader<T, DP, false, KEYS, ROW_THREADS>;
    constexpr u32 TILE_BYTES = KEYS * DP * 2;
    __shared__ __attribute__((aligned(512))) char lds[4 * TILE_BYTES];
    __shared__ __attribute__((aligned(16))) float starts[2][KEYS];
    const u32 lane = threadIdx.x & 63;
    const u32 half = lane / 32;
    const u32 id = blockIdx.x;
    const u32 row_tile = id % a.row_tiles;
    const u32 head = id / a.row_tiles % static_cast<u32>(a.state_heads);
    const u32 b = id / a.row_tiles / static_cast<u32>(a.state_heads);
    const u32 row = row_tile * GRAD_ROWS + threadIdx.x / 64 * 32 + lane % 32;
    const bool mine = row < a.rows;
    const u32 r = mine ? row : 0;
    vuint4 query[DP / 16];
    vuint4 grad[DP / 16];
    load_operand<DP>(query, a.queries.data + 2 * row_offset(a.queries, a, b, head, r), mine, static_cast<u32>(a.dim));
    load_operand<DP>(grad, g.grad_out.data + 2 * row_offset(g.grad_out, a, b, head, r), mine, static_cast<u32>(a.dim));
    const size_t flat = (static_cast<size_t>(b) * static_cast<u32>(a.state_heads) + head) * a.rows + r;
    const float top = mine ? exponent_base(a.lse[flat]) : __builtin_inff();
    const float delta = mine ? g.delta[flat] : 0.0F;
    vfloat16 sum[DP / 32];
    const u32 count = uniform(state_count(a, b));
    const u32 tiles = (count + KEYS - 1) / KEYS;
    const loader w{a, b, head, count};
    vuint4 keys[loader::LOADS];
    vuint4 values[loader::LOADS];
    typename loader::place next;
    typename loader::bits in = 0; // of the tile in the registers
    const auto fetch = [&](u32 t) {
        in = t < tiles ? w.taking_part(next, t) : 0;
        w.template load<true>(keys, next, t, in);
        w.template load<false>(values, next, t, in);
        w.look_up_state(next, t + 1);
    };
    const auto put = [&](u32 place) {
        w.template put<true>(lds + place * 2 * TILE_BYTES, keys, 1.0F);
        w.template put<false>(lds + place * 2 * TILE_BYTES + TILE_BYTES, values, 1.0F);
        if (threadIdx.x < KEYS)
        {
            starts[place][threadIdx.x] = ((in >> threadIdx.x) & 1) != 0 ? 0.0F : -__builtin_inff();
        }
    };
    const u32 row_at = row_address<DP>(lds, lane % 32);
    const u32 first_at = column_address<DP>(lds, 0);
    const u32 second_at = column_address<DP>(lds, 8);
    const auto walk = [&](auto in_range) {
        float power = 1.0F; // of the lane's row: times sum
#pragma unroll
        for (int n = 0; n < DP / 32; ++n)
        {
            sum[n] = vfloat16{};
        }
        if (tiles > 0)
        {
            w.look_up_state(next, 0);
            fetch(0);
            put(0);
            __syncthreads();
        }
        for (u32 tile = 0; tile < tiles; ++tile)
        {
            const u32 place = tile % 2;
            fetch(tile + 1);
#pragma unroll 1
            for (u32 u = 0; u < KEYS / 32; ++u)
            {
                const u32 at = place * 2 * TILE_BYTES + u * 32 * DP * 2;
                u32 row_to = row_at + at;
                u32 first = first_at + at;
                u32 second = second_at + at;
                // hidden from the compiler, as in the walk by states
                asm volatile("" : "+v"(row_to), "+v"(first), "+v"(second));
                vfloat16 p;
                vfloat16 slope = {};
#pragma unroll
                for (u32 q = 0; q < 4; ++q)
                {
                    const vfloat4 start = *reinterpret_cast<const vfloat4*>(starts[place] + 32 * u + 8 * q + 4 * half);
#pragma unroll
                    for (u32 i = 0; i < 4; ++i)
                    {
                        p[4 * q + i] = start[i];
                    }
                }
#pragma unroll
                for (u32 s = 0; s < DP / 16; ++s)
                {
                    p = mfma<T>::run(lds_read<vuint4>(row_to ^ (32 * s)), query[s], p);
                }
#pragma unroll
                for (u32 s = 0; s < DP / 16; ++s)
                {
                    slope = mfma<T>::run(lds_read<vuint4>((row_to ^ (32 * s)) + TILE_BYTES), grad[s], slope);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i], a.exponent_scale, -top));
                    slope[i] -= delta;
                }
                if constexpr (in_range())
                {
                    keep_in_range<DP>(p, slope, power, sum);
                }
                p *= slope;
                const vuint4 change[2] = {operand<T>(p, 0), operand<T>(p, 1)};
                const vuint4 rest[2] = {operand_rest<T>(p, 0, change[0]), operand_rest<T>(p, 1, change[1])};
#pragma unroll
                for (u32 n = 0; n < DP / 32; ++n)
                {
#pragma unroll
                    for (u32 s = 0; s < 2; ++s)
                    {
                        const u32 rows_on = 16 * s * DP * 2;
                        const vuint4 k = read_column((first ^ (64 * n)) + rows_on, (second ^ (64 * n)) + rows_on);
                        sum[n] = mfma<T>::run(k, change[s], sum[n]);
                        sum[n] = mfma<T>::run(k, rest[s], sum[n]);
                    }
                }
            }
            put(1 - place);
            __syncthreads();
        }
        if constexpr (in_range())
        {
            scale_sums<DP>(sum, 1.0F / power);
        }
    };
    walk(std::false_type{});
    if constexpr (RANGE<T>)
    {
        if (__syncthreads_or(mine && top != __builtin_inff() && !finite(sum[0][0])) != 0)
        {
            walk(std::true_type{});
        }
    }
    if (mine)
    {
        if (top == __builtin_inff())
        {
            // a row without any state: its zero weights times what it holds may be anything
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
            {
                sum[n] = vfloat16{};
            }
        }
        store_vector<T, DP>(g.grad_queries.data + 2 * row_offset(g.grad_queries, a, b, head, row), sum, a.scale,
                            static_cast<u32>(a.dim));
    }
}

template <typename T, int DP>
int launch(const attention_grad_args& g, size_t rows, u32 batch, hipStream_t stream)
{
    const u64 groups = static_cast<u64>(batch) * static_cast<u32>(g.f.state_heads);
    constexpr size_t per_group = 256 / (DP / 8);
    const size_t delta_groups = (rows + per_group - 1) / per_group;
    // all three before the first
    if (!fits_grid(delta_groups, 256) || !fits_grid(groups * g.f.row_tiles, ROW_THREADS) ||
        !fits_grid(groups * g.key_tiles, 64 * state_waves(DP)))
    {
        return fail(BITSKNN_ERR_UNSUPPORTED, "bitsknn_cross_attention_backward: too many rows");
    }
    if (rows > 0)
    {
        hipLaunchKernelGGL((attention_delta_kernel<T, DP>), dim3(static_cast<u32>(delta_groups)), dim3(256), 0, stream, g,
                           rows);
        BITSKNN_HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL((attention_grad_rows_kernel<T, DP>), dim3(static_cast<u32>(groups * g.f.row_tiles)),
                           dim3(ROW_THREADS), 0, stream, g);
        BITSKNN_HIP_CHECK(hipGetLastError());
    }
    if (g.f.states > 0)
    {
        hipLaunchKernelGGL((attention_grad_states_kernel<T, DP>), dim3(static_cast<u32>(groups * g.key_tiles)),
                           dim3(64 * state_waves(DP)), 0, stream, g);
        BITSKNN_HIP_CHECK(hipGetLastError());
    }
    return BITSKNN_OK;
}

size_t grad_workspace_bytes(const bitsknn_attention_shape& s)
{
    // one float per row, whole 16 bytes
    const size_t rows = static_cast<size_t>(s.batch) * static_cast<u32>(s.query_heads) * static_cast<u32>(s.queries);
    return (rows * sizeof(float) + 15) / 16 * 16;
}

} // namespace
} // namespace bitsknn

extern "C" size_t bitsknn_cross_attention_backward_workspace_bytes(const bitsknn_attention_shape* shape)
{
    using namespace bitsknn;
    clear_error();
    if (shape == nullptr || check_shape("bitsknn_cross_attention_backward_workspace_bytes", *shape) != BITSKNN_OK)
    {
        return 0;
    }
    return grad_workspace_bytes(*shape);
}

extern "C" int bitsknn_cross_attention_backward(const bitsknn_attention_shape* shape, const bitsknn_rows* grad_out,
                                                const bitsknn_rows* queries, const bitsknn_rows* keys,
                                                const bitsknn_rows* values, const bitsknn_rows* out, const float* lse,
                                                const int32_t* counts, const uint8_t* mask, size_t mask_stride,
                                                const bitsknn_rows* grad_queries, const bitsknn_rows* grad_keys,
                                                const bitsknn_rows* grad_values, void* workspace,
                                                size_t workspace_bytes, void* stream)
{
    using namespace bitsknn;
    clear_error();
    const char* name = "bitsknn_cross_attention_backward";
    if (shape == nullptr || grad_out == nullptr || queries == nullptr || keys == nullptr || values == nullptr ||
        out == nullptr || grad_queries == nullptr || grad_keys == nullptr || grad_values == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: null pointer", name);
    }
    const bitsknn_attention_shape& s = *shape;
    attention_grad_args g = {};
    attention_args& a = g.f;
    int status = check_shape(name, s);
    status = status != BITSKNN_OK ? status : fill_shape(a, s);
    const int h = s.query_heads;
    const int hs = s.state_heads;
    status = status != BITSKNN_OK ? status : check_rows(name, "grad_out", *grad_out, s, h, s.queries, false, g.grad_out);
    status = status != BITSKNN_OK ? status : check_rows(name, "queries", *queries, s, h, s.queries, false, a.queries);
    status = status != BITSKNN_OK ? status : check_rows(name, "keys", *keys, s, hs, s.states, false, a.keys);
    status = status != BITSKNN_OK ? status : check_rows(name, "values", *values, s, hs, s.states, false, a.values);
    status = status != BITSKNN_OK ? status : check_rows(name, "out", *out, s, h, s.queries, false, a.out);
    status = status != BITSKNN_OK ? status : check_rows(name, "grad_queries", *grad_queries, s, h, s.queries, true, g.grad_queries);
    status = status != BITSKNN_OK ? status : check_rows(name, "grad_keys", *grad_keys, s, hs, s.states, true, g.grad_keys);
    status = status != BITSKNN_OK ? status : check_rows(name, "grad_values", *grad_values, s, hs, s.states, true, g.grad_values);
    status = status != BITSKNN_OK ? status : check_mask(name, s, mask, mask_stride);
    status = status != BITSKNN_OK ? status : check_workspace(name, workspace);
    if (status != BITSKNN_OK || s.batch == 0)
    {
        return status;
    }
    const size_t rows = static_cast<size_t>(s.batch) * static_cast<u32>(h) * static_cast<u32>(s.queries);
    if (rows > 0 && lse == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: lse: null pointer", name);
    }
    const size_t need = grad_workspace_bytes(s);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    {
        return fail(BITSKNN_ERR_INVALID, "%s: a workspace of %zu bytes, %zu are needed", name,
                    workspace == nullptr ? size_t{0} : workspace_bytes, need);
    }
    const int padded = s.dim <= 64 ? 64 : (s.dim <= 128 ? 128 : 256);
    a.row_tiles = (a.rows + GRAD_ROWS - 1) / GRAD_ROWS;
    g.key_tiles = (a.states + states_per_group(padded) - 1) / states_per_group(padded);
    a.counts = counts;
    a.mask = mask;
    a.mask_stride = static_cast<std::int64_t>(mask_stride);
    a.lse = const_cast<float*>(lse);
    g.delta = static_cast<float*>(workspace);
    const auto st = static_cast<hipStream_t>(stream);
    const u32 batch = static_cast<u32>(s.batch);
    if (s.type == BITSKNN_BF16)
    {
        return padded == 64    ? launch<__bf16, 64>(g, rows, batch, st)
               : padded == 128 ? launch<__bf16, 128>(g, rows, batch, st)
                               : launch<__bf16, 256>(g, rows, batch, st);
    }
    return padded == 64    ? launch<_Float16, 64>(g, rows, batch, st)
           : padded == 128 ? launch<_Float16, 128>(g, rows, batch, st)
                           : launch<_Float16, 256>(g, rows, batch, st);
}
