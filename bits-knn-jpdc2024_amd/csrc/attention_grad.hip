// Gradients of attention over states of another length.
//
//   P = exp(scale q k - lse)      delta_i = sum(grad_out_i out_i)
//   grad_v = P^T grad_out         dS = P (grad_out v^T - delta)
//   grad_q = scale dS k           grad_k = scale dS^T q
//
// The scores are formed again from the log-sum-exps, nothing of their size is kept.  Two kernels walk
// the same score matrix, one by tiles of states with the sums of their gradients in registers, one by
// tiles of rows with those of the queries' gradients: seven products instead of the five of a single
// walk, and in return no sum is shared between workgroups: every result has one order of addition.
#include "attention_host.hpp"

namespace bitsknn
{
namespace
{

constexpr u32 WAVES = 4;
constexpr u32 GRAD_KEYS = 32 * WAVES; // states per workgroup of the walk by states
constexpr u32 GRAD_ROWS = 32 * WAVES; // rows per workgroup of the walk by rows
constexpr u32 TILE = 32;              // rows, or states, per step of either walk

// One row of delta per wave.
template <typename T>
__global__ void __launch_bounds__(256) attention_delta_kernel(const attention_grad_args g, size_t rows)
{
    const attention_args& a = g.f;
    const size_t flat = static_cast<size_t>(blockIdx.x) * 4 + threadIdx.x / 64;
    const u32 lane = threadIdx.x & 63;
    if (flat >= rows)
    {
        return;
    }
    const u32 row = static_cast<u32>(flat % a.rows);
    const u32 head = static_cast<u32>(flat / a.rows % static_cast<u32>(a.state_heads));
    const u32 b = static_cast<u32>(flat / a.rows / static_cast<u32>(a.state_heads));
    float sum = 0.0F;
    if (8 * lane < static_cast<u32>(a.dim))
    {
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
    for (int o = 16; o > 0; o /= 2)
    {
        sum += __shfl_xor(sum, o);
    }
    if (lane == 0)
    {
        g.delta[flat] = sum;
    }
}

// The log-sum-exp of a row in base-2 exponents; a row without any state has weights of zero.
__device__ __forceinline__ float exponent_base(float lse)
{
    return lse == -__builtin_inff() ? __builtin_inff() : lse * LOG2E;
}

// Two tiles of 32 rows (first of them `first`) of the row views x and y into LDS, and what a row's
// scores need: the base of its exponents and its delta.  Rows behind the last one are zero with
// weights of zero.
template <int DP>
__device__ __forceinline__ void stage_rows(char* x_tile, char* y_tile, float* base, float* delta,
                                           const attention_grad_args& g, u32 b, u32 head, u32 first)
{
    constexpr u32 CHUNKS = DP / 8;
    const attention_args& a = g.f;
#pragma unroll
    for (u32 c = threadIdx.x; c < TILE * CHUNKS; c += 64 * WAVES)
    {
        const u32 row = c / CHUNKS;
        const u32 chunk = c % CHUNKS;
        vuint4 x = {0, 0, 0, 0};
        vuint4 y = {0, 0, 0, 0};
        if (first + row < a.rows && chunk * 8 < static_cast<u32>(a.dim))
        {
            x = *reinterpret_cast<const vuint4*>(a.queries.data + 2 * row_offset(a.queries, a, b, head, first + row) +
                                                 16 * chunk);
            y = *reinterpret_cast<const vuint4*>(g.grad_out.data + 2 * row_offset(g.grad_out, a, b, head, first + row) +
                                                 16 * chunk);
        }
        *reinterpret_cast<vuint4*>(x_tile + tile_chunk<DP>(row, chunk)) = x;
        *reinterpret_cast<vuint4*>(y_tile + tile_chunk<DP>(row, chunk)) = y;
    }
    if (threadIdx.x < TILE)
    {
        const u32 row = first + threadIdx.x;
        const size_t flat = (static_cast<size_t>(b) * static_cast<u32>(a.state_heads) + head) * a.rows + row;
        base[threadIdx.x] = row < a.rows ? exponent_base(a.lse[flat]) : __builtin_inff();
        delta[threadIdx.x] = row < a.rows ? g.delta[flat] : 0.0F;
    }
}

// registers 8 s .. 8 s + 7 of a product as the operand of step s
template <typename T>
__device__ __forceinline__ vuint4 operand(const vfloat16& x, int s)
{
    return vuint4{pack2<T>(x[8 * s], x[8 * s + 1]), pack2<T>(x[8 * s + 2], x[8 * s + 3]),
                  pack2<T>(x[8 * s + 4], x[8 * s + 5]), pack2<T>(x[8 * s + 6], x[8 * s + 7])};
}

// one of 32 consecutive vectors in the operand layout of its lane
template <int DP>
__device__ __forceinline__ void load_vector(vuint4 (&x)[DP / 16], const char* at, bool in, u32 dim)
{
    const u32 half = (threadIdx.x & 63) / 32;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
    {
        const u32 column = 16 * s + 8 * half;
        x[s] = vuint4{0, 0, 0, 0};
        if (in && column < dim)
        {
            x[s] = *reinterpret_cast<const vuint4*>(at + 2 * column);
        }
    }
}

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
// rows that read them, those of all heads that share them.
template <typename T, int DP>
__global__ void __launch_bounds__(64 * WAVES) attention_grad_states_kernel(const attention_grad_args g)
{
    const attention_args& a = g.f;
    __shared__ __attribute__((aligned(16))) char query_tile[TILE * DP * 2];
    __shared__ __attribute__((aligned(16))) char grad_tile[TILE * DP * 2];
    __shared__ __attribute__((aligned(16))) float base[TILE];
    __shared__ __attribute__((aligned(16))) float delta[TILE];
    const u32 lane = threadIdx.x & 63;
    const u32 half = lane / 32;
    const u32 id = die_order(blockIdx.x, gridDim.x);
    const u32 key_tile = id % g.key_tiles;
    const u32 head = id / g.key_tiles % static_cast<u32>(a.state_heads);
    const u32 b = id / g.key_tiles / static_cast<u32>(a.state_heads);
    const u32 state = key_tile * GRAD_KEYS + threadIdx.x / 64 * 32 + lane % 32;
    const u32 count = state_count(a, b);
    bool in = state < count;
    if (a.mask != nullptr && in)
    {
        in = a.mask[static_cast<std::int64_t>(b) * a.mask_stride + state] != 0;
    }
    vuint4 key[DP / 16];
    vuint4 value[DP / 16];
    load_vector<DP>(key, a.keys.data + 2 * (b * a.keys.batch_stride + head * a.keys.head_stride + state * a.keys.row_stride),
                    in, static_cast<u32>(a.dim));
    load_vector<DP>(value, a.values.data + 2 * (b * a.values.batch_stride + head * a.values.head_stride + state * a.values.row_stride),
                    in, static_cast<u32>(a.dim));
    vfloat16 key_sum[DP / 32];
    vfloat16 value_sum[DP / 32];
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
    {
        key_sum[n] = vfloat16{};
        value_sum[n] = vfloat16{};
    }
    const u32 steps = __syncthreads_or(in) != 0 ? (a.rows + TILE - 1) / TILE : 0;
    for (u32 step = 0; step < steps; ++step)
    {
        __syncthreads();
        stage_rows<DP>(query_tile, grad_tile, base, delta, g, b, head, step * TILE);
        __syncthreads();
        vfloat16 p = {};
        vfloat16 slope = {};
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
        {
            p = mfma<T>::run(tile_row<DP>(query_tile, lane % 32, s), key[s], p);
        }
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
        {
            slope = mfma<T>::run(tile_row<DP>(grad_tile, lane % 32, s), value[s], slope);
        }
#pragma unroll
        for (int i = 0; i < 16; i += 4)
        {
            const vfloat4 top = *reinterpret_cast<const vfloat4*>(base + 2 * i + 4 * half);
            const vfloat4 d = *reinterpret_cast<const vfloat4*>(delta + 2 * i + 4 * half);
#pragma unroll
            for (int j = 0; j < 4; ++j)
            {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i + j], a.exponent_scale, -top[j]));
                p[i + j] = x;
                slope[i + j] = x * (slope[i + j] - d[j]);
            }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
        {
            const vuint4 weight = operand<T>(p, s);
            const vuint4 change = operand<T>(slope, s);
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
            {
                value_sum[n] = mfma<T>::run(tile_column<DP>(grad_tile, s, n), weight, value_sum[n]);
                key_sum[n] = mfma<T>::run(tile_column<DP>(query_tile, s, n), change, key_sum[n]);
            }
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
// queries' gradients, and walks over the states.
template <typename T, int DP>
__global__ void __launch_bounds__(64 * WAVES) attention_grad_rows_kernel(const attention_grad_args g)
{
    const attention_args& a = g.f;
    constexpr u32 CHUNKS = DP / 8;
    __shared__ __attribute__((aligned(16))) char key_tile[TILE * DP * 2];
    __shared__ __attribute__((aligned(16))) char value_tile[TILE * DP * 2];
    const u32 lane = threadIdx.x & 63;
    const u32 half = lane / 32;
    const u32 id = die_order(blockIdx.x, gridDim.x);
    const u32 row_tile = id % a.row_tiles;
    const u32 head = id / a.row_tiles % static_cast<u32>(a.state_heads);
    const u32 b = id / a.row_tiles / static_cast<u32>(a.state_heads);
    const u32 row = row_tile * GRAD_ROWS + threadIdx.x / 64 * 32 + lane % 32;
    const bool in = row < a.rows;
    const u32 r = in ? row : 0;
    vuint4 query[DP / 16];
    vuint4 grad[DP / 16];
    load_vector<DP>(query, a.queries.data + 2 * row_offset(a.queries, a, b, head, r), in, static_cast<u32>(a.dim));
    load_vector<DP>(grad, g.grad_out.data + 2 * row_offset(g.grad_out, a, b, head, r), in, static_cast<u32>(a.dim));
    const size_t flat = (static_cast<size_t>(b) * static_cast<u32>(a.state_heads) + head) * a.rows + r;
    const float top = in ? exponent_base(a.lse[flat]) : __builtin_inff();
    const float delta = in ? g.delta[flat] : 0.0F;
    vfloat16 sum[DP / 32];
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
    {
        sum[n] = vfloat16{};
    }
    const u32 count = state_count(a, b);
    for (u32 first = 0; first < count; first += TILE)
    {
        const u32 taking = static_cast<u32>(states_taking_part(a, b, count, first));
        if (taking == 0)
        {
            continue;
        }
        __syncthreads();
        const char* keys = a.keys.data + 2 * (b * a.keys.batch_stride + head * a.keys.head_stride + first * a.keys.row_stride);
        const char* values = a.values.data + 2 * (b * a.values.batch_stride + head * a.values.head_stride + first * a.values.row_stride);
#pragma unroll
        for (u32 c = threadIdx.x; c < TILE * CHUNKS; c += 64 * WAVES)
        {
            const u32 j = c / CHUNKS;
            const u32 chunk = c % CHUNKS;
            vuint4 x = {0, 0, 0, 0};
            vuint4 y = {0, 0, 0, 0};
            if (((taking >> j) & 1) != 0 && chunk * 8 < static_cast<u32>(a.dim))
            {
                x = *reinterpret_cast<const vuint4*>(keys + 2 * (j * a.keys.row_stride + chunk * 8));
                y = *reinterpret_cast<const vuint4*>(values + 2 * (j * a.values.row_stride + chunk * 8));
            }
            *reinterpret_cast<vuint4*>(key_tile + tile_chunk<DP>(j, chunk)) = x;
            *reinterpret_cast<vuint4*>(value_tile + tile_chunk<DP>(j, chunk)) = y;
        }
        __syncthreads();
        vfloat16 p = {};
        vfloat16 slope = {};
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
        {
            p = mfma<T>::run(tile_row<DP>(key_tile, lane % 32, s), query[s], p);
        }
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
        {
            slope = mfma<T>::run(tile_row<DP>(value_tile, lane % 32, s), grad[s], slope);
        }
        const u32 bits = taking >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
            float x = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i], a.exponent_scale, -top)) * (slope[i] - delta);
            if (taking != ~0U)
            {
                // a state that takes no part was staged as zero; its weight may be infinite
                x = ((bits >> (8 * (i / 4) + i % 4)) & 1) != 0 ? x : 0.0F;
            }
            p[i] = x;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
        {
            const vuint4 change = operand<T>(p, s);
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
            {
                sum[n] = mfma<T>::run(tile_column<DP>(key_tile, s, n), change, sum[n]);
            }
        }
    }
    if (in)
    {
        store_vector<T, DP>(g.grad_queries.data + 2 * row_offset(g.grad_queries, a, b, head, row), sum, a.scale,
                            static_cast<u32>(a.dim));
    }
}

template <typename T, int DP>
int launch(const attention_grad_args& g, size_t rows, u32 batch, hipStream_t stream)
{
    const u64 groups = static_cast<u64>(batch) * static_cast<u32>(g.f.state_heads);
    if (rows > 0)
    {
        hipLaunchKernelGGL(attention_delta_kernel<T>, dim3(static_cast<u32>((rows + 3) / 4)), dim3(256), 0, stream, g, rows);
        BITSKNN_HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL((attention_grad_rows_kernel<T, DP>), dim3(static_cast<u32>(groups * g.f.row_tiles)),
                           dim3(64 * WAVES), 0, stream, g);
        BITSKNN_HIP_CHECK(hipGetLastError());
    }
    if (g.f.states > 0)
    {
        hipLaunchKernelGGL((attention_grad_states_kernel<T, DP>), dim3(static_cast<u32>(groups * g.key_tiles)),
                           dim3(64 * WAVES), 0, stream, g);
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
    a.row_tiles = (a.rows + GRAD_ROWS - 1) / GRAD_ROWS;
    g.key_tiles = (a.states + GRAD_KEYS - 1) / GRAD_KEYS;
    const u64 groups = static_cast<u64>(s.batch) * static_cast<u32>(hs);
    if (groups * a.row_tiles > MOST_WORKGROUPS || groups * g.key_tiles > MOST_WORKGROUPS ||
        (rows + 3) / 4 > MOST_WORKGROUPS)
    {
        return fail(BITSKNN_ERR_UNSUPPORTED, "%s: too many rows", name);
    }
    a.counts = counts;
    a.mask = mask;
    a.mask_stride = static_cast<std::int64_t>(mask_stride);
    a.lse = const_cast<float*>(lse);
    g.delta = static_cast<float*>(workspace);
    const int padded = s.dim <= 64 ? 64 : (s.dim <= 128 ? 128 : 256);
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
