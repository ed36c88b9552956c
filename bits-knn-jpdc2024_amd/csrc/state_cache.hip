// Writing states into the 8-bit cache.
#include "attention_host.hpp"

namespace bitsknn
{
namespace
{

struct store_args
{
    rows_view states[2]; // keys, values
    std::uint8_t* codes[2];
    float* scales[2];
    std::int32_t* block_counts;
    const std::int32_t* counts;
    const std::int32_t* table;
    std::int64_t table_stride;
    u32 blocks;
    u32 block_shift;
    u32 state_heads;
    u32 dim;
    u32 states_per_head;
    u32 slots;
};

// eight values in 32 bits
template <typename T>
__device__ __forceinline__ void load8(const char* at, float (&x)[8])
{
    if constexpr (std::is_same_v<T, float>)
    {
        const vfloat4 lo = reinterpret_cast<const vfloat4*>(at)[0];
        const vfloat4 hi = reinterpret_cast<const vfloat4*>(at)[1];
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            x[i] = lo[i];
            x[4 + i] = hi[i];
        }
    }
    else
    {
        const auto v = *reinterpret_cast<const typename mfma<T>::v8*>(at);
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            x[i] = static_cast<float>(v[i]);
        }
    }
}

// One workgroup per block, head and kind (keys or values).  Bound by memory: the block is read once,
// kept in registers (CHUNKS times eight values a thread) while its largest magnitude is found, and
// written once.
template <typename T, int THREADS, int CHUNKS>
__global__ void __launch_bounds__(THREADS) cache_store_kernel(const store_args a)
{
    __shared__ u32 wave_top[THREADS / 64];
    const u32 kind = blockIdx.x % 2;
    const u32 head = blockIdx.x / 2 % a.state_heads;
    const u32 slot = blockIdx.x / 2 / a.state_heads % a.slots;
    const u32 b = blockIdx.x / 2 / a.state_heads / a.slots;
    u32 count = a.states_per_head;
    if (a.counts != nullptr)
    {
        const std::int32_t c = a.counts[b];
        count = c <= 0 ? 0 : (static_cast<u32>(c) < count ? static_cast<u32>(c) : count);
    }
    const u32 first = slot << a.block_shift;
    const u32 id = static_cast<u32>(a.table[b * a.table_stride + slot]);
    if (first >= count || id >= a.blocks)
    {
        return;
    }
    const u32 block = 1U << a.block_shift;
    const u32 held = count - first < block ? count - first : block;
    const rows_view& v = a.states[kind];
    const char* base = v.data + static_cast<std::int64_t>(sizeof(T)) *
                                    (b * v.batch_stride + head * v.head_stride + first * v.row_stride);
    const u32 per_row = a.dim / 8;
    const u32 step_rows = THREADS / per_row;
    const u32 step_chunks = THREADS % per_row;
    u32 row = threadIdx.x / per_row;
    u32 chunk = threadIdx.x % per_row;
    float x[CHUNKS][8];
    u32 top = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
    {
        if (row < held)
        {
            load8<T>(base + static_cast<std::int64_t>(sizeof(T)) * (row * v.row_stride + chunk * 8), x[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                const u32 bits = __builtin_bit_cast(u32, x[c][i]) & 0x7FFFFFFFU;
                top = bits < 0x7F800000U && bits > top ? bits : top;
            }
        }
        row += step_rows;
        chunk += step_chunks;
        if (chunk >= per_row)
        {
            chunk -= per_row;
            ++row;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o /= 2)
    {
        const u32 other = static_cast<u32>(__shfl_xor(static_cast<int>(top), o));
        top = other > top ? other : top;
    }
    if constexpr (THREADS > 64)
    {
        if (threadIdx.x % 64 == 0)
        {
            wave_top[threadIdx.x / 64] = top;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w)
        {
            top = wave_top[w] > top ? wave_top[w] : top;
        }
    }
    // 448 = 1.75 * 2^8: the smallest power of two that is at least top / 448 is 2^(exponent - 8) where
    // the mantissa is at most 1.75, else the next one
    int exponent = static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7FFFFFU) > 0x600000U ? 1 : 0);
    exponent = exponent < -126 ? -126 : exponent;
    const float scale = __builtin_bit_cast(float, static_cast<u32>(exponent + 127) << 23);
    const float inverse = __builtin_bit_cast(float, static_cast<u32>(127 - exponent) << 23);
    const size_t at = static_cast<size_t>(id) * a.state_heads + head;
    vuint2* out = reinterpret_cast<vuint2*>(a.codes[kind] + ((at << a.block_shift) * a.dim));
    const u32 chunks = held * per_row;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
    {
        const u32 n = threadIdx.x + c * THREADS;
        if (n < chunks)
        {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                const bool finite = (__builtin_bit_cast(u32, x[c][i]) & 0x7FFFFFFFU) < 0x7F800000U;
                y[i] = finite ? x[c][i] * inverse : __builtin_nanf("");
            }
            int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
            int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
            out[n] = vuint2{static_cast<u32>(lo), static_cast<u32>(hi)};
        }
    }
    if (threadIdx.x == 0)
    {
        a.scales[kind][at] = scale;
        if (head == 0 && kind == 0)
        {
            a.block_counts[id] = static_cast<std::int32_t>(held);
        }
    }
}

template <typename T>
int launch_store(const store_args& a, u64 groups, hipStream_t stream)
{
    const u32 chunks = (a.dim / 8) << a.block_shift;
    // threads per block of states: few enough that a thread has several chunks, enough that they fit
    // its registers
    const u32 threads = chunks <= 256 ? 64 : (chunks <= 1024 ? 256 : 1024);
    if (groups * threads > 0xFFFFFFFFULL)
    {
        return fail(BITSKNN_ERR_UNSUPPORTED, "bitsknn_cache_store: too many blocks");
    }
    const dim3 grid(static_cast<u32>(groups));
    if (threads == 64)
    {
        hipLaunchKernelGGL((cache_store_kernel<T, 64, 4>), grid, dim3(64), 0, stream, a);
    }
    else if (threads == 256)
    {
        hipLaunchKernelGGL((cache_store_kernel<T, 256, 4>), grid, dim3(256), 0, stream, a);
    }
    else
    {
        hipLaunchKernelGGL((cache_store_kernel<T, 1024, 8>), grid, dim3(1024), 0, stream, a);
    }
    BITSKNN_HIP_CHECK(hipGetLastError());
    return BITSKNN_OK;
}

} // namespace
} // namespace bitsknn

extern "C" int bitsknn_cache_store(const bitsknn_state_cache* cache, int32_t type, int32_t batch, int32_t states,
                                   const bitsknn_rows* keys, const bitsknn_rows* values, const int32_t* counts,
                                   const int32_t* table, size_t table_stride, void* stream)
{
    using namespace bitsknn;
    clear_error();
    const char* name = "bitsknn_cache_store";
    if (cache == nullptr || keys == nullptr || values == nullptr)
    {
        return fail(BITSKNN_ERR_INVALID, "%s: null pointer", name);
    }
    if (type != BITSKNN_BF16 && type != BITSKNN_FP16 && type != BITSKNN_F32)
    {
        return fail(BITSKNN_ERR_UNSUPPORTED, "%s: unknown type %d", name, type);
    }
    cache_view view = {};
    int status = check_cache(name, cache, view);
    if (status != BITSKNN_OK)
    {
        return status;
    }
    // a 16-bit type and a query head per state head fill the shape
    const bitsknn_attention_shape s = {type == BITSKNN_F32 ? BITSKNN_BF16 : type, cache->dim, batch, cache->state_heads,
                                       cache->state_heads, 0, states, 1.0F};
    const int bytes = type == BITSKNN_F32 ? 4 : 2;
    store_args a = {};
    status = check_shape(name, s);
    status = status != BITSKNN_OK ? status : check_rows(name, "keys", *keys, s, s.state_heads, states, false, a.states[0], bytes);
    status = status != BITSKNN_OK ? status : check_rows(name, "values", *values, s, s.state_heads, states, false, a.states[1], bytes);
    status = status != BITSKNN_OK ? status : check_table(name, table, table_stride, batch, states, view);
    if (status != BITSKNN_OK || batch == 0 || states == 0 || cache->blocks == 0)
    {
        return status;
    }
    a.codes[0] = view.key_codes;
    a.codes[1] = view.value_codes;
    a.scales[0] = view.key_scales;
    a.scales[1] = view.value_scales;
    a.block_counts = view.block_counts;
    a.counts = counts;
    a.table = view.table;
    a.table_stride = view.table_stride;
    a.blocks = view.blocks;
    a.block_shift = view.block_shift;
    a.state_heads = static_cast<u32>(cache->state_heads);
    a.dim = static_cast<u32>(cache->dim);
    a.states_per_head = static_cast<u32>(states);
    a.slots = (static_cast<u32>(states) + static_cast<u32>(cache->block) - 1) >> view.block_shift;
    const u64 groups = 2ULL * static_cast<u32>(batch) * a.slots * a.state_heads;
    const auto st = static_cast<hipStream_t>(stream);
    return type == BITSKNN_BF16   ? launch_store<__bf16>(a, groups, st)
           : type == BITSKNN_FP16 ? launch_store<_Float16>(a, groups, st)
                                  : launch_store<float>(a, groups, st);
}
