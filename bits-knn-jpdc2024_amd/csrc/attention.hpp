// What the attention kernels share: the matrix instruction for both 16-bit types, the layout of a
// tile in LDS, and the arguments.
//
// Every product is taken with v_mfma_f32_32x32x16 (fp32 sums).  Lane l = 32 h + c holds of
//   A (32 x 16): row c, the eight values k = 8 h ..     B (16 x 32): column c, k = 8 h ..
//   C (32 x 32): column c, register i = row 8 (i / 4) + 4 h + i % 4
// A product whose result is the right operand of the next one is arranged so that the next one sums
// over its rows: registers 8 s .. 8 s + 7 of C are then a B operand as they stand, the sixteen rows
// 16 s + 4 h + {0..3, 8..11} of step s in the order of the registers, and the A operand is read in the
// same order (tile_column).  No value crosses lanes between the two products.
#ifndef BITSKNN_CSRC_ATTENTION_HPP_
#define BITSKNN_CSRC_ATTENTION_HPP_

#include <type_traits>

#include "common.hpp"

namespace bitsknn
{

// batch x heads x rows vectors of 16-bit values; strides in elements
struct rows_view
{
    char* data;
    std::int64_t batch_stride;
    std::int64_t head_stride;
    std::int64_t row_stride;
};

struct cache_view
{
    std::uint8_t* key_codes;
    std::uint8_t* value_codes;
    float* key_scales;
    float* value_scales;
    std::int32_t* block_counts;
    const std::int32_t* table;
    std::int64_t table_stride;
    u32 blocks;
    u32 block_shift; // log2 of the states per block
};

struct attention_args
{
    rows_view queries;
    rows_view keys;
    rows_view values;
    rows_view out;
    cache_view cache;
    const std::int32_t* counts;
    const std::uint8_t* mask;
    std::int64_t mask_stride;
    float* lse;       // batch x query heads x rows, or null
    float* part;      // partial sums of the splits: rows x splits x padded dim
    float2* part_ml;  // rows x splits (maximum in base-2 exponents, sum)
    std::int32_t dim;
    std::int32_t state_heads;
    std::int32_t group;   // query heads per state head
    u32 queries_per_head;
    u32 rows;             // group * queries_per_head: the rows that read one state head
    u32 states;
    u32 row_tiles;
    u32 splits;
    float exponent_scale; // scale * log2(e)
    float scale;
};

struct attention_grad_args
{
    attention_args f;   // out, lse: what the forward pass returned
    rows_view grad_out;
    rows_view grad_queries;
    rows_view grad_keys;
    rows_view grad_values;
    float* delta;       // batch x query heads x rows: sum of grad_out * out
    u32 key_tiles;
};

namespace
{

typedef float vfloat16 __attribute__((ext_vector_type(16)));
typedef float vfloat4 __attribute__((ext_vector_type(4)));
typedef float vfloat2 __attribute__((ext_vector_type(2)));
typedef u32 vuint4 __attribute__((ext_vector_type(4)));
typedef u32 vuint2 __attribute__((ext_vector_type(2)));
typedef short vshort4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634F;
constexpr float LN2 = 0.6931471805599453F;

template <typename T>
struct mfma;

template <>
struct mfma<__bf16>
{
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ vfloat16 run(vuint4 a, vuint4 b, vfloat16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    // two e4m3 codes (the lower or the upper half of x) as two values, times the power of two of `power`
    // (its mantissa is ignored): exact
    template <bool UPPER>
    static __device__ __forceinline__ u32 decode(u32 x, float power)
    {
        return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, power, UPPER));
    }
};

template <>
struct mfma<_Float16>
{
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ vfloat16 run(vuint4 a, vuint4 b, vfloat16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    template <bool UPPER>
    static __device__ __forceinline__ u32 decode(u32 x, float power)
    {
        return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, power, UPPER));
    }
};

// two values rounded to nearest even
template <typename T>
__device__ __forceinline__ u32 pack2(float x, float y)
{
    return __builtin_bit_cast(u32, __builtin_convertvector((vfloat2{x, y}), typename mfma<T>::v2));
}

// eight e4m3 codes as eight 16-bit values, times the power of two of `power`
template <typename T>
__device__ __forceinline__ vuint4 decode8(vuint2 codes, float power)
{
    return vuint4{mfma<T>::template decode<false>(codes.x, power), mfma<T>::template decode<true>(codes.x, power),
                  mfma<T>::template decode<false>(codes.y, power), mfma<T>::template decode<true>(codes.y, power)};
}

// the value of the lane in the other half of the wave
__device__ __forceinline__ float other_half(float x)
{
    const u32 bits = __builtin_bit_cast(u32, x);
    const auto both = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 32) != 0 ? both[0] : both[1]);
}

// ---- a tile of rows x DP 16-bit values in LDS -------------------------------------------------
//
// Rows one after the other in chunks of 16 bytes, a row's chunks stored exclusive-or'ed with a number of
// the row.  LDS serves 256 bytes at a time, sixteen chunks from different banks, to two kinds of reads:
// sixteen consecutive rows at one chunk, and (transposed) four rows of which each gives four chunks side
// by side.  With the row's lowest two bits above its next two, both meet every bank once; in 64
// dimensions, where two rows fill the banks, the same holds for the bits above the lowest.
// (Twice the row modulo eight left 44 % of the LDS cycles to conflicts.)

template <int DP>
__device__ __forceinline__ constexpr u32 tile_swizzle(u32 row)
{
    return DP == 64 ? 4 * ((row / 2) % 2) + (row / 4) % 4 : 4 * (row % 4) + (row / 4) % 4;
}

// byte offset of a 16-byte chunk
template <int DP>
__device__ __forceinline__ constexpr u32 tile_chunk(u32 row, u32 chunk)
{
    return row * (DP * 2) + (chunk ^ tile_swizzle<DP>(row)) * 16;
}

// A operand: row `row` (its lane's), the eight values of step `step` of the row
template <int DP>
__device__ __forceinline__ vuint4 tile_row(const char* tile, u32 row, u32 step)
{
    const u32 half = (threadIdx.x & 63) / 32;
    return *reinterpret_cast<const vuint4*>(tile + tile_chunk<DP>(row, 2 * step + half));
}

// A operand of the transposed tile: the lane's column 32 block + c, the rows 16 step + 4 h + {0..3,
// 8..11}.  ds_read_b64_tr_b16 hands lane i of sixteen the values at place i of the 4 x 16 matrix
// whose rows are eight bytes each of lanes 4 j .. 4 j + 3.
template <int DP>
__device__ __forceinline__ vuint4 tile_column(const char* tile, u32 step, u32 block)
{
    typedef __attribute__((address_space(3))) vshort4* lds_ptr;
    const u32 lane = threadIdx.x & 63;
    const u32 row = 16 * step + 4 * (lane / 32) + (lane % 16) / 4;
    const u32 chunk = 4 * block + 2 * ((lane / 16) % 2) + (lane % 4) / 2;
    const char* first = tile + tile_chunk<DP>(row, chunk) + 8 * (lane % 2);
    const char* second = tile + tile_chunk<DP>(row + 8, chunk) + 8 * (lane % 2);
    const vshort4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)first);
    const vshort4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)second);
    const vuint2 lo = __builtin_bit_cast(vuint2, x);
    const vuint2 hi = __builtin_bit_cast(vuint2, y);
    return vuint4{lo.x, lo.y, hi.x, hi.y};
}

// The same reads from addresses that a lane works out once per tile: the steps and the blocks of a tile
// differ from the first in bits that an exclusive or sets, so one register stands for all of them
// (tiles that start at multiples of 512 bytes).
template <typename V>
__device__ __forceinline__ V lds_read(u32 at)
{
    typedef __attribute__((address_space(3))) const V* lds_ptr;
    return *(lds_ptr)(static_cast<std::uintptr_t>(at));
}

__device__ __forceinline__ u32 lds_address(const char* p)
{
    return static_cast<u32>(reinterpret_cast<std::uintptr_t>((__attribute__((address_space(3))) const char*)p));
}

// read row `row` at step s: row_address ^ (32 s)
template <int DP>
__device__ __forceinline__ u32 row_address(const char* tile, u32 row)
{
    return lds_address(tile) + tile_chunk<DP>(row, (threadIdx.x & 63) / 32);
}

// read the transposed step s at block n: column_address(0) ^ (64 n) and column_address(8) ^ (64 n), both
// plus 16 s rows
template <int DP>
__device__ __forceinline__ u32 column_address(const char* tile, u32 second)
{
    const u32 lane = threadIdx.x & 63;
    const u32 row = 4 * (lane / 32) + (lane % 16) / 4 + second;
    return lds_address(tile) + tile_chunk<DP>(row, 2 * ((lane / 16) % 2) + (lane % 4) / 2) + 8 * (lane % 2);
}

__device__ __forceinline__ vuint4 read_column(u32 first, u32 second)
{
    typedef __attribute__((address_space(3))) vshort4* lds_ptr;
    const vuint2 lo = __builtin_bit_cast(vuint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(static_cast<std::uintptr_t>(first))));
    const vuint2 hi = __builtin_bit_cast(vuint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(static_cast<std::uintptr_t>(second))));
    return vuint4{lo.x, lo.y, hi.x, hi.y};
}

// Between LDS writes and reads that lanes of one wave exchange: no instruction, an order for the compiler.
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

// ---- rows and states --------------------------------------------------------------------------

// a value that all lanes hold, in a scalar register
__device__ __forceinline__ u32 uniform(u32 x)
{
    return static_cast<u32>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
}

// The states [0, count) of sequence b
__device__ __forceinline__ u32 state_count(const attention_args& a, u32 b)
{
    if (a.counts == nullptr)
    {
        return a.states;
    }
    const std::int32_t c = a.counts[b];
    return c <= 0 ? 0 : (static_cast<u32>(c) < a.states ? static_cast<u32>(c) : a.states);
}

// Row r of the rows that read state head `head` of sequence b: the query heads of the group one after
// the other, so that the row's place among the log-sum-exps is (b * state_heads + head) * rows + r.
__device__ __forceinline__ std::int64_t row_offset(const rows_view& v, const attention_args& a, u32 b, u32 head, u32 r)
{
    const u32 in_group = r / a.queries_per_head;
    const u32 position = r - in_group * a.queries_per_head;
    return b * v.batch_stride + static_cast<std::int64_t>(head * static_cast<u32>(a.group) + in_group) * v.head_stride +
           position * v.row_stride;
}

// Workgroups are dealt to the eight dies in turn, and each die has an L2 of its own: neighbours in
// the returned order, which read the same states, land on one die.
__device__ __forceinline__ u32 die_order(u32 block, u32 total)
{
    constexpr u32 DIES = 8;
    const u32 die = block % DIES;
    const u32 base = total / DIES;
    const u32 rest = total % DIES;
    return die * base + (die < rest ? die : rest) + block / DIES;
}

} // namespace
} // namespace bitsknn

#endif // BITSKNN_CSRC_ATTENTION_HPP_
