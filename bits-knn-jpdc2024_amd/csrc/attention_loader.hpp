// How tiles of states reach LDS: from the caller's keys and values, or from the cache's codes.
#ifndef BITSKNN_CSRC_ATTENTION_LOADER_HPP_
#define BITSKNN_CSRC_ATTENTION_LOADER_HPP_

#include "attention.hpp"

namespace bitsknn
{
namespace
{

// THREADS threads bring tiles of KEYS states of one sequence and head into LDS, in steps that the
// caller spreads over its loop so that no step waits for the one before: the table entry (cache), what
// the block holds and its scales (or the mask byte), the vectors into registers, and from there into
// LDS, the codes decoded on the way.  Lane l of every wave knows state l % KEYS of a tile.
template <typename T, int DP, bool CACHE, u32 KEYS, u32 THREADS>
struct state_loader
{
    // 16 bytes of a row per load: eight values, or sixteen codes
    static constexpr u32 PER_LOAD = CACHE ? 16 : 8;
    static constexpr u32 CHUNKS = DP / PER_LOAD; // loads per row
    static constexpr bool SPARE = KEYS * CHUNKS < THREADS; // more threads than loads
    static constexpr int LOADS = SPARE ? 1 : KEYS * CHUNKS / THREADS; // per thread and matrix
    static constexpr int SIXTEENS = KEYS / 16;
    // the cache's keys are exact in either type; its values times their scale need the range of bf16, so
    // the second product is taken in bf16 (fp16 queries: a weight as two bf16 pieces, sixteen bits, so
    // that an fp16 result loses nothing)
    using V = std::conditional_t<CACHE, __bf16, T>;
    static constexpr bool PIECES = CACHE && std::is_same_v<T, _Float16>;
    using bits = std::conditional_t<KEYS == 64, u64, u32>;

    struct place
    {
        std::int32_t block = 0; // table entry (cache)
        std::int32_t held = 0;  // states in the block (cache); mask byte
        float key_scale = 1.0F;
        float value_scale = 1.0F;
    };

    struct scales
    {
        float key_factor = 1.0F;
        float value_scale = 1.0F; // its power of two counts
        float mantissa_log = 0.0F;
        float mantissa_inverse = 1.0F;
    };

    const attention_args& a;
    const u32 b;
    const u32 head;
    const u32 count;

    __device__ __forceinline__ u32 my_state(u32 tile) const { return tile * KEYS + threadIdx.x % KEYS; }

    // first step of the look-up: the table entry
    __device__ __forceinline__ void look_up_block(place& p, u32 tile) const
    {
        if constexpr (CACHE)
        {
            const u32 j = my_state(tile);
            p.block = -1;
            if (j < count)
            {
                p.block = a.cache.table[static_cast<std::int64_t>(b) * a.cache.table_stride + (j >> a.cache.block_shift)];
            }
        }
    }

    // second step: what the block holds, or the mask
    __device__ __forceinline__ void look_up_state(place& p, u32 tile) const
    {
        const u32 j = my_state(tile);
        p.held = 0;
        p.key_scale = 1.0F;
        p.value_scale = 1.0F;
        if constexpr (CACHE)
        {
            const u32 id = static_cast<u32>(p.block);
            if (id < a.cache.blocks)
            {
                const size_t at = static_cast<size_t>(id) * static_cast<u32>(a.state_heads) + head;
                p.held = a.cache.block_counts[id];
                p.key_scale = a.cache.key_scales[at];
                p.value_scale = a.cache.value_scales[at];
            }
        }
        else if (j < count)
        {
            p.held = a.mask == nullptr ? 1 : a.mask[static_cast<std::int64_t>(b) * a.mask_stride + j];
        }
    }

    // bit l: state l of the tile takes part
    __device__ __forceinline__ bits taking_part(const place& p, u32 tile) const
    {
        const u32 j = my_state(tile);
        bool in = j < count;
        if constexpr (CACHE)
        {
            in = in && static_cast<u32>(p.block) < a.cache.blocks &&
                 static_cast<std::int32_t>(j & ((1U << a.cache.block_shift) - 1)) < p.held;
        }
        else
        {
            in = in && p.held != 0;
        }
        return static_cast<bits>(__ballot(in));
    }

    static __device__ __forceinline__ float of_sixteen(float x, int g)
    {
        return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 16 * g));
    }

    // A lane's scales, ready for use.  States that take part are a block's first ones, so the first of a
    // sixteen has the scales of all that do; where it takes no part they are 1.  A key's scale
    // multiplies the factor from scores to exponents (at least the least normal number: a masked score
    // of -inf stays one; at most the largest: a score of zero stays one).  Of a value's scale the power of two goes into the decoded values, exactly
    // (bf16 has the exponents), and the mantissa into the exponents of the weights; the sum of weights
    // takes it out again.
    __device__ __forceinline__ scales ready(const place& p, bool in) const
    {
        scales s;
        if constexpr (CACHE)
        {
            const float key = in ? p.key_scale * a.exponent_scale : 1.0F;
            s.key_factor = key < 1.17549435e-38F ? 1.17549435e-38F : (key > 3.402823466e38F ? 3.402823466e38F : key);
            s.value_scale = in ? p.value_scale : 1.0F;
            const float mantissa =
                __builtin_bit_cast(float, (__builtin_bit_cast(u32, s.value_scale) & 0x007FFFFFU) | 0x3F800000U);
            s.mantissa_log = __builtin_amdgcn_logf(mantissa);
            s.mantissa_inverse = __builtin_amdgcn_rcpf(mantissa);
        }
        return s;
    }

    // The tile's vectors into registers: neighbouring threads take neighbouring chunks of a row.  What
    // takes no part is zero.
    template <bool KEY>
    __device__ __forceinline__ void load(vuint4 (&x)[LOADS], const place& p, u32 tile, bits in) const
    {
        const u32 t = threadIdx.x % THREADS;
        const u32 chunk = t % CHUNKS;
        const u32 dim = static_cast<u32>(a.dim);
        const char* base = nullptr;
        u32 stride = dim;
        if constexpr (!CACHE)
        {
            const rows_view& v = KEY ? a.keys : a.values;
            base = v.data + 2 * (b * v.batch_stride + head * v.head_stride +
                                 static_cast<std::int64_t>(tile) * KEYS * v.row_stride);
            stride = 2 * static_cast<u32>(v.row_stride);
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
        {
            u32 row = (static_cast<u32>(i) * THREADS + t) / CHUNKS;
            bool wanted = chunk * PER_LOAD < dim;
            if constexpr (SPARE)
            {
                wanted = wanted && row < KEYS;
            }
            const char* from = base;
            if constexpr (CACHE)
            {
                // the rows of a wave's load are of one sixteen, and a block holds whole sixteens; an
                // entry that names no block is never followed: none of its states takes part
                const int g = __builtin_amdgcn_readfirstlane(static_cast<int>(row / 16)) % SIXTEENS;
                const u32 id = static_cast<u32>(__builtin_amdgcn_readlane(p.block, 16 * g));
                const u32 within = (tile * KEYS + 16 * static_cast<u32>(g)) & ((1U << a.cache.block_shift) - 1);
                from = reinterpret_cast<const char*>(KEY ? a.cache.key_codes : a.cache.value_codes) +
                       (((static_cast<size_t>(id) * static_cast<u32>(a.state_heads) + head) << a.cache.block_shift) + within) * dim;
                wanted = wanted && ((in >> (row % KEYS)) & 1) != 0;
                row %= 16;
            }
            else
            {
                wanted = wanted && ((in >> (row % KEYS)) & 1) != 0;
            }
            x[i] = vuint4{0, 0, 0, 0};
            if (wanted)
            {
                const char* at = from + (row * stride + chunk * 16);
                if constexpr (CACHE)
                {
                    // the dimensions are whole eights: the last load of a row may be half a one
                    const vuint2 lo = reinterpret_cast<const vuint2*>(at)[0];
                    vuint2 hi = {0, 0};
                    if (chunk * 16 + 8 < dim)
                    {
                        hi = reinterpret_cast<const vuint2*>(at)[1];
                    }
                    x[i] = vuint4{lo.x, lo.y, hi.x, hi.y};
                }
                else
                {
                    x[i] = *reinterpret_cast<const vuint4*>(at);
                }
            }
        }
    }

    // Decoded codes are two chunks per load: a row's even chunks are written by one instruction, the odd ones
    // by the next, and two neighbouring rows meet in the same banks then (40 % of the LDS cycles of the cache's
    // stream kernel, 15 % of its tile kernel's; neither is bound by LDS).  The caller's states meet none.
    template <bool KEY>
    __device__ __forceinline__ void put(char* tile, const vuint4 (&x)[LOADS], float scale) const
    {
        using E = std::conditional_t<KEY, T, V>;
        const u32 t = threadIdx.x % THREADS;
        const u32 chunk = t % CHUNKS;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
        {
            const u32 row = (static_cast<u32>(i) * THREADS + t) / CHUNKS;
            if (SPARE && row >= KEYS)
            {
                break;
            }
            if constexpr (CACHE)
            {
                float power = 1.0F;
                if constexpr (!KEY)
                {
                    power = of_sixteen(scale, __builtin_amdgcn_readfirstlane(static_cast<int>(row / 16)) % SIXTEENS);
                }
                *reinterpret_cast<vuint4*>(tile + tile_chunk<DP>(row, 2 * chunk)) = decode8<E>(vuint2{x[i].x, x[i].y}, power);
                *reinterpret_cast<vuint4*>(tile + tile_chunk<DP>(row, 2 * chunk + 1)) = decode8<E>(vuint2{x[i].z, x[i].w}, power);
            }
            else
            {
                *reinterpret_cast<vuint4*>(tile + tile_chunk<DP>(row, chunk)) = x[i];
            }
        }
    }
};

// A wave's 32 rows of queries in the operand layout.
template <int DP>
__device__ __forceinline__ void load_operand(vuint4 (&x)[DP / 16], const char* row, bool in, u32 dim)
{
    const u32 half = (threadIdx.x & 63) / 32;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
    {
        const u32 at = 16 * s + 8 * half;
        x[s] = vuint4{0, 0, 0, 0};
        if (in && at < dim)
        {
            x[s] = *reinterpret_cast<const vuint4*>(row + 2 * at);
        }
    }
}

// Registers 8 s .. 8 s + 7 of a product as the operand of step s, in one piece or two.
template <typename V>
__device__ __forceinline__ vuint4 operand(const vfloat16& x, int s)
{
    return vuint4{pack2<V>(x[8 * s], x[8 * s + 1]), pack2<V>(x[8 * s + 2], x[8 * s + 3]),
                  pack2<V>(x[8 * s + 4], x[8 * s + 5]), pack2<V>(x[8 * s + 6], x[8 * s + 7])};
}

// what operand `p` leaves of its values, as an operand of its own
template <typename V>
__device__ __forceinline__ vuint4 operand_rest(const vfloat16& x, int s, vuint4 p)
{
    vuint4 rest;
#pragma unroll
    for (int k = 0; k < 4; ++k)
    {
        const u32 word = p[k]; // a copy: a bit cast of an element in place reads the vector's first
        float lo;
        float hi;
        if constexpr (std::is_same_v<V, __bf16>)
        {
            lo = __builtin_bit_cast(float, word << 16);
            hi = __builtin_bit_cast(float, word & 0xFFFF0000U);
        }
        else
        {
            const auto both = __builtin_bit_cast(typename mfma<V>::v2, word);
            lo = static_cast<float>(both[0]);
            hi = static_cast<float>(both[1]);
        }
        rest[k] = pack2<V>(x[8 * s + 2 * k] - lo, x[8 * s + 2 * k + 1] - hi);
    }
    return rest;
}

} // namespace
} // namespace bitsknn

#endif // BITSKNN_CSRC_ATTENTION_LOADER_HPP_
