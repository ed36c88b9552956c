// Attention of few rows: the states are streamed past tiles of at most 32 rows.
#ifndef BITSKNN_CSRC_ATTENTION_STREAM_HPP_
#define BITSKNN_CSRC_ATTENTION_STREAM_HPP_

#include "attention_loader.hpp"

namespace bitsknn
{
namespace
{

constexpr u32 STREAM_WAVES = 4;
constexpr u32 STREAM_KEYS = 32; // states per tile of a wave
constexpr u32 STREAM_ROWS = 32;

// Bound by memory.  All waves of a workgroup hold the same 32 rows and take tiles of 32 states in turn,
// each for itself: no barrier until the end, where their sums are joined in LDS.  A wave's loop is a
// pipeline over its tiles: while tile t is multiplied, the vectors of t + 1 are on their way into
// registers, and so is what has to be known before the vectors of t + 2 can be asked for (mask; block,
// its count and scales; the table entry of t + 3).  The vectors pass through LDS (the wave's own part)
// to reach the operands' layout.  A wave's LDS instructions are served in order, so lanes that exchange
// values there need no barrier, only a fence that keeps the compiler from moving them.  (Heads of 136 to 256
// dimensions: the query's operands and two tiles on their way do not fit beside the sums, 141 registers are
// kept in scratch memory; 188 us, 5.7 TB/s, for 64 x 16/4 heads, one token over 4096 states x 256.)
template <typename T, int DP, bool CACHE>
__global__ void __launch_bounds__(64 * STREAM_WAVES, DP <= 128 ? 2 : 1) attention_stream_kernel(const attention_args a)
{
    using wave_type = state_loader<T, DP, CACHE, STREAM_KEYS, 64>;
    using V = typename wave_type::V;
    constexpr u32 TILE_BYTES = STREAM_KEYS * DP * 2;
    // per wave: a tile of keys and one of values; at the end the wave's sums (the same size)
    __shared__ __attribute__((aligned(16))) char lds[STREAM_WAVES * 2 * TILE_BYTES];
    __shared__ float wave_top[STREAM_WAVES][STREAM_ROWS];
    __shared__ float wave_weight[STREAM_WAVES][STREAM_ROWS];
    const u32 lane = threadIdx.x % 64;
    const u32 half = lane / 32;
    const u32 wave = uniform(threadIdx.x / 64);
    char* const keys = lds + wave * 2 * TILE_BYTES;
    char* const values = keys + TILE_BYTES;
    const u32 id = die_order(blockIdx.x, gridDim.x);
    const u32 row_tile = id % a.row_tiles;
    const u32 split = id / a.row_tiles % a.splits;
    const u32 head = id / a.row_tiles / a.splits % static_cast<u32>(a.state_heads);
    const u32 b = id / a.row_tiles / a.splits / static_cast<u32>(a.state_heads);
    const u32 row = row_tile * STREAM_ROWS + lane % 32;
    vuint4 query[DP / 16];
    load_operand<DP>(query, a.queries.data + 2 * row_offset(a.queries, a, b, head, row < a.rows ? row : 0),
                     row < a.rows, static_cast<u32>(a.dim));
    vfloat16 sum[DP / 32];
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
    {
        sum[n] = vfloat16{};
    }
    float top = -__builtin_inff();
    float weight = 0.0F;

    const u32 count = state_count(a, b);
    const u32 tiles = (count + STREAM_KEYS - 1) / STREAM_KEYS;
    const u32 end = static_cast<u32>(static_cast<u64>(tiles) * (split + 1) / a.splits);
    u32 tile = static_cast<u32>(static_cast<u64>(tiles) * split / a.splits) + wave;
    const wave_type w{a, b, head, count};
    vuint4 next_keys[wave_type::LOADS];
    vuint4 next_values[wave_type::LOADS];
    typename wave_type::place now;   // of the tile whose vectors are in the registers
    typename wave_type::place next;  // of the tile after it
    typename wave_type::place after; // its table entry only
    u32 in = 0;
    if (tile < end)
    {
        w.look_up_block(now, tile);
        w.look_up_block(next, tile + STREAM_WAVES);
        w.look_up_block(after, tile + 2 * STREAM_WAVES);
        w.look_up_state(now, tile);
        w.look_up_state(next, tile + STREAM_WAVES);
        in = w.taking_part(now, tile);
        w.template load<true>(next_keys, now, tile, in);
        w.template load<false>(next_values, now, tile, in);
    }
    for (; tile < end; tile += STREAM_WAVES)
    {
        const u32 taking = in;
        const typename wave_type::scales scales = w.ready(now, ((taking >> (lane % 32)) & 1) != 0);
        wave_fence(); // behind the reads of the tile before
        w.template put<true>(keys, next_keys, 1.0F);
        w.template put<false>(values, next_values, scales.value_scale);
        wave_fence();
        now = next;
        next.block = after.block;
        in = w.taking_part(now, tile + STREAM_WAVES);
        w.look_up_block(after, tile + 3 * STREAM_WAVES);
        w.look_up_state(next, tile + 2 * STREAM_WAVES);
        if (tile + STREAM_WAVES < end)
        {
            w.template load<true>(next_keys, now, tile + STREAM_WAVES, in);
            w.template load<false>(next_values, now, tile + STREAM_WAVES, in);
        }
        if (taking == 0)
        {
            continue;
        }
        vfloat16 score = {};
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
        {
            score = mfma<T>::run(tile_row<DP>(keys, lane % 32, s), query[s], score);
        }
        if (taking != ~0U)
        {
            const u32 bits = taking >> (4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                score[i] = ((bits >> (8 * (i / 4) + i % 4)) & 1) != 0 ? score[i] : -__builtin_inff();
            }
        }
        // the factors of the two sixteens of the tile: registers 0 .. 7 and 8 .. 15
        const float factor[2] = {CACHE ? w.of_sixteen(scales.key_factor, 0) : a.exponent_scale,
                                 CACHE ? w.of_sixteen(scales.key_factor, 1) : a.exponent_scale};
        float largest[2] = {score[0], score[8]};
#pragma unroll
        for (int i = 1; i < 8; ++i)
        {
            largest[0] = fmaxf(largest[0], score[i]);
            largest[1] = fmaxf(largest[1], score[8 + i]);
        }
        float most = fmaxf(largest[0] * factor[0], largest[1] * factor[1]);
        most = fmaxf(most, other_half(most));
        // The reference of the exponents follows the maximum only where that has grown by more than 8:
        // weights stay below 2^8, and the sums are seldom rescaled.
        if (__any(most > top + 8.0F))
        {
            asm volatile(""); // stays a branch
            most = fmaxf(most, top);
            const float shrink = __builtin_amdgcn_exp2f(top - (most == -__builtin_inff() ? 0.0F : most));
            weight *= shrink;
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
            {
                sum[n] *= shrink;
            }
            top = most;
        }
        const float base = top == -__builtin_inff() ? 0.0F : top;
        float part[2] = {0.0F, 0.0F};
#pragma unroll
        for (int g = 0; g < 2; ++g)
        {
            const float from = CACHE ? w.of_sixteen(scales.mantissa_log, g) - base : -base;
#pragma unroll
            for (int i = 8 * g; i < 8 * g + 8; ++i)
            {
                score[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[i], factor[g], from));
                part[g] += score[i];
            }
            weight = CACHE ? __builtin_fmaf(part[g], w.of_sixteen(scales.mantissa_inverse, g), weight) : weight + part[g];
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
        {
            const vuint4 p = operand<V>(score, s);
            vuint4 rest;
            if constexpr (wave_type::PIECES)
            {
                rest = operand_rest<V>(score, s, p);
            }
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
            {
                const vuint4 v = tile_column<DP>(values, s, n);
                sum[n] = mfma<V>::run(v, p, sum[n]);
                if constexpr (wave_type::PIECES)
                {
                    sum[n] = mfma<V>::run(v, rest, sum[n]);
                }
            }
        }
    }

    // the waves' sums, row by row in LDS: 32 rows of DP floats fill a wave's part
    wave_fence();
    weight += other_half(weight);
    if (half == 0)
    {
        wave_top[wave][lane] = top;
        wave_weight[wave][lane] = weight;
    }
    float* const mine = reinterpret_cast<float*>(keys);
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
    {
#pragma unroll
        for (int g = 0; g < 4; ++g)
        {
            // four columns at a time, exclusive-or'ed with the row against bank conflicts
            const u32 quad = 8 * n + 2 * g + half;
            *reinterpret_cast<vfloat4*>(mine + (lane % 32) * DP + ((quad ^ (lane % 16)) * 4)) =
                vfloat4{sum[n][4 * g], sum[n][4 * g + 1], sum[n][4 * g + 2], sum[n][4 * g + 3]};
        }
    }
    __syncthreads();
    constexpr u32 QUADS = DP / 4;
    const u32 rows = a.rows - row_tile * STREAM_ROWS < STREAM_ROWS ? a.rows - row_tile * STREAM_ROWS : STREAM_ROWS;
    for (u32 n = threadIdx.x; n < rows * QUADS; n += 64 * STREAM_WAVES)
    {
        const u32 r = n / QUADS;
        const u32 quad = n % QUADS;
        float most = wave_top[0][r];
#pragma unroll
        for (u32 v = 1; v < STREAM_WAVES; ++v)
        {
            most = fmaxf(most, wave_top[v][r]);
        }
        const float base = most == -__builtin_inff() ? 0.0F : most;
        vfloat4 total = {};
        float all = 0.0F;
#pragma unroll
        for (u32 v = 0; v < STREAM_WAVES; ++v)
        {
            const float f = __builtin_amdgcn_exp2f(wave_top[v][r] - base);
            all += f * wave_weight[v][r];
            total += f * *reinterpret_cast<const vfloat4*>(reinterpret_cast<const float*>(lds + v * 2 * TILE_BYTES) + r * DP +
                                                          ((quad ^ (r % 16)) * 4));
        }
        const u32 out_row = row_tile * STREAM_ROWS + r;
        const size_t flat = (static_cast<size_t>(b) * static_cast<u32>(a.state_heads) + head) * a.rows + out_row;
        if (a.splits > 1)
        {
            const size_t at = flat * a.splits + split;
            *reinterpret_cast<vfloat4*>(a.part + at * DP + 4 * quad) = total;
            if (quad == 0)
            {
                a.part_ml[at] = float2{most, all};
            }
            continue;
        }
        if (quad == 0 && a.lse != nullptr)
        {
            a.lse[flat] = all == 0.0F ? -__builtin_inff() : (most + __builtin_log2f(all)) * LN2;
        }
        if (4 * quad < static_cast<u32>(a.dim))
        {
            const float inverse = all == 0.0F ? 0.0F : 1.0F / all;
            *reinterpret_cast<vuint2*>(a.out.data + 2 * (row_offset(a.out, a, b, head, out_row) + 4 * quad)) =
                vuint2{pack2<T>(total[0] * inverse, total[1] * inverse), pack2<T>(total[2] * inverse, total[3] * inverse)};
        }
    }
}

} // namespace
} // namespace bitsknn

#endif // BITSKNN_CSRC_ATTENTION_STREAM_HPP_
