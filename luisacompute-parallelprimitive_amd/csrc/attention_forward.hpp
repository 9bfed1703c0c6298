// The loop over keys that the packed forward kernel and the paged kernel for many rows share.
//
// A wave holds 32 query rows as B operands.  S^T = K Q^T leaves a row's scores in two lanes' registers (32 keys apart
// in halves), so the running maximum and sum cost one lane exchange a tile, and the weights go into O^T = V^T P^T as
// they stand.  Tiles of 64 keys are loaded straight into LDS, one ahead of the one in use.
#pragma once

#include "attention.hpp"

namespace lcpp_hip {
namespace attention {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr int kRowsPerWave = 32;
constexpr int kRowTile = kWaves * kRowsPerWave;  // query rows of a workgroup
constexpr int kKeyTile = 64;                     // keys in LDS at a time
// The running maximum that scales the sums follows the true one only when a row has outgrown it by this (as an exponent
// of 2): weights are then at most 2^8, within the 16-bit types, and the products are rescaled a few times a row at most
// (16,384 rows: 1,138 us, with a slack of 0 1,180; uneven prompts 157 and 165).
constexpr float kSlack = 8.f;
// Weights are taken times 2^kRaise, in f16 as far as the slack leaves room below 2^16: its normal numbers end at 2^-14, and a long
// row's many small weights would be rounded away or up together (100,000 keys e^-17 below one: the output was 9% off).  The
// factor is in the products and in their sum alike, and out of the latter for the lse.
template <typename T>
constexpr int kRaise = T::kNarrow ? 7 : 0;

// Direct loads of a tile by some waves side by side, a block of rows each: a lane's chunk is the same in all of them, and its
// row goes up by kRowStep.
template <int DP, int ROWS, int WAVES = kWaves>
struct TileLoads {
    static constexpr int kRowStep = WAVES * Tile<DP>::kBlockRows;
    static constexpr int kPerWave = ROWS / kRowStep;
    static_assert(kPerWave > 0 && ROWS % kRowStep == 0);
    __device__ __forceinline__ static int row() {
        return threadIdx.x % (WAVES * kWave) / kWave * Tile<DP>::kBlockRows + Tile<DP>::lane_row(threadIdx.x % kWave);
    }
    __device__ __forceinline__ static int chunk() { return Tile<DP>::lane_chunk(threadIdx.x % kWave); }
    __device__ __forceinline__ static char* place(char* tile, int i) {
        return tile + (i * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x % (WAVES * kWave) / kWave)) * Tile<DP>::kBlockBytes;
    }
};

__device__ __forceinline__ void load_to_lds(const char* from, char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)(from),
                                     (__attribute__((address_space(3))) uint32_t*)(to), 16, 0, 0);
}

// Zeros where a row of fewer items than DP has none; loads never touch those chunks.
template <int DP, int ROWS, int WAVES = kWaves>
__device__ __forceinline__ void clear_past(char* tile, int dim) {
    using Loads = TileLoads<DP, ROWS, WAVES>;
    if (Loads::chunk() * 8 < dim) return;
#pragma unroll
    for (int i = 0; i < Loads::kPerWave; ++i)
        *reinterpret_cast<U32x4*>(Loads::place(tile, i) + threadIdx.x % kWave * 16) = U32x4{0u, 0u, 0u, 0u};
}

// Rows of a packed sequence: those past its last are loaded as its last, and masked.  Addresses are a scalar base and a
// lane's offset of 32 bits without a sign, which stays the same from tile to tile: rows are less than 2^25 bytes apart (the host
// sees to it), and a tile has 128 of them at most, so that the last one's chunks begin below 127 * 2^25 + 256 < 2^32.
template <int DP, int ROWS, int WAVES = kWaves>
struct PackedRows {
    static_assert(ROWS <= 128, "a lane's offset within a tile has 32 bits");
    using Loads = TileLoads<DP, ROWS, WAVES>;
    const char* base;  // the sequence's first row of the head
    int64_t token_bytes;
    int size;
    uint32_t offset;
    bool has;
    __device__ __forceinline__ PackedRows(const char* first, int64_t bytes, int rows, int dim)
        : base(first), token_bytes(bytes), size(rows),
          offset(static_cast<uint32_t>(Loads::row()) * static_cast<uint32_t>(bytes) + Loads::chunk() * 16u),
          has(Loads::chunk() * 8 < dim) {}
    __device__ __forceinline__ void load(char* tile, int row0, int64_t more = 0) const {
        if (!has) return;
        const char* from = base + more + row0 * token_bytes;
        if (row0 + ROWS <= size) {
#pragma unroll
            for (int i = 0; i < Loads::kPerWave; ++i)
                load_to_lds(from + i * Loads::kRowStep * token_bytes + offset, Loads::place(tile, i));
        } else {
            const int last = size - 1 - row0;
#pragma unroll
            for (int i = 0; i < Loads::kPerWave; ++i) {
                int row = Loads::row() + i * Loads::kRowStep;
                row = row < last ? row : last;
                const uint32_t at = static_cast<uint32_t>(row) * static_cast<uint32_t>(token_bytes) + Loads::chunk() * 16u;
                load_to_lds(from + at, Loads::place(tile, i));
            }
        }
    }
};

// What a lane has for its row.
template <int DP>
struct RowState {
    F32x16 acc[DP / 32];
    float top;    // the scale of acc and total: at most kSlack / c below the largest score so far
    float total;  // of the lane's half of the keys
};

// Keys from k0 on that a row sees, when it sees the first `count` of its sequence.
__device__ __forceinline__ uint32_t first_keys(int count, int k0) {
    const int n = count - k0;
    return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
}

// Writes column `lane % 32` of a transposed result (rows are items of the head) times `factor`.
template <typename T, int DP>
__device__ __forceinline__ void store_row(const Rows& dst, int64_t token, int head, const F32x16 (&acc)[DP / 32], float factor,
                                          int dim) {
    const int half = threadIdx.x % kWave / 32;
    char* row = dst.at(token, head);
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = b * 32 + 8 * g + 4 * half;
            if (d >= dim) continue;
            const U32x2 v = {pack2<T>(acc[b][4 * g] * factor, acc[b][4 * g + 1] * factor),
                             pack2<T>(acc[b][4 * g + 2] * factor, acc[b][4 * g + 3] * factor)};
            *reinterpret_cast<U32x2*>(row + d * 2) = v;
        }
    }
}

// Moves the row's scale up to `high`, the largest score of the coming keys, where that has outgrown it.
template <int DP>
__device__ __forceinline__ void rescale(RowState<DP>& state, float high, float c) {
    const bool outgrown = (high - state.top) * c > kSlack;  // (from -inf: yes, unless the row still sees nothing)
    if (wave_ballot(outgrown) == 0) return;
    const float top = outgrown ? high : state.top;
    const float alpha = outgrown ? exp2_fast((state.top - top) * c) : 1.f;
    state.top = top;
    state.total *= alpha;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) state.acc[d] *= alpha;
}

// What a score's exponent is taken from (a row that sees nothing has no scale: its scores are -inf).
template <typename T>
__device__ __forceinline__ float weight_base(float top, float c) {
    return top == -INFINITY ? 0.f : top * c - kRaise<T>;
}

// One tile of keys.  `seen(k0)`: the 32 keys from k0 on that the lane's row sees, as bits; `masked`: some row of the
// workgroup does not see all of the tile.
template <typename T, int DP, typename Seen>
__device__ __forceinline__ void forward_tile(RowState<DP>& state, const char* k_tile, const char* v_tile, const U32x4 (&qf)[DP / 16],
                                             float c, int k0, bool masked, Seen seen) {
    constexpr int kBlocks = kKeyTile / 32;
    const int half = threadIdx.x % kWave / 32;
    F32x16 s[kBlocks] = {};
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) s[b] = T::mfma(read_rows<DP>(k_tile, b * 32, i), qf[i], s[b]);
    if (masked) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const uint32_t word = seen(k0 + 32 * b) >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] = word & (1u << acc_row(r, 0)) ? s[b][r] : -INFINITY;
        }
    }
    float high = s[0][0];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) high = fmaxf(high, s[b][r]);
    rescale(state, halves_max(high), c);
    const float base = weight_base<T>(state.top, c);
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[b][r] = exp2_fast(s[b][r] * c - base);
            sum += s[b][r];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const U32x4 p = pack_step<T>(s[b], i);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
                state.acc[d] = T::mfma(read_columns<DP>(v_tile, b * 32 + i * 16, d * 32), p, state.acc[d]);
        }
    }
    state.total += sum;
}

// Infinities and NaN in masked places.  A masked weight is zero, but zero times an infinity or NaN is NaN: in a tile of keys
// that only some rows see, the matrix product carries such a value to the others.  The kernels do not look for them (the
// guards in every tile's products cost a third of the registers): a wave whose sums come out as anything but finite numbers
// takes the tiles that all of its rows see again, and then the other keys without matrix instructions, one at a time, where
// a row adds only what it sees.  A lane keeps the row and the items of it that it has in the matrix products.

// Dot products of the lane's row (a B operand, half its items in each of two lanes) with one row of memory that the
// whole wave reads.
template <typename T, int DP, typename Operand>
__device__ __forceinline__ float careful_dot(Operand operand, const char* row, int dim) {
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        sum += dot8<T>(operand(s), load_chunk(row, 2 * s + threadIdx.x % kWave / 32, dim, true));
        if (s % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // four loads in flight: more would spill
    }
    return halves_sum(sum);
}

// acc += weight * the row, where `seen`.
template <typename T, int DP>
__device__ __forceinline__ void careful_add(F32x16 (&acc)[DP / 32], float weight, const char* row, int dim, bool seen) {
    const int half = threadIdx.x % kWave / 32;
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {
        const int d = 8 * i + 4 * half;
        if (8 * i >= dim || !seen) continue;
        const U32x2 v = *reinterpret_cast<const U32x2*>(row + d * 2);
        acc[i / 4][4 * (i % 4) + 0] += weight * item_low<T>(v[0]);
        acc[i / 4][4 * (i % 4) + 1] += weight * item_high<T>(v[0]);
        acc[i / 4][4 * (i % 4) + 2] += weight * item_low<T>(v[1]);
        acc[i / 4][4 * (i % 4) + 3] += weight * item_high<T>(v[1]);
        if (i % 8 == 7) __builtin_amdgcn_sched_barrier(0);
    }
}

// Whether any wave of the workgroup has `found`; `flag` was cleared before an earlier barrier.  Waits for LDS only, not
// for stores to memory that are on their way (__syncthreads_or in its place: 155 -> 162 us for 16 uneven prompts).
__device__ __forceinline__ bool block_any(bool found, int* flag) {
    if (wave_ballot(found) != 0 && threadIdx.x % kWave == 0) *flag = 1;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    return *flag != 0;
}

// The kernel's only argument, read again: what a rarely taken path needs of it then takes no registers of the usual one.
template <typename Args>
__device__ __forceinline__ Args arguments_again() {
    static_assert(sizeof(Args) % 4 == 0);
    struct Words {
        uint32_t word[sizeof(Args) / 4];
    } words;
    const auto* from = (const __attribute__((address_space(4))) uint32_t*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(from));
#pragma unroll
    for (unsigned i = 0; i < sizeof(Args) / 4; ++i) words.word[i] = from[i];
    return __builtin_bit_cast(Args, words);
}

// The end of the tiles from `begin` on that every row sees, when they see all keys below `full` of those below `end`.
__device__ __forceinline__ int clean_end(int begin, int full, int end) {
    return full < end ? begin + (full - begin) / kKeyTile * kKeyTile : end;
}

// One key for the lane's row; the whole wave has the same.
template <typename T, int DP>
__device__ __forceinline__ void careful_key(RowState<DP>& state, const U32x4 (&qf)[DP / 16], const char* key, const char* value,
                                            int dim, float c, bool seen) {
    const float dot = careful_dot<T, DP>([&](int i) { return qf[i]; }, key, dim), score = seen ? dot : -INFINITY;
    rescale(state, score, c);
    const float weight = exp2_fast(score * c - weight_base<T>(state.top, c));
    if (threadIdx.x % kWave < 32) state.total += weight;
    careful_add<T, DP>(state.acc, weight, value, dim, seen);
}

// (The hardware's logarithm, right to an ulp or so, as the sum it is taken of.)
template <typename T>
__device__ __forceinline__ float row_lse(float top, float total, float scale) {
    return total == 0.f ? -INFINITY : top * scale + __logf(ldexpf(total, -kRaise<T>));
}

// Runs the tiles from `begin` to `end`, SIZE apart, with two sets of buffers: while one is computed on, the other is loaded.
// The sets are distinct arrays, so that reads of one do not wait for loads of the other.
template <int SIZE, typename LoadEven, typename LoadOdd, typename StepEven, typename StepOdd>
__device__ __forceinline__ void pass_tiles(int begin, int end, LoadEven load_even, LoadOdd load_odd, StepEven step_even,
                                           StepOdd step_odd) {
    if (begin >= end) return;
    load_even(begin);
    __syncthreads();
    for (int at = begin;; at += 2 * SIZE) {
        if (at + SIZE < end) load_odd(at + SIZE);
        step_even(at);
        if (at + SIZE >= end) break;
        __syncthreads();
        if (at + 2 * SIZE < end) load_even(at + 2 * SIZE);
        step_odd(at + SIZE);
        if (at + 2 * SIZE >= end) break;
        __syncthreads();
    }
}

// All keys in [begin, end), whose tiles the workgroup's waves load together.  Tiles that pass `full` are masked; a wave
// whose rows see nothing from `wave_end` on leaves the rest to the others.
template <typename T, int DP, typename Keys, typename Seen>
__device__ __forceinline__ void forward_keys(RowState<DP>& state, char* k_even, char* v_even, char* k_odd, char* v_odd, const Keys& keys,
                                             const Keys& values, const U32x4 (&qf)[DP / 16], float c, int begin, int end, int wave_end,
                                             int full, Seen seen) {
    const auto load = [&](char* k_tile, char* v_tile, int k0) {
        keys.load(k_tile, k0);
        values.load(v_tile, k0);
    };
    const auto step = [&](const char* k_tile, const char* v_tile, int k0) {
        if (k0 < wave_end) forward_tile<T, DP>(state, k_tile, v_tile, qf, c, k0, k0 + kKeyTile > full, seen);
    };
    pass_tiles<kKeyTile>(begin, end, [&](int k0) { load(k_even, v_even, k0); }, [&](int k0) { load(k_odd, v_odd, k0); },
                         [&](int k0) { step(k_even, v_even, k0); }, [&](int k0) { step(k_odd, v_odd, k0); });
}

}  // namespace attention
}  // namespace lcpp_hip
