// Building blocks of the attention kernels (packed and paged): 16-bit operand types and their matrix
// instruction, staging of rows into LDS, fragment reads in both directions, and the map from a workgroup to its
// tile of a ragged batch.
//
// Matrix instruction: 32x32x16, f32 accumulators.  Lane l = 32 h + c holds of the A operand row c, of the B
// operand column c, at contraction indices 8 h .. 8 h + 7; of the result column c, rows acc_row(r, h), r < 16.
// A contraction may run over its index in any order that both operands share.  Products are arranged so that
// the softmax axis of a result lies in a lane's own registers and the result feeds the next product as its B
// operand as it stands: step s of 16 contraction indices takes registers 8 s .. 8 s + 7, which are rows
// 16 s + 4 h + {0..3} and 16 s + 8 + 4 h + {0..3}; the A operand is read in that order (read_columns).
#pragma once

#include "common.hpp"
#include "../../include/lcpp_hip.h"

namespace lcpp_hip {
namespace attention {

using F32x16 = float __attribute__((ext_vector_type(16)));
using F32x4 = float __attribute__((ext_vector_type(4)));
using F32x2 = float __attribute__((ext_vector_type(2)));
using U32x4 = uint32_t __attribute__((ext_vector_type(4)));
using U32x2 = uint32_t __attribute__((ext_vector_type(2)));
using S16x4 = short __attribute__((ext_vector_type(4)));

// kNarrow: exponents are too few for what products make as it comes, and operands are taken times powers of two.
struct Bf16 {
    static constexpr bool kNarrow = false;
    using Item = __bf16;
    using Vec2 = Item __attribute__((ext_vector_type(2)));
    using Vec8 = Item __attribute__((ext_vector_type(8)));
    __device__ static F32x16 mfma(U32x4 a, U32x4 b, F32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Vec8, a), __builtin_bit_cast(Vec8, b), c, 0, 0, 0);
    }
};

struct F16 {
    static constexpr bool kNarrow = true;
    using Item = _Float16;
    using Vec2 = Item __attribute__((ext_vector_type(2)));
    using Vec8 = Item __attribute__((ext_vector_type(8)));
    __device__ static F32x16 mfma(U32x4 a, U32x4 b, F32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(Vec8, a), __builtin_bit_cast(Vec8, b), c, 0, 0, 0);
    }
};

// Two floats rounded to nearest even, in one word.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const F32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, typename T::Vec2));
}

template <typename T>
__device__ __forceinline__ float item_low(uint32_t w) {
    return static_cast<float>(__builtin_bit_cast(typename T::Vec2, w)[0]);
}
template <typename T>
__device__ __forceinline__ float item_high(uint32_t w) {
    return static_cast<float>(__builtin_bit_cast(typename T::Vec2, w)[1]);
}

// The sum of eight products of 16-bit items.
template <typename T>
__device__ __forceinline__ float dot8(U32x4 a, U32x4 b) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sum += item_low<T>(a[i]) * item_low<T>(b[i]);
        sum += item_high<T>(a[i]) * item_high<T>(b[i]);
    }
    return sum;
}

// Row of a 32x32 result that register r of a lane in half h holds.
__device__ __forceinline__ constexpr int acc_row(int r, int h) { return 8 * (r / 4) + 4 * h + r % 4; }

// Registers 8 s .. 8 s + 7 of a result, rounded to 16 bits: the B operand of contraction step s.
template <typename T>
__device__ __forceinline__ U32x4 pack_step(const F32x16& p, int s) {
    return U32x4{pack2<T>(p[8 * s + 0], p[8 * s + 1]), pack2<T>(p[8 * s + 2], p[8 * s + 3]),
                 pack2<T>(p[8 * s + 4], p[8 * s + 5]), pack2<T>(p[8 * s + 6], p[8 * s + 7])};
}

// Whether any of a lane's sums is an infinity or NaN.
template <int N>
__device__ __forceinline__ bool any_not_finite(const F32x16 (&acc)[N]) {
    float zero = 0.f;
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) zero += acc[d][r] * 0.f;
    return !(zero == 0.f);
}

// A value of this lane and of the lane 32 away: the lower lane's first.  (The two words are copied out before they are
// reinterpreted: a bit cast of a vector's element would take its first.)
struct Halves {
    float low, high;
};
__device__ __forceinline__ Halves halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t low = r[0], high = r[1];
    return {__builtin_bit_cast(float, low), __builtin_bit_cast(float, high)};
}
__device__ __forceinline__ float halves_max(float x) {
    const Halves h = halves(x);
    return fmaxf(h.low, h.high);
}
__device__ __forceinline__ float halves_sum(float x) {
    const Halves h = halves(x);
    return h.low + h.high;
}

// (An ulp or so; results below the least normal number are 0, which is 2^-126 of a row's largest weight.)
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr uint64_t kMostKeys = 0x7FFFF000;  // of a sequence: a few tiles below what a position may be

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Rows of 16-bit items: one of a [tokens][heads][dim] array with the last axis contiguous.
struct Rows {
    char* data;
    int64_t token_bytes;
    int64_t head_bytes;
    __device__ __forceinline__ char* at(int64_t token, int head) const {
        return data + token * token_bytes + static_cast<int64_t>(head) * head_bytes;
    }
};

// Rows of a paged cache: [pages][page size][heads][dim] in any order of the first three axes.
struct Pages {
    char* data;
    int64_t page_bytes;
    int64_t token_bytes;
    int64_t head_bytes;
    __device__ __forceinline__ char* at(int64_t page, int64_t slot, int head) const {
        return data + page * page_bytes + slot * token_bytes + static_cast<int64_t>(head) * head_bytes;
    }
};

// Division of 32-bit numbers by one that the host knows, without the compiler's twenty-odd instructions: with l the least
// power that 2^l >= d and m = floor(2^32 (2^l - d) / d) + 1, x / d = (t + (x - t) / 2) / 2^(l - 1) where t is the high word
// of m x (Granlund and Montgomery, "Division by invariant integers using multiplication"); d = 1 takes no shift.
struct Divider {
    uint32_t by, factor, shift1, shift2;
    explicit Divider(uint32_t d) : by(d) {
        uint32_t l = 0;
        while (l < 32 && (uint64_t{1} << l) < d) ++l;
        factor = static_cast<uint32_t>((uint64_t{1} << 32) * ((uint64_t{1} << l) - d) / d + 1);
        shift1 = l < 1 ? 0 : 1;
        shift2 = l < 1 ? 0 : l - 1;
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const {
        const uint32_t t = __umulhi(factor, x);
        return (t + ((x - t) >> shift1)) >> shift2;
    }
};

// What the 16-byte loads and stores of rows need.
inline bool usable(const lcpp_hip_rows* r) {
    return r != nullptr && r->data != nullptr && reinterpret_cast<uintptr_t>(r->data) % 16 == 0 && r->token_stride >= 0 &&
           r->head_stride >= 0 && r->token_stride % 8 == 0 && r->head_stride % 8 == 0;
}
inline bool usable(const lcpp_hip_pages* c) {
    return c != nullptr && c->data != nullptr && reinterpret_cast<uintptr_t>(c->data) % 16 == 0 && c->page_stride >= 0 &&
           c->token_stride >= 0 && c->head_stride >= 0 && c->page_stride % 8 == 0 && c->token_stride % 8 == 0 &&
           c->head_stride % 8 == 0;
}
inline int unusable(const char* what) {
    return set_error(kInvalidArgument, "%s: rows must be there and 16-byte aligned, their strides multiples of 8 items", what);
}
inline Rows rows_of(const lcpp_hip_rows* r) { return {static_cast<char*>(r->data), r->token_stride * 2, r->head_stride * 2}; }
inline Pages pages_of(const lcpp_hip_pages* c) {
    return {static_cast<char*>(c->data), c->page_stride * 2, c->token_stride * 2, c->head_stride * 2};
}

// A tile of rows in LDS: DP items a row (the head size rounded up; zeros past it), in chunks of 16 bytes, with room for 64
// or 128 items.  A wave's direct load writes 64 chunks in lane order: 4 rows of 128 items, or 8 of 64.  Within these four
// chunks of a row lie side by side (64 bytes that a load reads together), then the same four of the next row; and from one
// 4 rows to the next a chunk moves by 16 bytes, by padding or by exchanging neighbours.  So the same chunk of 16 rows (a
// read along rows), and four chunks of four rows (a transposed read), fill the 64 banks of 4 bytes once; and a lane's
// addresses in one tile differ by constants.
template <int DP>
struct Tile {
    static_assert(DP % 32 == 0 && DP <= 128);
    static constexpr bool kWide = DP > 64;
    static constexpr int kBlockRows = kWide ? 4 : 8;
    static constexpr int kBlockBytes = 1024 + (kWide ? 16 : 32);
    static constexpr int bytes(int rows) { return rows / kBlockRows * kBlockBytes; }
    __device__ __forceinline__ static int place(int row, int chunk) {
        const int group = kWide ? 0 : row / 4 % 2;
        return row / kBlockRows * kBlockBytes + group * 512 + chunk / 4 * 256 + row % 4 * 64 + (chunk % 4 ^ group) * 16;
    }
    // The row of its block and the chunk that a lane's direct load writes.
    __device__ __forceinline__ static int lane_row(int lane) { return (kWide ? 0 : lane / 32 * 4) + lane % 16 / 4; }
    __device__ __forceinline__ static int lane_chunk(int lane) {
        return kWide ? lane / 16 * 4 + lane % 4 : lane / 16 % 2 * 4 + (lane % 4 ^ lane / 32);
    }
};

// Contraction step s of row c (A operand of 32 rows from `row0`, a multiple of 16): 8 items at 16 s + 8 h.
template <int DP>
__device__ __forceinline__ U32x4 read_rows(const char* tile, int row0, int s) {
    const int lane = threadIdx.x % kWave;
    const char* p = tile + Tile<DP>::place(lane % 32, lane / 32);
    return *reinterpret_cast<const U32x4*>(p + Tile<DP>::bytes(row0) + s / 2 * 256 + s % 2 * 32);
}

// A operand of the transposed tile: 32 columns from `col0`, contraction over the 16 rows from `row0` (a multiple of 16)
// in the order of pack_step.  A transposed read hands each of 16 lanes the four items of its column from four rows.
template <int DP>
__device__ __forceinline__ U32x4 read_columns(const char* tile, int row0, int col0) {
    using LdsPtr = __attribute__((address_space(3))) S16x4*;
    const int lane = threadIdx.x % kWave;
    // One offset, which the compiler does not take apart: behind more than a few steps of address arithmetic it no longer knows
    // which array is read, and waits for the loads into all of them.
    int at = Tile<DP>::place(4 * (lane / 32) + lane % 16 / 4, 2 * (lane / 16 % 2) + lane % 4 / 2) + lane % 2 * 8;
    asm("" : "+v"(at));
    const char* p = tile + at + (Tile<DP>::bytes(row0) + col0 / 32 * 256);
    const S16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(p));
    const S16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(p + Tile<DP>::bytes(8)));
    const U32x2 x = __builtin_bit_cast(U32x2, a), y = __builtin_bit_cast(U32x2, b);
    return U32x4{x[0], x[1], y[0], y[1]};
}

// 16 bytes of a row, or zeros past the row's items or for a row that is not there.
__device__ __forceinline__ U32x4 load_chunk(const char* row, int chunk, int dim, bool there) {
    U32x4 v = {0u, 0u, 0u, 0u};
    if (there && chunk * 8 < dim) v = *reinterpret_cast<const U32x4*>(row + chunk * 16);
    return v;
}

// Places of a ragged batch's tiles.  Sequence b with rows [offsets[b], offsets[b + 1]) has its tiles of `size` rows
// from number offsets[b] / size + b on: numbers never collide, because floor(x / size) + 1 more tiles than any
// sequence of x rows needs are set aside, and there are at most total / size + count of them.  The tile's owner is
// the last b whose first number is not above it; a number past its owner's rows has no tile.
struct TilePlace {
    int sequence;
    int tile;
};

// The last of `count` ascending numbers that is not above `number` (-1: none): a wave tests 64 at a time.
template <typename Number, typename Key>
__device__ __forceinline__ int find_last(int count, Number number, Key key) {
    const int lane = threadIdx.x % kWave;
    int low = 0, high = count;
    while (high - low > 0) {
        const int step = (high - low + kWave - 1) / kWave;
        const int at = low + lane * step;
        const int passed = __popcll(wave_ballot(at < high && key(at) <= number));
        if (passed == 0) return -1;
        low += (passed - 1) * step;
        if (step == 1) break;
        high = low + step < high ? low + step : high;
    }
    return __builtin_amdgcn_readfirstlane(low);
}

// (Offsets that do not ascend from 0 give wrong tiles, but none before a sequence's first row.)
__device__ __forceinline__ TilePlace find_tile(const int32_t* offsets, int count, int scale, int size, int number) {
    const auto first = [&](int b) { return static_cast<int64_t>(offsets[b] > 0 ? offsets[b] : 0) * scale / size + b; };
    const int owner = find_last<int64_t>(count, number, first);
    const int64_t tile = owner < 0 ? -1 : number - first(owner);
    return {tile < 0 ? -1 : owner, static_cast<int>(tile)};
}

}  // namespace attention
}  // namespace lcpp_hip
