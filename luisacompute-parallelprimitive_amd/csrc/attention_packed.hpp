// What the packed forward and backward kernels share: the batch's shape, a sequence's rows and keys, what a row sees, and the
// host's checks.
#pragma once

#include "attention_forward.hpp"

namespace lcpp_hip {
namespace attention {

constexpr int kTeams = 2;  // of four waves, in the gradients' workgroups

struct Shape {
    int sequences;
    int q_tokens;
    int k_tokens;
    int q_heads;
    int kv_heads;
    int dim;
    float scale;
    int causal;
};

struct Span {
    int begin;
    int size;
};

__device__ __forceinline__ Span span_of(const int32_t* offsets, int sequence, int tokens) {
    int begin = offsets[sequence], end = offsets[sequence + 1];
    begin = begin < 0 ? 0 : begin > tokens ? tokens : begin;
    end = end < begin ? begin : end > tokens ? tokens : end;
    return {begin, end - begin};
}

// The calling lane's row as a B operand: column lane % 32, all contraction steps.
template <int DP>
__device__ __forceinline__ void load_row(U32x4 (&f)[DP / 16], const Rows& src, int64_t token, int head, bool there, int dim) {
    const char* row = src.at(there ? token : 0, head);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) f[s] = load_chunk(row, 2 * s + threadIdx.x % kWave / 32, dim, there);
}

// Keys that a row sees (the first `count`), that every row of its workgroup sees, and that any does, or any of its wave.
struct RowRange {
    int count, full, end, wave_end;
    __device__ __forceinline__ RowRange(const Shape& shape, const Span& rows, const Span& keys, int row0, int row) {
        const int shift = keys.size - rows.size + 1;
        const int last = row0 + kRowTile < rows.size ? row0 + kRowTile - 1 : rows.size - 1;
        const auto seen = [&](int r) { return !shape.causal || r + shift > keys.size ? keys.size : r + shift > 0 ? r + shift : 0; };
        count = seen(row);
        full = seen(row0);
        end = seen(last);
        const int wave_row0 = row0 + __builtin_amdgcn_readfirstlane(threadIdx.x % kBlock / kWave) * kRowsPerWave;
        const int wave_last = wave_row0 + kRowsPerWave - 1;
        wave_end = wave_row0 < rows.size ? seen(wave_last < last ? wave_last : last) : 0;
    }
};

// Tiles of a batch of at most 64 sequences in the order of the work that they are, the most first: a workgroup of a long
// sequence's last rows takes half of an uneven batch's time, and has to start early.  16 uneven prompts: 154 us in the
// tiles' order, 148 so.  Gradients of 8 sequences of 500 rows (32 heads of 128 on 8): 121 and 111 us; of six from 700 to 4,096
// rows 807 to 853, by their place in the batch, and 811 to 820.  Finding the place takes half a microsecond more, which
// is not spent where all workgroups run at once.  A lane holds a sequence; its tiles are at consecutive levels from
// `first` on, or all at that one, and the level of number `number` is found by halving.
struct OrderedTile {
    int lane;   // of its sequence, -1: none
    int index;  // how far above `first` it is, or its number among those of one level
    __device__ __forceinline__ OrderedTile(int tiles, int first, bool consecutive, int number) : lane(-1), index(0) {
        const auto from = [&](int level) {  // tiles at this level or above
            if (!consecutive) return level <= first ? tiles : 0;
            const int n = first + tiles - level;
            return n < 0 ? 0 : n < tiles ? n : tiles;
        };
        if (wave_reduce(tiles, SumOp{}) <= number) return;
        int low = -wave_reduce(tiles ? -first : -INT32_MAX, MaxValueOp{}), high = wave_reduce(tiles ? first + tiles : -INT32_MAX, MaxValueOp{});
        int above = 0;  // tiles at `high` or above: not more than number; at `low` there are more
        while (high - low > 1) {
            const int level = low + (high - low) / 2, n = wave_reduce(from(level), SumOp{});
            if (n > number) low = level;
            else high = level, above = n;
        }
        const int mine = from(low) - from(high), before = wave_inclusive_scan(mine, SumOp{}) - mine, rest = number - above - before;
        lane = __ffsll(static_cast<unsigned long long>(wave_ballot(rest >= 0 && rest < mine))) - 1;
        index = wave_read_lane(consecutive ? low - first : rest, lane);
    }
};

__device__ __forceinline__ Span read_span(const Span& s, int lane) { return {wave_read_lane(s.begin, lane), wave_read_lane(s.size, lane)}; }

// The spans of a lane's sequence.
__device__ __forceinline__ void lane_spans(const int32_t* q_offsets, const int32_t* k_offsets, const Shape& shape, Span& rows, Span& keys) {
    const int lane = threadIdx.x % kWave, sequence = lane < shape.sequences ? lane : shape.sequences - 1;
    rows = span_of(q_offsets, sequence, shape.q_tokens);
    keys = span_of(k_offsets, sequence, shape.k_tokens);
    if (lane >= shape.sequences) rows.size = keys.size = 0;
}

// A tile of SIZE rows, by the keys that it sees.
template <int SIZE>
__device__ __forceinline__ bool take_ordered_tile(const int32_t* q_offsets, const int32_t* k_offsets, const Shape& shape, int number,
                                                  Span& rows, Span& keys, int& row0) {
    Span r, k;
    lane_spans(q_offsets, k_offsets, shape, r, k);
    const int seen = shape.causal ? k.size - r.size : k.size;
    const OrderedTile tile((r.size + SIZE - 1) / SIZE, seen >= 0 ? seen / SIZE : -((SIZE - 1 - seen) / SIZE), shape.causal, number);
    if (tile.lane < 0) return false;
    rows = read_span(r, tile.lane), keys = read_span(k, tile.lane), row0 = tile.index * SIZE;
    return true;
}

// A tile of SIZE keys, by the rows that see it: the first of a causal sequence's are seen by the most.
template <int SIZE>
__device__ __forceinline__ bool take_ordered_keys(const int32_t* q_offsets, const int32_t* k_offsets, const Shape& shape, int number,
                                                  Span& rows, Span& keys, int& key0) {
    Span r, k;
    lane_spans(q_offsets, k_offsets, shape, r, k);
    const int tiles = (k.size + SIZE - 1) / SIZE;
    const OrderedTile tile(tiles, shape.causal ? 0 : r.size / SIZE, shape.causal, number);
    if (tile.lane < 0) return false;
    rows = read_span(r, tile.lane), keys = read_span(k, tile.lane);
    key0 = (shape.causal ? wave_read_lane(tiles, tile.lane) - 1 - tile.index : tile.index) * SIZE;
    return true;
}

inline int check_shape(const char* what, uint32_t sequences, uint64_t q_tokens, uint64_t k_tokens, uint32_t q_heads,
                uint32_t kv_heads, uint32_t dim, float scale) {
    if (q_heads == 0 || kv_heads == 0 || q_heads % kv_heads != 0 || q_heads > 65535)
        return set_error(kInvalidArgument, "%s: query heads must be a multiple of the key heads, and at most 65535", what);
    if (dim == 0 || dim % 8 != 0 || dim > 128)
        return set_error(kUnsupported, "%s: the head size must be a multiple of 8 up to 128", what);
    if (q_tokens > 0x7FFFFFFFull || k_tokens > kMostKeys || sequences > 0x7FFFFFFu)
        return set_error(kInvalidArgument, "%s: too many tokens or sequences", what);
    if (!(scale > 0.f) || scale == INFINITY) return set_error(kInvalidArgument, "%s: the scale must be positive and finite", what);
    return kOk;
}

// Rows so far apart that a lane's offset within a tile would not fit its 32 bits (PackedRows).
inline bool too_wide(const lcpp_hip_rows* r) { return r != nullptr && r->token_stride >= 1 << 24; }
inline int refuse_wide(const char* what) { return set_error(kUnsupported, "%s: token strides must be below 2^24 items", what); }

// Tiles that a ragged batch may have, and the launch over (tile, head).
inline int check_grid(const char* what, uint64_t tokens, int tile_rows, uint32_t sequences, uint32_t heads, unsigned& tiles,
                      unsigned& grid) {
    const uint64_t t = tokens / tile_rows + sequences;
    if (t * heads > 0x7FFFFFFFull / (kTeams * kBlock)) return set_error(kInvalidArgument, "%s: too many tiles", what);
    tiles = static_cast<unsigned>(t);
    grid = static_cast<unsigned>(t * heads);
    return kOk;
}

}  // namespace attention
}  // namespace lcpp_hip
