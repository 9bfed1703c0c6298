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

// A tile's bytes fit 31 bits.
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
