// Gradients of attention over packed sequences:
//
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - rowsum(dO O)),  dQ = scale dS K,  dK = scale dS^T Q,
//
// with P = exp(S - lse) taken again from the scores and the forward pass's lse.  Two roles, of which each has its sums in
// registers and one order for them, so that no atomic additions are needed: dK and dV of a tile of keys as rows pass by (four
// products), dQ of a tile of rows as keys pass by (three, two of them the same again).  Both are workgroups of one launch,
// the longer ones (keys) first: those of the other role fill the device as they end (two launches in turn: 55 us for five
// examples of up to 517 rows, one: 47).
//
// Rounded to 16 bits: P and dS, as operands of the products with 16-bit rows; and O, from which rowsum(dO O) is taken, as
// the forward pass stored it.  The last is rowsum(P dP) with O's rounding error, which a second pass over the keys would
// cost to avoid; with it dQ and dK differ from the formula by 0.3 to 0.4% of their size in bf16, where the rounding of P, dS
// and the results alone makes 0.2%.  Sums, dP and dP - rowsum are f32.
//
// 10 * dim operations a pair of row and key if S and dP were made once, 14 with both roles; bound by the matrix cores and by
// what feeds them: 11,059 tokens in six sequences (32 heads of 128 on 8) take 926 us, 865 TFLOP/s of what runs, 620 of
// what has to.  LDS holds the tiles that pass by, twice, and 128 keys' values (101 KB at 128 items: one workgroup of eight
// waves a compute unit, two waves a SIMD).  At 128 items a wave has all of its 256 registers and keeps two values in scratch memory
// over the loops.
#include "attention_packed.hpp"

namespace lcpp_hip {
namespace attention {
namespace {

// f16 holds normal numbers from 2^-14 to 2^16 only: weights of long rows are below, and dS goes with the sizes of dO and V, which
// training scales at will.  (With P and dS as they come, 3,000 rows and dO of width 1e-4: dQ 0.9% from the formula, where
// rounding the result makes 0.25%; and a dS past 65,504 was an infinity.)  So P is taken times 2^kWeightRaise, which leaves room
// for weights of 16, where the lse of very large scores is off; and dS times a power of two that a lane has for its row (dQ)
// or key (dK).  That one starts at 2^kFirstRaise and comes down with the running sums, as a softmax's scale does, whenever a
// |dS| would pass 2^15.  Both are undone in f32.  (The maxima and products cost 3% of a training step: 11,059 tokens in six
// sequences 1,206 -> 1,244 us, five short examples 46.3 -> 47.9.)
template <typename T>
constexpr int kWeightRaise = T::kNarrow ? 12 : 0;
constexpr int kFirstRaise = 32;

// By how many powers of two a lane's values, of a row or key that it shares with the lane 32 away, have to come down: none up to
// 2^15, else to 2^8, so that sums are seldom rescaled.  (Infinities stay: the sums of their row or key are not finite either.)
__device__ __forceinline__ int too_large_by(const F32x16& x) {
    float most = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(x[r]));
    most = halves_max(most);
    return most > 32768.f && most < INFINITY ? __builtin_amdgcn_frexp_expf(most) - 8 : 0;
}

// What the gradients need of a row: stats[h][t] = lse in powers of 2, less kWeightRaise (infinity for a row that saw nothing: its
// weights are then 2^-inf = 0), and behind all of those delta[h][t] = sum over the head's items of dO * O.  16 lanes a row.  Bound
// by memory (the rows of O and dO, 181 MB for 11,059 tokens of 32 heads: 34 us, 5.3 TB/s).
template <typename T>
__global__ __launch_bounds__(kBlock) void attention_row_stats_kernel(Rows out, Rows dout, const float* __restrict__ lse,
                                                                     float* __restrict__ stats, int q_tokens, int q_heads, int dim) {
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (kBlock / 16) + threadIdx.x / 16;
    const int64_t rows = static_cast<int64_t>(q_tokens) * q_heads;
    if (item >= rows) return;
    const int64_t token = item / q_heads;
    const int head = static_cast<int>(item % q_heads), chunk = threadIdx.x % 16;
    const U32x4 a = load_chunk(out.at(token, head), chunk, dim, true);
    const U32x4 b = load_chunk(dout.at(token, head), chunk, dim, true);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sum += item_low<T>(a[i]) * item_low<T>(b[i]);
        sum += item_high<T>(a[i]) * item_high<T>(b[i]);
    }
#pragma unroll
    for (int step = 8; step > 0; step /= 2) sum += __shfl_xor(sum, step);
    if (chunk == 0) {
        const int64_t at = static_cast<int64_t>(head) * q_tokens + token;
        const float l = lse[at];
        stats[at] = l == -INFINITY ? INFINITY : l * kLog2e - kWeightRaise<T>;
        stats[rows + at] = sum;
    }
}

constexpr int kQueryTile = 32;  // rows that pass by at a time: the next ones are loaded while these are worked on
constexpr int kAllWaves = kTeams * kWaves;

// LDS of a gradient workgroup.  Distinct arrays: reads of one do not wait for loads of another.
template <int DP>
struct GradientMemory {
    static constexpr int kTileBytes = Tile<DP>::bytes(kKeyTile);  // of keys or values, or two teams' rows that pass by
    static_assert(kTileBytes >= kTeams * Tile<DP>::bytes(kQueryTile));
    static_assert(DP / 32 * kBlock * 16 <= kTileBytes, "a quarter of a team's sums fits where a tile was");
    char *a, *b, *c, *d;
    char* values;  // kRowTile rows
    float *stats_even, *stats_odd;
    int* broken;  // whether the sums of some wave are not finite
};

struct GradientArgs {
    Rows q, k, v, dout, dq, dk, dv;
    const float* stats;
    float* part_sums;
    const int32_t* q_offsets;
    const int32_t* k_offsets;
    Shape shape;
    int row_tiles;    // tiles of rows, and workgroups of keys and parts of each
    int key_blocks;
    int parts;
    bool ordered_tiles;
};

// dQ: two teams of four waves share the keys' and values' tiles.  They take a tile of rows of two heads of one key head, or
// where its group is odd two tiles of rows of one head (which sequences of up to 128 rows leave half empty; 4 heads on one
// key head, long sequences: 885 us the first way, 898 the second).
template <typename T, int DP>
__device__ __forceinline__ void dq_block(const GradientArgs& g, const GradientMemory<DP>& memory, int block) {
    const Shape& shape = g.shape;
    const int group = shape.q_heads / shape.kv_heads;
    const bool two_heads = group % 2 == 0;
    const int team = __builtin_amdgcn_readfirstlane(threadIdx.x / kBlock);
    const int units = two_heads ? shape.q_heads / 2 : shape.q_heads, unit = block % units;
    const int kv_head = unit % shape.kv_heads;
    const int head = kv_head * group + (two_heads ? unit / shape.kv_heads * 2 + team : unit / shape.kv_heads);
    const int tile_rows = two_heads ? kRowTile : kTeams * kRowTile;
    Span rows, keys;
    int first_row;
    if (g.ordered_tiles) {
        if (!(two_heads ? take_ordered_tile<kRowTile>(g.q_offsets, g.k_offsets, shape, block / units, rows, keys, first_row)
                        : take_ordered_tile<kTeams * kRowTile>(g.q_offsets, g.k_offsets, shape, block / units, rows, keys, first_row)))
            return;
    } else {
        const TilePlace place = find_tile(g.q_offsets, shape.sequences, 1, tile_rows, g.row_tiles - 1 - block / units);
        if (place.sequence < 0) return;
        rows = span_of(g.q_offsets, place.sequence, shape.q_tokens);
        keys = span_of(g.k_offsets, place.sequence, shape.k_tokens);
        first_row = place.tile * tile_rows;
    }
    if (first_row >= rows.size) return;
    const int lane = threadIdx.x % kWave, half = lane / 32;
    const int row0 = two_heads ? first_row : first_row + team * kRowTile;
    const int row = row0 + threadIdx.x % kBlock / kWave * kRowsPerWave + lane % 32;
    const bool there = row < rows.size;
    const RowRange range(shape, rows, keys, row0, row);
    // Keys that any row of either team sees: the later team's, if it has rows.
    const int end = two_heads || first_row + kRowTile >= rows.size ? RowRange(shape, rows, keys, first_row, row).end
                                                                   : RowRange(shape, rows, keys, first_row + kRowTile, row).end;
    const float c = shape.scale * kLog2e;
    char* k_even = memory.a;
    char* v_even = memory.b;
    char* k_odd = memory.c;
    char* v_odd = memory.d;

    U32x4 qf[DP / 16], of[DP / 16];
    load_row<DP>(qf, g.q, rows.begin + row, head, there, shape.dim);
    load_row<DP>(of, g.dout, rows.begin + row, head, there, shape.dim);
    const int64_t stat = static_cast<int64_t>(head) * shape.q_tokens + rows.begin + row;
    const float row_base = there ? g.stats[stat] : INFINITY;
    float base = row_base;  // of dS, `raise` powers of two lower
    int raise = kWeightRaise<T>;
    const float delta = there ? g.stats[static_cast<int64_t>(shape.q_heads) * shape.q_tokens + stat] : 0.f;
    for (char* tile : {k_even, v_even, k_odd, v_odd}) clear_past<DP, kKeyTile, kAllWaves>(tile, shape.dim);
    F32x16 acc[DP / 32];
    const PackedRows<DP, kKeyTile, kAllWaves> key_rows(g.k.at(keys.begin, kv_head), g.k.token_bytes, keys.size, shape.dim);
    const PackedRows<DP, kKeyTile, kAllWaves> value_rows(g.v.at(keys.begin, kv_head), g.v.token_bytes, keys.size, shape.dim);
    const auto load = [&](char* k_tile, char* v_tile, int k0) {
        key_rows.load(k_tile, k0);
        value_rows.load(v_tile, k0);
    };
    const auto step = [&](const char* k_tile, const char* v_tile, int k0) {
        if (k0 >= range.wave_end) return;
#pragma unroll
        for (int b = 0; b < kKeyTile / 32; ++b) {
            F32x16 s = {}, dp = {};
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                s = T::mfma(read_rows<DP>(k_tile, b * 32, i), qf[i], s);
                dp = T::mfma(read_rows<DP>(v_tile, b * 32, i), of[i], dp);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = exp2_fast(s[r] * c - base) * (dp[r] - delta);
            if (k0 + kKeyTile > range.full) {
                const uint32_t word = first_keys(range.count, k0 + 32 * b) >> (4 * half);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = word & (1u << acc_row(r, 0)) ? s[r] : 0.f;
            }
            if constexpr (T::kNarrow) {
                const int down = too_large_by(s);
                if (wave_ballot(down != 0) != 0) {
                    const float f = ldexpf(1.f, -down);
                    base += down, raise -= down;
                    s *= f;
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) acc[d] *= f;
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const U32x4 ds = pack_step<T>(s, i);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d)
                    acc[d] = T::mfma(read_columns<DP>(k_tile, b * 32 + i * 16, d * 32), ds, acc[d]);
            }
        }
    };
    const int clean = clean_end(0, two_heads ? range.full : RowRange(shape, rows, keys, first_row, row).full, end);
    const auto pass = [&](int stop) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = F32x16{};
        if constexpr (T::kNarrow) base = row_base - kFirstRaise, raise = kWeightRaise<T> + kFirstRaise;
        pass_tiles<kKeyTile>(0, stop, [&](int k0) { load(k_even, v_even, k0); }, [&](int k0) { load(k_odd, v_odd, k0); },
                             [&](int k0) { step(k_even, v_even, k0); }, [&](int k0) { step(k_odd, v_odd, k0); });
    };
    const auto store = [&] {
        if (there) store_row<T, DP>(g.dq, rows.begin + row, head, acc, ldexpf(shape.scale, -raise), shape.dim);
    };
    pass(end);
    store();  // (before waves wait for each other)
    if (clean < end && block_any(any_not_finite(acc), memory.broken)) {
        pass(clean);
        for (int j = clean; j < range.wave_end; ++j) {
            const char* key = g.k.at(keys.begin + static_cast<int64_t>(j), kv_head);
            const char* value = g.v.at(keys.begin + static_cast<int64_t>(j), kv_head);
            const float s = careful_dot<T, DP>([&](int i) { return qf[i]; }, key, shape.dim);
            const float dp = careful_dot<T, DP>([&](int i) { return of[i]; }, value, shape.dim);
            careful_add<T, DP>(acc, exp2_fast(s * c - base) * (dp - delta), key, shape.dim, j < range.count);
        }
        store();
    }
}

struct RowTiles {  // of one team: which head of the group, which row
    int head, row0, start, size;
    __device__ __forceinline__ void skip(int count) {
        for (row0 += count * kQueryTile; row0 >= size; row0 -= round()) ++head;
    }
    __device__ __forceinline__ int round() const { return (size - start + kQueryTile - 1) / kQueryTile * kQueryTile; }
};

// dK and dV of a tile of keys of one key head: the rows of every query head of its group pass by, so that the sum
// over the group is taken in registers and in one order.  The tiles of rows, of one head after the other, are dealt to two
// teams of four waves, which hold the same keys and add their sums at the end: a tile of keys that many rows see is done
// sooner, and each of a SIMD's two waves has products to run while the other's exponentials do.  Where there are few tiles
// of keys, the rows are split further over `parts` workgroups, whose sums go to memory in 32 bits.
template <typename T, int DP>
__device__ __forceinline__ void dkv_block(const GradientArgs& args, const GradientMemory<DP>& memory, int block, int part) {
    constexpr int kTileBytes = Tile<DP>::bytes(kQueryTile);
    const auto& [q, k, v, dout, dq, dk, dv, stats, part_sums, q_offsets, k_offsets, shape, row_tiles, key_blocks, parts, ordered_tiles] = args;
    const int kv_head = block % shape.kv_heads;
    Span rows, keys;
    int key0;
    if (ordered_tiles) {
        if (!take_ordered_keys<kRowTile>(q_offsets, k_offsets, shape, block / shape.kv_heads, rows, keys, key0)) return;
    } else {
        const TilePlace place = find_tile(k_offsets, shape.sequences, 1, kRowTile, block / shape.kv_heads);
        if (place.sequence < 0) return;
        keys = span_of(k_offsets, place.sequence, shape.k_tokens);
        rows = span_of(q_offsets, place.sequence, shape.q_tokens);
        key0 = place.tile * kRowTile;
    }
    if (key0 >= keys.size) return;
    const int group = shape.q_heads / shape.kv_heads;
    const int lane = threadIdx.x % kWave, half = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x % kBlock / kWave);
    const int team = __builtin_amdgcn_readfirstlane(threadIdx.x / kBlock);
    char* q_even = memory.a + team * kTileBytes;
    char* o_even = memory.b + team * kTileBytes;
    char* q_odd = memory.c + team * kTileBytes;
    char* o_odd = memory.d + team * kTileBytes;
    float* s_even = memory.stats_even + team * 2 * kQueryTile;
    float* s_odd = memory.stats_odd + team * 2 * kQueryTile;
    const int key = key0 + wave * kRowsPerWave + lane % 32;
    const bool there = key < keys.size;
    const int shift = keys.size - rows.size;
    // The first row that sees the key, that sees any of the workgroup's, and from which on rows see all of them.
    const int first = shape.causal && key - shift > 0 ? key - shift : 0;
    int start = shape.causal && key0 - shift > 0 ? key0 - shift : 0;
    start -= start % kQueryTile;
    const int full = shape.causal && key0 + kRowTile - 1 - shift > 0 ? key0 + kRowTile - 1 - shift : 0;
    const int wave_key0 = key0 + wave * kRowsPerWave;
    const int wave_start = wave_key0 >= keys.size ? rows.size : shape.causal ? wave_key0 - shift : 0;
    const float c = shape.scale * kLog2e;

    // Keys in registers; values in LDS, where both teams read them (in registers they left no room for fragments of the rows
    // to be read ahead).  Rows past the last are its copies; their sums are not stored.
    U32x4 kf[DP / 16];
    load_row<DP>(kf, k, keys.begin + key, kv_head, there, shape.dim);
    clear_past<DP, kRowTile, kAllWaves>(memory.values, shape.dim);
    PackedRows<DP, kRowTile, kAllWaves>(v.at(keys.begin, kv_head), v.token_bytes, keys.size, shape.dim).load(memory.values, key0);
    const char* values = memory.values + Tile<DP>::bytes(kRowsPerWave) * wave;
    for (char* tile : {q_even, o_even, q_odd, o_odd}) clear_past<DP, kQueryTile>(tile, shape.dim);
    F32x16 dk_acc[DP / 32], dv_acc[DP / 32];
    float lift = 1.f;  // of dS
    const int all = rows.size > start ? (rows.size - start + kQueryTile - 1) / kQueryTile * group : 0;
    const int per = (all + parts - 1) / parts;
    const int from = part * per, to = from + per < all ? from + per : all;
    RowTiles loads, steps;
    const PackedRows<DP, kQueryTile> q_rows(q.at(rows.begin, 0), q.token_bytes, rows.size, shape.dim);
    const PackedRows<DP, kQueryTile> o_rows(dout.at(rows.begin, 0), dout.token_bytes, rows.size, shape.dim);
    const float* s_rows = stats + static_cast<int64_t>(half) * shape.q_heads * shape.q_tokens + rows.begin;
    const auto load = [&](char* q_tile, char* o_tile, float* s_tile, int at) {
        if (at + team >= to) return;
        q_rows.load(q_tile, loads.row0, loads.head * q.head_bytes);
        o_rows.load(o_tile, loads.row0, loads.head * dout.head_bytes);
        if (wave == 0) {  // lse by the lower half of the wave, delta by the upper
            const int row = loads.row0 + lane % 32 < rows.size ? loads.row0 + lane % 32 : rows.size - 1;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)(
                                                 s_rows + static_cast<int64_t>(loads.head) * shape.q_tokens + row),
                                             (__attribute__((address_space(3))) uint32_t*)(s_tile), 4, 0, 0);
        }
        loads.skip(kTeams);
    };
    // `clean` leaves out tiles of rows of which some do not see some key.
    const auto step = [&](const char* q_tile, const char* o_tile, const float* s_tile, int at, bool clean) {
        if (at + team >= to) return;
        const int tile_row0 = steps.row0;
        steps.skip(kTeams);
#pragma unroll
        for (int b = 0; b < kQueryTile / 32; ++b) {
            const int r0 = tile_row0 + 32 * b;
            if (r0 + 32 <= wave_start || r0 >= rows.size || (clean && r0 < full)) continue;
            F32x16 s = {}, dp = {};
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                s = T::mfma(read_rows<DP>(q_tile, 32 * b, i), kf[i], s);
                dp = T::mfma(read_rows<DP>(o_tile, 32 * b, i), read_rows<DP>(values, 0, i), dp);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const F32x4 l = *reinterpret_cast<const F32x4*>(&s_tile[32 * b + acc_row(4 * j, half)]);
                const F32x4 e = *reinterpret_cast<const F32x4*>(&s_tile[kQueryTile + 32 * b + acc_row(4 * j, half)]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 4 * j + i;
                    s[r] = exp2_fast(s[r] * c - l[i]);
                    dp[r] = s[r] * (T::kNarrow ? (dp[r] - e[i]) * lift : dp[r] - e[i]);
                }
            }
            if (r0 < full || r0 + 32 > rows.size) {
                const uint32_t word = (first_keys(rows.size, r0) & ~first_keys(first, r0)) >> (4 * half);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool seen = word & (1u << acc_row(r, 0));
                    s[r] = seen ? s[r] : 0.f;
                    dp[r] = seen ? dp[r] : 0.f;
                }
            }
            if constexpr (T::kNarrow) {
                const int down = too_large_by(dp);
                if (wave_ballot(down != 0) != 0) {
                    const float f = ldexpf(1.f, -down);
                    lift *= f;
                    dp *= f;
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) dk_acc[d] *= f;
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const U32x4 pf = pack_step<T>(s, i), sf = pack_step<T>(dp, i);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) {
                    dv_acc[d] = T::mfma(read_columns<DP>(o_tile, 32 * b + i * 16, d * 32), pf, dv_acc[d]);
                    dk_acc[d] = T::mfma(read_columns<DP>(q_tile, 32 * b + i * 16, d * 32), sf, dk_acc[d]);
                }
            }
        }
    };
    const auto pass = [&](bool clean) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) dk_acc[d] = dv_acc[d] = F32x16{};
        if constexpr (T::kNarrow) lift = ldexpf(1.f, kFirstRaise);
        loads = {kv_head * group, start, start, rows.size};
        if (from < to) loads.skip(from + team);
        steps = loads;
        pass_tiles<kTeams>(from, to, [&](int x) { load(q_even, o_even, s_even, x); },
                           [&](int x) { load(q_odd, o_odd, s_odd, x); },
                           [&](int x) { step(q_even, o_even, s_even, x, clean); },
                           [&](int x) { step(q_odd, o_odd, s_odd, x, clean); });
    };
    pass(false);
    const bool clean = start < full && block_any(any_not_finite(dk_acc) || any_not_finite(dv_acc), memory.broken);
    if (clean) pass(true);
    if constexpr (T::kNarrow) {
        const float f = 1.f / lift;  // (a power of two)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) dk_acc[d] *= f;
    }
    // The first team ends with dK, the second with dV; each hands the other its share.
    // (Over the tiles, which nothing is loaded into any more: a quarter of the sums in each of the four arrays.)
    const auto join_at = [&](int i) {
        constexpr int kQuarter = DP / 32;
        char* to = i < kQuarter ? memory.a : i < 2 * kQuarter ? memory.b : i < 3 * kQuarter ? memory.c : memory.d;
        return reinterpret_cast<F32x4*>(to + (i % kQuarter * kBlock + threadIdx.x % kBlock) * 16);
    };
    const auto give = [&](const F32x16(&acc)[DP / 32]) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
            *join_at(i) = F32x4{acc[i / 4][4 * (i % 4)], acc[i / 4][4 * (i % 4) + 1], acc[i / 4][4 * (i % 4) + 2], acc[i / 4][4 * (i % 4) + 3]};
    };
    const auto take = [&](F32x16(&acc)[DP / 32]) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
            const F32x4 other = *join_at(i);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i / 4][4 * (i % 4) + j] += other[j];
        }
    };
    const auto store = [&](const Rows& dst, const F32x16(&acc)[DP / 32], float factor, int which) {
        if (!there) return;
        if (parts == 1) {
            store_row<T, DP>(dst, keys.begin + key, kv_head, acc, factor, shape.dim);
            return;
        }
        const int64_t row = (static_cast<int64_t>(part) * 2 + which) * shape.k_tokens * shape.kv_heads +
                            static_cast<int64_t>(keys.begin + key) * shape.kv_heads + kv_head;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
            const int d = 8 * i + 4 * half;
            if (d < shape.dim)
                *reinterpret_cast<F32x4*>(part_sums + row * shape.dim + d) =
                    F32x4{acc[i / 4][4 * (i % 4)], acc[i / 4][4 * (i % 4) + 1], acc[i / 4][4 * (i % 4) + 2], acc[i / 4][4 * (i % 4) + 3]} * factor;
        }
    };
    // The rows that a clean pass left out, of both teams.
    const auto add_left_out = [&](F32x16(&acc)[DP / 32], bool of_keys) {
        const GradientArgs again = arguments_again<GradientArgs>();
        RowTiles tile{kv_head * group, start, start, rows.size};
        if (from < to) tile.skip(from);
        for (int at = from; at < to; ++at, tile.skip(1)) {
            if (tile.row0 >= full) continue;
            const int end = tile.row0 + kQueryTile < rows.size ? tile.row0 + kQueryTile : rows.size;
            for (int row = tile.row0 > wave_start ? tile.row0 : wave_start; row < end; ++row) {
                const char* q_row = again.q.at(rows.begin + static_cast<int64_t>(row), tile.head);
                const char* o_row = again.dout.at(rows.begin + static_cast<int64_t>(row), tile.head);
                const int64_t stat = static_cast<int64_t>(tile.head) * again.shape.q_tokens + rows.begin + row;
                const float p = exp2_fast(careful_dot<T, DP>([&](int i) { return kf[i]; }, q_row, again.shape.dim) * c - again.stats[stat]);
                if (of_keys) {
                    const float dp = careful_dot<T, DP>([&](int i) { return read_rows<DP>(values, 0, i); }, o_row, again.shape.dim);
                    const float delta = again.stats[static_cast<int64_t>(again.shape.q_heads) * again.shape.q_tokens + stat];
                    careful_add<T, DP>(acc, p * (dp - delta), q_row, again.shape.dim, row >= first);
                } else {
                    careful_add<T, DP>(acc, p, o_row, again.shape.dim, row >= first);
                }
            }
        }
    };
    __syncthreads();
    if (team == 1) give(dk_acc);
    __syncthreads();
    if (team == 0) {
        take(dk_acc);
        if (clean) add_left_out(dk_acc, true);
        store(dk, dk_acc, ldexpf(shape.scale, -kWeightRaise<T>), 0);
    }
    __syncthreads();
    if (team == 0) give(dv_acc);
    __syncthreads();
    if (team == 1) {
        take(dv_acc);
        if (clean) add_left_out(dv_acc, false);
        store(dv, dv_acc, ldexpf(1.f, -kWeightRaise<T>), 1);
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(kTeams* kBlock, 2) void attention_gradients_kernel(GradientArgs args) {
    __shared__ __attribute__((aligned(16))) char a[GradientMemory<DP>::kTileBytes];
    __shared__ __attribute__((aligned(16))) char b[GradientMemory<DP>::kTileBytes];
    __shared__ __attribute__((aligned(16))) char c[GradientMemory<DP>::kTileBytes];
    __shared__ __attribute__((aligned(16))) char d[GradientMemory<DP>::kTileBytes];
    __shared__ __attribute__((aligned(16))) char values[Tile<DP>::bytes(kRowTile)];
    __shared__ __attribute__((aligned(16))) float stats_even[kTeams * 2 * kQueryTile];
    __shared__ __attribute__((aligned(16))) float stats_odd[kTeams * 2 * kQueryTile];
    __shared__ int broken;
    if (threadIdx.x == 0) broken = 0;
    const GradientMemory<DP> memory{a, b, c, d, values, stats_even, stats_odd, &broken};
    const int of_keys = args.key_blocks * args.parts, block = static_cast<int>(blockIdx.x);
    if (block < of_keys) dkv_block<T, DP>(args, memory, block % args.key_blocks, block / args.key_blocks);
    else dq_block<T, DP>(args, memory, block - of_keys);
}

// Adds the parts of dK and dV, in the parts' order: a thread per four items.
template <typename T>
__global__ __launch_bounds__(kBlock) void attention_dkv_join_kernel(Rows dk, Rows dv, const float* __restrict__ part_sums, int parts,
                                                                    const int32_t* __restrict__ k_offsets, Shape shape) {
    const int quads = shape.dim / 4;
    const int64_t rows = static_cast<int64_t>(shape.k_tokens) * shape.kv_heads;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    if (at >= rows * quads) return;
    const int64_t row = at / quads, token = row / shape.kv_heads;
    if (token < k_offsets[0] || token >= k_offsets[shape.sequences]) return;
    const int head = static_cast<int>(row % shape.kv_heads), quad = static_cast<int>(at % quads);
    const float* from = part_sums + (blockIdx.y * rows + row) * shape.dim + quad * 4;
    F32x4 sum = {};
    for (int i = 0; i < parts; ++i) sum += *reinterpret_cast<const F32x4*>(from + 2 * i * rows * shape.dim);
    const Rows& dst = blockIdx.y == 0 ? dk : dv;
    *reinterpret_cast<U32x2*>(dst.at(token, head) + quad * 8) = U32x2{pack2<T>(sum[0], sum[1]), pack2<T>(sum[2], sum[3])};
}

// ---- host side ---------------------------------------------------------------------------------------------------
constexpr uint64_t kResident = 256;  // workgroups that run at once, one a compute unit

// Workgroups that share a tile of keys: as many as there are compute units, while each still has a few tiles of rows (one
// sequence of 1,024 rows, 32 heads on 8 keys' heads: 130 us unsplit, 86 so, 104 with twice as many; on one: 835, 90, 111).
constexpr uint64_t kKeyGrid = 256;
constexpr uint64_t kLeastSteps = 8;

uint64_t key_parts(uint64_t sequences, uint64_t q_tokens, uint64_t k_tokens, uint64_t q_heads, uint64_t kv_heads) {
    if (sequences == 0 || kv_heads == 0) return 1;
    // Tiles of keys that there are about, and steps that each has: its sequence's rows for every head of the group.
    const uint64_t tiles = (k_tokens / kRowTile > sequences ? k_tokens / kRowTile : sequences) * kv_heads;
    const uint64_t steps = ceil_div(q_tokens / sequences, kQueryTile) * (q_heads / kv_heads);
    const uint64_t wanted = kKeyGrid / tiles, most = steps / kLeastSteps;
    const uint64_t parts = wanted < most ? wanted : most;
    return parts > 1 ? parts : 1;
}

size_t stats_bytes(uint64_t q_tokens, uint64_t q_heads) { return align_up(q_tokens * q_heads * 2 * sizeof(float), kViewAlign); }

size_t backward_bytes(uint64_t sequences, uint64_t q_tokens, uint64_t k_tokens, uint64_t q_heads, uint64_t kv_heads, uint64_t dim) {
    const uint64_t parts = key_parts(sequences, q_tokens, k_tokens, q_heads, kv_heads);
    return stats_bytes(q_tokens, q_heads) +
           (parts > 1 ? align_up(parts * 2 * k_tokens * kv_heads * dim * sizeof(float), kViewAlign) : 0);
}

template <typename T>
int packed_backward(void* temp, size_t temp_bytes, const lcpp_hip_rows* q, const lcpp_hip_rows* k, const lcpp_hip_rows* v,
                    const lcpp_hip_rows* out, const float* lse, const lcpp_hip_rows* dout, const int32_t* q_offsets,
                    const int32_t* k_offsets, const lcpp_hip_rows* dq, const lcpp_hip_rows* dk, const lcpp_hip_rows* dv,
                    uint32_t sequences, uint64_t q_tokens, uint64_t k_tokens, uint32_t q_heads, uint32_t kv_heads,
                    uint32_t dim, float scale, int causal, void* stream_ptr) {
    const char* what = "attention_packed_backward";
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (int st = check_shape(what, sequences, q_tokens, k_tokens, q_heads, kv_heads, dim, scale); st != kOk) return st;
    if (sequences == 0 || (q_tokens == 0 && k_tokens == 0)) return kOk;
    if (q_tokens * (q_heads / kv_heads) > kMostKeys) return set_error(kInvalidArgument, "%s: too many tokens or sequences", what);
    if (!q_offsets || !k_offsets) return set_error(kInvalidArgument, "%s: null offsets", what);
    if (q_tokens && !lse) return set_error(kInvalidArgument, "%s: null lse, which the forward pass gives", what);
    if (q_tokens && (!usable(q) || !usable(out) || !usable(dout) || !usable(dq)))
        return unusable(what);
    if (k_tokens && (!usable(k) || !usable(v) || !usable(dk) || !usable(dv)))
        return unusable(what);
    const size_t needed = backward_bytes(sequences, q_tokens, k_tokens, q_heads, kv_heads, dim);
    if (temp_bytes < needed || (needed && !temp))
        return set_error(kTempTooSmall, "%s: temp storage too small", what);
    if ((k_tokens && (too_wide(k) || too_wide(v))) || (q_tokens && (too_wide(q) || too_wide(dout)))) return refuse_wide(what);
    unsigned tiles, grid, key_tiles, key_grid;
    const bool two_heads = q_heads / kv_heads % 2 == 0;
    if (int st = check_grid(what, q_tokens, two_heads ? kRowTile : kTeams * kRowTile, sequences, two_heads ? q_heads / 2 : q_heads, tiles, grid);
        st != kOk)
        return st;
    if (int st = check_grid(what, k_tokens, kRowTile, sequences, kv_heads, key_tiles, key_grid); st != kOk) return st;
    const uint64_t parts = key_parts(sequences, q_tokens, k_tokens, q_heads, kv_heads);
    const uint64_t blocks = (q_tokens ? grid : 0) + (k_tokens ? key_grid * parts : 0);
    if (blocks > 0x7FFFFFFFull / (kTeams * kBlock)) return set_error(kInvalidArgument, "%s: too many tiles", what);
    float* stats = static_cast<float*>(temp);
    const Rows none{nullptr, 0, 0};
    const auto rows = [&](uint64_t tokens, const lcpp_hip_rows* r) { return tokens ? rows_of(r) : none; };
    const GradientArgs args{rows(q_tokens, q), rows(k_tokens, k), rows(k_tokens, v), rows(q_tokens, dout), rows(q_tokens, dq),
                            rows(k_tokens, dk), rows(k_tokens, dv), stats,
                            reinterpret_cast<float*>(static_cast<char*>(temp) + stats_bytes(q_tokens, q_heads)), q_offsets, k_offsets,
                            Shape{static_cast<int>(sequences), static_cast<int>(q_tokens), static_cast<int>(k_tokens),
                                  static_cast<int>(q_heads), static_cast<int>(kv_heads), static_cast<int>(dim), scale, causal != 0},
                            static_cast<int>(tiles), k_tokens ? static_cast<int>(key_grid) : 0, static_cast<int>(parts),
                            sequences > 1 && sequences <= kWave && blocks > kResident};
    if (q_tokens) {
        LaunchScope scope("attention_row_stats", stream);
        const uint64_t stat_blocks = ceil_div(q_tokens * q_heads, kBlock / 16);
        if (stat_blocks > 0x7FFFFFFFull / kBlock) return set_error(kInvalidArgument, "%s: too many rows", what);
        attention_row_stats_kernel<T><<<static_cast<unsigned>(stat_blocks), kBlock, 0, stream>>>(
            rows_of(out), args.dout, lse, stats, args.shape.q_tokens, args.shape.q_heads, args.shape.dim);
        if (int st = check_hip(hipGetLastError(), "attention_row_stats launch"); st != kOk) return st;
    }
    {
        LaunchScope scope("attention_gradients", stream);
        auto* kernel = dim <= 64   ? attention_gradients_kernel<T, 64>
                       : dim <= 96 ? attention_gradients_kernel<T, 96>
                                   : attention_gradients_kernel<T, 128>;
        kernel<<<static_cast<unsigned>(blocks), kTeams * kBlock, 0, stream>>>(args);
        if (int st = check_hip(hipGetLastError(), "attention_gradients launch"); st != kOk) return st;
    }
    if (parts == 1 || k_tokens == 0) return kOk;
    const uint64_t join_blocks = ceil_div(k_tokens * kv_heads * (dim / 4), kBlock);
    if (join_blocks > 0x7FFFFFFFull / kBlock) return set_error(kInvalidArgument, "%s: too many rows", what);
    LaunchScope scope("attention_dkv_join", stream);
    attention_dkv_join_kernel<T><<<dim3(static_cast<unsigned>(join_blocks), 2), kBlock, 0, stream>>>(
        args.dk, args.dv, args.part_sums, args.parts, k_offsets, args.shape);
    return check_hip(hipGetLastError(), "attention_dkv_join launch");
}

}  // namespace
}  // namespace attention
}  // namespace lcpp_hip

using namespace lcpp_hip;

extern "C" {

size_t lcpp_hip_attention_packed_backward_temp_bytes(uint32_t sequences, uint64_t q_tokens, uint64_t k_tokens, uint32_t q_heads,
                                                     uint32_t kv_heads, uint32_t head_dim) {
    return attention::backward_bytes(sequences, q_tokens, k_tokens, q_heads, kv_heads, head_dim);
}

#define LCPP_HIP_DEFINE_ATTENTION_BACKWARD(S, T)                                                                            \
    int lcpp_hip_attention_packed_backward_##S(                                                                             \
        void* temp, size_t temp_bytes, const lcpp_hip_rows* q, const lcpp_hip_rows* k, const lcpp_hip_rows* v,              \
        const lcpp_hip_rows* out, const float* lse, const lcpp_hip_rows* dout, const int32_t* q_offsets,                    \
        const int32_t* k_offsets, const lcpp_hip_rows* dq, const lcpp_hip_rows* dk, const lcpp_hip_rows* dv,                \
        uint32_t sequences, uint64_t q_tokens, uint64_t k_tokens, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim,   \
        float scale, int causal, void* stream) {                                                                            \
        return attention::packed_backward<attention::T>(temp, temp_bytes, q, k, v, out, lse, dout, q_offsets, k_offsets,    \
                                                        dq, dk, dv, sequences, q_tokens, k_tokens, q_heads, kv_heads,       \
                                                        head_dim, scale, causal, stream);                                   \
    }
LCPP_HIP_DEFINE_ATTENTION_BACKWARD(bf16, Bf16)
LCPP_HIP_DEFINE_ATTENTION_BACKWARD(f16, F16)
#undef LCPP_HIP_DEFINE_ATTENTION_BACKWARD

}  // extern "C"
