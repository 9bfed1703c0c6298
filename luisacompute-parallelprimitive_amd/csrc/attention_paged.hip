// Attention of a few new tokens of every request over a paged cache of keys and values.
//
// Request r has kv_lengths[r] keys, position p of them in page block_table[r][p / page] at p % page, and its last n
// keys belong to its n new tokens.  New token i sees every key before those, and new key j where bit j of its tree
// word is set (without a tree: j <= i).  n = 1 is plain decoding.
//
// The n * group rows of a request that share a key head are one matrix of rows, so a key is read once for all of them.
// Reading the cache bounds the call: 4 * dim bytes a key and key head.  256 requests of 200 to 4,000 keys, 8 key heads of
// 128: 1.38 GB in 281 us, 4.9 TB/s, where reads alone reach 7.0 on this card.  One request of 131,000: 537 MB in 98 us,
// 5.5 TB/s, and 7 us to join.
//
// Few rows (attention_paged_kernel): a workgroup takes 32 rows and a part of the keys, its four waves take 32 keys in turn,
// each with its own running maximum, sum and products, and join them at the end.  More (attention_paged_wide_kernel): four
// waves of 32 rows share tiles of 64 keys, as the packed kernel's do.  Weights are rounded to 16 bits as there, and parts
// are joined in f32.
#include "attention_forward.hpp"

namespace lcpp_hip {
namespace attention {
namespace {

constexpr int kNarrowRows = 32;
constexpr int kWaveKeys = 32;                  // keys of a wave at a time
constexpr int kKeyStep = kWaves * kWaveKeys;   // keys of a workgroup at a time
constexpr int kPartKeys = 256;  // at least so many keys make a part: two turns of a workgroup (1,024 took the same time)
// Workgroups wanted at most, if all requests were the longest.  Narrow: two for each compute unit, which is what is resident
// (one request of 131,000 keys: 119 us with 1,024, 116 with 512, 120 with 256).  Wide: three times as many, because a long
// request's parts are few and end together (24 trees: 116 us with 512, 113 with 1,024, 105 with 1,536).  The parts are
// rounded down: one more would pass that number (a chunk of 4,096 rows, which then has no parts, 213 us where two parts
// take 265, 11 requests of 30,000 keys 265 and 300, 24 of 4,000 94 and 102; 40 of 4,000 150 and 145).
constexpr int kNarrowGrid = 512;
constexpr int kWideGrid = 1536;

struct Paged {
    int requests;
    int q_tokens;
    int q_heads;
    int kv_heads;
    int dim;
    Divider page_size;
    int pages;
    int table_stride;
    int table_width;
    int parts;   // at most, of a request as long as stated
    int stated;  // the longest request's keys, as the caller said
    float scale;
};

__device__ __forceinline__ int slot_of(const Paged& p, uint32_t position) {
    return static_cast<int>(position - p.page_size(position) * p.page_size.by);
}

__device__ __forceinline__ int whole_steps(int keys) { return (keys + kKeyStep - 1) / kKeyStep * kKeyStep; }

// Keys of one part: the same for every request, so that parts are alike and a short request is one.  The longest request decides
// it, not what the caller stated: a table's width, or a maximum that a recorded graph was given, may be far more (one request
// of 8,000 keys, 131,072 stated: 39 us by the statement, 17 so; four of 2,000 to 8,000: 116 and 35), and the same
// parts make the same bits.  Where there are parts, requests are some hundred at most, a few loads a lane.
__device__ __forceinline__ int part_of(const int32_t* kv_lengths, const Paged& p) {
    int longest = p.stated;
    if (p.parts > 1) {
        int length = 1;
        for (int r = threadIdx.x % kWave; r < p.requests; r += kWave) length = kv_lengths[r] > length ? kv_lengths[r] : length;
        length = wave_reduce(length, MaxValueOp{});
        longest = length < longest ? length : longest;
    }
    const int part = whole_steps((longest - 1) / p.parts + 1);
    return part > kPartKeys ? part : kPartKeys;
}

// More where a request is longer than the caller said.
__device__ __forceinline__ int part_keys(int length, const Paged& p, int part) {
    const int64_t held = static_cast<int64_t>(part) * p.parts;
    return length <= held ? part : whole_steps((length - 1) / p.parts + 1);
}

struct Work {
    int request;
    int token0;   // first new token of the request
    int tokens;   // new tokens
    int row0;     // first row of the tile
    int rows;     // rows of the request
    int length;   // keys that the table holds
    int ahead;    // keys before the new tokens' own; negative where there are fewer than new tokens
};

__device__ __forceinline__ void take_request(Work& w, const int32_t* q_offsets, const int32_t* kv_lengths, const Paged& p,
                                             int request) {
    int begin = q_offsets[request], end = q_offsets[request + 1];
    begin = begin < 0 ? 0 : begin > p.q_tokens ? p.q_tokens : begin;
    end = end < begin ? begin : end > p.q_tokens ? p.q_tokens : end;
    w.request = request;
    w.token0 = begin;
    w.tokens = end - begin;
    w.rows = w.tokens * (p.q_heads / p.kv_heads);
    int64_t most = static_cast<int64_t>(p.table_width) * p.page_size.by;
    most = most < static_cast<int64_t>(kMostKeys) ? most : static_cast<int64_t>(kMostKeys);
    const int length = kv_lengths[request] < 0 ? 0 : kv_lengths[request];
    w.length = length > most ? static_cast<int>(most) : length;
    w.ahead = length - w.tokens;
}

// Tile `number` of `tile_rows` rows.
__device__ __forceinline__ bool find_work(Work& w, const int32_t* q_offsets, const int32_t* kv_lengths, const Paged& p,
                                          int tile_rows, int number) {
    const TilePlace place = find_tile(q_offsets, p.requests, p.q_heads / p.kv_heads, tile_rows, number);
    if (place.sequence < 0) return false;
    take_request(w, q_offsets, kv_lengths, p, place.sequence);
    w.row0 = place.tile * tile_rows;
    return w.row0 < w.rows;
}

// A part's keys as a tile of rows sees them.
struct Sight {
    int begin;     // of the part
    int end;       // keys in [begin, end) that some row of the tile sees
    int full;      // and those before are seen by all, if their pages are there
    int wave_end;  // keys that some row of the wave sees
    bool whole;    // the request has no other part
    // False where the part holds nothing of the request (and another one writes its rows).
    __device__ __forceinline__ bool find(const Work& w, const Paged& p, int keys, int part, int tile_rows, bool tree_given, int wave_row0,
                                         int wave_rows) {
        const int per = part_keys(w.length, p, keys), group = p.q_heads / p.kv_heads;
        const int64_t first = static_cast<int64_t>(part) * per;
        if (first >= w.length && part > 0) return false;
        begin = static_cast<int>(first);
        whole = w.length <= per;
        const int part_end = w.length - begin > per ? begin + per : w.length;
        // Keys that a row sees, at most and (without a tree) exactly.
        const auto seen = [&](int row) {
            const int64_t last = w.ahead + (tree_given ? int64_t{64} : int64_t{row < w.rows ? row : w.rows - 1} / group + 1);
            return static_cast<int>(last < begin ? begin : last < part_end ? last : part_end);
        };
        end = seen(w.row0 + tile_rows - 1);
        full = tree_given ? (w.ahead < begin ? begin : w.ahead < end ? w.ahead : end) : seen(w.row0);
        wave_end = wave_row0 < w.rows ? seen(wave_row0 + wave_rows - 1) : begin;
        return true;
    }
};

// Bit b: whether the row sees key k0 + b, of 32, as far as new tokens go.  `ahead` keys lie before the new ones.
__device__ __forceinline__ uint32_t seen_word(uint64_t tree, int k0, int ahead) {
    const int shift = k0 - ahead;
    if (shift <= -32) return ~0u;
    if (shift < 0) return static_cast<uint32_t>(tree << -shift) | ((1u << -shift) - 1u);
    return shift < 64 ? static_cast<uint32_t>(tree >> shift) : 0u;
}

// What the row of a lane is.
struct PagedRow {
    bool there;
    int token, head;  // token of its request
    uint64_t tree;
    __device__ __forceinline__ PagedRow(const Work& w, const Paged& p, const uint64_t* words, int kv_head, int row) {
        const int group = p.q_heads / p.kv_heads;
        there = row < w.rows;
        token = there ? row / group : 0;
        head = kv_head * group + (there ? row % group : 0);
        tree = words != nullptr && there ? words[w.token0 + token] : 0;
    }
    __device__ __forceinline__ uint32_t seen(bool tree_given, int k0, int ahead) const {
        return tree_given ? seen_word(tree, k0, ahead) : first_keys(ahead + token + 1, k0);
    }
};

// 16 bytes of a part's sums, or of the output.
template <typename T>
__device__ __forceinline__ void store_items(char* to, const F32x4& a, const F32x4& b, float f) {
    *reinterpret_cast<U32x4*>(to) = U32x4{pack2<T>(a[0] * f, a[1] * f), pack2<T>(a[2] * f, a[3] * f),
                                          pack2<T>(b[0] * f, b[1] * f), pack2<T>(b[2] * f, b[3] * f)};
}

// Where a part's results go, and the row's when one part is all.
struct Parts {
    float* out;      // [parts][q_heads][q_tokens][dim], unnormalised
    F32x2* stats;    // [parts][q_heads][q_tokens]: scale and sum
    __device__ __forceinline__ int64_t row(const Paged& p, int part, int head, int64_t token) const {
        return (static_cast<int64_t>(part) * p.q_heads + head) * p.q_tokens + token;
    }
};

// The wave's keys [k0, end), 32 every `step`: those that a row sees and whose page is there.
template <typename T, int DP>
__device__ __forceinline__ void careful_keys(RowState<DP>& state, const U32x4 (&qf)[DP / 16], const Pages& key_cache, const Pages& value_cache,
                                             const int32_t* table, const PagedRow& row, const uint64_t* tree, const Paged& p,
                                             const Work& w, int kv_head, int k0, int end, int step) {
    for (; k0 < end; k0 += step) {
        const uint32_t seen = row.seen(tree != nullptr, k0, w.ahead);
        for (int j = 0; j < kWaveKeys && k0 + j < end; ++j) {
            const int cell = static_cast<int>(p.page_size(k0 + j)), page = table[cell];
            if (page < 0 || page >= p.pages) continue;
            const int64_t slot = slot_of(p, k0 + j);
            careful_key<T, DP>(state, qf, key_cache.at(page, slot, kv_head), value_cache.at(page, slot, kv_head), p.dim, p.scale * kLog2e,
                               seen >> j & 1);
        }
    }
}

// Tiles go through registers to LDS: what is in flight is then as much as registers hold (a tile of keys and values, 16 KB
// a wave and eight waves a compute unit), and page numbers are known two tiles ahead.  256 requests take 283 us; with tiles
// loaded straight into LDS they took 475, and through registers with a lane a key (16 bytes of a row at a time) 411.
template <typename T, int DP>
__global__ __launch_bounds__(kBlock, 2) void attention_paged_kernel(Rows q, Pages key_cache, Pages value_cache, Rows out,
                                                                    float* __restrict__ lse, Parts parts,
                                                                    const int32_t* __restrict__ block_table,
                                                                    const int32_t* __restrict__ q_offsets,
                                                                    const int32_t* __restrict__ kv_lengths,
                                                                    const uint64_t* __restrict__ tree, Paged p) {
    constexpr int kTileBytes = Tile<DP>::bytes(kWaveKeys);
    constexpr int kJoinStride = DP + 4;  // floats
    constexpr int kJoinBytes = kWaves * kNarrowRows * kJoinStride * 4;
    constexpr int kTilesBytes = kWaves * 2 * kTileBytes;
    constexpr int kLoads = kWaveKeys / Tile<DP>::kBlockRows;
    __shared__ __attribute__((aligned(16))) char tiles[kTilesBytes > kJoinBytes ? kTilesBytes : kJoinBytes];
    __shared__ float stats[2][kWaves][kNarrowRows];
    const int kv_head = blockIdx.x % p.kv_heads;
    const int part = part_of(kv_lengths, p);
    Work w;
    if (!find_work(w, q_offsets, kv_lengths, p, kNarrowRows, blockIdx.x / p.kv_heads)) return;
    Sight sight;
    if (!sight.find(w, p, part, blockIdx.y, kNarrowRows, tree != nullptr, w.row0, kNarrowRows)) return;
    const int begin = sight.begin, end = sight.end;
    const bool whole = sight.whole;
    const int group = p.q_heads / p.kv_heads;
    const int lane = threadIdx.x % kWave, half = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const PagedRow row(w, p, tree, kv_head, w.row0 + lane % 32);
    const float c = p.scale * kLog2e;
    const int32_t* table = block_table + static_cast<int64_t>(w.request) * p.table_stride;
    const char* keys = key_cache.at(0, 0, kv_head);
    const char* values = value_cache.at(0, 0, kv_head);

    U32x4 qf[DP / 16];
    const char* q_row = q.at(w.token0 + row.token, row.head);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) qf[s] = load_chunk(q_row, 2 * s + half, p.dim, row.there);
    char* k_tile = tiles + wave * 2 * kTileBytes;
    char* v_tile = k_tile + kTileBytes;
    // Lane l and l + 32 look key l of a tile up; the tile's rows are then read four lanes to 64 bytes.  Tiles are in
    // registers one ahead of the one in LDS, page numbers two ahead.
    const bool alike = key_cache.page_bytes == value_cache.page_bytes && key_cache.token_bytes == value_cache.token_bytes;
    const bool has = Tile<DP>::lane_chunk(lane) * 8 < p.dim;
    const auto page_of = [&](int k0) {
        const int position = k0 + lane % 32;
        return position < end ? table[p.page_size(position)] : -1;
    };
    U32x4 kf[kLoads], vf[kLoads];
    // Loads tile k0; the keys that are there, as bits.
    const auto load = [&](int page, int k0) {
        const bool here = page >= 0 && page < p.pages;
        const uint32_t held = static_cast<uint32_t>(wave_ballot(here));
        const int64_t pg = here ? page : 0, slot = here ? slot_of(p, k0 + lane % 32) : 0;
        const int64_t k_at = pg * key_cache.page_bytes + slot * key_cache.token_bytes;
        const int64_t v_at = alike ? k_at : pg * value_cache.page_bytes + slot * value_cache.token_bytes;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int key = i * Tile<DP>::kBlockRows + Tile<DP>::lane_row(lane);
            const int64_t k_from = __shfl(k_at, key), v_from = alike ? k_from : __shfl(v_at, key);
            const bool there = has && (held >> key & 1);
            kf[i] = vf[i] = U32x4{0u, 0u, 0u, 0u};
            if (there) {
                kf[i] = *reinterpret_cast<const U32x4*>(keys + k_from + Tile<DP>::lane_chunk(lane) * 16);
                vf[i] = *reinterpret_cast<const U32x4*>(values + v_from + Tile<DP>::lane_chunk(lane) * 16);
            }
        }
        return held;
    };
    RowState<DP> state;
    int k0 = begin + wave * kWaveKeys;
    uint32_t next_held;
    int page;
    const auto start = [&] {
        state = {};
        state.top = -INFINITY;
        k0 = begin + wave * kWaveKeys;
        next_held = load(page_of(k0), k0);
        page = page_of(k0 + kKeyStep);
    };
    const auto step = [&] {
        const uint32_t held = next_held;
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            *reinterpret_cast<U32x4*>(k_tile + i * Tile<DP>::kBlockBytes + lane * 16) = kf[i];
            *reinterpret_cast<U32x4*>(v_tile + i * Tile<DP>::kBlockBytes + lane * 16) = vf[i];
        }
        wave_lds_order();
        next_held = load(page, k0 + kKeyStep);
        page = page_of(k0 + 2 * kKeyStep);
        F32x16 s = {};
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) s = T::mfma(read_rows<DP>(k_tile, 0, i), qf[i], s);
        if (held != ~0u || k0 + kWaveKeys > sight.full) {
            const uint32_t seen = (held & row.seen(tree != nullptr, k0, w.ahead)) >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = seen & (1u << acc_row(r, 0)) ? s[r] : -INFINITY;
        }
        float high = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) high = fmaxf(high, s[r]);
        rescale(state, halves_max(high), c);
        const float base = weight_base<T>(state.top, c);
        float sum = 0.f;  // (a weight alone may be below the last bit of a long row's total)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = exp2_fast(s[r] * c - base);
            sum += s[r];
        }
        state.total += sum;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const U32x4 pf = pack_step<T>(s, i);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
                state.acc[d] = T::mfma(read_columns<DP>(v_tile, i * 16, d * 32), pf, state.acc[d]);
        }
    };
    start();
    for (; k0 < end; k0 += kKeyStep) step();
    if (sight.full < end && wave_ballot(any_not_finite(state.acc)) != 0) {
        start();
        for (; k0 + kWaveKeys <= sight.full; k0 += kKeyStep) step();
        careful_keys<T, DP>(state, qf, key_cache, value_cache, table, row, tree, p, w, kv_head, k0, end, kKeyStep);
    }
    const float total = halves_sum(state.total);
    if (half == 0) {
        stats[0][wave][lane] = state.top;
        stats[1][wave][lane] = total;
    }
    __syncthreads();
    // The waves' products, scaled to the rows' common maximum, side by side over the tiles.
    float all_top = -INFINITY, all_total = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) all_top = fmaxf(all_top, stats[0][i][lane % 32]);
    const float base = all_top == -INFINITY ? 0.f : all_top * c;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) all_total += stats[1][i][lane % 32] * exp2_fast(stats[0][i][lane % 32] * c - base);
    const float mine = exp2_fast(state.top * c - base);
    float* join = reinterpret_cast<float*>(tiles);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const F32x4 v = {state.acc[d][4 * g], state.acc[d][4 * g + 1], state.acc[d][4 * g + 2], state.acc[d][4 * g + 3]};
            *reinterpret_cast<F32x4*>(join + (wave * kNarrowRows + lane % 32) * kJoinStride + d * 32 + 8 * g + 4 * half) = v * mine;
        }
    __syncthreads();
    if (threadIdx.x < kNarrowRows) {
        stats[0][0][lane] = all_total;
        if (row.there && whole && lse != nullptr)
            lse[static_cast<int64_t>(row.head) * p.q_tokens + w.token0 + row.token] = row_lse<T>(all_top, all_total, p.scale);
        if (row.there && !whole) parts.stats[parts.row(p, blockIdx.y, row.head, w.token0 + row.token)] = F32x2{all_top, all_total};
    }
    __syncthreads();
    for (int item = threadIdx.x; item < kNarrowRows * DP / 8; item += kBlock) {
        const int r = item / (DP / 8), chunk = item % (DP / 8);
        if (w.row0 + r >= w.rows || chunk * 8 >= p.dim) continue;
        F32x4 a = {}, b = {};
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            const float* from = join + (i * kNarrowRows + r) * kJoinStride + chunk * 8;
            a += *reinterpret_cast<const F32x4*>(from);
            b += *reinterpret_cast<const F32x4*>(from + 4);
        }
        const int64_t t = w.token0 + (w.row0 + r) / group;
        const int h = kv_head * group + (w.row0 + r) % group;
        if (whole) {
            const float sum = stats[0][0][r];
            store_items<T>(out.at(t, h) + chunk * 16, a, b, sum == 0.f ? 0.f : 1.f / sum);
        } else {
            float* to = parts.out + parts.row(p, blockIdx.y, h, t) * p.dim + chunk * 8;
            *reinterpret_cast<F32x4*>(to) = a;
            *reinterpret_cast<F32x4*>(to + 4) = b;
        }
    }
}

// A row of zeros, for a page that is not there.
__device__ __attribute__((aligned(16))) const uint32_t zero_row[64] = {};

// Direct loads of tiles of keys and values from the cache.  Positions past the last are loaded as the last, and masked; rows
// of a page that is not there are loaded from a row of zeros.
template <int DP>
struct PagedTiles {
    using Loads = TileLoads<DP, kKeyTile>;
    const char* keys;
    const char* values;
    const Pages& key_cache;
    const Pages& value_cache;
    const int32_t* table;
    const Paged& p;
    int end;
    int page[Loads::kPerWave];  // of the tile to load next
    __device__ __forceinline__ int position(int k0, int i) const {
        const int at = k0 + Loads::row() + i * Loads::kRowStep;
        return at < end ? at : end - 1;
    }
    __device__ __forceinline__ void look_up(int k0) {
#pragma unroll
        for (int i = 0; i < Loads::kPerWave; ++i) page[i] = table[p.page_size(position(k0, i))];
    }
    __device__ __forceinline__ void load(char* k_tile, char* v_tile, int k0) {
        const int chunk = Loads::chunk();
        if (chunk * 8 < p.dim) {
#pragma unroll
            for (int i = 0; i < Loads::kPerWave; ++i) {
                const int64_t slot = slot_of(p, position(k0, i));
                const bool there = page[i] >= 0 && page[i] < p.pages;
                const char* key = keys + page[i] * key_cache.page_bytes + slot * key_cache.token_bytes;
                const char* value = values + page[i] * value_cache.page_bytes + slot * value_cache.token_bytes;
                load_to_lds((there ? key : reinterpret_cast<const char*>(zero_row)) + chunk * 16, Loads::place(k_tile, i));
                load_to_lds((there ? value : reinterpret_cast<const char*>(zero_row)) + chunk * 16, Loads::place(v_tile, i));
            }
        }
        if (k0 + kKeyTile < end) look_up(k0 + kKeyTile);
    }
};

// Many rows of a request: 24 trees of 5 to 48 tokens over 500 to 8,000 keys, 4 heads a key head: 302 MB in 91 us,
// 3.3 TB/s, and 11 us to join.  Bound by the latency of a tile: a workgroup has one in flight while it works on another.
template <typename T, int DP>
__global__ __launch_bounds__(kBlock, DP <= 64 ? 3 : 2) void attention_paged_wide_kernel(Rows q, Pages key_cache, Pages value_cache, Rows out,
                                                                         float* __restrict__ lse, Parts parts,
                                                                         const int32_t* __restrict__ block_table,
                                                                         const int32_t* __restrict__ q_offsets,
                                                                         const int32_t* __restrict__ kv_lengths,
                                                                         const uint64_t* __restrict__ tree, Paged p) {
    constexpr int kTileBytes = Tile<DP>::bytes(kKeyTile);
    __shared__ __attribute__((aligned(16))) char k_even[kTileBytes];
    __shared__ __attribute__((aligned(16))) char v_even[kTileBytes];
    __shared__ __attribute__((aligned(16))) char k_odd[kTileBytes];
    __shared__ __attribute__((aligned(16))) char v_odd[kTileBytes];
    __shared__ int broken;  // whether the sums of some wave are not finite
    if (threadIdx.x == 0) broken = 0;
    const int kv_head = blockIdx.x % p.kv_heads;
    const int part = part_of(kv_lengths, p);
    Work w;
    // Without a tree later tiles see more keys: they come first.
    if (!find_work(w, q_offsets, kv_lengths, p, kRowTile, static_cast<int>((gridDim.x - 1 - blockIdx.x) / p.kv_heads))) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wave_row0 = w.row0 + wave * kRowsPerWave;
    Sight sight;
    if (!sight.find(w, p, part, blockIdx.y, kRowTile, tree != nullptr, wave_row0, kRowsPerWave)) return;
    const int begin = sight.begin, end = sight.end, wave_end = sight.wave_end;
    const bool whole = sight.whole;
    const int lane = threadIdx.x % kWave, half = lane / 32;
    const PagedRow row(w, p, tree, kv_head, wave_row0 + lane % 32);
    const float c = p.scale * kLog2e;
    const int32_t* table = block_table + static_cast<int64_t>(w.request) * p.table_stride;
    // A page that is not there: every tile is masked, by what the table says of its keys.  (Each wave looks for itself, so
    // that nothing waits for it.)
    bool lost = false;
    if (begin < end)
        for (int i = static_cast<int>(p.page_size(begin)) + lane; i <= static_cast<int>(p.page_size(end - 1)); i += kWave)
            lost |= table[i] < 0 || table[i] >= p.pages;
    lost = wave_ballot(lost) != 0;

    U32x4 qf[DP / 16];
    const char* q_row = q.at(w.token0 + row.token, row.head);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) qf[s] = load_chunk(q_row, 2 * s + half, p.dim, row.there);
    for (char* tile : {k_even, v_even, k_odd, v_odd}) clear_past<DP, kKeyTile>(tile, p.dim);
    RowState<DP> state;
    const auto seen = [&](int k0) {
        uint32_t word = row.seen(tree != nullptr, k0, w.ahead) & first_keys(end, k0);
        if (lost) {
            const int position = k0 + lane % 32;
            const int page = position < end ? table[p.page_size(position)] : -1;
            word &= static_cast<uint32_t>(wave_ballot(page >= 0 && page < p.pages));
        }
        return word;
    };
    PagedTiles<DP> source{key_cache.at(0, 0, kv_head), value_cache.at(0, 0, kv_head), key_cache, value_cache, table, p, end, {}};
    const int full = lost ? begin : sight.full;
    const auto step = [&](const char* k_tile, const char* v_tile, int k0) {
        if (k0 < wave_end) forward_tile<T, DP>(state, k_tile, v_tile, qf, c, k0, k0 + kKeyTile > full, seen);
    };
    const int clean = clean_end(begin, sight.full, end);
    const auto pass = [&](RowState<DP>& state, int stop) {
        state = {};
        state.top = -INFINITY;
        if (begin < stop) source.look_up(begin);
        pass_tiles<kKeyTile>(begin, stop, [&](int k0) { source.load(k_even, v_even, k0); }, [&](int k0) { source.load(k_odd, v_odd, k0); },
                             [&](int k0) { step(k_even, v_even, k0); }, [&](int k0) { step(k_odd, v_odd, k0); });
    };
    const auto store = [&](const RowState<DP>& state) {
        const float total = halves_sum(state.total);
        if (!row.there) return;
        const int64_t t = w.token0 + row.token;
        if (whole) {
            store_row<T, DP>(out, t, row.head, state.acc, total == 0.f ? 0.f : 1.f / total, p.dim);
            if (lse != nullptr && half == 0) lse[static_cast<int64_t>(row.head) * p.q_tokens + t] = row_lse<T>(state.top, total, p.scale);
            return;
        }
        const int64_t at = parts.row(p, blockIdx.y, row.head, t);
        if (half == 0) parts.stats[at] = F32x2{state.top, total};
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
            const int d = 8 * i + 4 * half;
            const F32x16& acc = state.acc[i / 4];
            if (d < p.dim)
                *reinterpret_cast<F32x4*>(parts.out + at * p.dim + d) =
                    F32x4{acc[4 * (i % 4)], acc[4 * (i % 4) + 1], acc[4 * (i % 4) + 2], acc[4 * (i % 4) + 3]};
        }
    };
    pass(state, end);
    store(state);  // (before waves wait for each other)
    if (clean < end && block_any(any_not_finite(state.acc), &broken)) {
        pass(state, clean);
        careful_keys<T, DP>(state, qf, key_cache, value_cache, table, row, tree, p, w, kv_head, clean, wave_end, kWaveKeys);
        store(state);
    }
}

// Joins the parts of a token's rows, in the parts' order: with t the largest of the parts' scales, O = sum exp(t_i - t) A_i /
// sum exp(t_i - t) l_i.  16 lanes take a row's items; GROUPS such groups every GROUPS-th part of it, and a workgroup's rows
// are heads of one token.  Bound by latency (64 parts of 32 rows, 16 groups: 7 us; one group: 51).
template <typename T, int GROUPS>
__global__ __launch_bounds__(kBlock) void attention_paged_join_kernel(Rows out, float* __restrict__ lse, Parts parts,
                                                                      const int32_t* __restrict__ q_offsets,
                                                                      const int32_t* __restrict__ kv_lengths, Paged p) {
    constexpr int kHeads = kBlock / 16 / GROUPS;
    __shared__ F32x4 sums[2][GROUPS][kHeads][16];
    __shared__ F32x2 group_stats[GROUPS][kHeads];
    const int blocks = (p.q_heads + kHeads - 1) / kHeads, part = part_of(kv_lengths, p);
    const int64_t token = blockIdx.x / blocks;
    const int request = find_last(p.requests, token, [&](int r) { return static_cast<int64_t>(q_offsets[r]); });
    if (request < 0) return;
    Work w;
    take_request(w, q_offsets, kv_lengths, p, request);
    const int per = part_keys(w.length, p, part);
    if (token >= w.token0 + w.tokens || w.length <= per) return;
    const int count = (w.length + per - 1) / per;
    const int chunk = threadIdx.x % 16, group = threadIdx.x / 16 % GROUPS, local = threadIdx.x / 16 / GROUPS;
    const int head = blockIdx.x % blocks * kHeads + local;
    const bool there = head < p.q_heads;
    const float c = p.scale * kLog2e;
    float top = -INFINITY, total = 0.f;
    F32x4 a = {}, b = {};
    if (there) {
        for (int i = group; i < count; i += GROUPS) top = fmaxf(top, parts.stats[parts.row(p, i, head, token)][0]);
        const float base = top == -INFINITY ? 0.f : top * c;
#pragma unroll 2
        for (int i = group; i < count; i += GROUPS) {
            const int64_t row = parts.row(p, i, head, token);
            const F32x2 st = parts.stats[row];
            const float f = exp2_fast(st[0] * c - base);
            total += st[1] * f;
            if (chunk * 8 < p.dim) {
                const float* from = parts.out + row * p.dim + chunk * 8;
                a += *reinterpret_cast<const F32x4*>(from) * f;
                b += *reinterpret_cast<const F32x4*>(from + 4) * f;
            }
        }
    }
    if constexpr (GROUPS > 1) {
        sums[0][group][local][chunk] = a;
        sums[1][group][local][chunk] = b;
        if (chunk == 0) group_stats[group][local] = F32x2{top, total};
        __syncthreads();
        for (int i = 0; i < GROUPS; ++i) top = fmaxf(top, group_stats[i][local][0]);
        const float base = top == -INFINITY ? 0.f : top * c;
        a = F32x4{}, b = F32x4{}, total = 0.f;
        for (int i = 0; i < GROUPS; ++i) {
            const float f = exp2_fast(group_stats[i][local][0] * c - base);
            total += group_stats[i][local][1] * f;
            a += sums[0][i][local][chunk] * f;
            b += sums[1][i][local][chunk] * f;
        }
    }
    if (!there || group != 0) return;
    if (chunk * 8 < p.dim) store_items<T>(out.at(token, head) + chunk * 16, a, b, total == 0.f ? 0.f : 1.f / total);
    if (chunk == 0 && lse != nullptr) lse[static_cast<int64_t>(head) * p.q_tokens + token] = row_lse<T>(top, total, p.scale);
}

// ---- host side ---------------------------------------------------------------------------------------------------
// Rows of a tile: 32 while a request has no more on average, else 128 (4 rows a request: 285 us with 32, 329 with 128; 20 to
// 190: 119 and 98).
uint64_t tile_rows(uint64_t requests, uint64_t q_tokens, uint64_t group) {
    return q_tokens * group > requests * kNarrowRows ? kRowTile : kNarrowRows;
}

uint64_t parts_of(uint64_t requests, uint64_t q_tokens, uint64_t max_kv, uint64_t q_heads, uint64_t kv_heads) {
    if (kv_heads == 0 || q_heads < kv_heads) return 1;
    // Tiles that have rows: as many as the rows make, or one a request.
    const uint64_t group = q_heads / kv_heads;
    const uint64_t rows = ceil_div(q_tokens * group, tile_rows(requests, q_tokens, group));
    const uint64_t busy = (rows > requests ? rows : requests) * kv_heads;
    const uint64_t most = ceil_div(max_kv, kPartKeys);
    const uint64_t target = tile_rows(requests, q_tokens, group) == kNarrowRows ? kNarrowGrid : kWideGrid;
    uint64_t parts = target / (busy ? busy : 1);
    parts = parts < most ? parts : most;
    return parts ? parts : 1;
}

size_t stats_bytes(uint64_t parts, uint64_t rows) { return align_up(parts * rows * sizeof(F32x2), kViewAlign); }

size_t paged_bytes(uint64_t requests, uint64_t q_tokens, uint64_t max_kv, uint64_t q_heads, uint64_t kv_heads, uint64_t dim) {
    const uint64_t parts = parts_of(requests, q_tokens, max_kv, q_heads, kv_heads);
    if (parts == 1) return 0;
    return stats_bytes(parts, q_tokens * q_heads) + align_up(parts * q_tokens * q_heads * dim * sizeof(float), kViewAlign);
}

template <typename T>
int paged(void* temp, size_t temp_bytes, const lcpp_hip_rows* q, const lcpp_hip_pages* key_cache,
          const lcpp_hip_pages* value_cache, const int32_t* block_table, uint32_t table_stride, uint32_t table_width,
          const int32_t* q_offsets, const int32_t* kv_lengths, const uint64_t* tree, const lcpp_hip_rows* out, float* lse,
          uint32_t requests, uint64_t q_tokens, uint64_t max_kv_length, uint32_t q_heads, uint32_t kv_heads, uint32_t dim,
          uint32_t page_size, uint32_t pages, float scale, void* stream_ptr) {
    const char* what = "attention_paged";
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (q_heads == 0 || kv_heads == 0 || q_heads % kv_heads != 0 || q_heads > 65535)
        return set_error(kInvalidArgument, "%s: query heads must be a multiple of the key heads, and at most 65535", what);
    if (dim == 0 || dim % 8 != 0 || dim > 128)
        return set_error(kUnsupported, "%s: the head size must be a multiple of 8 up to 128", what);
    if (page_size == 0 || page_size > 0x7FFFFFFFu || pages > 0x7FFFFFFFu)
        return set_error(kInvalidArgument, "%s: page size or page count out of range", what);
    if (table_width > table_stride || table_stride > 0x7FFFFFFFu)
        return set_error(kInvalidArgument, "%s: a block table's row must hold its width", what);
    if (q_tokens > 0x7FFFFFFFull || q_tokens * (q_heads / kv_heads) > kMostKeys || requests > 0x7FFFFFFu)
        return set_error(kInvalidArgument, "%s: too many tokens or requests", what);
    if (max_kv_length > kMostKeys) return set_error(kInvalidArgument, "%s: requests too long", what);
    if (!(scale > 0.f) || scale == INFINITY) return set_error(kInvalidArgument, "%s: the scale must be positive and finite", what);
    if (requests == 0 || q_tokens == 0) return kOk;
    if (!q_offsets || !kv_lengths || (table_width && !block_table))
        return set_error(kInvalidArgument, "%s: null offsets, lengths or block table", what);
    if (!usable(q) || !usable(out) || !usable(key_cache) || !usable(value_cache))
        return unusable(what);
    const uint64_t parts = parts_of(requests, q_tokens, max_kv_length, q_heads, kv_heads);
    const size_t needed = paged_bytes(requests, q_tokens, max_kv_length, q_heads, kv_heads, dim);
    if (temp_bytes < needed || (needed && !temp)) return set_error(kTempTooSmall, "%s: temp storage too small", what);
    const uint64_t rows = tile_rows(requests, q_tokens, q_heads / kv_heads);
    const uint64_t blocks = (q_tokens * (q_heads / kv_heads) / rows + requests) * kv_heads;
    if (blocks * parts > 0x7FFFFFFFull / kBlock || parts > 65535 || (parts > 1 && q_tokens * q_heads > 0x7FFFFFFFull / kBlock))
        return set_error(kInvalidArgument, "%s: too many tiles", what);
    const Paged p{static_cast<int>(requests), static_cast<int>(q_tokens), static_cast<int>(q_heads), static_cast<int>(kv_heads),
                  static_cast<int>(dim), Divider(page_size), static_cast<int>(pages), static_cast<int>(table_stride),
                  static_cast<int>(table_width), static_cast<int>(parts), static_cast<int>(max_kv_length ? max_kv_length : 1), scale};
    Parts sums{nullptr, static_cast<F32x2*>(temp)};
    if (parts > 1) sums.out = reinterpret_cast<float*>(static_cast<char*>(temp) + stats_bytes(parts, q_tokens * q_heads));
    {
        LaunchScope scope("attention_paged", stream);
        auto* narrow = dim <= 64   ? attention_paged_kernel<T, 64>
                       : dim <= 96 ? attention_paged_kernel<T, 96>
                                   : attention_paged_kernel<T, 128>;
        auto* wide = dim <= 64   ? attention_paged_wide_kernel<T, 64>
                     : dim <= 96 ? attention_paged_wide_kernel<T, 96>
                                 : attention_paged_wide_kernel<T, 128>;
        auto* kernel = rows == kNarrowRows ? narrow : wide;
        kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(parts)), kBlock, 0, stream>>>(
            rows_of(q), pages_of(key_cache), pages_of(value_cache), rows_of(out), lse, sums, block_table, q_offsets, kv_lengths, tree, p);
        if (int st = check_hip(hipGetLastError(), "attention_paged launch"); st != kOk) return st;
    }
    if (parts == 1) return kOk;
    LaunchScope scope("attention_paged_join", stream);
    const bool many = parts > kBlock / 16;
    auto* join = many ? attention_paged_join_kernel<T, kBlock / 16> : attention_paged_join_kernel<T, 1>;
    const uint64_t join_blocks = q_tokens * (many ? q_heads : ceil_div(q_heads, kBlock / 16));
    join<<<static_cast<unsigned>(join_blocks), kBlock, 0, stream>>>(rows_of(out), lse, sums, q_offsets, kv_lengths, p);
    return check_hip(hipGetLastError(), "attention_paged_join launch");
}

}  // namespace
}  // namespace attention
}  // namespace lcpp_hip

using namespace lcpp_hip;

extern "C" {

size_t lcpp_hip_attention_paged_temp_bytes(uint32_t requests, uint64_t q_tokens, uint64_t max_kv_length, uint32_t q_heads,
                                           uint32_t kv_heads, uint32_t head_dim) {
    return attention::paged_bytes(requests, q_tokens, max_kv_length, q_heads, kv_heads, head_dim);
}

#define LCPP_HIP_DEFINE_ATTENTION_PAGED(S, T)                                                                                \
    int lcpp_hip_attention_paged_##S(                                                                                        \
        void* temp, size_t temp_bytes, const lcpp_hip_rows* q, const lcpp_hip_pages* key_cache,                              \
        const lcpp_hip_pages* value_cache, const int32_t* block_table, uint32_t table_stride, uint32_t table_width,          \
        const int32_t* q_offsets, const int32_t* kv_lengths, const uint64_t* tree, const lcpp_hip_rows* out, float* lse,     \
        uint32_t requests, uint64_t q_tokens, uint64_t max_kv_length, uint32_t q_heads, uint32_t kv_heads,                   \
        uint32_t head_dim, uint32_t page_size, uint32_t pages, float scale, void* stream) {                                  \
        return attention::paged<attention::T>(temp, temp_bytes, q, key_cache, value_cache, block_table, table_stride,        \
                                              table_width, q_offsets, kv_lengths, tree, out, lse, requests, q_tokens,        \
                                              max_kv_length, q_heads, kv_heads, head_dim, page_size, pages, scale, stream);  \
    }
LCPP_HIP_DEFINE_ATTENTION_PAGED(bf16, Bf16)
LCPP_HIP_DEFINE_ATTENTION_PAGED(f16, F16)
#undef LCPP_HIP_DEFINE_ATTENTION_PAGED

}  // extern "C"
