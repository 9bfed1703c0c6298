// Attention of a few new tokens of every request over a paged cache of keys and values.
//
// Request r has kv_lengths[r] keys, position p of them in page block_table[r][p / page] at p % page, and its last n
// keys belong to its n new tokens.  New token i sees every key before those, and new key j where bit j of its tree
// word is set (without a tree: j <= i).  n = 1 is plain decoding.
//
// The n * group rows of a request that share a key head are one matrix of rows, so a key is read once for all of them.
// Reading the cache bounds the call; a workgroup takes 32 rows and a part of the keys, its four waves take 32 keys in
// turn, each with its own running maximum, sum and products, and join them at the end.
#include "attention.hpp"

namespace lcpp_hip {
namespace attention {
namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr int kRowTile = 32;
constexpr int kKeyTile = 32;                  // keys of a wave at a time
constexpr int kKeyStep = kWaves * kKeyTile;   // keys of a workgroup at a time
constexpr int kPartKeys = 256;                // at least so many keys make a part
constexpr int kGridTarget = 1024;             // workgroups that fill the device

struct Paged {
    int requests;
    int q_tokens;
    int q_heads;
    int kv_heads;
    int dim;
    int page_size;
    int pages;
    int table_stride;
    int table_width;
    int parts;  // of a long request
    float scale;
};

// Keys of one part of a request: the same for every part, a multiple of a workgroup's step.
__device__ __forceinline__ int part_keys(int length, int parts) {
    int per = (length + parts - 1) / parts;
    per = per > kPartKeys ? per : kPartKeys;
    return (per + kKeyStep - 1) / kKeyStep * kKeyStep;
}

struct Work {
    int request;
    int token0;   // first new token of the request
    int tokens;   // new tokens
    int row0;     // first row of the tile
    int rows;     // rows of the request
    int length;   // keys
};

__device__ __forceinline__ bool find_work(Work& w, const int32_t* q_offsets, const int32_t* kv_lengths, const Paged& p,
                                          int number) {
    const int group = p.q_heads / p.kv_heads;
    const TilePlace place = find_tile(q_offsets, p.requests, group, kRowTile, number);
    if (place.sequence < 0) return false;
    int begin = q_offsets[place.sequence], end = q_offsets[place.sequence + 1];
    begin = begin < 0 ? 0 : begin > p.q_tokens ? p.q_tokens : begin;
    end = end < begin ? begin : end > p.q_tokens ? p.q_tokens : end;
    w.request = place.sequence;
    w.token0 = begin;
    w.tokens = end - begin;
    w.row0 = place.tile * kRowTile;
    w.rows = w.tokens * group;
    const int64_t most = static_cast<int64_t>(p.table_width) * p.page_size;
    const int length = kv_lengths[place.sequence];
    w.length = length < 0 ? 0 : length > most ? static_cast<int>(most) : length;
    return w.row0 < w.rows;
}

// Bit b: whether the row sees key k0 + b, of 32, as far as new tokens go.  `ahead` keys lie before the new ones.
__device__ __forceinline__ uint32_t seen_word(uint64_t tree, int k0, int ahead) {
    const int shift = k0 - ahead;
    if (shift <= -32) return ~0u;
    if (shift < 0) return static_cast<uint32_t>(tree << -shift) | ((1u << -shift) - 1u);
    return shift < 64 ? static_cast<uint32_t>(tree >> shift) : 0u;
}
__device__ __forceinline__ uint32_t chain_word(int token, int k0, int ahead) {
    const int count = ahead + token + 1 - k0;  // keys from k0 on that the row sees
    return count >= 32 ? ~0u : count <= 0 ? 0u : (1u << count) - 1u;
}

template <typename T, int DP>
__global__ __launch_bounds__(kBlock) void attention_paged_kernel(Rows q, Pages key_cache, Pages value_cache, Rows out,
                                                                 float* __restrict__ lse, float* __restrict__ part_out,
                                                                 F32x2* __restrict__ part_stats,
                                                                 const int32_t* __restrict__ block_table,
                                                                 const int32_t* __restrict__ q_offsets,
                                                                 const int32_t* __restrict__ kv_lengths,
                                                                 const uint64_t* __restrict__ tree, Paged p) {
    constexpr int kTileBytes = Tile<DP>::bytes(kKeyTile);
    constexpr int kJoinStride = DP + 4;  // floats
    constexpr int kJoinBytes = kWaves * kRowTile * kJoinStride * 4;
    __shared__ __attribute__((aligned(16))) char tiles[kWaves * 2 * kTileBytes > kJoinBytes ? kWaves * 2 * kTileBytes : kJoinBytes];
    __shared__ float stats[2][kWaves][kRowTile];
    const int kv_head = blockIdx.x % p.kv_heads;
    Work w;
    if (!find_work(w, q_offsets, kv_lengths, p, blockIdx.x / p.kv_heads)) return;
    const int per = part_keys(w.length, p.parts);
    const int begin = blockIdx.y * per;
    if (begin >= w.length && blockIdx.y > 0) return;
    const int end = begin + per < w.length ? begin + per : w.length;
    const bool whole = w.length <= per;
    const int group = p.q_heads / p.kv_heads;
    const int lane = threadIdx.x % kWave, half = lane / 32, wave = threadIdx.x / kWave;
    const int row = w.row0 + lane % 32;
    const bool there = row < w.rows;
    const int token = there ? row / group : 0;
    const int head = kv_head * group + (there ? row % group : 0);
    const int ahead = w.length - w.tokens;
    const uint64_t word = tree != nullptr && there ? tree[w.token0 + token] : 0;
    const float c = p.scale * kLog2e;
    const int32_t* table = block_table + static_cast<int64_t>(w.request) * p.table_stride;

    U32x4 qf[DP / 16];
    const char* q_row = q.at(w.token0 + token, head);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) qf[s] = load_chunk(q_row, 2 * s + half, p.dim, there);
    char* k_tile = tiles + wave * 2 * kTileBytes;
    char* v_tile = k_tile + kTileBytes;
    F32x16 acc[DP / 32] = {};
    float top = -INFINITY, total = 0.f;
    for (int k0 = begin + wave * kKeyTile; k0 < end; k0 += kKeyStep) {
        // Lane l < 32 finds the page of key k0 + l.
        const int position = k0 + lane % 32;
        int page = -1;
        if (position < end) page = table[position / p.page_size];
        const bool held = page >= 0 && page < p.pages;
        const int slot = position % p.page_size;
        const uint32_t held_word = static_cast<uint32_t>(wave_ballot(held));
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < kKeyTile * DP / 8 / kWave; ++i) {
            const int at = i * kWave + lane;
            const int key = at / (DP / 8), chunk = at % (DP / 8);
            const int from_page = __shfl(page, key), from_slot = __shfl(slot, key);
            const bool here = held_word >> key & 1;
            const int64_t pg = here ? from_page : 0, sl = here ? from_slot : 0;
            const U32x4 kc = load_chunk(key_cache.at(pg, sl, kv_head), chunk, p.dim, here);
            const U32x4 vc = load_chunk(value_cache.at(pg, sl, kv_head), chunk, p.dim, here);
            *reinterpret_cast<U32x4*>(k_tile + Tile<DP>::place(key, chunk)) = kc;
            *reinterpret_cast<U32x4*>(v_tile + Tile<DP>::place(key, chunk)) = vc;
        }
        wave_lds_order();
        F32x16 s = {};
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) s = T::mfma(read_rows<DP>(k_tile, 0, i), qf[i], s);
        const uint32_t seen = held_word & (tree != nullptr ? seen_word(word, k0, ahead) : chain_word(token, k0, ahead));
        float high = top;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if (!(seen >> acc_row(r, half) & 1)) s[r] = -INFINITY;
            high = fmaxf(high, s[r]);
        }
        high = halves_max(high);
        const float base = high == -INFINITY ? 0.f : high * c;
        const float alpha = exp2_fast(top * c - base);
        top = high;
        total *= alpha;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] *= alpha;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = exp2_fast(s[r] * c - base);
            total += s[r];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const U32x4 pf = pack_step<T>(s, i);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) acc[d] = T::mfma(read_columns<DP>(v_tile, i * 16, d * 32), pf, acc[d]);
        }
    }
    total = halves_sum(total);
    if (half == 0) {
        stats[0][wave][lane] = top;
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
    const float mine = exp2_fast(top * c - base);
    float* join = reinterpret_cast<float*>(tiles);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const F32x4 v = {acc[d][4 * g] * mine, acc[d][4 * g + 1] * mine, acc[d][4 * g + 2] * mine, acc[d][4 * g + 3] * mine};
            *reinterpret_cast<F32x4*>(join + (wave * kRowTile + lane % 32) * kJoinStride + d * 32 + 8 * g + 4 * half) = v;
        }
    __syncthreads();
    if (wave == 0 && half == 0) stats[0][0][lane] = all_total;
    const int64_t stat = static_cast<int64_t>(head) * p.q_tokens + w.token0 + token;
    if (wave == 0 && half == 0 && there) {
        if (whole) {
            if (lse != nullptr) lse[stat] = all_total == 0.f ? -INFINITY : all_top * p.scale + __logf(all_total);
        } else {
            part_stats[static_cast<int64_t>(blockIdx.y) * p.q_tokens * p.q_heads + stat] = F32x2{all_top, all_total};
        }
    }
    __syncthreads();
    for (int at = threadIdx.x; at < kRowTile * DP / 8; at += kBlock) {
        const int r = at / (DP / 8), chunk = at % (DP / 8);
        if (w.row0 + r >= w.rows || chunk * 8 >= p.dim) continue;
        F32x4 a = {}, b = {};
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            const float* from = join + (i * kRowTile + r) * kJoinStride + chunk * 8;
            a += *reinterpret_cast<const F32x4*>(from);
            b += *reinterpret_cast<const F32x4*>(from + 4);
        }
        const int64_t t = w.token0 + (w.row0 + r) / group;
        const int h = kv_head * group + (w.row0 + r) % group;
        if (whole) {
            const float sum = stats[0][0][r];
            const float f = sum == 0.f ? 0.f : 1.f / sum;
            *reinterpret_cast<U32x4*>(out.at(t, h) + chunk * 16) =
                U32x4{pack2<T>(a[0] * f, a[1] * f), pack2<T>(a[2] * f, a[3] * f), pack2<T>(b[0] * f, b[1] * f),
                      pack2<T>(b[2] * f, b[3] * f)};
        } else {
            float* to = part_out + ((static_cast<int64_t>(blockIdx.y) * p.q_heads + h) * p.q_tokens + t) * p.dim + chunk * 8;
            *reinterpret_cast<F32x4*>(to) = a;
            *reinterpret_cast<F32x4*>(to + 4) = b;
        }
    }
}

// Joins the parts of a tile's rows, in the parts' order.
template <typename T>
__global__ __launch_bounds__(kBlock) void attention_paged_join_kernel(Rows out, float* __restrict__ lse,
                                                                      const float* __restrict__ part_out,
                                                                      const F32x2* __restrict__ part_stats,
                                                                      const int32_t* __restrict__ q_offsets,
                                                                      const int32_t* __restrict__ kv_lengths, Paged p) {
    const int kv_head = blockIdx.x % p.kv_heads;
    Work w;
    if (!find_work(w, q_offsets, kv_lengths, p, blockIdx.x / p.kv_heads)) return;
    const int per = part_keys(w.length, p.parts);
    if (w.length <= per) return;
    const int parts = (w.length + per - 1) / per;
    const int group = p.q_heads / p.kv_heads;
    const float c = p.scale * kLog2e;
    // 16 lanes a row, 8 items each.
    for (int r = threadIdx.x / 16; r < kRowTile && w.row0 + r < w.rows; r += kBlock / 16) {
        const int64_t t = w.token0 + (w.row0 + r) / group;
        const int h = kv_head * group + (w.row0 + r) % group;
        const int chunk = threadIdx.x % 16;
        const int64_t rows = static_cast<int64_t>(p.q_tokens) * p.q_heads, stat = static_cast<int64_t>(h) * p.q_tokens + t;
        float top = -INFINITY, total = 0.f;
        for (int i = 0; i < parts; ++i) top = fmaxf(top, part_stats[i * rows + stat][0]);
        const float base = top == -INFINITY ? 0.f : top * c;
        F32x4 a = {}, b = {};
        for (int i = 0; i < parts; ++i) {
            const F32x2 st = part_stats[i * rows + stat];
            const float f = exp2_fast(st[0] * c - base);
            total += st[1] * f;
            if (chunk * 8 < p.dim) {
                const float* from = part_out + (i * rows + stat) * p.dim + chunk * 8;
                a += *reinterpret_cast<const F32x4*>(from) * f;
                b += *reinterpret_cast<const F32x4*>(from + 4) * f;
            }
        }
        const float f = total == 0.f ? 0.f : 1.f / total;
        if (chunk * 8 < p.dim)
            *reinterpret_cast<U32x4*>(out.at(t, h) + chunk * 16) =
                U32x4{pack2<T>(a[0] * f, a[1] * f), pack2<T>(a[2] * f, a[3] * f), pack2<T>(b[0] * f, b[1] * f),
                      pack2<T>(b[2] * f, b[3] * f)};
        if (chunk == 0 && lse != nullptr) lse[stat] = total == 0.f ? -INFINITY : top * p.scale + __logf(total);
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------
uint64_t tiles_of(uint64_t requests, uint64_t q_tokens, uint64_t group) { return q_tokens * group / kRowTile + requests; }

uint64_t parts_of(uint64_t requests, uint64_t q_tokens, uint64_t max_kv, uint64_t q_heads, uint64_t kv_heads) {
    if (kv_heads == 0 || q_heads < kv_heads) return 1;
    // Tiles that have rows: as many as the rows make, or one a request.
    const uint64_t rows = ceil_div(q_tokens * (q_heads / kv_heads), kRowTile);
    const uint64_t busy = (rows > requests ? rows : requests) * kv_heads;
    const uint64_t most = ceil_div(max_kv, kPartKeys);
    uint64_t parts = ceil_div(kGridTarget, busy ? busy : 1);
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
    if (q_tokens > 0x7FFFFFFFull || q_tokens * (q_heads / kv_heads) > 0x7FFFFFFFull || requests > 0x7FFFFFFu)
        return set_error(kInvalidArgument, "%s: too many tokens or requests", what);
    if (max_kv_length > 0x7FFFFFFFull) return set_error(kInvalidArgument, "%s: requests too long", what);
    if (!(scale > 0.f) || scale == INFINITY) return set_error(kInvalidArgument, "%s: the scale must be positive and finite", what);
    if (requests == 0 || q_tokens == 0) return kOk;
    if (!q_offsets || !kv_lengths || (table_width && !block_table))
        return set_error(kInvalidArgument, "%s: null offsets, lengths or block table", what);
    if (!usable(q) || !usable(out) || !usable(key_cache) || !usable(value_cache))
        return unusable(what);
    const uint64_t parts = parts_of(requests, q_tokens, max_kv_length, q_heads, kv_heads);
    const size_t needed = paged_bytes(requests, q_tokens, max_kv_length, q_heads, kv_heads, dim);
    if (temp_bytes < needed || (needed && !temp)) return set_error(kTempTooSmall, "%s: temp storage too small", what);
    const uint64_t blocks = tiles_of(requests, q_tokens, q_heads / kv_heads) * kv_heads;
    if (blocks * parts > 0x7FFFFFFFull / kBlock || parts > 65535) return set_error(kInvalidArgument, "%s: too many tiles", what);
    const Paged p{static_cast<int>(requests), static_cast<int>(q_tokens), static_cast<int>(q_heads), static_cast<int>(kv_heads),
                  static_cast<int>(dim), static_cast<int>(page_size), static_cast<int>(pages), static_cast<int>(table_stride),
                  static_cast<int>(table_width), static_cast<int>(parts), scale};
    F32x2* part_stats = static_cast<F32x2*>(temp);
    float* part_out = parts > 1 ? reinterpret_cast<float*>(static_cast<char*>(temp) + stats_bytes(parts, q_tokens * q_heads)) : nullptr;
    {
        LaunchScope scope("attention_paged", stream);
        auto* kernel = dim <= 64 ? attention_paged_kernel<T, 64> : dim <= 96 ? attention_paged_kernel<T, 96> : attention_paged_kernel<T, 128>;
        kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(parts)), kBlock, 0, stream>>>(
            rows_of(q), pages_of(key_cache), pages_of(value_cache), rows_of(out), lse, part_out, part_stats, block_table,
            q_offsets, kv_lengths, tree, p);
        if (int st = check_hip(hipGetLastError(), "attention_paged launch"); st != kOk) return st;
    }
    if (parts == 1) return kOk;
    LaunchScope scope("attention_paged_join", stream);
    attention_paged_join_kernel<T><<<static_cast<unsigned>(blocks), kBlock, 0, stream>>>(rows_of(out), lse, part_out, part_stats,
                                                                                         q_offsets, kv_lengths, p);
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
