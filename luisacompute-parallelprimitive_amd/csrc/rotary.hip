// Rotary positions: every pair of items of a query's or key's head is turned by its position's angle,
//
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),   t = (position + shift) f_i,
//
// with a frequency f_i for each pair and one magnitude m.  A pair is the items i and i + R / 2 (halves), or 2 i and 2 i + 1
// (interleaved); items from R on are copied.  The gradient is the turn by -t.  The paged form puts the turned keys, and the
// values as they are, into the step's slots.
//
// An angle of a far position has more bits than 32-bit floats hold: the turns, t / 2 pi, and what is left of them after whole
// ones, are taken in 64 bits.  Turning is f32, rounded once.  A pair's sine and cosine serve all heads of a token.
//
// Memory bounds the large calls: each item is read and written once.  11,059 tokens of 32 + 8 heads of 128: 226 MB in 41.5 us,
// 5.5 TB/s, where the library's copy of 1 GiB reaches 6.0; 32,749 tokens of 16 heads and 4 + 4 into pages: 403 MB in 74 us, 5.5.
// A decoding step of 64 tokens takes 3.5 us, two or three dependent loads.  Where half a rotation is no multiple of 8 items go one
// by one, loaded after the table is made: 14,000 tokens of 32 + 8 heads of 96, 24 items turned, 112 us where 32 items take 44.
#include "attention.hpp"

#include <cmath>

namespace lcpp_hip {
namespace attention {
namespace {

constexpr int kTurnBlock = 256;
constexpr uint32_t kMostDim = 1024;

struct Turn {
    int64_t tokens;
    int q_heads;
    int kv_heads;
    int dim;
    int half;     // pairs
    bool inverse;
    float factor;
    int num_shifts;
    Divider units;      // of a token
    Divider per_head;   // units of a head
    Divider pairs;
    int group;          // tokens of a workgroup
};

// Where rows come from and go to; values only in the paged form, whose keys and values go to slots.
struct TurnRows {
    Rows q, k, v, q_out, k_out;
    Pages key_cache, value_cache;
    const int64_t* slots;
    int32_t* slot_positions;
    Divider page_size;
    int64_t pages;
};

// How a head is cut into units, one a thread: kHalves, 8 items and the 8 that are half a rotation further, or 8 items past the
// rotation; kInterleaved, 8 items (four pairs, some past the rotation); kOdd, as kHalves where half a rotation is no multiple
// of 8, so that items are read and written by themselves.  Units share no items: rows may be turned in place.
enum class Layout { kHalves, kInterleaved, kOdd };

__host__ __device__ constexpr int units_per_head(Layout layout, int dim, int half) {
    return layout == Layout::kInterleaved ? dim / 8 : (half + 7) / 8 + (dim - 2 * half + 7) / 8;
}

__device__ __forceinline__ int64_t position_of(const int32_t* positions, const int32_t* requests, const int32_t* shifts, int num_shifts,
                                               int64_t token) {
    int64_t position = positions[token];
    if (shifts != nullptr) {
        const int64_t request = requests[token];
        if (request >= 0 && request < num_shifts) position += shifts[request];
    }
    return position;
}

template <typename T>
__device__ __forceinline__ void turn2(uint32_t& x, uint32_t& y, F32x2 cs0, F32x2 cs1) {
    const float a0 = item_low<T>(x), a1 = item_high<T>(x), b0 = item_low<T>(y), b1 = item_high<T>(y);
    x = pack2<T>(a0 * cs0[0] - b0 * cs0[1], a1 * cs1[0] - b1 * cs1[1]);
    y = pack2<T>(a0 * cs0[1] + b0 * cs0[0], a1 * cs1[1] + b1 * cs1[0]);
}

// (Each item is read once: loads that stay out of the caches take 83 us where ordinary ones take 99, 11,059 tokens in both directions.)
__device__ __forceinline__ U32x4 load_once(const char* p) { return __builtin_nontemporal_load(reinterpret_cast<const U32x4*>(p)); }

// What a token's rows need to know: where its slot is (in the paged form), and whether they are written at all.
struct TokenPlace {
    int64_t key_bytes, value_bytes;
    bool rows, slot;
};

// EACH units a thread of `group` tokens, or of a part of a token's (blockIdx.y).  Rows are loaded first; while they come, some
// threads make the workgroup's table of cosines and sines and others look up the tokens' slots.  (With the slots looked up
// before the rows were loaded, 32,749 tokens took 294 us.)
template <typename T, Layout LAYOUT, bool PAGED, int EACH>
__global__ __launch_bounds__(kTurnBlock) void rotary_kernel(TurnRows rows, const int32_t* __restrict__ positions,
                                                            const int32_t* __restrict__ requests, const int32_t* __restrict__ shifts,
                                                            const double* __restrict__ frequencies, Turn p) {
    using Item = typename T::Item;
    extern __shared__ __attribute__((aligned(16))) char shared[];
    const int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.group;
    const int count = static_cast<int>(p.tokens - token0 < p.group ? p.tokens - token0 : p.group);
    TokenPlace* places = reinterpret_cast<TokenPlace*>(shared);
    F32x2* table = reinterpret_cast<F32x2*>(places + p.group);
    const uint32_t all = static_cast<uint32_t>(count) * p.units.by;
    const uint32_t first = blockIdx.y * (kTurnBlock * EACH) + threadIdx.x;
    const int pair_units = LAYOUT == Layout::kOdd ? (p.half + 7) / 8 : p.half / 8;

    U32x4 x[EACH], y[EACH];
    const char* from[EACH];
    int unit[EACH], local[EACH], head[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        // (Past the last unit, the last one again, which is not written.)
        const uint32_t at = first + e * kTurnBlock < all ? first + e * kTurnBlock : all - 1;
        local[e] = static_cast<int>(p.units(at));
        const int rest = static_cast<int>(at - local[e] * p.units.by);
        head[e] = static_cast<int>(p.per_head(rest));
        unit[e] = rest - head[e] * static_cast<int>(p.per_head.by);
        const int64_t token = token0 + local[e];
        const int kv_head = head[e] - p.q_heads;
        from[e] = kv_head < 0 ? rows.q.at(token, head[e]) : !PAGED || kv_head < p.kv_heads ? rows.k.at(token, kv_head)
                                                                                           : rows.v.at(token, kv_head - p.kv_heads);
        if constexpr (LAYOUT == Layout::kInterleaved) {
            x[e] = load_once(from[e] + unit[e] * 16);
        } else if constexpr (LAYOUT == Layout::kHalves) {
            const int more = unit[e] < pair_units ? 0 : p.half * 2;
            x[e] = load_once(from[e] + more + unit[e] * 16);
            if (more == 0) y[e] = load_once(from[e] + p.half * 2 + unit[e] * 16);
        }
    }
    for (int i = threadIdx.x; i < count * p.half; i += kTurnBlock) {
        const int t = static_cast<int>(p.pairs(i)), pair = i - t * p.half;
        const double position = static_cast<double>(position_of(positions, requests, shifts, p.num_shifts, token0 + t));
        double turns = position * frequencies[pair] * 0.15915494309189533577;
        turns -= rint(turns);
        float s, c;
        sincospif(2.f * static_cast<float>(turns), &s, &c);
        table[i] = F32x2{c * p.factor, (p.inverse ? -s : s) * p.factor};
    }
    for (int t = kTurnBlock - 1 - static_cast<int>(threadIdx.x); t < count; t += kTurnBlock) {
        const int64_t token = token0 + t;
        TokenPlace place{0, 0, requests == nullptr || requests[token] >= 0, false};
        if constexpr (PAGED) {
            const int64_t slot = rows.slots[token];
            if (place.rows && slot >= 0) {
                const int64_t page = slot <= 0xFFFFFFFFll ? rows.page_size(static_cast<uint32_t>(slot)) : slot / rows.page_size.by;
                if (page < rows.pages) {
                    const int64_t within = slot - page * rows.page_size.by;
                    place.slot = true;
                    place.key_bytes = page * rows.key_cache.page_bytes + within * rows.key_cache.token_bytes;
                    place.value_bytes = page * rows.value_cache.page_bytes + within * rows.value_cache.token_bytes;
                    if (rows.slot_positions != nullptr && blockIdx.y == 0)
                        rows.slot_positions[slot] = static_cast<int32_t>(position_of(positions, requests, shifts, p.num_shifts, token));
                }
            }
        }
        places[t] = place;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        if (first + e * kTurnBlock >= all) continue;
        const TokenPlace place = places[local[e]];
        const int64_t token = token0 + local[e];
        const int kv_head = head[e] - p.q_heads;
        const bool turned = !PAGED || kv_head < p.kv_heads;
        char* to;
        if (kv_head < 0) {
            if (!place.rows) continue;
            to = rows.q_out.at(token, head[e]);
        } else if constexpr (PAGED) {
            if (!place.slot) continue;
            to = turned ? rows.key_cache.data + place.key_bytes + kv_head * rows.key_cache.head_bytes
                        : rows.value_cache.data + place.value_bytes + (kv_head - p.kv_heads) * rows.value_cache.head_bytes;
        } else {
            if (!place.rows) continue;
            to = rows.k_out.at(token, kv_head);
        }
        const F32x2* cs = table + local[e] * p.half;
        if constexpr (LAYOUT == Layout::kInterleaved) {
            if (turned && 4 * unit[e] < p.half) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int pair = 4 * unit[e] + i;
                    const float a = item_low<T>(x[e][i]), b = item_high<T>(x[e][i]);
                    const F32x2 t = cs[pair < p.half ? pair : 0];
                    const uint32_t turn = pack2<T>(a * t[0] - b * t[1], a * t[1] + b * t[0]);
                    x[e][i] = pair < p.half ? turn : x[e][i];
                }
            }
            *reinterpret_cast<U32x4*>(to + unit[e] * 16) = x[e];
        } else if constexpr (LAYOUT == Layout::kHalves) {
            if (unit[e] >= pair_units) {
                *reinterpret_cast<U32x4*>(to + p.half * 2 + unit[e] * 16) = x[e];
                continue;
            }
            if (turned) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t a = x[e][i], b = y[e][i];
                    turn2<T>(a, b, cs[8 * unit[e] + 2 * i], cs[8 * unit[e] + 2 * i + 1]);
                    x[e][i] = a;
                    y[e][i] = b;
                }
            }
            *reinterpret_cast<U32x4*>(to + unit[e] * 16) = x[e];
            *reinterpret_cast<U32x4*>(to + p.half * 2 + unit[e] * 16) = y[e];
        } else {
            const Item* in = reinterpret_cast<const Item*>(from[e]);
            Item* out = reinterpret_cast<Item*>(to);
            for (int i = 0; i < 8; ++i) {
                if (unit[e] < pair_units) {
                    const int pair = 8 * unit[e] + i;
                    if (pair >= p.half) break;
                    const Item first_item = in[pair], second_item = in[pair + p.half];
                    const float a = static_cast<float>(first_item), b = static_cast<float>(second_item);
                    const F32x2 t = cs[pair];
                    out[pair] = turned ? static_cast<Item>(a * t[0] - b * t[1]) : first_item;
                    out[pair + p.half] = turned ? static_cast<Item>(a * t[1] + b * t[0]) : second_item;
                } else {
                    const int at = 2 * p.half + 8 * (unit[e] - pair_units) + i;
                    if (at >= p.dim) break;
                    out[at] = in[at];
                }
            }
        }
    }
}

// Units a thread: four where that leaves four workgroups for every compute unit, else one: fewer tables, and more bytes on their way
// in each wave, against more waves for a few tokens.  (32 + 8 heads of 128: 64 tokens one 3.1 us, four 4.7; 1,024: 5.7 and 6.8; 4,096: 20.1
// and 18.9; 8,192: 36.3 and 32.0.)
constexpr int kEach = 4;
constexpr uint64_t kManyBlocks = 1024;
constexpr uint64_t kMostPairs = 2048;  // of a workgroup's table, 16 KB

template <typename T, bool PAGED>
int launch(const char* what, const TurnRows& rows, const int32_t* positions, const int32_t* requests, const int32_t* shifts,
           uint32_t num_shifts, const double* frequencies, uint64_t tokens, uint32_t q_heads, uint32_t kv_heads, uint32_t dim,
           uint32_t rotary_dim, bool interleaved, bool inverse, float factor, hipStream_t stream) {
    const int half = static_cast<int>(rotary_dim / 2);
    const Layout layout = interleaved ? Layout::kInterleaved : half % 8 == 0 ? Layout::kHalves : Layout::kOdd;
    const uint64_t per_head = units_per_head(layout, dim, half);
    const uint64_t units = per_head * (q_heads + static_cast<uint64_t>(kv_heads) * (PAGED ? 2 : 1));
    const bool many = tokens * units >= kManyBlocks * kTurnBlock * kEach;
    const uint64_t block_units = kTurnBlock * (many ? kEach : 1);
    uint64_t group = units >= block_units ? 1 : block_units / units;
    if (group * half > kMostPairs) group = half < kMostPairs ? kMostPairs / half : 1;
    if (group > kTurnBlock) group = kTurnBlock;
    const uint64_t blocks = ceil_div(tokens, group), parts = ceil_div(group * units, block_units);
    if (blocks > 0x7FFFFFFFull / kTurnBlock || parts > 65535)
        return set_error(kInvalidArgument, "%s: too many tokens or heads", what);
    const Turn p{static_cast<int64_t>(tokens), static_cast<int>(q_heads), static_cast<int>(kv_heads), static_cast<int>(dim), half,
                 inverse, factor, static_cast<int>(num_shifts), Divider(static_cast<uint32_t>(units)),
                 Divider(static_cast<uint32_t>(per_head)), Divider(static_cast<uint32_t>(half)), static_cast<int>(group)};
    const size_t lds = group * (half * sizeof(F32x2) + sizeof(TokenPlace));
    const auto run = [&](auto kernel) {
        kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(parts)), kTurnBlock, lds, stream>>>(
            rows, positions, requests, shifts, frequencies, p);
    };
    const auto choose = [&](auto each) {
        constexpr int kUnits = decltype(each)::value;
        if (layout == Layout::kInterleaved) run(rotary_kernel<T, Layout::kInterleaved, PAGED, kUnits>);
        else if (layout == Layout::kHalves) run(rotary_kernel<T, Layout::kHalves, PAGED, kUnits>);
        else run(rotary_kernel<T, Layout::kOdd, PAGED, kUnits>);
    };
    LaunchScope scope(what, stream);
    if (many) choose(std::integral_constant<int, kEach>{});
    else choose(std::integral_constant<int, 1>{});
    return check_hip(hipGetLastError(), what);
}

int check_sizes(const char* what, uint64_t tokens, uint32_t q_heads, uint32_t kv_heads, uint32_t dim, uint32_t rotary_dim, float factor,
                const int32_t* requests, const int32_t* shifts, uint32_t num_shifts) {
    if (dim == 0 || dim % 8 != 0 || dim > kMostDim)
        return set_error(kUnsupported, "%s: the head size must be a multiple of 8 up to %u", what, kMostDim);
    if (rotary_dim == 0 || rotary_dim % 2 != 0 || rotary_dim > dim)
        return set_error(kInvalidArgument, "%s: the turned items must be an even number, at most the head size", what);
    if (q_heads > 65535 || kv_heads > 65535 || q_heads + kv_heads == 0)
        return set_error(kInvalidArgument, "%s: no heads, or more than 65535", what);
    if (tokens > 0x7FFFFFFFull || num_shifts > 0x7FFFFFFFu) return set_error(kInvalidArgument, "%s: too many tokens or requests", what);
    if (shifts && !requests) return set_error(kInvalidArgument, "%s: shifts need the rows' requests", what);
    if (!std::isfinite(factor)) return set_error(kInvalidArgument, "%s: the factor must be finite", what);
    return kOk;
}

// The same rows, or others.
bool same_or_apart(const lcpp_hip_rows* in, const lcpp_hip_rows* out) {
    return in->data != out->data || (in->token_stride == out->token_stride && in->head_stride == out->head_stride);
}

template <typename T>
int rotary(const lcpp_hip_rows* q, const lcpp_hip_rows* k, const int32_t* positions, const int32_t* requests, const int32_t* shifts,
           uint32_t num_shifts, const double* frequencies, const lcpp_hip_rows* q_out, const lcpp_hip_rows* k_out, uint64_t tokens,
           uint32_t q_heads, uint32_t kv_heads, uint32_t dim, uint32_t rotary_dim, int interleaved, int inverse, float factor,
           void* stream_ptr) {
    const char* what = "rotary";
    if (int st = check_sizes(what, tokens, q_heads, kv_heads, dim, rotary_dim, factor, requests, shifts, num_shifts); st != kOk) return st;
    if (tokens == 0) return kOk;
    if (!positions || !frequencies) return set_error(kInvalidArgument, "%s: null positions or frequencies", what);
    TurnRows rows{{}, {}, {}, {}, {}, {}, {}, nullptr, nullptr, Divider(1), 0};
    if (q_heads) {
        if (!usable(q) || !usable(q_out)) return unusable(what);
        if (!same_or_apart(q, q_out)) return set_error(kInvalidArgument, "%s: rows turned in place keep their strides", what);
        rows.q = rows_of(q);
        rows.q_out = rows_of(q_out);
    }
    if (kv_heads) {
        if (!usable(k) || !usable(k_out)) return unusable(what);
        if (!same_or_apart(k, k_out)) return set_error(kInvalidArgument, "%s: rows turned in place keep their strides", what);
        rows.k = rows_of(k);
        rows.k_out = rows_of(k_out);
    }
    return launch<T, false>(what, rows, positions, requests, shifts, num_shifts, frequencies, tokens, q_heads, kv_heads, dim, rotary_dim,
                            interleaved != 0, inverse != 0, factor, static_cast<hipStream_t>(stream_ptr));
}

template <typename T>
int paged_write_rotary(const lcpp_hip_rows* q, const lcpp_hip_rows* key, const lcpp_hip_rows* value, const int32_t* positions,
                       const int32_t* requests, const int32_t* shifts, uint32_t num_shifts, const double* frequencies,
                       const int64_t* slots, const lcpp_hip_rows* q_out, const lcpp_hip_pages* key_cache,
                       const lcpp_hip_pages* value_cache, int32_t* slot_positions, uint64_t tokens, uint32_t q_heads, uint32_t kv_heads,
                       uint32_t dim, uint32_t rotary_dim, int interleaved, float factor, uint32_t page_size, uint32_t pages,
                       void* stream_ptr) {
    const char* what = "paged_write_rotary";
    if (int st = check_sizes(what, tokens, q_heads, kv_heads, dim, rotary_dim, factor, requests, shifts, num_shifts); st != kOk) return st;
    if (kv_heads == 0) return set_error(kInvalidArgument, "%s: no key heads", what);
    if (page_size == 0 || page_size > 0x7FFFFFFFu) return set_error(kInvalidArgument, "%s: page size out of range", what);
    if (tokens == 0) return kOk;
    if (!positions || !frequencies || !slots) return set_error(kInvalidArgument, "%s: null positions, frequencies or slots", what);
    if (!usable(key) || !usable(value) || !usable(key_cache) || !usable(value_cache)) return unusable(what);
    TurnRows rows{{}, rows_of(key), rows_of(value), {}, {}, pages_of(key_cache), pages_of(value_cache), slots, slot_positions,
                  Divider(page_size), static_cast<int64_t>(pages)};
    if (q_heads) {
        if (!usable(q) || !usable(q_out)) return unusable(what);
        if (!same_or_apart(q, q_out)) return set_error(kInvalidArgument, "%s: rows turned in place keep their strides", what);
        rows.q = rows_of(q);
        rows.q_out = rows_of(q_out);
    }
    return launch<T, true>(what, rows, positions, requests, shifts, num_shifts, frequencies, tokens, q_heads, kv_heads, dim, rotary_dim,
                           interleaved != 0, false, factor, static_cast<hipStream_t>(stream_ptr));
}

// Frequencies of the pairs, in radians a position: base^(-2 i / R), or stretched for contexts `scale` times as long as the
// trained ones.
int rotary_frequencies(double* out, uint32_t rotary_dim, double base, int scaling, double scale, double trained, double low, double high) {
    const char* what = "rotary_frequencies";
    if (!out || rotary_dim == 0 || rotary_dim % 2 != 0) return set_error(kInvalidArgument, "%s: an even number of items is needed", what);
    if (!(base > 0.0) || !std::isfinite(base) || !(scale > 0.0) || !std::isfinite(scale))
        return set_error(kInvalidArgument, "%s: base and scale must be positive and finite", what);
    if (scaling < LCPP_HIP_ROTARY_PLAIN || scaling > LCPP_HIP_ROTARY_BANDS)
        return set_error(kInvalidArgument, "%s: unknown scaling", what);
    if (scaling == LCPP_HIP_ROTARY_BANDS && !(trained > 0.0 && std::isfinite(trained) && low >= 0.0 && high > low && std::isfinite(high)))
        return set_error(kInvalidArgument, "%s: bands need a trained length and 0 <= low < high", what);
    if (scaling == LCPP_HIP_ROTARY_BASE && rotary_dim < 4)
        return set_error(kInvalidArgument, "%s: a stretched base needs four items", what);
    constexpr double kTurn = 6.283185307179586477;
    const double dim = rotary_dim;
    if (scaling == LCPP_HIP_ROTARY_BASE) base *= std::pow(scale, dim / (dim - 2.0));
    for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / dim);
        out[i] = f;
        if (scaling == LCPP_HIP_ROTARY_LINEAR) out[i] = f / scale;
        if (scaling == LCPP_HIP_ROTARY_BANDS) {
            const double turns = trained * f / kTurn;
            const double kept = turns <= low ? 0.0 : turns >= high ? 1.0 : (turns - low) / (high - low);
            out[i] = f * (kept + (1.0 - kept) / scale);
        }
    }
    return kOk;
}

}  // namespace
}  // namespace attention
}  // namespace lcpp_hip

using namespace lcpp_hip;

extern "C" {

int lcpp_hip_rotary_frequencies(double* out, uint32_t rotary_dim, double base, int scaling, double scale, double trained, double low,
                                double high) {
    return attention::rotary_frequencies(out, rotary_dim, base, scaling, scale, trained, low, high);
}

#define LCPP_HIP_DEFINE_ROTARY(S, T)                                                                                          \
    int lcpp_hip_rotary_##S(const lcpp_hip_rows* q, const lcpp_hip_rows* k, const int32_t* positions, const int32_t* requests, \
                            const int32_t* shifts, uint32_t num_shifts, const double* frequencies, const lcpp_hip_rows* q_out, \
                            const lcpp_hip_rows* k_out, uint64_t tokens, uint32_t q_heads, uint32_t kv_heads,                 \
                            uint32_t head_dim, uint32_t rotary_dim, int interleaved, int inverse, float factor, void* stream) { \
        return attention::rotary<attention::T>(q, k, positions, requests, shifts, num_shifts, frequencies, q_out, k_out, tokens, \
                                               q_heads, kv_heads, head_dim, rotary_dim, interleaved, inverse, factor, stream); \
    }                                                                                                                         \
    int lcpp_hip_paged_write_rotary_##S(                                                                                      \
        const lcpp_hip_rows* q, const lcpp_hip_rows* key, const lcpp_hip_rows* value, const int32_t* positions,               \
        const int32_t* requests, const int32_t* shifts, uint32_t num_shifts, const double* frequencies, const int64_t* slots, \
        const lcpp_hip_rows* q_out, const lcpp_hip_pages* key_cache, const lcpp_hip_pages* value_cache,                       \
        int32_t* slot_positions, uint64_t tokens, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim,                     \
        uint32_t rotary_dim, int interleaved, float factor, uint32_t page_size, uint32_t pages, void* stream) {               \
        return attention::paged_write_rotary<attention::T>(q, key, value, positions, requests, shifts, num_shifts, frequencies, \
                                                           slots, q_out, key_cache, value_cache, slot_positions, tokens,      \
                                                           q_heads, kv_heads, head_dim, rotary_dim, interleaved, factor,      \
                                                           page_size, pages, stream);                                         \
    }
LCPP_HIP_DEFINE_ROTARY(bf16, Bf16)
LCPP_HIP_DEFINE_ROTARY(f16, F16)
#undef LCPP_HIP_DEFINE_ROTARY

}  // extern "C"
