// Causal or full attention over packed sequences with grouped heads.
//
//   S = scale q k^T,  row i of n sees key j of m where j <= i + m - n (causal) or any j,
//   P = softmax(S),  O = P V,  lse = log sum exp S;  a row that sees nothing has O = 0 and lse = -inf.
//
// One pass over the keys: with t the running maximum of a row's scores, l = sum exp(S - t) and A = sum exp(S - t) v are
// scaled by exp(t - t') where t moves to t', and O = A / l, lse = t + log l.  S, t, l and A are f32; the weights exp(S - t)
// are rounded to 16 bits for the product with V, whose operands are 16 bits wide (l adds them up unrounded).
//
// 4 * dim operations a pair of row and key, and little to read (each row of K and V once for 128 query rows): long
// sequences are bound by the matrix cores.  One of 16,384 rows, 16 heads of 128: 1,080 to 1,120 us, 980 to 1,020 TFLOP/s,
// where a large library product reaches 1,186; the clock falls as low as 1.7 GHz under it, so what is left is power.
// Uneven prompts of 60 to 2,500 rows (32 heads of 128) take 145 to 165 us, 630 to 710 TFLOP/s: their last tiles are part empty, and a
// workgroup of few keys is latency.  Seven prompts of up to 200 rows: 8.2 us, all of it latency.
//
// A workgroup: four waves of 32 rows and 64 keys at a time, keys and values shared in LDS (33 KB a set of buffers at 128
// items, two sets, so two workgroups a compute unit).  Eight waves a workgroup, and a wave's products and exponentials
// interleaved by hand, took the same time; raised wave priority too.
#include "attention_packed.hpp"

namespace lcpp_hip {
namespace attention {
namespace {

// DP, the head size that registers and LDS are laid out for: 64, 96 or 128 (heads of 80 in 96 items 16.8 us, in 128 18.9;
// of 64 in 64 items 9.8 us, in 128 11.8).  At 64, three waves a SIMD need no scratch; four took the same time.
template <typename T, int DP>
__global__ __launch_bounds__(kBlock, DP <= 64 ? 3 : 2) void attention_packed_kernel(Rows q, Rows k, Rows v, Rows out, float* __restrict__ lse,
                                                                     const int32_t* __restrict__ q_offsets,
                                                                     const int32_t* __restrict__ k_offsets, Shape shape,
                                                                     int tiles, bool ordered_tiles) {
    constexpr int kTileBytes = Tile<DP>::bytes(kKeyTile);
    __shared__ __attribute__((aligned(16))) char k_even[kTileBytes];
    __shared__ __attribute__((aligned(16))) char v_even[kTileBytes];
    __shared__ __attribute__((aligned(16))) char k_odd[kTileBytes];
    __shared__ __attribute__((aligned(16))) char v_odd[kTileBytes];
    __shared__ int broken;  // whether the sums of some wave are not finite
    if (threadIdx.x == 0) broken = 0;
    // Workgroups go to the 8 XCDs in turn: with the key head as the fastest number, those of a key head share an L2.
    // Tiles that see more keys come first.
    const int group = shape.q_heads / shape.kv_heads;
    const int kv_head = blockIdx.x % shape.kv_heads;
    const int head = kv_head * group + blockIdx.x / shape.kv_heads % group;
    const int number = static_cast<int>(blockIdx.x / shape.q_heads);
    Span rows, keys;
    int row0;
    if (ordered_tiles) {
        if (!take_ordered_tile<kRowTile>(q_offsets, k_offsets, shape, number, rows, keys, row0)) return;
    } else {
        const TilePlace place = find_tile(q_offsets, shape.sequences, 1, kRowTile, tiles - 1 - number);
        if (place.sequence < 0) return;
        rows = span_of(q_offsets, place.sequence, shape.q_tokens);
        keys = span_of(k_offsets, place.sequence, shape.k_tokens);
        row0 = place.tile * kRowTile;
    }
    if (row0 >= rows.size) return;
    const int lane = threadIdx.x % kWave, half = lane / 32;
    const int row = row0 + threadIdx.x / kWave * kRowsPerWave + lane % 32;
    const bool there = row < rows.size;
    const RowRange range(shape, rows, keys, row0, row);
    const float c = shape.scale * kLog2e;

    U32x4 qf[DP / 16];
    load_row<DP>(qf, q, rows.begin + row, head, there, shape.dim);
    for (char* tile : {k_even, v_even, k_odd, v_odd}) clear_past<DP, kKeyTile>(tile, shape.dim);
    const PackedRows<DP, kKeyTile> key_rows(k.at(keys.begin, kv_head), k.token_bytes, keys.size, shape.dim);
    const PackedRows<DP, kKeyTile> value_rows(v.at(keys.begin, kv_head), v.token_bytes, keys.size, shape.dim);
    const auto pass = [&](RowState<DP>& state, int stop) {
        state = {};
        state.top = -INFINITY;
        forward_keys<T, DP>(state, k_even, v_even, k_odd, v_odd, key_rows, value_rows, qf, c, 0, stop, range.wave_end, range.full,
                            [&](int k0) { return first_keys(range.count, k0); });
    };
    const auto store = [&](const RowState<DP>& state) {
        const float total = halves_sum(state.total);
        if (!there) return;
        store_row<T, DP>(out, rows.begin + row, head, state.acc, total == 0.f ? 0.f : 1.f / total, shape.dim);
        if (lse != nullptr && half == 0)
            lse[static_cast<int64_t>(head) * shape.q_tokens + rows.begin + row] = row_lse<T>(state.top, total, shape.scale);
    };
    RowState<DP> state;
    pass(state, range.end);
    store(state);  // (before waves wait for each other)
    const int clean = clean_end(0, range.full, range.end);
    if (clean < range.end && block_any(any_not_finite(state.acc), &broken)) {
        pass(state, clean);
        for (int j = clean; j < range.wave_end; ++j)
            careful_key<T, DP>(state, qf, k.at(keys.begin + static_cast<int64_t>(j), kv_head), v.at(keys.begin + static_cast<int64_t>(j), kv_head),
                               shape.dim, c, j < range.count);
        store(state);
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------
constexpr unsigned kResident = 512;  // workgroups that run at once, two a compute unit

template <typename T>
int packed(const lcpp_hip_rows* q, const lcpp_hip_rows* k, const lcpp_hip_rows* v, const int32_t* q_offsets,
           const int32_t* k_offsets, const lcpp_hip_rows* out, float* lse, uint32_t sequences, uint64_t q_tokens,
           uint64_t k_tokens, uint32_t q_heads, uint32_t kv_heads, uint32_t dim, float scale, int causal, void* stream_ptr) {
    const char* what = "attention_packed";
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (int st = check_shape(what, sequences, q_tokens, k_tokens, q_heads, kv_heads, dim, scale); st != kOk) return st;
    if (sequences == 0 || q_tokens == 0) return kOk;
    if (!q_offsets || !k_offsets) return set_error(kInvalidArgument, "%s: null offsets", what);
    if (!usable(q) || !usable(out) || (k_tokens && (!usable(k) || !usable(v))))
        return unusable(what);
    if (k_tokens && (too_wide(k) || too_wide(v))) return refuse_wide(what);
    unsigned tiles, grid;
    if (int st = check_grid(what, q_tokens, kRowTile, sequences, q_heads, tiles, grid); st != kOk) return st;
    const Shape shape{static_cast<int>(sequences), static_cast<int>(q_tokens), static_cast<int>(k_tokens),
                      static_cast<int>(q_heads), static_cast<int>(kv_heads), static_cast<int>(dim), scale, causal != 0};
    // Several sequences, one for each lane of a wave at most, and more workgroups than run at once: see OrderedTile.
    const bool ordered_tiles = sequences > 1 && sequences <= kWave && grid > kResident;
    const Rows none{nullptr, 0, 0};
    const Rows kr = k_tokens ? rows_of(k) : none, vr = k_tokens ? rows_of(v) : none;
    LaunchScope scope("attention_packed", stream);
    auto* kernel = dim <= 64   ? attention_packed_kernel<T, 64>
                   : dim <= 96 ? attention_packed_kernel<T, 96>
                               : attention_packed_kernel<T, 128>;
    kernel<<<grid, kBlock, 0, stream>>>(rows_of(q), kr, vr, rows_of(out), lse, q_offsets, k_offsets, shape, tiles, ordered_tiles);
    return check_hip(hipGetLastError(), "attention_packed launch");
}

}  // namespace
}  // namespace attention
}  // namespace lcpp_hip

using namespace lcpp_hip;

extern "C" {

size_t lcpp_hip_attention_packed_temp_bytes(uint32_t sequences, uint64_t q_tokens, uint64_t k_tokens, uint32_t q_heads,
                                            uint32_t kv_heads, uint32_t head_dim) {
    (void)sequences, (void)q_tokens, (void)k_tokens, (void)q_heads, (void)kv_heads, (void)head_dim;
    return 0;
}

#define LCPP_HIP_DEFINE_ATTENTION(S, T)                                                                                     \
    int lcpp_hip_attention_packed_##S(void* temp, size_t temp_bytes, const lcpp_hip_rows* q, const lcpp_hip_rows* k,        \
                                      const lcpp_hip_rows* v, const int32_t* q_offsets, const int32_t* k_offsets,           \
                                      const lcpp_hip_rows* out, float* lse, uint32_t sequences, uint64_t q_tokens,          \
                                      uint64_t k_tokens, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim,            \
                                      float scale, int causal, void* stream) {                                              \
        (void)temp, (void)temp_bytes;                                                                                       \
        return attention::packed<attention::T>(q, k, v, q_offsets, k_offsets, out, lse, sequences, q_tokens, k_tokens,      \
                                               q_heads, kv_heads, head_dim, scale, causal, stream);                         \
    }
LCPP_HIP_DEFINE_ATTENTION(bf16, Bf16)
LCPP_HIP_DEFINE_ATTENTION(f16, F16)
#undef LCPP_HIP_DEFINE_ATTENTION

}  // extern "C"
