// Softmax weights that a step's rows gave to each key of a paged cache, added to the keys' sums:
//
//   w_j = decay * w_j (keys that had a sum) + sum over heads h and rows i that see j of exp(scale q_ih k_jg - lse_ih)
//
// with the log-sums that attention over the same pages gave, and g the key head of h.  Scores, exponentials and sums are f32;
// nothing is rounded to 16 bits.  Each key's sum has one owner and one order.
//
// Each key is read once; 2 * dim operations a row, head and key.  Matrix instruction: 16x16x32, rows of queries by keys: lane
// l has key l % 16 of the result, rows 4 (l / 16) .. + 3, so that a key's weights of 16 rows lie in four lanes' registers and are
// added up there; lanes meet once, at the end.
#include "attention.hpp"

namespace lcpp_hip {
namespace attention {
namespace {

constexpr int kWeightWaves = 4;
constexpr int kWeightBlock = kWeightWaves * kWave;
constexpr int kUnitKeys = 64;           // of a workgroup at a time
constexpr int kGroups = kUnitKeys / 16;  // matrix products side by side
constexpr int kRowsAtOnce = 16;

using Acc = F32x4;

template <typename T>
__device__ __forceinline__ Acc product(U32x4 a, U32x4 b, Acc c) {
    if constexpr (std::is_same_v<T, Bf16>)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(typename T::Vec8, a), __builtin_bit_cast(typename T::Vec8, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(typename T::Vec8, a), __builtin_bit_cast(typename T::Vec8, b), c, 0,
                                                      0, 0);
}

struct Weigh {
    int requests;
    int q_tokens;
    int q_heads;
    int kv_heads;
    int dim;
    Divider group;
    Divider page_size;
    int pages;
    int64_t table_stride;
    int table_width;
    uint32_t parts;  // workgroups of a request
    int splits;  // waves that share a key head's rows
    float scale;
    float decay;
};

template <typename T, int DP>
__global__ __launch_bounds__(kWeightBlock) void attention_weights_kernel(Rows q, Pages key_cache, const int32_t* __restrict__ block_table,
                                                                         const int32_t* __restrict__ q_offsets,
                                                                         const int32_t* __restrict__ kv_lengths,
                                                                         const int32_t* __restrict__ known_lengths,
                                                                         const uint64_t* __restrict__ tree, const float* __restrict__ lse,
                                                                         const float* weights_in, float* weights_out, Weigh p) {
    constexpr int kSteps = DP / 32;
    __shared__ float sums[kWeightWaves][kUnitKeys];
    const int request = static_cast<int>(blockIdx.x / p.parts), part = static_cast<int>(blockIdx.x % p.parts), lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    int begin = q_offsets[request], end = q_offsets[request + 1];
    begin = begin < 0 ? 0 : begin > p.q_tokens ? p.q_tokens : begin;
    end = end < begin ? begin : end > p.q_tokens ? p.q_tokens : end;
    const int group = p.q_heads / p.kv_heads, rows = (end - begin) * group;
    const int length = kv_lengths[request] < 0 ? 0 : kv_lengths[request];
    const int64_t room = static_cast<int64_t>(p.table_width) * p.page_size.by;
    const int held = length < room ? length : static_cast<int>(room);
    const int ahead = length - (end - begin);  // keys before the new tokens' own
    const int known = known_lengths != nullptr ? known_lengths[request] : ahead;
    const int32_t* table = block_table + request * p.table_stride;
    const float c = p.scale * kLog2e;
    const int column = lane % 16, quarter = lane / 16;

    for (int64_t unit = part; unit * kUnitKeys < held; unit += p.parts) {
        const int key0 = static_cast<int>(unit) * kUnitKeys;
        const char* key[kGroups];
        bool there[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int j = key0 + 16 * g + column, at = j < held ? j : held - 1;
            const uint32_t cell = p.page_size(at);
            const int page = table[cell];
            there[g] = page >= 0 && page < p.pages;
            key[g] = key_cache.at(there[g] ? page : 0, there[g] ? at - static_cast<int>(cell * p.page_size.by) : 0, 0);
        }
        // Rows that see every key of the unit need no masks.
        const bool masked = key0 + kUnitKeys - 1 > (tree != nullptr ? ahead - 1 : ahead);
        float sum[kGroups] = {};
        for (int job = wave; job < p.kv_heads * p.splits; job += kWeightWaves) {
            const int kv_head = job % p.kv_heads, split = job / p.kv_heads;
            U32x4 k[kGroups][kSteps];
#pragma unroll
            for (int g = 0; g < kGroups; ++g)
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
                    k[g][s] = load_chunk(key[g] + kv_head * key_cache.head_bytes, 4 * s + quarter, p.dim, there[g]);
            for (int row0 = split * kRowsAtOnce; row0 < rows; row0 += p.splits * kRowsAtOnce) {
                const int mine = row0 + column;
                const int my_token = static_cast<int>(p.group(mine));
                const char* q_row = q.at(begin + my_token, kv_head * group + mine - my_token * group);
                U32x4 a[kSteps];
#pragma unroll
                for (int s = 0; s < kSteps; ++s) a[s] = load_chunk(q_row, 4 * s + quarter, p.dim, mine < rows);
                float base[4];
                bool none[4];
                int token[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = row0 + 4 * quarter + r;
                    token[r] = static_cast<int>(p.group(row));
                    float l = -INFINITY;
                    if (row < rows)
                        l = lse[static_cast<int64_t>(kv_head * group + row - token[r] * group) * p.q_tokens + begin + token[r]];
                    none[r] = l == -INFINITY;
                    base[r] = none[r] ? INFINITY : l * kLog2e;  // rows that are not there, or see nothing, weigh nothing
                }
                Acc acc[kGroups] = {};
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) acc[g] = product<T>(a[s], k[g][s], acc[g]);
                if (!masked && row0 + kRowsAtOnce <= rows) {
#pragma unroll
                    for (int g = 0; g < kGroups; ++g)
#pragma unroll
                        for (int r = 0; r < 4; ++r) sum[g] += exp2_fast(acc[g][r] * c - base[r]);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool real = row0 + 4 * quarter + r < rows && !none[r];
                        const uint64_t word = real && tree != nullptr ? tree[begin + token[r]] : 0;
#pragma unroll
                        for (int g = 0; g < kGroups; ++g) {
                            const int fresh = key0 + 16 * g + column - ahead;  // which of the new keys
                            const bool seen = tree == nullptr ? fresh <= token[r] : fresh < 0 || (fresh < 64 && (word >> fresh & 1) != 0);
                            sum[g] += real && seen ? exp2_fast(acc[g][r] * c - base[r]) : 0.f;
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            sum[g] += __shfl_xor(sum[g], 16);
            sum[g] += __shfl_xor(sum[g], 32);
            if (quarter == 0) sums[wave][16 * g + column] = sum[g];
        }
        __syncthreads();
        if (threadIdx.x < kUnitKeys) {
            const int j = key0 + static_cast<int>(threadIdx.x);
            float total = 0.f;
#pragma unroll
            for (int w = 0; w < kWeightWaves; ++w) total += sums[w][threadIdx.x];
            if (j < held) {
                const uint32_t cell = p.page_size(j);
                const int page = table[cell];
                if (page >= 0 && page < p.pages) {
                    const int64_t slot = static_cast<int64_t>(page) * p.page_size.by + (j - cell * p.page_size.by);
                    weights_out[slot] = j < known && weights_in != nullptr ? weights_in[slot] * p.decay + total : total;
                }
            }
        }
        __syncthreads();
    }
}

// Workgroups wanted: a request's units are dealt out to so many that all requests make about this number.
constexpr uint64_t kWeightGrid = 8192;

template <typename T>
int paged_weights(void* temp, size_t temp_bytes, const lcpp_hip_rows* q, const lcpp_hip_pages* key_cache, const int32_t* block_table,
                  uint64_t table_stride, uint32_t table_width, const int32_t* q_offsets, const int32_t* kv_lengths,
                  const int32_t* known_lengths, const uint64_t* tree, const float* lse, const float* weights_in, float* weights_out,
                  uint32_t requests, uint64_t q_tokens, uint64_t max_kv_length, uint32_t q_heads, uint32_t kv_heads, uint32_t dim,
                  uint32_t page_size, uint32_t pages, float scale, float decay, void* stream_ptr) {
    const char* what = "attention_paged_weights";
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (q_heads == 0 || kv_heads == 0 || q_heads % kv_heads != 0 || q_heads > 65535)
        return set_error(kInvalidArgument, "%s: query heads must be a multiple of the key heads, and at most 65535", what);
    if (dim == 0 || dim % 8 != 0 || dim > 128)
        return set_error(kUnsupported, "%s: the head size must be a multiple of 8 up to 128", what);
    if (page_size == 0 || page_size > 0x7FFFFFFFu || pages > 0x7FFFFFFFu)
        return set_error(kInvalidArgument, "%s: page size or page count out of range", what);
    if (table_width > table_stride || table_width > 0x7FFFFFFFu || table_stride > 0x7FFFFFFFFFFull)
        return set_error(kInvalidArgument, "%s: a block table's row must hold its width", what);
    if (q_tokens > 0x7FFFFFFFull || q_tokens * (q_heads / kv_heads) > kMostKeys || requests > 0x7FFFFFu)
        return set_error(kInvalidArgument, "%s: too many tokens or requests", what);
    if (max_kv_length > kMostKeys || static_cast<uint64_t>(table_width) * page_size > kMostKeys)
        return set_error(kInvalidArgument, "%s: requests too long", what);
    if (!(scale > 0.f) || scale == INFINITY) return set_error(kInvalidArgument, "%s: the scale must be positive and finite", what);
    if (!(decay >= 0.f) || decay == INFINITY) return set_error(kInvalidArgument, "%s: the decay must be finite, and not negative", what);
    if (requests == 0) return kOk;
    if (!q_offsets || !kv_lengths || (table_width && !block_table) || !weights_out)
        return set_error(kInvalidArgument, "%s: null offsets, lengths, block table or sums", what);
    if (!usable(key_cache)) return unusable(what);
    if (q_tokens && (!usable(q) || !lse))
        return usable(q) ? set_error(kInvalidArgument, "%s: null lse", what) : unusable(what);
    const size_t needed = lcpp_hip_attention_paged_weights_temp_bytes(requests, q_tokens, max_kv_length, q_heads, kv_heads, dim);
    if (temp_bytes < needed || (needed && !temp)) return set_error(kTempTooSmall, "%s: temp storage too small", what);
    const uint64_t units = ceil_div(max_kv_length ? max_kv_length : 1, kUnitKeys), wanted = ceil_div(kWeightGrid, requests);
    const int splits = kv_heads >= kWeightWaves ? 1 : static_cast<int>(kWeightWaves / kv_heads);
    const Weigh p{static_cast<int>(requests), static_cast<int>(q_tokens), static_cast<int>(q_heads), static_cast<int>(kv_heads),
                  static_cast<int>(dim), Divider(q_heads / kv_heads), Divider(page_size), static_cast<int>(pages),
                  static_cast<int64_t>(table_stride), static_cast<int>(table_width),
                  static_cast<uint32_t>(units < wanted ? units : wanted), splits, scale, decay};
    const Rows q_rows = q_tokens ? rows_of(q) : Rows{};
    LaunchScope scope(what, stream);
    auto* kernel = dim <= 64   ? attention_weights_kernel<T, 64>
                   : dim <= 96 ? attention_weights_kernel<T, 96>
                               : attention_weights_kernel<T, 128>;
    kernel<<<p.parts * requests, kWeightBlock, 0, stream>>>(
        q_rows, pages_of(key_cache), block_table, q_offsets, kv_lengths, known_lengths, tree, lse, weights_in, weights_out, p);
    return check_hip(hipGetLastError(), "attention_paged_weights launch");
}

}  // namespace
}  // namespace attention
}  // namespace lcpp_hip

using namespace lcpp_hip;

extern "C" {

size_t lcpp_hip_attention_paged_weights_temp_bytes(uint32_t, uint64_t, uint64_t, uint32_t, uint32_t, uint32_t) { return 0; }

#define LCPP_HIP_DEFINE_ATTENTION_WEIGHTS(S, T)                                                                               \
    int lcpp_hip_attention_paged_weights_##S(                                                                                 \
        void* temp, size_t temp_bytes, const lcpp_hip_rows* q, const lcpp_hip_pages* key_cache, const int32_t* block_table,   \
        uint64_t table_stride, uint32_t table_width, const int32_t* q_offsets, const int32_t* kv_lengths,                     \
        const int32_t* known_lengths, const uint64_t* tree, const float* lse, const float* weights_in, float* weights_out,    \
        uint32_t requests, uint64_t q_tokens, uint64_t max_kv_length, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, \
        uint32_t page_size, uint32_t pages, float scale, float decay, void* stream) {                                         \
        return attention::paged_weights<attention::T>(temp, temp_bytes, q, key_cache, block_table, table_stride, table_width, \
                                                      q_offsets, kv_lengths, known_lengths, tree, lse, weights_in, weights_out, \
                                                      requests, q_tokens, max_kv_length, q_heads, kv_heads, head_dim,         \
                                                      page_size, pages, scale, decay, stream);                                \
    }
LCPP_HIP_DEFINE_ATTENTION_WEIGHTS(bf16, Bf16)
LCPP_HIP_DEFINE_ATTENTION_WEIGHTS(f16, F16)
#undef LCPP_HIP_DEFINE_ATTENTION_WEIGHTS

}  // extern "C"
