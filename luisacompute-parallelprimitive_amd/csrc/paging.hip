// The paged cache's bookkeeping: one step's offsets, positions, pages and slots from the requests' lengths, and the
// step's rows into their slots.
#include "attention.hpp"

namespace lcpp_hip {
namespace {

constexpr int kScanBlock = 1024;
constexpr int kTokenBlock = 256;

struct Plan {
    int requests;
    int page_size;
    int num_free;
    int table_width;
    int64_t table_stride;
    int64_t max_tokens;
};

__device__ __forceinline__ int length_at(const int32_t* lengths, int i) { return lengths[i] > 0 ? lengths[i] : 0; }

// Pages of the table that `length` tokens fill or begin.
__device__ __forceinline__ uint32_t pages_of(int64_t length, const Plan& p) {
    const int64_t n = (length + p.page_size - 1) / p.page_size;
    return static_cast<uint32_t>(n < p.table_width ? n : p.table_width);
}

// One workgroup: prefix sums of new tokens (low word) and of new pages (high word) together.
__global__ __launch_bounds__(kScanBlock) void page_plan_scan_kernel(const int32_t* __restrict__ cached,
                                                                    const int32_t* __restrict__ fresh, uint32_t* __restrict__ first_page,
                                                                    int32_t* __restrict__ offsets, int32_t* __restrict__ kv_lengths,
                                                                    int32_t* __restrict__ counts, Plan p) {
    __shared__ uint64_t wave_sums[kScanBlock / kWave];
    uint64_t carry = 0;
    for (int base = 0; base < p.requests; base += kScanBlock) {
        const int r = base + static_cast<int>(threadIdx.x);
        uint64_t mine = 0;
        if (r < p.requests) {
            const int64_t held = length_at(cached, r), add = length_at(fresh, r), all = held + add;
            kv_lengths[r] = static_cast<int32_t>(all < INT32_MAX ? all : INT32_MAX);
            mine = static_cast<uint64_t>(pages_of(all, p) - pages_of(held, p)) << 32 | static_cast<uint64_t>(add);
        }
        const uint64_t inclusive = wave_inclusive_scan(mine, SumOp{});
        if (threadIdx.x % kWave == kWave - 1) wave_sums[threadIdx.x / kWave] = inclusive;
        __syncthreads();
        uint64_t before = carry, all = 0;
        for (int i = 0; i < kScanBlock / kWave; ++i) {
            if (i < static_cast<int>(threadIdx.x / kWave)) before += wave_sums[i];
            all += wave_sums[i];
        }
        __syncthreads();
        const uint64_t exclusive = before + inclusive - mine;
        if (r < p.requests) {
            offsets[r] = static_cast<int32_t>(exclusive);
            first_page[r] = static_cast<uint32_t>(exclusive >> 32);
        }
        carry += all;
    }
    if (threadIdx.x == 0) {
        offsets[p.requests] = static_cast<int32_t>(carry);
        counts[0] = static_cast<int32_t>(carry);
        counts[1] = static_cast<int32_t>(carry >> 32);
    }
}

// A thread per token.  A page is new to the table where it begins at or past the cached length, and then its first
// position is a new token's: that token enters it.
__global__ __launch_bounds__(kTokenBlock) void page_plan_tokens_kernel(
    const int32_t* __restrict__ cached, const uint32_t* __restrict__ first_page, const int32_t* __restrict__ offsets,
    const int32_t* __restrict__ free_pages, int32_t* __restrict__ block_table, int32_t* __restrict__ token_request,
    int32_t* __restrict__ token_position, int64_t* __restrict__ token_slot, Plan p) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kTokenBlock + threadIdx.x;
    if (t >= p.max_tokens) return;
    if (t >= offsets[p.requests]) {
        token_request[t] = -1;
        token_position[t] = 0;
        token_slot[t] = -1;
        return;
    }
    // The last request that begins at or before t: empty requests before it share its beginning.
    int low = 0, high = p.requests;
    while (high - low > 1) {
        const int middle = low + (high - low) / 2;
        if (offsets[middle] <= t) low = middle;
        else high = middle;
    }
    const int64_t held = length_at(cached, low), position = held + t - offsets[low];
    const int64_t cell = position / p.page_size;
    const int within = static_cast<int>(position - cell * p.page_size);
    int page = -1;
    if (cell >= 0 && cell < p.table_width) {
        int32_t* entry = block_table + low * p.table_stride + cell;
        const uint32_t have = pages_of(held, p);
        if (cell >= have) {
            const uint32_t index = first_page[low] + static_cast<uint32_t>(cell) - have;
            if (index < static_cast<uint32_t>(p.num_free)) page = free_pages[index];
            if (within == 0) *entry = page;
        } else {
            page = *entry;
        }
    }
    token_request[t] = low;
    token_position[t] = static_cast<int32_t>(position);
    token_slot[t] = page < 0 ? -1 : static_cast<int64_t>(page) * p.page_size + within;
}

// ---- rows into pages ---------------------------------------------------------------------------------------------
__global__ __launch_bounds__(kTokenBlock) void paged_write_kernel(attention::Rows key, attention::Rows value,
                                                                  attention::Pages key_cache, attention::Pages value_cache, const int64_t* __restrict__ slots,
                                                                  int64_t tokens, int heads, int chunks, int page_size, int64_t pages) {
    using attention::U32x4;
    const int per = heads * chunks;
    const int64_t items = tokens * per, stride = static_cast<int64_t>(gridDim.x) * kTokenBlock;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * kTokenBlock + threadIdx.x; at < items; at += stride) {
        const int64_t token = at / per;
        const int rest = static_cast<int>(at - token * per), head = rest / chunks, chunk = rest % chunks;
        const int64_t slot = slots[token];
        if (slot < 0) continue;
        const int64_t page = slot / page_size, within = slot % page_size;
        if (page >= pages) continue;
        const U32x4 k = *reinterpret_cast<const U32x4*>(key.at(token, head) + chunk * 16);
        const U32x4 v = *reinterpret_cast<const U32x4*>(value.at(token, head) + chunk * 16);
        *reinterpret_cast<U32x4*>(key_cache.at(page, within, head) + chunk * 16) = k;
        *reinterpret_cast<U32x4*>(value_cache.at(page, within, head) + chunk * 16) = v;
    }
}

int page_plan(void* temp, size_t temp_bytes, const int32_t* cached, const int32_t* fresh, uint32_t requests, uint32_t page_size,
              const int32_t* free_pages, uint32_t num_free, int32_t* block_table, uint64_t table_stride, uint32_t table_width,
              int32_t* offsets, int32_t* kv_lengths, int32_t* token_request, int32_t* token_position, int64_t* token_slot,
              uint64_t max_tokens, int32_t* counts, void* stream_ptr) {
    const char* what = "page_plan";
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (page_size == 0 || page_size > 0x7FFFFFFFu) return set_error(kInvalidArgument, "%s: page size out of range", what);
    if (requests > 0x7FFFFFFu || num_free > 0x7FFFFFFFu || max_tokens > 0x7FFFFFFFull)
        return set_error(kInvalidArgument, "%s: too many requests, pages or tokens", what);
    if (table_width > table_stride || table_width > 0x7FFFFFFFu)
        return set_error(kInvalidArgument, "%s: a block table's row must hold its width", what);
    if (!offsets || !counts) return set_error(kInvalidArgument, "%s: null offsets or counts", what);
    if (requests && (!cached || !fresh || !kv_lengths)) return set_error(kInvalidArgument, "%s: null lengths", what);
    if (requests && table_width && !block_table) return set_error(kInvalidArgument, "%s: null block table", what);
    if (num_free && !free_pages) return set_error(kInvalidArgument, "%s: null free list", what);
    if (max_tokens && (!token_request || !token_position || !token_slot))
        return set_error(kInvalidArgument, "%s: null token outputs", what);
    const size_t needed = lcpp_hip_page_plan_temp_bytes(requests);
    if (temp_bytes < needed || (needed && !temp)) return set_error(kTempTooSmall, "%s: temp storage too small", what);
    const Plan p{static_cast<int>(requests), static_cast<int>(page_size), static_cast<int>(num_free), static_cast<int>(table_width),
                 static_cast<int64_t>(table_stride), static_cast<int64_t>(max_tokens)};
    uint32_t* first_page = static_cast<uint32_t*>(temp);
    {
        LaunchScope scope("page_plan_scan", stream);
        page_plan_scan_kernel<<<1, kScanBlock, 0, stream>>>(cached, fresh, first_page, offsets, kv_lengths, counts, p);
        if (int st = check_hip(hipGetLastError(), "page_plan scan launch"); st != kOk) return st;
    }
    if (max_tokens == 0) return kOk;
    LaunchScope scope("page_plan_tokens", stream);
    page_plan_tokens_kernel<<<static_cast<unsigned>(ceil_div(max_tokens, kTokenBlock)), kTokenBlock, 0, stream>>>(
        cached, first_page, offsets, free_pages, block_table, token_request, token_position, token_slot, p);
    return check_hip(hipGetLastError(), "page_plan tokens launch");
}

int paged_write(const lcpp_hip_rows* key, const lcpp_hip_rows* value, const int64_t* slots, uint64_t tokens,
                const lcpp_hip_pages* key_cache, const lcpp_hip_pages* value_cache, uint32_t kv_heads, uint32_t dim,
                uint32_t page_size, uint32_t pages, void* stream_ptr) {
    const char* what = "paged_write";
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (dim == 0 || dim % 8 != 0 || dim > 65536) return set_error(kUnsupported, "%s: the head size must be a multiple of 8", what);
    if (kv_heads == 0 || kv_heads > 65535) return set_error(kInvalidArgument, "%s: no heads, or too many", what);
    if (static_cast<uint64_t>(kv_heads) * (dim / 8) > 0x7FFFFFFFull)
        return set_error(kInvalidArgument, "%s: rows too long", what);
    if (page_size == 0 || page_size > 0x7FFFFFFFu) return set_error(kInvalidArgument, "%s: page size out of range", what);
    if (tokens > 0x7FFFFFFFull) return set_error(kInvalidArgument, "%s: too many tokens", what);
    if (tokens == 0) return kOk;
    if (!slots) return set_error(kInvalidArgument, "%s: null slots", what);
    if (!attention::usable(key) || !attention::usable(value) || !attention::usable(key_cache) || !attention::usable(value_cache))
        return attention::unusable(what);
    const int chunks = static_cast<int>(dim / 8);
    const uint64_t blocks = ceil_div(tokens * kv_heads * chunks, kTokenBlock);
    const uint64_t most = static_cast<uint64_t>(device_cu_count()) * 32;
    LaunchScope scope("paged_write", stream);
    paged_write_kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), kTokenBlock, 0, stream>>>(
        attention::rows_of(key), attention::rows_of(value), attention::pages_of(key_cache), attention::pages_of(value_cache), slots, static_cast<int64_t>(tokens),
        static_cast<int>(kv_heads), chunks, static_cast<int>(page_size), static_cast<int64_t>(pages));
    return check_hip(hipGetLastError(), "paged_write launch");
}

}  // namespace
}  // namespace lcpp_hip

using namespace lcpp_hip;

extern "C" {

size_t lcpp_hip_page_plan_temp_bytes(uint32_t requests) { return align_up(static_cast<size_t>(requests) * sizeof(uint32_t), kViewAlign); }

int lcpp_hip_page_plan(void* temp, size_t temp_bytes, const int32_t* cached_lengths, const int32_t* new_lengths, uint32_t requests,
                       uint32_t page_size, const int32_t* free_pages, uint32_t num_free, int32_t* block_table,
                       uint64_t table_stride, uint32_t table_width, int32_t* query_offsets, int32_t* kv_lengths,
                       int32_t* token_request, int32_t* token_position, int64_t* token_slot, uint64_t max_tokens,
                       int32_t* counts, void* stream) {
    return page_plan(temp, temp_bytes, cached_lengths, new_lengths, requests, page_size, free_pages, num_free, block_table,
                     table_stride, table_width, query_offsets, kv_lengths, token_request, token_position, token_slot,
                     max_tokens, counts, stream);
}

#define LCPP_HIP_DEFINE_PAGED_WRITE(S)                                                                                       \
    int lcpp_hip_paged_write_##S(const lcpp_hip_rows* key, const lcpp_hip_rows* value, const int64_t* slots, uint64_t tokens, \
                                 const lcpp_hip_pages* key_cache, const lcpp_hip_pages* value_cache, uint32_t kv_heads,      \
                                 uint32_t head_dim, uint32_t page_size, uint32_t pages, void* stream) {                      \
        return paged_write(key, value, slots, tokens, key_cache, value_cache, kv_heads, head_dim, page_size, pages, stream); \
    }
LCPP_HIP_DEFINE_PAGED_WRITE(bf16)
LCPP_HIP_DEFINE_PAGED_WRITE(f16)
#undef LCPP_HIP_DEFINE_PAGED_WRITE

}  // extern "C"
