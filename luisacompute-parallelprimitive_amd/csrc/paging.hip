// The paged cache's bookkeeping: one step's offsets, positions, pages and slots from the requests' lengths, and the
// step's rows into their slots.
#include "attention.hpp"

namespace lcpp_hip {
namespace {

constexpr int kScanBlock = 1024;
constexpr int kTokenBlock = 256;
// Requests that every workgroup scans for itself, so that a plan is one launch; more are scanned by one workgroup first.
// (64 requests: 5.3 us for two launches, 3.3 us for one; 4,096 requests and tokens: 9.0 and 6.1.)  Twelve bytes of LDS a
// request leave room for two workgroups on a compute unit.
constexpr int kRequestsPerThread = 5;
constexpr int kFusedRequests = kRequestsPerThread * kScanBlock;
// Where there are tokens for every compute unit at that (kFusedTokens): 250,000 tokens take 7.0 us with one a thread, 9.2
// with four, 600,000 13.5 and 10.1, 1.2 million 20 and 12.6.
constexpr int kTokensPerThread = 4;
constexpr uint64_t kFusedTokens = 256 * kScanBlock;

struct Plan {
    int requests;
    attention::Divider page_size;
    int num_free;
    int table_width;
    int64_t table_stride;
    int64_t max_tokens;
};

__device__ __forceinline__ uint32_t length_at(const int32_t* lengths, int i) {
    return static_cast<uint32_t>(lengths[i] > 0 ? lengths[i] : 0);
}

// Pages of the table that `length` tokens fill or begin.  Lengths and positions, sums of two lengths, are below 2^32: they are
// divided in 32 bits (divisions in 64 bits were most of a plan's time).
__device__ __forceinline__ uint32_t pages_of(uint32_t length, const Plan& p) {
    const uint32_t full = p.page_size(length), n = full + (length != full * p.page_size.by);
    return n < static_cast<uint32_t>(p.table_width) ? n : static_cast<uint32_t>(p.table_width);
}

// A request's lengths, new tokens (low word) and new pages (high word).
struct Request {
    uint32_t held, add;
    __device__ __forceinline__ void load(const int32_t* cached, const int32_t* fresh, int r) {
        held = length_at(cached, r);
        add = length_at(fresh, r);
    }
    __device__ __forceinline__ uint64_t needs(const Plan& p) const {
        return static_cast<uint64_t>(pages_of(held + add, p) - pages_of(held, p)) << 32 | add;
    }
    __device__ __forceinline__ int32_t kv_length() const { return static_cast<int32_t>(held + add < INT32_MAX ? held + add : INT32_MAX); }
};

// Exclusive sums over kFusedRequests requests, request i * kScanBlock + thread in needs[i], and the sum of all.  Waves scan
// their 64 of each row; the first wave scans the waves' sums, of which there are 64 and 16 more.
struct FusedScan {
    static constexpr int kWavesPerRow = kScanBlock / kWave;
    static constexpr int kSums = kRequestsPerThread * kWavesPerRow;
    static_assert(kSums > kWave && kSums <= 2 * kWave);
    uint64_t sums[kSums];
    uint64_t all;
    __device__ __forceinline__ void run(uint64_t (&needs)[kRequestsPerThread], int count) {
        const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
        uint64_t inclusive[kRequestsPerThread];
#pragma unroll
        for (int i = 0; i < kRequestsPerThread; ++i) {
            inclusive[i] = i * kScanBlock < count ? wave_inclusive_scan(needs[i], SumOp{}) : 0;
            if (lane == kWave - 1) sums[i * kWavesPerRow + wave] = inclusive[i];
        }
        __syncthreads();
        if (wave == 0) {
            const uint64_t first = sums[lane], second = lane < kSums - kWave ? sums[kWave + lane] : 0;
            const uint64_t a = wave_inclusive_scan(first, SumOp{}), half = wave_read_lane(a, kWave - 1);
            const uint64_t b = half + (count > kWave * kWave ? wave_inclusive_scan(second, SumOp{}) : 0);
            sums[lane] = a - first;
            if (lane < kSums - kWave) sums[kWave + lane] = b - second;
            if (lane == kWave - 1) all = b;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kRequestsPerThread; ++i) needs[i] = sums[i * kWavesPerRow + wave] + inclusive[i] - needs[i];
    }
};

// Pages of one request as its tokens come in order.  A page is new to the table where it begins at or past the cached
// length, and then its first position is a new token's: that token enters it.
struct RequestPages {
    uint32_t position, cell, within;
    int page;
    __device__ __forceinline__ void look_up(int r, uint32_t held, uint32_t first_page, const int32_t* free_pages, int32_t* block_table,
                                            const Plan& p) {
        page = -1;
        if (cell >= static_cast<uint32_t>(p.table_width)) return;
        int32_t* entry = block_table + r * p.table_stride + cell;
        const uint32_t have = pages_of(held, p);
        if (cell < have) {
            page = *entry;
            return;
        }
        const uint32_t index = first_page + cell - have;
        if (index < static_cast<uint32_t>(p.num_free)) page = free_pages[index];
        if (within == 0) *entry = page;
    }
    __device__ __forceinline__ void start(uint32_t at, const Plan& p) {
        position = at;
        cell = p.page_size(at);
        within = at - cell * p.page_size.by;
    }
    __device__ __forceinline__ bool next(const Plan& p) {  // whether a page begins
        ++position;
        if (++within < p.page_size.by) return false;
        within = 0;
        ++cell;
        return true;
    }
    __device__ __forceinline__ int64_t slot(const Plan& p) const {
        return page < 0 ? -1 : static_cast<int64_t>(page) * p.page_size.by + within;
    }
};

__device__ __forceinline__ void no_token(int64_t t, int32_t* token_request, int32_t* token_position, int64_t* token_slot) {
    token_request[t] = -1;
    token_position[t] = 0;
    token_slot[t] = -1;
}

// The last request that begins at or before t: empty requests before it share its beginning.
template <typename Token, typename Offset>
__device__ __forceinline__ int owner_of(Token t, int low, int high, Offset offset) {
    while (high - low > 1) {
        const int middle = low + (high - low) / 2;
        if (offset(middle) <= t) low = middle;
        else high = middle;
    }
    return low;
}

// A plan of at most kFusedRequests requests.  Every workgroup scans all of them into LDS, a few consecutive requests a
// thread; the first writes the requests' outputs, and each places its tokens, EACH consecutive ones a thread: the tokens of
// a wave lie between the owners of its first and its last, which it finds together.  Bound by latency up to some hundred
// thousand tokens, then by the instructions a token takes: 1.2 million tokens, 19.8 MB, take 12.6 us, 1.6 TB/s.
template <int EACH>
__global__ __launch_bounds__(kScanBlock) void page_plan_kernel(const int32_t* __restrict__ cached, const int32_t* __restrict__ fresh,
                                                               const int32_t* __restrict__ free_pages, int32_t* __restrict__ block_table,
                                                               int32_t* __restrict__ offsets, int32_t* __restrict__ kv_lengths,
                                                               int32_t* __restrict__ token_request, int32_t* __restrict__ token_position,
                                                               int64_t* __restrict__ token_slot, int32_t* __restrict__ counts, bool vectors, Plan p) {
    __shared__ uint32_t begins[kFusedRequests];
    __shared__ uint32_t first_pages[kFusedRequests];
    __shared__ uint32_t helds[kFusedRequests];
    __shared__ FusedScan scan;
    // All loads first (past the last request, its own again): one wait, not one a request.
    Request requests[kRequestsPerThread];
#pragma unroll
    for (int i = 0; i < kRequestsPerThread; ++i) {
        const int r = i * kScanBlock + static_cast<int>(threadIdx.x);
        if (i * kScanBlock < p.requests) requests[i].load(cached, fresh, r < p.requests ? r : p.requests - 1);
    }
    uint64_t needs[kRequestsPerThread];
#pragma unroll
    for (int i = 0; i < kRequestsPerThread; ++i)
        needs[i] = i * kScanBlock + static_cast<int>(threadIdx.x) < p.requests ? requests[i].needs(p) : 0;
    scan.run(needs, p.requests);
    const uint64_t all = scan.all;
#pragma unroll
    for (int i = 0; i < kRequestsPerThread; ++i) {
        const int r = i * kScanBlock + static_cast<int>(threadIdx.x);
        if (r < p.requests) {
            begins[r] = static_cast<uint32_t>(needs[i]);
            first_pages[r] = static_cast<uint32_t>(needs[i] >> 32);
            helds[r] = requests[i].held;
            if (blockIdx.x == 0) {
                offsets[r] = static_cast<int32_t>(needs[i]);
                kv_lengths[r] = requests[i].kv_length();
            }
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        offsets[p.requests] = counts[0] = static_cast<int32_t>(all);
        counts[1] = static_cast<int32_t>(all >> 32);
    }
    __syncthreads();
    const auto begin_of = [&](int r) { return begins[r]; };
    // Tokens past max_tokens (below 2^31) are left out, also where there are more.
    const uint32_t most = static_cast<uint32_t>(p.max_tokens);
    const uint32_t total = static_cast<uint32_t>(all) < most ? static_cast<uint32_t>(all) : most;
    const uint32_t wave_first = (blockIdx.x * kScanBlock + threadIdx.x / kWave * kWave) * EACH;
    const uint32_t t0 = wave_first + threadIdx.x % kWave * EACH;
    if (wave_first >= most) return;
    int32_t request[EACH], position[EACH];
    int64_t slot[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) request[i] = -1, position[i] = 0, slot[i] = -1;
    if (wave_first < total) {
        const uint32_t wave_last = wave_first + kWave * EACH < total ? wave_first + kWave * EACH - 1 : total - 1;
        const int low = attention::find_last(p.requests, wave_first, begin_of);
        const int high = attention::find_last(p.requests, wave_last, begin_of) + 1;
        if (t0 < total) {
            int r = low;
            uint32_t end = 0, held = 0;
            RequestPages pages{};
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const uint32_t t = t0 + i;
                if (t >= total) break;
                bool begins_page = true;
                if (t >= end) {
                    r = owner_of(t, r, high, begin_of);
                    end = r + 1 < p.requests ? begin_of(r + 1) : ~0u;
                    held = helds[r];
                    pages.start(held + (t - begin_of(r)), p);
                } else {
                    begins_page = pages.next(p);
                }
                if (begins_page) pages.look_up(r, held, first_pages[r], free_pages, block_table, p);
                request[i] = r;
                position[i] = static_cast<int32_t>(pages.position);
                slot[i] = pages.slot(p);
            }
        }
    }
    if (EACH == 4 && vectors && t0 + EACH <= most) {
        using I32x4 = int32_t __attribute__((ext_vector_type(4)));
        using I64x2 = int64_t __attribute__((ext_vector_type(2)));
        *reinterpret_cast<I32x4*>(token_request + t0) = I32x4{request[0], request[1 % EACH], request[2 % EACH], request[3 % EACH]};
        *reinterpret_cast<I32x4*>(token_position + t0) = I32x4{position[0], position[1 % EACH], position[2 % EACH], position[3 % EACH]};
        *reinterpret_cast<I64x2*>(token_slot + t0) = I64x2{slot[0], slot[1 % EACH]};
        *reinterpret_cast<I64x2*>(token_slot + t0 + 2) = I64x2{slot[2 % EACH], slot[3 % EACH]};
        return;
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (t0 + i >= most) break;
        token_request[t0 + i] = request[i];
        token_position[t0 + i] = position[i];
        token_slot[t0 + i] = slot[i];
    }
}

// More requests: one workgroup's scan, then a thread a token, which finds its request by halving.  Bound by the scan's
// rounds, each waiting for its loads (a token a request: 5,120 requests 7.4 us in one launch, 5,121 11.5 in two, 11,000 14.9,
// 100,000 64).
__global__ __launch_bounds__(kScanBlock) void page_plan_scan_kernel(const int32_t* __restrict__ cached,
                                                                    const int32_t* __restrict__ fresh, uint32_t* __restrict__ first_page,
                                                                    int32_t* __restrict__ offsets, int32_t* __restrict__ kv_lengths,
                                                                    int32_t* __restrict__ counts, Plan p) {
    __shared__ FusedScan scan;
    uint64_t carry = 0;
    for (int base = 0; base < p.requests; base += kFusedRequests) {
        Request requests[kRequestsPerThread];
        uint64_t needs[kRequestsPerThread];
#pragma unroll
        for (int i = 0; i < kRequestsPerThread; ++i) {
            const int r = base + i * kScanBlock + static_cast<int>(threadIdx.x);
            requests[i].load(cached, fresh, r < p.requests ? r : p.requests - 1);
        }
#pragma unroll
        for (int i = 0; i < kRequestsPerThread; ++i)
            needs[i] = base + i * kScanBlock + static_cast<int>(threadIdx.x) < p.requests ? requests[i].needs(p) : 0;
        scan.run(needs, kFusedRequests);
#pragma unroll
        for (int i = 0; i < kRequestsPerThread; ++i) {
            const int r = base + i * kScanBlock + static_cast<int>(threadIdx.x);
            if (r < p.requests) {
                kv_lengths[r] = requests[i].kv_length();
                offsets[r] = static_cast<int32_t>(carry + needs[i]);
                first_page[r] = static_cast<uint32_t>((carry + needs[i]) >> 32);
            }
        }
        carry += scan.all;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        offsets[p.requests] = counts[0] = static_cast<int32_t>(carry);
        counts[1] = static_cast<int32_t>(carry >> 32);
    }
}

__global__ __launch_bounds__(kTokenBlock) void page_plan_tokens_kernel(
    const int32_t* __restrict__ cached, const uint32_t* __restrict__ first_page, const int32_t* __restrict__ offsets,
    const int32_t* __restrict__ free_pages, int32_t* __restrict__ block_table, int32_t* __restrict__ token_request,
    int32_t* __restrict__ token_position, int64_t* __restrict__ token_slot, Plan p) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kTokenBlock + threadIdx.x;
    if (t >= p.max_tokens) return;
    if (t >= offsets[p.requests]) return no_token(t, token_request, token_position, token_slot);
    const int r = owner_of(t, 0, p.requests, [&](int i) { return offsets[i]; });
    const uint32_t held = length_at(cached, r);
    RequestPages pages;
    pages.start(held + static_cast<uint32_t>(t - offsets[r]), p);
    pages.look_up(r, held, first_page[r], free_pages, block_table, p);
    token_request[t] = r;
    token_position[t] = static_cast<int32_t>(pages.position);
    token_slot[t] = pages.slot(p);
}

// ---- rows into pages ---------------------------------------------------------------------------------------------
// A copy: a thread a 16-byte chunk of a token's key and value, neighbours next to each other.  A row has `per` chunks; a
// workgroup takes `group` short rows, or one of blockIdx.y parts of a long one.  Bound by memory (65,521 tokens of 8 x 128
// items, 537 MB, from a cold cache: 95 us, 5.6 TB/s; four tokens a thread: 102 us), and
// by latency for a step's few tokens (256 of them: 2.2 us; four a thread: 3.5 us).
__global__ __launch_bounds__(kTokenBlock) void paged_write_kernel(attention::Rows key, attention::Rows value,
                                                                  attention::Pages key_cache, attention::Pages value_cache,
                                                                  const int64_t* __restrict__ slots, int64_t tokens, int per,
                                                                  int chunks, int group, attention::Divider page_size, int64_t pages) {
    using attention::U32x4;
    const int rest = static_cast<int>(blockIdx.y) * kTokenBlock + static_cast<int>(threadIdx.x) % (group > 1 ? per : kTokenBlock);
    const int mine = group > 1 ? static_cast<int>(threadIdx.x) / per : 0;
    if (rest >= per || mine >= group) return;
    const int64_t token = static_cast<int64_t>(blockIdx.x) * group + mine;
    if (token >= tokens) return;
    const int64_t slot = slots[token];
    if (slot < 0) return;
    const int head = rest / chunks, chunk = rest % chunks;
    const U32x4 k = __builtin_nontemporal_load(reinterpret_cast<const U32x4*>(key.at(token, head) + chunk * 16));
    const U32x4 v = __builtin_nontemporal_load(reinterpret_cast<const U32x4*>(value.at(token, head) + chunk * 16));
    // Division in 32 bits where the slot allows.
    const int64_t page = slot <= 0xFFFFFFFFll ? page_size(static_cast<uint32_t>(slot)) : slot / page_size.by;
    if (page >= pages) return;
    const int64_t within = slot - page * page_size.by;
    *reinterpret_cast<U32x4*>(key_cache.at(page, within, head) + chunk * 16) = k;
    *reinterpret_cast<U32x4*>(value_cache.at(page, within, head) + chunk * 16) = v;
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
    const Plan p{static_cast<int>(requests), attention::Divider(page_size), static_cast<int>(num_free), static_cast<int>(table_width),
                 static_cast<int64_t>(table_stride), static_cast<int64_t>(max_tokens)};
    if (requests <= kFusedRequests) {
        const bool many = max_tokens > kFusedTokens;
        const bool vectors = (reinterpret_cast<uintptr_t>(token_request) | reinterpret_cast<uintptr_t>(token_position) |
                              reinterpret_cast<uintptr_t>(token_slot)) % 16 == 0;
        const uint64_t blocks = ceil_div(max_tokens, static_cast<uint64_t>(kScanBlock) * (many ? kTokensPerThread : 1));
        auto* kernel = many ? page_plan_kernel<kTokensPerThread> : page_plan_kernel<1>;
        LaunchScope scope("page_plan", stream);
        kernel<<<static_cast<unsigned>(blocks ? blocks : 1), kScanBlock, 0, stream>>>(
            cached, fresh, free_pages, block_table, offsets, kv_lengths, token_request, token_position, token_slot, counts, vectors, p);
        return check_hip(hipGetLastError(), "page_plan launch");
    }
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
    const int chunks = static_cast<int>(dim / 8), per = static_cast<int>(kv_heads) * chunks;
    const int group = per <= kTokenBlock / 2 ? kTokenBlock / per : 1;
    const uint64_t splits = ceil_div(per, kTokenBlock);
    if (splits > 65535) return set_error(kInvalidArgument, "%s: rows too long", what);
    const uint64_t most = 0x7FFFFFFFull / kTokenBlock / splits * group;  // tokens of a launch
    LaunchScope scope("paged_write", stream);
    attention::Rows k = attention::rows_of(key), v = attention::rows_of(value);
    for (uint64_t first = 0; first < tokens; first += most) {
        const uint64_t count = tokens - first < most ? tokens - first : most;
        const unsigned blocks = static_cast<unsigned>(ceil_div(count, static_cast<uint64_t>(group)));
        paged_write_kernel<<<dim3(blocks, static_cast<unsigned>(splits)), kTokenBlock, 0, stream>>>(
            k, v, attention::pages_of(key_cache), attention::pages_of(value_cache), slots + first, static_cast<int64_t>(count), per,
            chunks, group, attention::Divider(page_size), static_cast<int64_t>(pages));
        k.data += static_cast<int64_t>(count) * k.token_bytes;
        v.data += static_cast<int64_t>(count) * v.token_bytes;
    }
    return check_hip(hipGetLastError(), "paged_write launch");
}

}  // namespace
}  // namespace lcpp_hip

using namespace lcpp_hip;

extern "C" {

size_t lcpp_hip_page_plan_temp_bytes(uint32_t requests) {
    return requests <= kFusedRequests ? 0 : align_up(static_cast<size_t>(requests) * sizeof(uint32_t), kViewAlign);
}

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
