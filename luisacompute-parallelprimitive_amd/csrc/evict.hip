// Eviction from a paged cache: which of a request's keys stay, where they go, and the pages that come free.
//
// A request of n keys that is to keep K of them keeps those of the largest sums of weights, and before them all that are
// protected: the first positions and the latest ones.  Keys are turned by their own positions already, and attention does not
// ask in which order they lie: a kept key past the new end moves into the place of one that goes, nothing else moves, and
// no place is both read and written.
//
// The K-th largest of a request's sums is found by a radix selection over the bits of the sums, highest first, so it is exact;
// equal sums go by the lower index.
#include "attention.hpp"

namespace lcpp_hip {
namespace attention {
namespace {

constexpr int kEvictBlock = 1024;
constexpr int kEvictWaves = kEvictBlock / kWave;

// ---- lengths and pages -------------------------------------------------------------------------------------------
struct Release {
    int requests;
    Divider page_size;
    int64_t table_stride;
    int table_width;
    int64_t most_moves;
    int64_t capacity;
};

__device__ __forceinline__ int64_t at_least_0(int32_t x) { return x > 0 ? x : 0; }

__device__ __forceinline__ int64_t kept_of(int64_t n, int64_t keep, int64_t most_moves) {
    if (keep >= n) return n;
    return (keep < n - keep ? keep : n - keep) > most_moves ? n : keep;
}

__device__ __forceinline__ int64_t cells_of(int64_t length, const Release& p) {
    const uint32_t full = p.page_size(static_cast<uint32_t>(length));
    const int64_t n = full + (static_cast<uint32_t>(length) != full * p.page_size.by);
    return n < p.table_width ? n : p.table_width;
}

// Exclusive sums over a workgroup's threads, and the sum of all.
struct BlockScan {
    int64_t sums[kEvictWaves];
    __device__ __forceinline__ int64_t run(int64_t x, int64_t& all) {
        const int wave = threadIdx.x / kWave;
        const int64_t inclusive = wave_inclusive_scan(x, SumOp{});
        __syncthreads();
        if (threadIdx.x % kWave == kWave - 1) sums[wave] = inclusive;
        __syncthreads();
        int64_t before = 0;
        all = 0;
#pragma unroll
        for (int w = 0; w < kEvictWaves; ++w) {
            before += w < wave ? sums[w] : 0;
            all += sums[w];
        }
        return before + inclusive - x;
    }
};

// One workgroup: 1,024 requests at a time, then their free cells, four a thread at a time, in the requests' order.
__global__ __launch_bounds__(kEvictBlock) void page_release_kernel(const int32_t* __restrict__ kv_lengths,
                                                                   const int32_t* __restrict__ keep_lengths,
                                                                   const int32_t* __restrict__ block_table, const int32_t* shifts,
                                                                   int32_t* __restrict__ kept_lengths, int32_t* shifts_out,
                                                                   int32_t* __restrict__ released, int32_t* __restrict__ counts,
                                                                   Release p) {
    constexpr int kCells = 4;
    __shared__ BlockScan scan;
    __shared__ int64_t begins[kEvictBlock];
    __shared__ int32_t first_cells[kEvictBlock];
    int64_t given = 0, all_kept = 0;
    for (int base = 0; base < p.requests; base += kEvictBlock) {
        const int r = base + static_cast<int>(threadIdx.x);
        int64_t cells = 0, kept = 0, first_cell = 0;
        if (r < p.requests) {
            const int64_t n = at_least_0(kv_lengths[r]);
            kept = kept_of(n, at_least_0(keep_lengths[r]), p.most_moves);
            kept_lengths[r] = static_cast<int32_t>(kept);
            if (shifts_out != nullptr) shifts_out[r] = static_cast<int32_t>((shifts != nullptr ? shifts[r] : 0) + n - kept);
            first_cell = cells_of(kept, p);
            cells = cells_of(n, p) - first_cell;
        }
        int64_t all, total;
        const int64_t begin = scan.run(cells, total);
        begins[threadIdx.x] = begin;
        first_cells[threadIdx.x] = static_cast<int32_t>(first_cell);
        scan.run(kept, all);
        all_kept += all;
        const int count = p.requests - base < kEvictBlock ? p.requests - base : kEvictBlock;
        for (int64_t c0 = 0; c0 < total; c0 += kEvictBlock * kCells) {
            int32_t page[kCells];
            int valid = 0;
            const int64_t mine = c0 + static_cast<int64_t>(threadIdx.x) * kCells;
            int low = 0, high = count;
            while (high - low > 1) {
                const int middle = low + (high - low) / 2;
                if (begins[middle] <= mine) low = middle;
                else high = middle;
            }
#pragma unroll
            for (int i = 0; i < kCells; ++i) {
                page[i] = -1;
                if (mine + i >= total) continue;
                while (low + 1 < count && begins[low + 1] <= mine + i) ++low;
                page[i] = block_table[(base + low) * p.table_stride + first_cells[low] + (mine + i - begins[low])];
                valid += page[i] >= 0;
            }
            int64_t found;
            int64_t at = given + scan.run(valid, found);
#pragma unroll
            for (int i = 0; i < kCells; ++i)
                if (page[i] >= 0) {
                    if (at < p.capacity) released[at] = page[i];
                    ++at;
                }
            given += found;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        counts[0] = static_cast<int32_t>(given);
        counts[1] = static_cast<int32_t>(all_kept);
    }
}

// ---- which keys stay ---------------------------------------------------------------------------------------------
struct Evict {
    Divider page_size;
    int64_t table_stride;
    int table_width;
    int pages;
    int64_t width;  // moves that a request has room for
    int first;
    int recent;
};

// A sum of weights as a number of the same order: 0 for a key whose page is not there, 1 for NaN, the largest for a
// protected one; -0 as 0.
__device__ __forceinline__ uint32_t order_of(float weight, bool safe, bool there) {
    const float w = weight + 0.f;
    const uint32_t bits = __builtin_bit_cast(uint32_t, w);
    uint32_t order = bits >> 31 ? ~bits : bits | 0x80000000u;
    order = w == w ? order : 1u;
    order = safe ? ~0u : order;
    return there ? order : 0u;
}

// One request's keys.
struct Keys {
    const float* weights;
    const int32_t* positions;
    const int32_t* table;
    int64_t late;  // positions from here on are protected
    const Evict& p;
    __device__ __forceinline__ int64_t slot(int j) const {
        const uint32_t cell = p.page_size(static_cast<uint32_t>(j));
        const int page = table[cell];
        return page < 0 || page >= p.pages ? -1 : static_cast<int64_t>(page) * p.page_size.by + (j - cell * p.page_size.by);
    }
    __device__ __forceinline__ uint32_t order(int j) const {
        const int64_t at = slot(j);
        if (at < 0) return 0u;
        bool safe = false;
        if (positions != nullptr) {
            const int64_t position = positions[at];
            safe = position < p.first || position >= late;
        }
        return order_of(weights[at], safe, true);
    }
};

// A workgroup a request.  Wave w has the keys [w per, (w + 1) per), so that counts of the waves before give a key its rank.
__global__ __launch_bounds__(kEvictBlock) void evict_plan_kernel(const float* __restrict__ weights, const int32_t* __restrict__ positions,
                                                                 const int32_t* __restrict__ block_table,
                                                                 const int32_t* __restrict__ kv_lengths,
                                                                 const int32_t* __restrict__ kept_lengths,
                                                                 const int32_t* __restrict__ shifts, int64_t* __restrict__ move_from,
                                                                 int64_t* __restrict__ move_to, Evict p) {
    __shared__ uint32_t bins[256];
    __shared__ uint32_t chosen, wanted;
    __shared__ int32_t tie_sums[kEvictWaves], mover_sums[kEvictWaves], hole_sums[kEvictWaves];
    const int request = blockIdx.x, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int64_t length = at_least_0(kv_lengths[request]);
    const int64_t room = static_cast<int64_t>(p.table_width) * p.page_size.by;
    const int n = static_cast<int>(length < room ? length : room);
    const int64_t asked = at_least_0(kept_lengths[request]);
    const int keep = static_cast<int>(asked < n ? asked : n);
    int64_t* from = move_from + request * p.width;
    int64_t* to = move_to + request * p.width;
    if (keep == 0 || keep == n) {
        for (int64_t i = threadIdx.x; i < p.width; i += kEvictBlock) from[i] = to[i] = -1;
        return;
    }
    const Keys keys{weights, positions, block_table + request * p.table_stride,
                    p.recent ? (shifts != nullptr ? shifts[request] : 0) + length - p.recent : INT64_MAX, p};
    // The keep-th largest: the bytes of its order, highest first.
    uint32_t prefix = 0, need = static_cast<uint32_t>(keep);
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) bins[threadIdx.x] = 0;
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += kEvictBlock) {
            const uint32_t order = keys.order(j);
            if (shift == 24 || order >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&bins[order >> shift & 255], 1u);
        }
        __syncthreads();
        if (wave == 0) {  // bins from the largest down, four a lane
            uint32_t own[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += own[i] = bins[255 - (4 * lane + i)];
            uint32_t before = wave_inclusive_scan(sum, SumOp{}) - sum;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (before < need && need <= before + own[i]) {
                    chosen = 255 - (4 * lane + i);
                    wanted = need - before;
                }
                before += own[i];
            }
        }
        __syncthreads();
        prefix |= chosen << shift;
        need = wanted;
    }
    const int per = ((n + kEvictWaves - 1) / kEvictWaves + kWave - 1) / kWave * kWave;
    const int begin = wave * per, end = begin + per < n ? begin + per : n;
    // Of the keys equal to it, the first `need` stay.
    int ties = 0;
    for (int j0 = begin; j0 < end; j0 += kWave) ties += __popcll(wave_ballot(j0 + lane < end && keys.order(j0 + lane) == prefix));
    if (lane == 0) tie_sums[wave] = ties;
    __syncthreads();
    int tie_base = 0;
    for (int w = 0; w < wave; ++w) tie_base += tie_sums[w];
    const auto sweep = [&](auto emit) {
        int tie = tie_base;
        for (int j0 = begin; j0 < end; j0 += kWave) {
            const int j = j0 + lane;
            const uint32_t order = j < end ? keys.order(j) : 0u;
            const uint64_t equal = wave_ballot(j < end && order == prefix);
            const bool stays = order > prefix || (order == prefix && tie + static_cast<int>(popc_lanes_below(equal)) < static_cast<int>(need));
            tie += __popcll(equal);
            const bool mover = j < end && stays && j >= keep, hole = j < end && !stays && j < keep;
            emit(j, mover, hole);
        }
    };
    int movers = 0, holes = 0;
    sweep([&](int, bool mover, bool hole) {
        movers += __popcll(wave_ballot(mover));
        holes += __popcll(wave_ballot(hole));
    });
    if (lane == 0) {
        mover_sums[wave] = movers;
        hole_sums[wave] = holes;
    }
    __syncthreads();
    int64_t mover_at = 0, hole_at = 0, moves = 0;
    for (int w = 0; w < kEvictWaves; ++w) {
        if (w < wave) {
            mover_at += mover_sums[w];
            hole_at += hole_sums[w];
        }
        moves += mover_sums[w];
    }
    sweep([&](int j, bool mover, bool hole) {
        const uint64_t moving = wave_ballot(mover), open = wave_ballot(hole);
        if (mover) {
            const int64_t at = mover_at + popc_lanes_below(moving);
            if (at < p.width) from[at] = keys.slot(j);
        }
        if (hole) {
            const int64_t at = hole_at + popc_lanes_below(open);
            if (at < p.width) to[at] = keys.slot(j);
        }
        mover_at += __popcll(moving);
        hole_at += __popcll(open);
    });
    for (int64_t i = moves + threadIdx.x; i < p.width; i += kEvictBlock) from[i] = to[i] = -1;
}

// ---- rows from slot to slot --------------------------------------------------------------------------------------
constexpr int kMoveBlock = 256;

// A thread a 16-byte chunk of a move's key and value.
__global__ __launch_bounds__(kMoveBlock) void paged_move_kernel(Pages key_cache, Pages value_cache, float* weights, int32_t* positions,
                                                                const int64_t* __restrict__ from, const int64_t* __restrict__ to,
                                                                int64_t moves, int per, Divider chunks, int group, Divider page_size,
                                                                int64_t pages) {
    const int rest = static_cast<int>(blockIdx.y) * kMoveBlock + static_cast<int>(threadIdx.x) % (group > 1 ? per : kMoveBlock);
    const int mine = group > 1 ? static_cast<int>(threadIdx.x) / per : 0;
    if (rest >= per || mine >= group) return;
    const int64_t move = static_cast<int64_t>(blockIdx.x) * group + mine;
    if (move >= moves) return;
    const int64_t source = from[move], target = to[move];
    if (source < 0 || target < 0) return;
    const auto page_of = [&](int64_t slot) {
        return slot <= 0xFFFFFFFFll ? static_cast<int64_t>(page_size(static_cast<uint32_t>(slot))) : slot / page_size.by;
    };
    const int64_t source_page = page_of(source), target_page = page_of(target);
    if (source_page >= pages || target_page >= pages) return;
    const int64_t source_at = source - source_page * page_size.by, target_at = target - target_page * page_size.by;
    const int head = static_cast<int>(chunks(rest)), chunk = rest - head * static_cast<int>(chunks.by);
    const U32x4 k = *reinterpret_cast<const U32x4*>(key_cache.at(source_page, source_at, head) + chunk * 16);
    const U32x4 v = *reinterpret_cast<const U32x4*>(value_cache.at(source_page, source_at, head) + chunk * 16);
    if (rest == 0) {
        if (weights != nullptr) weights[target] = weights[source];
        if (positions != nullptr) positions[target] = positions[source];
    }
    *reinterpret_cast<U32x4*>(key_cache.at(target_page, target_at, head) + chunk * 16) = k;
    *reinterpret_cast<U32x4*>(value_cache.at(target_page, target_at, head) + chunk * 16) = v;
}

// ---- host side ---------------------------------------------------------------------------------------------------
int check_pages(const char* what, uint32_t requests, uint32_t page_size, uint64_t table_stride, uint32_t table_width) {
    if (page_size == 0 || page_size > 0x7FFFFFFFu) return set_error(kInvalidArgument, "%s: page size out of range", what);
    if (requests > 0x7FFFFFFu) return set_error(kInvalidArgument, "%s: too many requests", what);
    if (table_width > table_stride || table_width > 0x7FFFFFFFu || table_stride > 0x7FFFFFFFFFFull)
        return set_error(kInvalidArgument, "%s: a block table's row must hold its width", what);
    return kOk;
}

int page_release(const int32_t* kv_lengths, const int32_t* keep_lengths, uint32_t requests, uint32_t page_size,
                 const int32_t* block_table, uint64_t table_stride, uint32_t table_width, uint64_t most_moves, const int32_t* shifts,
                 int32_t* kept_lengths, int32_t* shifts_out, int32_t* released, uint64_t max_released, int32_t* counts, void* stream_ptr) {
    const char* what = "page_release";
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (int st = check_pages(what, requests, page_size, table_stride, table_width); st != kOk) return st;
    if (max_released > 0x7FFFFFFFull) return set_error(kInvalidArgument, "%s: too many pages", what);
    if (!counts) return set_error(kInvalidArgument, "%s: null counts", what);
    if (requests && (!kv_lengths || !keep_lengths || !kept_lengths)) return set_error(kInvalidArgument, "%s: null lengths", what);
    if (requests && table_width && !block_table) return set_error(kInvalidArgument, "%s: null block table", what);
    if (max_released && !released) return set_error(kInvalidArgument, "%s: null list of pages", what);
    const Release p{static_cast<int>(requests), Divider(page_size), static_cast<int64_t>(table_stride), static_cast<int>(table_width),
                    static_cast<int64_t>(most_moves > 0x7FFFFFFFull ? 0x7FFFFFFFull : most_moves), static_cast<int64_t>(max_released)};
    LaunchScope scope(what, stream);
    page_release_kernel<<<1, kEvictBlock, 0, stream>>>(kv_lengths, keep_lengths, block_table, shifts, kept_lengths, shifts_out, released,
                                                       counts, p);
    return check_hip(hipGetLastError(), "page_release launch");
}

int evict_plan(void* temp, size_t temp_bytes, const float* weights, const int32_t* positions, const int32_t* block_table,
               uint64_t table_stride, uint32_t table_width, const int32_t* kv_lengths, const int32_t* kept_lengths, const int32_t* shifts,
               uint32_t requests, uint64_t max_kv_length, uint32_t page_size, uint32_t pages, uint32_t first, uint32_t recent,
               int64_t* move_from, int64_t* move_to, uint64_t width, void* stream_ptr) {
    const char* what = "evict_plan";
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (int st = check_pages(what, requests, page_size, table_stride, table_width); st != kOk) return st;
    if (pages > 0x7FFFFFFFu || width > 0x7FFFFFFFull) return set_error(kInvalidArgument, "%s: too many pages or moves", what);
    if (first > 0x7FFFFFFFu || recent > 0x7FFFFFFFu) return set_error(kInvalidArgument, "%s: too many protected keys", what);
    if (max_kv_length > kMostKeys || static_cast<uint64_t>(table_width) * page_size > kMostKeys)
        return set_error(kInvalidArgument, "%s: requests too long", what);
    if (requests == 0) return kOk;
    if (!weights || !kv_lengths || !kept_lengths || (table_width && !block_table))
        return set_error(kInvalidArgument, "%s: null sums, lengths or block table", what);
    if (!positions && (first || recent)) return set_error(kInvalidArgument, "%s: protected keys need the positions", what);
    if (width && (!move_from || !move_to)) return set_error(kInvalidArgument, "%s: null moves", what);
    const size_t needed = lcpp_hip_evict_plan_temp_bytes(requests, max_kv_length);
    if (temp_bytes < needed || (needed && !temp)) return set_error(kTempTooSmall, "%s: temp storage too small", what);
    const Evict p{Divider(page_size), static_cast<int64_t>(table_stride), static_cast<int>(table_width), static_cast<int>(pages),
                  static_cast<int64_t>(width), static_cast<int>(first), static_cast<int>(recent)};
    LaunchScope scope(what, stream);
    evict_plan_kernel<<<requests, kEvictBlock, 0, stream>>>(weights, positions, block_table, kv_lengths, kept_lengths, shifts, move_from,
                                                            move_to, p);
    return check_hip(hipGetLastError(), "evict_plan launch");
}

int paged_move(const int64_t* move_from, const int64_t* move_to, uint64_t moves, const lcpp_hip_pages* key_cache,
               const lcpp_hip_pages* value_cache, float* weights, int32_t* positions, uint32_t kv_heads, uint32_t dim, uint32_t page_size,
               uint32_t pages, void* stream_ptr) {
    const char* what = "paged_move";
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (dim == 0 || dim % 8 != 0 || dim > 65536) return set_error(kUnsupported, "%s: the head size must be a multiple of 8", what);
    if (kv_heads == 0 || kv_heads > 65535) return set_error(kInvalidArgument, "%s: no heads, or too many", what);
    if (static_cast<uint64_t>(kv_heads) * (dim / 8) > 0xFFFF00ull) return set_error(kInvalidArgument, "%s: rows too long", what);
    if (page_size == 0 || page_size > 0x7FFFFFFFu) return set_error(kInvalidArgument, "%s: page size out of range", what);
    if (moves > 0x7FFFFFFFull) return set_error(kInvalidArgument, "%s: too many moves", what);
    if (moves == 0) return kOk;
    if (!move_from || !move_to) return set_error(kInvalidArgument, "%s: null moves", what);
    if (!usable(key_cache) || !usable(value_cache)) return unusable(what);
    const int chunks = static_cast<int>(dim / 8), per = static_cast<int>(kv_heads) * chunks;
    const int group = per <= kMoveBlock / 2 ? kMoveBlock / per : 1;
    const uint64_t splits = ceil_div(per, kMoveBlock);
    const uint64_t most = 0x7FFFFFFFull / kMoveBlock / splits * group;  // moves of a launch
    LaunchScope scope(what, stream);
    for (uint64_t at = 0; at < moves; at += most) {
        const uint64_t count = moves - at < most ? moves - at : most;
        paged_move_kernel<<<dim3(static_cast<unsigned>(ceil_div(count, static_cast<uint64_t>(group))), static_cast<unsigned>(splits)),
                            kMoveBlock, 0, stream>>>(pages_of(key_cache), pages_of(value_cache), weights, positions, move_from + at,
                                                     move_to + at, static_cast<int64_t>(count), per, Divider(static_cast<uint32_t>(chunks)),
                                                     group, Divider(page_size), static_cast<int64_t>(pages));
    }
    return check_hip(hipGetLastError(), "paged_move launch");
}

}  // namespace
}  // namespace attention
}  // namespace lcpp_hip

using namespace lcpp_hip;

extern "C" {

int lcpp_hip_page_release(const int32_t* kv_lengths, const int32_t* keep_lengths, uint32_t requests, uint32_t page_size,
                          const int32_t* block_table, uint64_t table_stride, uint32_t table_width, uint64_t most_moves,
                          const int32_t* shifts, int32_t* kept_lengths, int32_t* shifts_out, int32_t* released, uint64_t max_released,
                          int32_t* counts, void* stream) {
    return attention::page_release(kv_lengths, keep_lengths, requests, page_size, block_table, table_stride, table_width, most_moves,
                                   shifts, kept_lengths, shifts_out, released, max_released, counts, stream);
}

size_t lcpp_hip_evict_plan_temp_bytes(uint32_t, uint64_t) { return 0; }

int lcpp_hip_evict_plan(void* temp, size_t temp_bytes, const float* weights, const int32_t* positions, const int32_t* block_table,
                        uint64_t table_stride, uint32_t table_width, const int32_t* kv_lengths, const int32_t* kept_lengths,
                        const int32_t* shifts, uint32_t requests, uint64_t max_kv_length, uint32_t page_size, uint32_t pages,
                        uint32_t first, uint32_t recent, int64_t* move_from, int64_t* move_to, uint64_t width, void* stream) {
    return attention::evict_plan(temp, temp_bytes, weights, positions, block_table, table_stride, table_width, kv_lengths, kept_lengths,
                                 shifts, requests, max_kv_length, page_size, pages, first, recent, move_from, move_to, width, stream);
}

#define LCPP_HIP_DEFINE_PAGED_MOVE(S)                                                                                         \
    int lcpp_hip_paged_move_##S(const int64_t* move_from, const int64_t* move_to, uint64_t moves,                             \
                                const lcpp_hip_pages* key_cache, const lcpp_hip_pages* value_cache, float* weights,           \
                                int32_t* positions, uint32_t kv_heads, uint32_t head_dim, uint32_t page_size, uint32_t pages, \
                                void* stream) {                                                                               \
        return attention::paged_move(move_from, move_to, moves, key_cache, value_cache, weights, positions, kv_heads, head_dim, \
                                     page_size, pages, stream);                                                               \
    }
LCPP_HIP_DEFINE_PAGED_MOVE(bf16)
LCPP_HIP_DEFINE_PAGED_MOVE(f16)
#undef LCPP_HIP_DEFINE_PAGED_MOVE

}  // extern "C"
