// Eviction from a paged cache: which of a request's keys stay, where they go, and the pages that come free.
//
// A request of n keys that is to keep K of them keeps those of the largest sums of weights, and before them all that are
// protected: the first positions and the latest ones.  Keys are turned by their own positions already, and attention does not
// ask in which order they lie: a kept key past the new end moves into the place of one that goes, nothing else moves, and
// no place is both read and written.
//
// The K-th largest of a request's sums is found by a radix selection over the bits of the sums, highest first, so it is exact;
// equal sums go by the lower index.
//
// Bound by latency: 256 requests of 1,025 to 1,040 keys are planned in 9.1 us; 16 of 2,000 to 131,000 (4.5 MB to read and write) in six
// launches of 2 to 14 us, 47 together, where one workgroup a request took 455.  Moves are bound by memory: 396 MB in 80 us, 5.0 TB/s
// (a copy reaches 6.0).
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
template <typename T, int WAVES>
struct BlockScan {
    T sums[WAVES];
    __device__ __forceinline__ T run(T x, T& all) {
        const int wave = threadIdx.x / kWave;
        const T inclusive = wave_inclusive_scan(x, SumOp{});
        __syncthreads();
        if (threadIdx.x % kWave == kWave - 1) sums[wave] = inclusive;
        __syncthreads();
        T before = 0;
        all = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            before += w < wave ? sums[w] : 0;
            all += sums[w];
        }
        return before + inclusive - x;
    }
};

// One workgroup: 1,024 requests at a time, then their free cells, four a thread at a time, in the requests' order.  Latency: 256
// requests 6 us, 16 that give 10,000 pages 8.
__global__ __launch_bounds__(kEvictBlock) void page_release_kernel(const int32_t* __restrict__ kv_lengths,
                                                                   const int32_t* __restrict__ keep_lengths,
                                                                   const int32_t* __restrict__ block_table, const int32_t* shifts,
                                                                   int32_t* __restrict__ kept_lengths, int32_t* shifts_out,
                                                                   int32_t* __restrict__ released, int32_t* __restrict__ counts,
                                                                   Release p) {
    constexpr int kCells = 4;
    __shared__ BlockScan<int64_t, kEvictWaves> scan;
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

// A request's lengths.
struct Lengths {
    int n, keep;
    int64_t late;  // positions from here on are protected
    __device__ __forceinline__ Lengths(const int32_t* kv_lengths, const int32_t* kept_lengths, const int32_t* shifts, int request,
                                       const Evict& p) {
        const int64_t length = at_least_0(kv_lengths[request]), asked = at_least_0(kept_lengths[request]);
        const int64_t room = static_cast<int64_t>(p.table_width) * p.page_size.by;
        n = static_cast<int>(length < room ? length : room);
        keep = static_cast<int>(asked < n ? asked : n);
        late = p.recent ? (shifts != nullptr ? shifts[request] : 0) + length - p.recent : INT64_MAX;
    }
    __device__ __forceinline__ bool as_it_is() const { return keep == 0 || keep == n; }
};

// Radix selection: 11, 11 and 10 bits of the orders, the highest first.  (11 bits of a float reach into its fraction, so that
// sums of like size spread over the bins.)
constexpr int kDigits = 3;
constexpr int kBins = 2048;
constexpr int kShifts[kDigits] = {21, 10, 0};

// What a digit's counts say: the bin that holds the need-th largest, and which of the bin's it is.
template <int WAVES>
struct Chooser {
    BlockScan<uint32_t, WAVES> scan;
    uint32_t bin, need;
    __device__ __forceinline__ void run(const uint32_t* bins, uint32_t wanted) {
        constexpr int kEach = kBins / (WAVES * kWave);
        uint32_t own[kEach], sum = 0, all;
#pragma unroll
        for (int i = 0; i < kEach; ++i) sum += own[i] = bins[kBins - 1 - (threadIdx.x * kEach + i)];
        uint32_t before = scan.run(sum, all);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (before < wanted && wanted <= before + own[i]) {
                bin = kBins - 1 - (threadIdx.x * kEach + i);
                need = wanted - before;
            }
            before += own[i];
        }
        __syncthreads();
    }
};

// Of a wave's keys in order: which stay, with `tie` of the threshold's equals before them, and what moves.
struct Sorted {
    uint32_t threshold, need;
    int keep, tie;
    __device__ __forceinline__ void next(int j, bool there, uint32_t order, bool& mover, bool& hole) {
        const uint64_t equal = wave_ballot(there && order == threshold);
        const bool stays = order > threshold || (order == threshold && tie + static_cast<int>(popc_lanes_below(equal)) < static_cast<int>(need));
        tie += __popcll(equal);
        mover = there && stays && j >= keep;
        hole = there && !stays && j < keep;
    }
};

// A wave's keys [begin, end): ITEMS of a lane's orders stay in registers, a longer run is read again each time.
template <int ITEMS>
struct Run {
    int begin, end;
    bool held;
    uint32_t orders[ITEMS];
    __device__ __forceinline__ Run(const Keys& keys, int first, int last) : begin(first), end(last), held(last - first <= ITEMS * kWave) {
        if (!held) return;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int j = begin + i * kWave + static_cast<int>(threadIdx.x % kWave);
            orders[i] = j < end ? keys.order(j) : 0u;
        }
    }
    // 64 keys at a time: f(index, whether there is one, order).
    template <typename F>
    __device__ __forceinline__ void each(const Keys& keys, F f) const {
        const int lane = threadIdx.x % kWave;
        if (held) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (begin + i * kWave < end) f(begin + i * kWave + lane, begin + i * kWave + lane < end, orders[i]);
        } else {
            for (int j = begin + lane; j - lane < end; j += kWave) f(j, j < end, j < end ? keys.order(j) : 0u);
        }
    }
};

// Slots of movers and holes, each from its own number on.
struct Emitter {
    int64_t* from;
    int64_t* to;
    int64_t mover_at, hole_at;
    __device__ __forceinline__ void put(const Keys& keys, int64_t width, int j, bool mover, bool hole) {
        const uint64_t moving = wave_ballot(mover), open = wave_ballot(hole);
        if (mover) {
            const int64_t at = mover_at + popc_lanes_below(moving);
            if (at < width) from[at] = keys.slot(j);
        }
        if (hole) {
            const int64_t at = hole_at + popc_lanes_below(open);
            if (at < width) to[at] = keys.slot(j);
        }
        mover_at += __popcll(moving);
        hole_at += __popcll(open);
    }
};

// A workgroup a request.  Wave w has the keys [w per, (w + 1) per), so that counts of the waves before give a key its rank.  ITEMS
// of a lane's orders stay in registers; a request that has more is read again each time.
template <int ITEMS>
__global__ __launch_bounds__(kEvictBlock) void evict_plan_kernel(const float* __restrict__ weights, const int32_t* __restrict__ positions,
                                                                 const int32_t* __restrict__ block_table,
                                                                 const int32_t* __restrict__ kv_lengths,
                                                                 const int32_t* __restrict__ kept_lengths,
                                                                 const int32_t* __restrict__ shifts, int64_t* __restrict__ move_from,
                                                                 int64_t* __restrict__ move_to, Evict p) {
    __shared__ uint32_t bins[kBins];
    __shared__ Chooser<kEvictWaves> chooser;
    __shared__ int32_t tie_sums[kEvictWaves], mover_sums[kEvictWaves], hole_sums[kEvictWaves];
    const int request = blockIdx.x, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const Lengths lengths(kv_lengths, kept_lengths, shifts, request, p);
    const int n = lengths.n;
    int64_t* from = move_from + request * p.width;
    int64_t* to = move_to + request * p.width;
    if (lengths.as_it_is()) {
        for (int64_t i = threadIdx.x; i < p.width; i += kEvictBlock) from[i] = to[i] = -1;
        return;
    }
    const Keys keys{weights, positions, block_table + request * p.table_stride, lengths.late, p};
    const int per = ((n + kEvictWaves - 1) / kEvictWaves + kWave - 1) / kWave * kWave;
    const int begin = wave * per < n ? wave * per : n, end = begin + per < n ? begin + per : n;
    const Run<ITEMS> run(keys, begin, end);
    const auto each = [&](auto f) { run.each(keys, f); };
    Sorted sorted{0, static_cast<uint32_t>(lengths.keep), lengths.keep, 0};
#pragma unroll 1
    for (int digit = 0; digit < kDigits; ++digit) {
        const int shift = digit == 0 ? kShifts[0] : digit == 1 ? kShifts[1] : kShifts[2];
        const uint32_t above = digit == 0 ? 0u : digit == 1 ? ~0u << kShifts[0] : ~0u << kShifts[1];
        for (int i = threadIdx.x; i < kBins; i += kEvictBlock) bins[i] = 0;
        __syncthreads();
        each([&](int, bool there, uint32_t order) {
            if (there && (order & above) == sorted.threshold) atomicAdd(&bins[(order & ~above) >> shift], 1u);
        });
        __syncthreads();
        chooser.run(bins, sorted.need);
        sorted.threshold |= chooser.bin << shift;
        sorted.need = chooser.need;
    }
    // Of the keys equal to it, the first `need` stay.
    int ties = 0;
    each([&](int, bool there, uint32_t order) { ties += __popcll(wave_ballot(there && order == sorted.threshold)); });
    if (lane == 0) tie_sums[wave] = ties;
    __syncthreads();
    for (int w = 0; w < wave; ++w) sorted.tie += tie_sums[w];
    const int first_tie = sorted.tie;
    int movers = 0, holes = 0;
    each([&](int j, bool there, uint32_t order) {
        bool mover, hole;
        sorted.next(j, there, order, mover, hole);
        movers += __popcll(wave_ballot(mover));
        holes += __popcll(wave_ballot(hole));
    });
    if (lane == 0) {
        mover_sums[wave] = movers;
        hole_sums[wave] = holes;
    }
    __syncthreads();
    Emitter emitter{from, to, 0, 0};
    int64_t moves = 0;
    for (int w = 0; w < kEvictWaves; ++w) {
        if (w < wave) {
            emitter.mover_at += mover_sums[w];
            emitter.hole_at += hole_sums[w];
        }
        moves += mover_sums[w];
    }
    sorted.tie = first_tie;
    each([&](int j, bool there, uint32_t order) {
        bool mover, hole;
        sorted.next(j, there, order, mover, hole);
        if (wave_ballot(mover || hole) != 0) emitter.put(keys, p.width, j, mover, hole);
    });
    for (int64_t i = moves + threadIdx.x; i < p.width; i += kEvictBlock) from[i] = to[i] = -1;
}

// Long requests: `parts` workgroups a request, each a run of its keys, in launches that each end a step: the counts of a digit
// (three times), the counts of what stays, and the moves.
constexpr int kPartBlock = 256;
constexpr int kPartWaves = kPartBlock / kWave;
constexpr int kPartItems = 8;
constexpr int kPartKeys = kPartItems * kPartBlock;  // keys of a part, of a request as long as stated
constexpr int kPartLeast = 1024;                    // and at least, of a shorter one

struct PartCounts {
    int32_t low, low_equal, high, high_equal;  // above the threshold, or equal to it; before the new end, or past it
};

struct Parts {
    uint32_t* bins;      // [requests][kDigits][kBins]
    PartCounts* counts;  // [requests][parts]
    int parts;
};

// A part's keys [begin, end), a run of each wave's.
struct PartRange {
    int begin, end, wave_begin, wave_end;
    __device__ __forceinline__ PartRange(int n, int parts, int part) {
        int64_t per = (static_cast<int64_t>(n) + parts - 1) / parts;
        per = per < kPartLeast ? kPartLeast : (per + kPartBlock - 1) / kPartBlock * kPartBlock;
        const auto bound = [](int64_t x, int64_t most) { return static_cast<int>(x < most ? x : most); };
        begin = bound(part * per, n);
        end = bound(part * per + per, n);
        const int64_t run = per / kPartWaves, wave = threadIdx.x / kWave;
        wave_begin = bound(begin + wave * run, end);
        wave_end = bound(begin + wave * run + run, end);
    }
};

// The threshold as far as the digits before `digit` say.
template <int DIGIT>
__device__ __forceinline__ void threshold_of(Chooser<kPartWaves>& chooser, const Parts& parts, int request, Sorted& sorted) {
    const uint32_t* bins = parts.bins + static_cast<int64_t>(request) * kDigits * kBins;
#pragma unroll
    for (int d = 0; d < DIGIT; ++d) {
        chooser.run(bins + d * kBins, sorted.need);
        sorted.threshold |= chooser.bin << kShifts[d];
        sorted.need = chooser.need;
        __syncthreads();
    }
}

struct EvictArrays {
    const float* weights;
    const int32_t* positions;
    const int32_t* block_table;
    const int32_t* kv_lengths;
    const int32_t* kept_lengths;
    const int32_t* shifts;
};

template <int DIGIT>
__global__ __launch_bounds__(kPartBlock) void evict_digit_kernel(EvictArrays a, Parts parts, Evict p) {
    __shared__ uint32_t bins[kBins];
    __shared__ Chooser<kPartWaves> chooser;
    const int request = static_cast<int>(blockIdx.x / parts.parts), part = static_cast<int>(blockIdx.x % parts.parts);
    const Lengths lengths(a.kv_lengths, a.kept_lengths, a.shifts, request, p);
    const PartRange range(lengths.n, parts.parts, part);
    if (lengths.as_it_is() || range.begin >= range.end) return;
    const Keys keys{a.weights, a.positions, a.block_table + request * p.table_stride, lengths.late, p};
    const Run<kPartItems> run(keys, range.wave_begin, range.wave_end);
    for (int i = threadIdx.x; i < kBins; i += kPartBlock) bins[i] = 0;
    __syncthreads();
    Sorted sorted{0, static_cast<uint32_t>(lengths.keep), lengths.keep, 0};
    threshold_of<DIGIT>(chooser, parts, request, sorted);
    constexpr uint32_t kAbove = DIGIT == 0 ? 0u : ~0u << kShifts[DIGIT > 0 ? DIGIT - 1 : 0];
    run.each(keys, [&](int, bool there, uint32_t order) {
        if (there && (order & kAbove) == sorted.threshold) atomicAdd(&bins[(order & ~kAbove) >> kShifts[DIGIT]], 1u);
    });
    __syncthreads();
    uint32_t* all = parts.bins + (static_cast<int64_t>(request) * kDigits + DIGIT) * kBins;
    for (int i = threadIdx.x; i < kBins; i += kPartBlock)
        if (bins[i] != 0) atomic_add_agent(&all[i], bins[i]);
}

__global__ __launch_bounds__(kPartBlock) void evict_count_kernel(EvictArrays a, Parts parts, Evict p) {
    __shared__ Chooser<kPartWaves> chooser;
    __shared__ PartCounts sums[kPartWaves];
    const int request = static_cast<int>(blockIdx.x / parts.parts), part = static_cast<int>(blockIdx.x % parts.parts);
    const Lengths lengths(a.kv_lengths, a.kept_lengths, a.shifts, request, p);
    const PartRange range(lengths.n, parts.parts, part);
    if (lengths.as_it_is()) return;
    PartCounts mine{0, 0, 0, 0};
    if (range.begin < range.end) {
        const Keys keys{a.weights, a.positions, a.block_table + request * p.table_stride, lengths.late, p};
        const Run<kPartItems> run(keys, range.wave_begin, range.wave_end);
        Sorted sorted{0, static_cast<uint32_t>(lengths.keep), lengths.keep, 0};
        threshold_of<kDigits>(chooser, parts, request, sorted);
        run.each(keys, [&](int j, bool there, uint32_t order) {
            const bool low = j < lengths.keep, above = there && order > sorted.threshold, equal = there && order == sorted.threshold;
            mine.low += __popcll(wave_ballot(above && low));
            mine.high += __popcll(wave_ballot(above && !low));
            mine.low_equal += __popcll(wave_ballot(equal && low));
            mine.high_equal += __popcll(wave_ballot(equal && !low));
        });
    }
    if (threadIdx.x % kWave == 0) sums[threadIdx.x / kWave] = mine;
    __syncthreads();
    if (threadIdx.x != 0) return;
#pragma unroll
    for (int w = 1; w < kPartWaves; ++w) {
        mine.low += sums[w].low;
        mine.low_equal += sums[w].low_equal;
        mine.high += sums[w].high;
        mine.high_equal += sums[w].high_equal;
    }
    parts.counts[static_cast<int64_t>(request) * parts.parts + part] = mine;
}

__global__ __launch_bounds__(kPartBlock) void evict_moves_kernel(EvictArrays a, Parts parts, int64_t* __restrict__ move_from,
                                                                 int64_t* __restrict__ move_to, Evict p) {
    __shared__ Chooser<kPartWaves> chooser;
    __shared__ int32_t tie_sums[kPartWaves], mover_sums[kPartWaves], hole_sums[kPartWaves];
    const int request = static_cast<int>(blockIdx.x / parts.parts), part = static_cast<int>(blockIdx.x % parts.parts);
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const Lengths lengths(a.kv_lengths, a.kept_lengths, a.shifts, request, p);
    int64_t* from = move_from + request * p.width;
    int64_t* to = move_to + request * p.width;
    const int64_t stride = static_cast<int64_t>(parts.parts) * kPartBlock, own = static_cast<int64_t>(part) * kPartBlock + threadIdx.x;
    if (lengths.as_it_is()) {
        for (int64_t i = own; i < p.width; i += stride) from[i] = to[i] = -1;
        return;
    }
    const PartRange range(lengths.n, parts.parts, part);
    const Keys keys{a.weights, a.positions, a.block_table + request * p.table_stride, lengths.late, p};
    const Run<kPartItems> run(keys, range.wave_begin, range.wave_end);
    Sorted sorted{0, static_cast<uint32_t>(lengths.keep), lengths.keep, 0};
    threshold_of<kDigits>(chooser, parts, request, sorted);
    // What the parts before this one hold, and all of them: ties stay from the first on until enough do.
    Emitter emitter{from, to, 0, 0};
    int64_t moves = 0;
    int ties = 0;
    for (int first = 0; first < parts.parts; first += kWave) {
        const int other = first + lane;
        PartCounts c{0, 0, 0, 0};
        int low = 0;
        if (other < parts.parts) {
            c = parts.counts[static_cast<int64_t>(request) * parts.parts + other];
            const PartRange at(lengths.n, parts.parts, other);
            low = (at.end < lengths.keep ? at.end : lengths.keep) - at.begin;
            low = low > 0 ? low : 0;
        }
        const int equal = c.low_equal + c.high_equal, through = wave_inclusive_scan(equal, SumOp{});
        const int ahead = ties + through - equal, left = static_cast<int>(sorted.need) - ahead;
        const int staying = left <= 0 ? 0 : left < equal ? left : equal, staying_low = staying < c.low_equal ? staying : c.low_equal;
        const int movers = c.high + staying - staying_low, holes = low - c.low - staying_low;
        const bool before = other < part;
        emitter.mover_at += wave_reduce(before ? movers : 0, SumOp{});
        emitter.hole_at += wave_reduce(before ? holes : 0, SumOp{});
        sorted.tie += wave_reduce(before ? equal : 0, SumOp{});
        moves += wave_reduce(movers, SumOp{});
        ties += wave_read_lane(through, kWave - 1);
    }
    for (int64_t i = moves + own; i < p.width; i += stride) from[i] = to[i] = -1;
    if (range.begin >= range.end) return;
    // Then the waves before this one.
    const auto each = [&](auto f) { run.each(keys, f); };
    int equal = 0;
    each([&](int, bool there, uint32_t order) { equal += __popcll(wave_ballot(there && order == sorted.threshold)); });
    if (lane == 0) tie_sums[wave] = equal;
    __syncthreads();
    for (int w = 0; w < wave; ++w) sorted.tie += tie_sums[w];
    const int first_tie = sorted.tie;
    int movers = 0, holes = 0;
    each([&](int j, bool there, uint32_t order) {
        bool mover, hole;
        sorted.next(j, there, order, mover, hole);
        movers += __popcll(wave_ballot(mover));
        holes += __popcll(wave_ballot(hole));
    });
    if (lane == 0) {
        mover_sums[wave] = movers;
        hole_sums[wave] = holes;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        emitter.mover_at += mover_sums[w];
        emitter.hole_at += hole_sums[w];
    }
    sorted.tie = first_tie;
    each([&](int j, bool there, uint32_t order) {
        bool mover, hole;
        sorted.next(j, there, order, mover, hole);
        if (wave_ballot(mover || hole) != 0) emitter.put(keys, p.width, j, mover, hole);
    });
}

// ---- rows from slot to slot --------------------------------------------------------------------------------------
constexpr int kMoveBlock = 256;

// A thread a 16-byte chunk of a key and of a value, of EACH moves: their slots first, then all rows, then all writes.
template <int EACH>
__global__ __launch_bounds__(kMoveBlock) void paged_move_kernel(Pages key_cache, Pages value_cache, float* weights, int32_t* positions,
                                                                const int64_t* __restrict__ from, const int64_t* __restrict__ to,
                                                                int64_t moves, int per, Divider chunks, int group, Divider page_size,
                                                                int64_t pages) {
    const int rest = static_cast<int>(blockIdx.y) * kMoveBlock + static_cast<int>(threadIdx.x) % (group > 1 ? per : kMoveBlock);
    const int mine = group > 1 ? static_cast<int>(threadIdx.x) / per : 0;
    if (rest >= per || mine >= group) return;
    const int head = static_cast<int>(chunks(rest)), chunk = rest - head * static_cast<int>(chunks.by);
    const auto page_of = [&](int64_t slot) {
        return slot <= 0xFFFFFFFFll ? static_cast<int64_t>(page_size(static_cast<uint32_t>(slot))) : slot / page_size.by;
    };
    int64_t source[EACH], target[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int64_t move = (static_cast<int64_t>(blockIdx.x) * EACH + e) * group + mine;
        source[e] = move < moves ? from[move] : -1;
        target[e] = move < moves ? to[move] : -1;
    }
    U32x4 k[EACH], v[EACH];
    char* k_to[EACH];
    char* v_to[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        k_to[e] = nullptr;
        if (source[e] < 0 || target[e] < 0) continue;
        const int64_t source_page = page_of(source[e]), target_page = page_of(target[e]);
        if (source_page >= pages || target_page >= pages) continue;
        const int64_t source_at = source[e] - source_page * page_size.by, target_at = target[e] - target_page * page_size.by;
        const auto* k_from = reinterpret_cast<const U32x4*>(key_cache.at(source_page, source_at, head) + chunk * 16);
        const auto* v_from = reinterpret_cast<const U32x4*>(value_cache.at(source_page, source_at, head) + chunk * 16);
        k[e] = EACH > 1 ? __builtin_nontemporal_load(k_from) : *k_from;
        v[e] = EACH > 1 ? __builtin_nontemporal_load(v_from) : *v_from;
        k_to[e] = key_cache.at(target_page, target_at, head) + chunk * 16;
        v_to[e] = value_cache.at(target_page, target_at, head) + chunk * 16;
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        if (k_to[e] == nullptr) continue;
        if (rest == 0) {
            if (weights != nullptr) weights[target[e]] = weights[source[e]];
            if (positions != nullptr) positions[target[e]] = positions[source[e]];
        }
        *reinterpret_cast<U32x4*>(k_to[e]) = k[e];
        *reinterpret_cast<U32x4*>(v_to[e]) = v[e];
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------
// Workgroups of a request: one up to kLongRequest keys, then one for every kPartKeys.  (16 requests of 8,192 keys: one 18 us, parts 42; of
// 16,384: 36 and 42; of 32,768: 55 and 43; of 65,536, more than registers hold: 224 and 48.)  The stated length decides, so one far
// above what requests hold costs time: 256 requests of 1,040 keys 8.1 us stated as such, 17.8 as 16,384, 55 as 16,385, 106 as 32,768
// and 220 as 131,072.
constexpr uint64_t kLongRequest = 16384;
uint64_t parts_of(uint64_t max_kv_length) { return max_kv_length <= kLongRequest ? 1 : ceil_div(max_kv_length, kPartKeys); }
size_t bins_bytes(uint64_t requests) { return align_up(requests * kDigits * kBins * sizeof(uint32_t), kViewAlign); }
size_t plan_bytes(uint64_t requests, uint64_t max_kv_length) {
    const uint64_t parts = parts_of(max_kv_length);
    return requests == 0 || parts == 1 ? 0 : bins_bytes(requests) + align_up(requests * parts * sizeof(PartCounts), kViewAlign);
}

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
    const uint64_t count = parts_of(max_kv_length);
    if (count == 1) {
        LaunchScope scope(what, stream);
        auto* kernel = max_kv_length <= 2 * kEvictBlock ? evict_plan_kernel<2> : max_kv_length <= 8 * kEvictBlock ? evict_plan_kernel<8>
                                                                                                                 : evict_plan_kernel<32>;
        kernel<<<requests, kEvictBlock, 0, stream>>>(weights, positions, block_table, kv_lengths, kept_lengths, shifts, move_from, move_to, p);
        return check_hip(hipGetLastError(), "evict_plan launch");
    }
    if (requests * count > 0x7FFFFFFFull / kPartBlock) return set_error(kInvalidArgument, "%s: too many requests of such length", what);
    if (reinterpret_cast<uintptr_t>(temp) % sizeof(PartCounts) != 0)
        return set_error(kInvalidArgument, "%s: temp storage must be 16-byte aligned", what);
    const EvictArrays a{weights, positions, block_table, kv_lengths, kept_lengths, shifts};
    const Parts parts{static_cast<uint32_t*>(temp), reinterpret_cast<PartCounts*>(static_cast<char*>(temp) + bins_bytes(requests)),
                      static_cast<int>(count)};
    if (int st = launch_fill_u32(parts.bins, static_cast<uint64_t>(requests) * kDigits * kBins, 0, stream); st != kOk) return st;
    const unsigned blocks = static_cast<unsigned>(requests * count);
    LaunchScope scope(what, stream);
    evict_digit_kernel<0><<<blocks, kPartBlock, 0, stream>>>(a, parts, p);
    evict_digit_kernel<1><<<blocks, kPartBlock, 0, stream>>>(a, parts, p);
    evict_digit_kernel<2><<<blocks, kPartBlock, 0, stream>>>(a, parts, p);
    evict_count_kernel<<<blocks, kPartBlock, 0, stream>>>(a, parts, p);
    evict_moves_kernel<<<blocks, kPartBlock, 0, stream>>>(a, parts, move_from, move_to, p);
    return check_hip(hipGetLastError(), "evict_plan launch");
}

// Moves a thread: two where that leaves 64 workgroups for every compute unit, else one (rows of 8 heads of 128: 4,096 moves one 6.0 us,
// two 7.6; 32,768: 43.0 and 45.4; 65,536: 114 and 86; the lists of 16 long prompts, most of them empty: 105 and 77, four 103, eight 229).
constexpr int kMovesEach = 2;
constexpr uint64_t kManyMoves = 32768;

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
    const bool many = moves * per >= kManyMoves * kMoveBlock;
    const int each = many ? kMovesEach : 1;
    auto* kernel = many ? paged_move_kernel<kMovesEach> : paged_move_kernel<1>;
    const uint64_t most = 0x7FFFFFFFull / kMoveBlock / splits * group * each;  // moves of a launch
    LaunchScope scope(what, stream);
    for (uint64_t at = 0; at < moves; at += most) {
        const uint64_t count = moves - at < most ? moves - at : most;
        const uint64_t blocks = ceil_div(count, static_cast<uint64_t>(group) * each);
        kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(splits)), kMoveBlock, 0, stream>>>(
            pages_of(key_cache), pages_of(value_cache), weights, positions, move_from + at, move_to + at, static_cast<int64_t>(count), per,
            Divider(static_cast<uint32_t>(chunks)), group, Divider(page_size), static_cast<int64_t>(pages));
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

size_t lcpp_hip_evict_plan_temp_bytes(uint32_t requests, uint64_t max_kv_length) {
    return attention::plan_bytes(requests, max_kv_length);
}

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
