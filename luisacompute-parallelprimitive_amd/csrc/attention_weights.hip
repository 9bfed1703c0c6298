// Softmax weights that a step's rows gave to each key of a paged cache, added to the keys' sums:
//
//   w_j = decay * w_j (keys that had a sum) + sum over heads h and rows i that see j of exp(scale q_ih k_jg - lse_ih)
//
// with the log-sums that attention over the same pages gave, and g the key head of h.  Scores, exponentials and sums are f32;
// nothing is rounded to 16 bits.  Each key's sum has one owner and one order.
//
// Each key is read once, and that bounds a decoding step: 256 requests of 200 to 4,000 keys (8 key heads of 128, 32 query heads), 669 MB in
// 124 us, 5.4 TB/s, where reads alone reach 6.7.  The last 32 rows of three prompts of 9,000 to 60,000 keys: 22 GFLOP and 175 MB in
// 60 us, bound by the latency of a tile: two or three waves a SIMD fit the registers.
//
// Key heads are what waves share out (many rows) or go through with the next one's keys on their way (few): with fewer than four key
// heads waves of the first have nothing to do (windows of 32 rows of one key head: 122 us for 107 MB), and with one the second waits
// for each tile of keys (256 requests of one key head, 684 MB: 270 us where eight heads of the same bytes take 136).
//
// 2 * dim operations a row, head and key.  Matrix instruction: 16x16x32, rows of queries by keys: lane
// l has key l % 16 of the result, rows 4 (l / 16) .. + 3, so that a key's weights of 16 rows lie in four lanes' registers and are
// added up there; lanes meet once, at the end.
#include "attention.hpp"

namespace lcpp_hip {
namespace attention {
namespace {

constexpr int kWeightWaves = 4;
constexpr int kWeightBlock = kWeightWaves * kWave;
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
    int few;      // rows of a key head that make a request one of few
    int splits;   // workgroups that share the rows of a unit, if there are at most `units` units
    int64_t units;
    int each;     // workgroups of each request, where they are not dealt out over all
    float scale;
    float decay;
};

struct WeighArrays {
    const int32_t* block_table;
    const int32_t* q_offsets;
    const int32_t* kv_lengths;
    const int32_t* known_lengths;
    const uint64_t* tree;
    const float* lse;
    const float* weights_in;
    float* weights_out;
};

// A request's rows and keys.
struct Request {
    int begin, group, rows;
    int held;    // keys that the table has room for
    int ahead;   // keys before the new tokens' own
    int known;   // keys that have a sum to add to
    const int32_t* table;
    __device__ __forceinline__ Request(const WeighArrays& a, const Weigh& p, int request) {
        begin = a.q_offsets[request];
        int end = a.q_offsets[request + 1];
        begin = begin < 0 ? 0 : begin > p.q_tokens ? p.q_tokens : begin;
        end = end < begin ? begin : end > p.q_tokens ? p.q_tokens : end;
        group = p.q_heads / p.kv_heads;
        rows = (end - begin) * group;
        const int length = a.kv_lengths[request] < 0 ? 0 : a.kv_lengths[request];
        const int64_t room = static_cast<int64_t>(p.table_width) * p.page_size.by;
        held = length < room ? length : static_cast<int>(room);
        ahead = length - (end - begin);
        known = a.known_lengths != nullptr ? a.known_lengths[request] : ahead;
        table = a.block_table + request * p.table_stride;
    }
    // The address of row `row` of a key head, and its log-sum as a power of two (infinity where it gives no weight).
    __device__ __forceinline__ const char* row_at(const Rows& q, const Weigh& p, int kv_head, int row) const {
        const int token = static_cast<int>(p.group(row));
        return q.at(begin + token, kv_head * group + row - token * group);
    }
    __device__ __forceinline__ float base_of(const WeighArrays& a, const Weigh& p, int kv_head, int row) const {
        const int token = static_cast<int>(p.group(row));
        const float l = a.lse[static_cast<int64_t>(kv_head * group + row - token * group) * p.q_tokens + begin + token];
        return l == -INFINITY ? INFINITY : l * kLog2e;
    }
    __device__ __forceinline__ int64_t slot(const Weigh& p, int j) const {
        const uint32_t cell = p.page_size(j);
        const int page = table[cell];
        return page < 0 || page >= p.pages ? -1 : static_cast<int64_t>(page) * p.page_size.by + (j - cell * p.page_size.by);
    }
    __device__ __forceinline__ void put(const WeighArrays& a, const Weigh& p, int j, float total) const {
        if (j >= held) return;
        const int64_t at = slot(p, j);
        if (at >= 0) a.weights_out[at] = j < known && a.weights_in != nullptr ? a.weights_in[at] * p.decay + total : total;
    }
};

// Units of KEYS keys of the requests of a kind: each request's by `each` workgroups of its own, or (FLAT) numbered over all requests.
// Then a workgroup counts them for itself, kWeightBlock requests at a time, and takes every gridDim.x-th, so that long and short
// requests fill the device alike.  f(request, its unit, the unit's number, which of the workgroups that share its rows, how many do).
template <int KEYS, bool FEW, bool FLAT>
struct Units {
    template <typename F>
    __device__ __forceinline__ void each(const WeighArrays& a, const Weigh& p, F f) {
        const int r = blockIdx.x / p.each;
        const Request request(a, p, r);
        if ((request.rows <= p.few) != FEW) return;
        const int all = (request.held + KEYS - 1) / KEYS;
        for (int unit = blockIdx.x % p.each; unit < all; unit += p.each) f(r, unit, int64_t{0}, 0, 1);
    }
};
template <int KEYS, bool FEW>
struct Units<KEYS, FEW, true> {
    int64_t sums[kWeightWaves];
    int64_t begins[kWeightBlock];
    template <typename F>
    __device__ __forceinline__ void each(const WeighArrays& a, const Weigh& p, F f) {
        const int wave = threadIdx.x / kWave;
        int64_t before = 0, next = blockIdx.x;
        for (int base = 0; base < p.requests; base += kWeightBlock) {
            const int r = base + static_cast<int>(threadIdx.x);
            int64_t mine = 0;
            if (r < p.requests) {
                const Request request(a, p, r);
                if ((request.rows <= p.few) == FEW) mine = (request.held + KEYS - 1) / KEYS;
            }
            const int64_t inclusive = wave_inclusive_scan(mine, SumOp{});
            __syncthreads();
            if (threadIdx.x % kWave == kWave - 1) sums[wave] = inclusive;
            __syncthreads();
            int64_t begin = inclusive - mine, total = 0;
#pragma unroll
            for (int w = 0; w < kWeightWaves; ++w) {
                begin += w < wave ? sums[w] : 0;
                total += sums[w];
            }
            begins[threadIdx.x] = begin;
            __syncthreads();
            // (Splits are for a few requests alone, which are all counted here.)
            const int splits = p.splits > 1 && total <= p.units ? p.splits : 1;
            for (; next < before + total * splits; next += gridDim.x) {
                const int64_t number = (next - before) / splits;
                int low = 0, high = kWeightBlock;
                while (high - low > 1) {
                    const int middle = low + (high - low) / 2;
                    if (begins[middle] <= number) low = middle;
                    else high = middle;
                }
                low = __builtin_amdgcn_readfirstlane(low);
                f(base + low, static_cast<int>(number - begins[low]), number, static_cast<int>((next - before) % splits), splits);
            }
            before += total * splits;
        }
    }
};

// 16 rows on their way from memory to a matrix instruction's operand.  Lanes side by side load a row's 16-byte chunks side by side (a
// load of 16 rows at a time takes the cache four times as long), write them to LDS, and read back row lane % 16, chunk lane / 16 of
// every four.  Rows in LDS are 16 bytes further apart than they are long: 16 lanes read 64 banks.  Loads have no branch, so that
// those in flight are not waited for where paths meet: past a row's items its first ones are loaded, and taken as zeros.
template <int DP, bool EXACT>
struct Stage {
    static constexpr int kSteps = DP / 32;
    static constexpr int kPerRow = DP > 64 ? 16 : 8;
    static constexpr int kAtOnce = kWave / kPerRow;
    static constexpr int kLoads = 16 / kAtOnce;
    static constexpr int kRowBytes = DP * 2 + 16;
    static constexpr int kBytes = 16 * kRowBytes;
    using Chunks = U32x4[kLoads];
    using Operand = U32x4[kSteps];
    // The row of load i that a lane reads.
    __device__ __forceinline__ static int row(int i) { return i * kAtOnce + static_cast<int>(threadIdx.x % kWave) / kPerRow; }
    __device__ __forceinline__ static int chunk() { return static_cast<int>(threadIdx.x) % kPerRow; }
    __device__ __forceinline__ static U32x4 load(const char* row, int dim) {
        return *reinterpret_cast<const U32x4*>(row + (EXACT && DP != 96 ? chunk() : chunk() * 8 < dim ? chunk() : 0) * 16);
    }
    __device__ __forceinline__ static void write(char* tile, const Chunks& x, int dim) {
        if (DP == 96 && chunk() >= DP / 8) return;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            U32x4 v = x[i];
            if constexpr (!EXACT) {
#pragma unroll
                for (int w = 0; w < 4; ++w) v[w] = chunk() * 8 < dim ? v[w] : 0u;
            }
            *reinterpret_cast<U32x4*>(tile + row(i) * kRowBytes + chunk() * 16) = v;
        }
    }
    __device__ __forceinline__ static void read(const char* tile, Operand& x) {
        const int lane = threadIdx.x % kWave;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) x[s] = *reinterpret_cast<const U32x4*>(tile + lane % 16 * kRowBytes + lane / 16 * 16 + s * 64);
    }
};

// Where key key0 + lane of a unit lies; of the last one past the end, and of any that is there where its page is not.
__device__ __forceinline__ int64_t key_at(const Pages& cache, const Request& r, const Weigh& p, int key0, int keys) {
    const int j = key0 + static_cast<int>(threadIdx.x % kWave) % keys, at = j < r.held ? j : r.held - 1;
    const uint32_t cell = p.page_size(at);
    const int page = r.table[cell];
    const bool there = page >= 0 && page < p.pages;
    return there ? page * cache.page_bytes + (at - static_cast<int>(cell * p.page_size.by)) * cache.token_bytes : 0;
}

// Whether a workgroup's rows have some without a log-sum among them: they give no weight whatever they hold, an infinity or NaN
// too, and take the way of masked rows.  note: each thread's own, between the barriers that its log-sums are written between; any:
// after them.
struct Without {
    int waves[kWeightWaves];
    __device__ __forceinline__ void note(bool mine) {
        const bool some = wave_ballot(mine) != 0;
        if (threadIdx.x % kWave == 0) waves[threadIdx.x / kWave] = some;
    }
    __device__ __forceinline__ bool any() const {
        int all = 0;
#pragma unroll
        for (int w = 0; w < kWeightWaves; ++w) all |= waves[w];
        return __builtin_amdgcn_readfirstlane(all) != 0;
    }
};

// Adds a tile of rows' weights to the sums of the lane's keys; `row0` is the lane's first row of four, `base` their log-sums.
template <typename T, int GROUPS, int STEPS>
__device__ __forceinline__ void weigh(float (&sum)[GROUPS], const U32x4 (&a)[STEPS], const U32x4 (&k)[GROUPS][STEPS], F32x4 base, float c,
                                      bool masked, const WeighArrays& arrays, const Request& request, const Weigh& p, int row0, int key0) {
    Acc acc[GROUPS] = {};
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) acc[g] = product<T>(a[s], k[g][s], acc[g]);
    if (!masked) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[g] += exp2_fast(acc[g][r] * c - base[r]);
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = row0 + r, token = static_cast<int>(p.group(row));
        const bool real = row < request.rows && base[r] != INFINITY;
        const uint64_t word = real && arrays.tree != nullptr ? arrays.tree[request.begin + token] : 0;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const int fresh = key0 + 16 * g + static_cast<int>(threadIdx.x % 16) - request.ahead;  // which of the new keys
            const bool seen = arrays.tree == nullptr ? fresh <= token : fresh < 0 || (fresh < 64 && (word >> fresh & 1) != 0);
            const float w = exp2_fast(acc[g][r] * c - base[r]);
            sum[g] += real && seen ? w : 0.f;
        }
    }
}

// Four lanes have the sums of a key's rows.
template <int GROUPS>
__device__ __forceinline__ void meet(float (&sum)[GROUPS]) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        sum[g] += __shfl_xor(sum[g], 16);
        sum[g] += __shfl_xor(sum[g], 32);
    }
}

// Requests of few rows: a wave goes through the key heads of 16 keys, a tile of 16 rows at a time, the next head's keys on their way
// while it works on one.  (256 requests: 16 keys a wave 124 us, 32 keys 215, 64 keys 203, as more fit fewer waves; with lanes on a key each
// instead of side by side on it 218.)
constexpr int kFewKeys = 16;
constexpr int kFewHeads = 32;  // key heads whose log-sums lie in LDS at once

template <typename T, int DP, bool EXACT, bool FLAT>
__global__ __launch_bounds__(kWeightBlock) void attention_weights_few_kernel(Rows q, Pages key_cache, WeighArrays arrays, Weigh p) {
    using S = Stage<DP, EXACT>;
    constexpr int kGroups = kFewKeys / 16;
    __shared__ __attribute__((aligned(16))) char staged[kWeightWaves][kGroups * S::kBytes];
    __shared__ __attribute__((aligned(16))) float bases[kFewHeads * kRowsAtOnce];
    __shared__ Without without;
    __shared__ Units<kFewKeys * kWeightWaves, true, FLAT> units;
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), column = lane % 16, quarter = lane / 16;
    const float c = p.scale * kLog2e;
    char* tile = staged[wave];
    units.each(arrays, p, [&](int index, int unit, int64_t, int, int) {
        const Request request(arrays, p, index);
        const int key0 = (unit * kWeightWaves + wave) * kFewKeys;
        const bool some = key0 < request.held;
        // Rows that see every key of the unit need no masks.
        const bool masked = key0 + kFewKeys - 1 > (arrays.tree != nullptr ? request.ahead - 1 : request.ahead);
        const int64_t own = key_at(key_cache, request, p, some ? key0 : 0, kFewKeys);
        float sum[kGroups] = {};
        for (int row_base = 0; row_base < request.rows; row_base += kRowsAtOnce) {
            // (Rows that are not there are the tile's first one with a log-sum of infinity: they weigh nothing.)
            const int mine = row_base + column < request.rows ? row_base + column : row_base;
            for (int head_base = 0; head_base < p.kv_heads; head_base += kFewHeads) {
                const int heads = p.kv_heads - head_base < kFewHeads ? p.kv_heads - head_base : kFewHeads;
                __syncthreads();
                bool out = false;
                for (int i = threadIdx.x; i < heads * kRowsAtOnce; i += kWeightBlock) {
                    const int row = row_base + i % kRowsAtOnce;
                    bases[i] = row < request.rows ? request.base_of(arrays, p, head_base + i / kRowsAtOnce, row) : INFINITY;
                    out |= row < request.rows && bases[i] == INFINITY;
                }
                without.note(out);
                __syncthreads();
                if (!some) continue;
                const bool any_masked = masked || without.any();
                const char* from[kGroups][S::kLoads];
#pragma unroll
                for (int g = 0; g < kGroups; ++g)
#pragma unroll
                    for (int i = 0; i < S::kLoads; ++i)
                        from[g][i] = key_cache.data + head_base * key_cache.head_bytes + __shfl(own, 16 * g + S::row(i));
                typename S::Chunks keys[kGroups];
                typename S::Operand a, next;
                const auto load = [&](int local) {
                    const char* row = request.row_at(q, p, head_base + local, mine);
#pragma unroll
                    for (int s = 0; s < S::kSteps; ++s) {
                        const int chunk = 4 * s + quarter;  // (past a row's items: any, the keys' are zeros)
                        next[s] = *reinterpret_cast<const U32x4*>(row + (EXACT || chunk * 8 < p.dim ? chunk : 0) * 16);
                    }
#pragma unroll
                    for (int g = 0; g < kGroups; ++g)
#pragma unroll
                        for (int i = 0; i < S::kLoads; ++i) keys[g][i] = S::load(from[g][i] + local * key_cache.head_bytes, p.dim);
                    __builtin_amdgcn_sched_barrier(0);
                };
                load(0);
                for (int local = 0; local < heads; ++local) {
                    wave_lds_order();
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) S::write(tile + g * S::kBytes, keys[g], p.dim);
#pragma unroll
                    for (int s = 0; s < S::kSteps; ++s) a[s] = next[s];
                    wave_lds_order();
                    load(local + 1 < heads ? local + 1 : local);  // (the last one again: a load, but no branch)
                    typename S::Operand k[kGroups];
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) S::read(tile + g * S::kBytes, k[g]);
                    const F32x4 base = *reinterpret_cast<const F32x4*>(&bases[local * kRowsAtOnce + 4 * quarter]);
                    weigh<T>(sum, a, k, base, c, any_masked, arrays, request, p, row_base + 4 * quarter, key0);
                }
            }
        }
        meet(sum);
        float total = sum[0];  // of group `quarter`
#pragma unroll
        for (int g = 1; g < kGroups; ++g) total = quarter == g ? sum[g] : total;
        if (quarter < kGroups) request.put(arrays, p, key0 + lane, total);
    });
}

// Requests of more rows: a workgroup has 48 keys, its waves take the key heads in turn and go through their rows, the next tile on
// its way while they work on one; the waves' sums meet in LDS.  (Three windows of 32 rows: 48 keys 59 us, 64 keys, which fill the
// registers of two waves a SIMD, 62, 32 keys, which read the rows more often, 69.)
constexpr int kManyKeys = 48;
constexpr int kTableHeads = 64;  // key heads that the table of rows holds at once
constexpr int kTableRows = 2048;

// Where each row of a few key heads lies, after the request's first, and its log-sum.  Rows that are not there are the table's first
// one, with a log-sum of infinity.
struct RowTable {
    int64_t at[kTableRows];
    __attribute__((aligned(16))) float base[kTableRows];
};

template <typename T, int DP, bool EXACT, bool FLAT>
__global__ __launch_bounds__(kWeightBlock, 3) void attention_weights_many_kernel(Rows q, Pages key_cache, WeighArrays arrays, float* partial,
                                                                              Weigh p) {
    using S = Stage<DP, EXACT>;
    constexpr int kGroups = kManyKeys / 16;
    __shared__ RowTable table;
    __shared__ __attribute__((aligned(16))) char staged[kWeightWaves][S::kBytes];
    __shared__ float sums[kWeightWaves][kManyKeys];
    __shared__ Without without;
    __shared__ Units<kManyKeys, false, FLAT> units;
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), column = lane % 16, quarter = lane / 16;
    const float c = p.scale * kLog2e;
    char* stage = staged[wave];
    const int heads_at_once = p.kv_heads < kTableHeads ? p.kv_heads : kTableHeads;
    const int most_rows = kTableRows / heads_at_once / kRowsAtOnce * kRowsAtOnce;
    int held_request = -1;  // whose rows all lie in the table
    bool held_without = false;
    units.each(arrays, p, [&](int index, int unit, int64_t number, int split, int splits) {
        const Request request(arrays, p, index);
        const char* first_row = q.at(request.begin, 0);
        const int key0 = unit * kManyKeys;
        const bool masked = key0 + kManyKeys - 1 > (arrays.tree != nullptr ? request.ahead - 1 : request.ahead);
        const int64_t own = key_at(key_cache, request, p, key0, kManyKeys);
        // The split's tiles of rows.
        const int all_tiles = (request.rows + kRowsAtOnce - 1) / kRowsAtOnce, per = (all_tiles + splits - 1) / splits;
        const int first_tile = split * per < all_tiles ? split * per : all_tiles;
        const int tile_end = first_tile + per < all_tiles ? first_tile + per : all_tiles;
        const int row_first = first_tile * kRowsAtOnce, row_end = tile_end < all_tiles ? tile_end * kRowsAtOnce : request.rows;
        float sum[kGroups] = {};
        for (int row_base = row_first; row_base < row_end; row_base += most_rows) {
            const int some = row_end - row_base < most_rows ? row_end - row_base : most_rows;
            const int tiles = (some + kRowsAtOnce - 1) / kRowsAtOnce, table_rows = tiles * kRowsAtOnce;
            for (int head_base = 0; head_base < p.kv_heads; head_base += heads_at_once) {
                const int heads = p.kv_heads - head_base < heads_at_once ? p.kv_heads - head_base : heads_at_once;
                if (held_request != index) {
                    __syncthreads();
                    bool out = false;
                    for (int i = threadIdx.x; i < heads * table_rows; i += kWeightBlock) {
                        const int local = i / table_rows, row = i - local * table_rows;
                        const bool real = row < some;
                        const int at = real ? row_base + row : row_base;
                        table.at[i] = request.row_at(q, p, head_base + local, at) - first_row;
                        table.base[i] = real ? request.base_of(arrays, p, head_base + local, at) : INFINITY;
                        out |= real && table.base[i] == INFINITY;
                    }
                    without.note(out);
                    __syncthreads();
                    held_without = without.any();
                    held_request = splits == 1 && some == request.rows && heads == p.kv_heads ? index : -1;
                }
                for (int local = wave; local < heads; local += kWeightWaves) {
                    typename S::Operand k[kGroups], a;
                    typename S::Chunks rows;
                    {
                        typename S::Chunks keys[kGroups];
#pragma unroll
                        for (int g = 0; g < kGroups; ++g)
#pragma unroll
                            for (int i = 0; i < S::kLoads; ++i)
                                keys[g][i] = S::load(key_cache.at(0, 0, head_base + local) + __shfl(own, 16 * g + S::row(i)), p.dim);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int g = 0; g < kGroups; ++g) {
                            wave_lds_order();
                            S::write(stage, keys[g], p.dim);
                            wave_lds_order();
                            S::read(stage, k[g]);
                        }
                    }
                    const auto load = [&](int tile) {
#pragma unroll
                        for (int i = 0; i < S::kLoads; ++i)
                            rows[i] = S::load(first_row + table.at[local * table_rows + tile * kRowsAtOnce + S::row(i)], p.dim);
                        __builtin_amdgcn_sched_barrier(0);
                    };
                    load(0);
                    for (int tile = 0; tile < tiles; ++tile) {
                        wave_lds_order();
                        S::write(stage, rows, p.dim);
                        wave_lds_order();
                        load(tile + 1 < tiles ? tile + 1 : tile);
                        S::read(stage, a);
                        const int row0 = tile * kRowsAtOnce + 4 * quarter;
                        const F32x4 base = *reinterpret_cast<const F32x4*>(&table.base[local * table_rows + row0]);
                        weigh<T>(sum, a, k, base, c, masked || held_without, arrays, request, p, row_base + row0, key0);
                    }
                }
            }
        }
        meet(sum);
        __syncthreads();
        if (quarter == 0)
#pragma unroll
            for (int g = 0; g < kGroups; ++g) sums[wave][16 * g + column] = sum[g];
        __syncthreads();
        if (threadIdx.x < kManyKeys) {
            float total = 0.f;
#pragma unroll
            for (int w = 0; w < kWeightWaves; ++w) total += sums[w][threadIdx.x];
            if (FLAT && splits > 1) partial[(split * p.units + number) * kManyKeys + threadIdx.x] = total;
            else request.put(arrays, p, key0 + static_cast<int>(threadIdx.x), total);
        }
    });
}

// Adds up the splits of each unit, in their order.
__global__ __launch_bounds__(kWeightBlock) void attention_weights_join_kernel(const float* __restrict__ partial, WeighArrays arrays, Weigh p) {
    __shared__ Units<kManyKeys, false, true> units;
    units.each(arrays, p, [&](int index, int unit, int64_t number, int split, int splits) {
        if (splits == 1 || split != 0 || threadIdx.x >= kManyKeys) return;
        float total = 0.f;
        for (int i = 0; i < splits; ++i) total += partial[(i * p.units + number) * kManyKeys + threadIdx.x];
        const Request request(arrays, p, index);
        request.put(arrays, p, unit * kManyKeys + static_cast<int>(threadIdx.x), total);
    });
}

// Workgroups of each request: as many as it has units at the stated length, as long as all have so many together (256 requests of
// one token and up to 4,000 keys: 124 us; three windows of 32 rows, 683 a request: 59).
constexpr uint64_t kFewOwn = 16384;
constexpr uint64_t kManyOwn = 2048;
// Where that leaves a request fewer than it has units and than the device has compute units, the longest would decide, and all units
// are dealt out to so many workgroups: twice and once what the device holds at a time (256 requests of a token: 138 us with 768, 132
// with 1,536, 145 with 8,192; 64 of 16 tokens: 85 us with 512, 97 with 768, 89 with 2,048).  A request of 500 tokens over 8,000 keys
// among 255 of one: 445 us, by request 2,891; 256 requests of one token over 1,300 keys each: 138 us, by request 130.
constexpr uint64_t kFlatBelow = 256;
constexpr uint64_t kFewGrid = 1536;
constexpr uint64_t kManyGrid = 512;
// Workgroups wanted where rows are split (one request of 4,096 tokens over 8,192 keys: 2,481 us unsplit, 1,344 with 512, 862 with
// 1,024; at 867 us 240 TFLOP/s: each tile of 16 rows passes LDS for each 48 keys).
constexpr uint64_t kSplitGrid = 1024;
// Rows of a key head up to which a request counts as one of few.
constexpr int kFewRows = 16;

bool is_few(uint64_t requests, uint64_t q_tokens, uint64_t group) {
    return (q_tokens <= requests && group <= kFewRows) || q_tokens * group <= kFewRows;
}

// Workgroups that share a unit's rows: as many as the grid has for each unit, where there are few units of many rows (in requests of
// the stated length, at most kWeightBlock of them), and each has four tiles of rows at least.
struct Split {
    uint64_t splits, units;
    Split(uint64_t requests, uint64_t q_tokens, uint64_t max_kv_length, uint64_t q_heads, uint64_t kv_heads) {
        units = requests * ceil_div(max_kv_length ? max_kv_length : 1, kManyKeys);
        const uint64_t rows = kv_heads ? q_tokens * (q_heads / kv_heads) : 0, tiles = rows / (4 * kRowsAtOnce);
        splits = requests == 0 || requests > kWeightBlock || units > kSplitGrid / 2 ? 1 : kSplitGrid / units;
        splits = splits < tiles ? splits : tiles ? tiles : 1;
    }
    size_t bytes() const { return splits > 1 ? align_up(splits * units * kManyKeys * sizeof(float), kViewAlign) : 0; }
};

template <typename T, int DP, bool EXACT>
void launch_weights(const Rows& q, const Pages& key_cache, const WeighArrays& arrays, float* partial, const Weigh& p, uint64_t max_kv_length,
                    bool few, bool many, hipStream_t stream) {
    const auto launch = [&](auto own_kernel, auto flat_kernel, uint64_t keys, uint64_t most_own, uint64_t most, int splits, auto... arguments) {
        const uint64_t each = ceil_div(max_kv_length ? max_kv_length : 1, keys), units = p.requests * each * splits;
        const uint64_t share = ceil_div(most_own, uint64_t(p.requests)), parts = share < each ? share : each;
        Weigh by = p;
        by.splits = splits;
        by.each = static_cast<int>(parts);
        if (splits > 1 || (parts < each && parts < kFlatBelow))
            flat_kernel<<<static_cast<unsigned>(splits > 1 || units < most ? units : most), kWeightBlock, 0, stream>>>(arguments..., by);
        else
            own_kernel<<<static_cast<unsigned>(parts * p.requests), kWeightBlock, 0, stream>>>(arguments..., by);
    };
    if (few)
        launch(attention_weights_few_kernel<T, DP, EXACT, false>, attention_weights_few_kernel<T, DP, EXACT, true>,
               kFewKeys * kWeightWaves, kFewOwn, kFewGrid, 1, q, key_cache, arrays);
    if (many)
        launch(attention_weights_many_kernel<T, DP, EXACT, false>, attention_weights_many_kernel<T, DP, EXACT, true>, kManyKeys, kManyOwn,
               kManyGrid, p.splits, q, key_cache, arrays, partial);
    if (many && p.splits > 1)
        launch(attention_weights_join_kernel, attention_weights_join_kernel, kManyKeys, kManyOwn, kManyGrid, p.splits, partial, arrays);
}

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
    if (needed && reinterpret_cast<uintptr_t>(temp) % alignof(float) != 0)
        return set_error(kInvalidArgument, "%s: temp storage must be 4-byte aligned", what);
    // A cache of no pages has no slot to add to, and not the first page that the kernels read in place of one that is not there.
    if (pages == 0) return kOk;
    // One token a request on average, or no more than a tile of rows in all: all requests count as ones of few rows.  More than
    // that on average: all as ones of many.  Otherwise each goes by its own rows, in two launches.  (256 requests of one token: 130 us,
    // 135 with the second launch; a request of 200 tokens over 8,000 keys among 255 of none: 320 us, 130 with it.)
    const uint64_t group = q_heads / kv_heads;
    const bool all_few = is_few(requests, q_tokens, group), all_many = q_tokens * group > uint64_t{requests} * kFewRows;
    const Split split(requests, all_few ? 0 : q_tokens, max_kv_length, q_heads, kv_heads);
    const Weigh p{static_cast<int>(requests), static_cast<int>(q_tokens), static_cast<int>(q_heads), static_cast<int>(kv_heads),
                  static_cast<int>(dim), Divider(q_heads / kv_heads), Divider(page_size), static_cast<int>(pages),
                  static_cast<int64_t>(table_stride), static_cast<int>(table_width),
                  all_few ? INT32_MAX : all_many ? -1 : kFewRows,
                  static_cast<int>(split.splits), static_cast<int64_t>(split.units), 0, scale, decay};
    const WeighArrays arrays{block_table, q_offsets, kv_lengths, known_lengths, tree, lse, weights_in, weights_out};
    const Rows q_rows = q_tokens ? rows_of(q) : Rows{};
    LaunchScope scope(what, stream);
    auto* launch = dim == 64    ? launch_weights<T, 64, true>
                   : dim < 64   ? launch_weights<T, 64, false>
                   : dim == 96  ? launch_weights<T, 96, true>
                   : dim < 96   ? launch_weights<T, 96, false>
                   : dim == 128 ? launch_weights<T, 128, true>
                                : launch_weights<T, 128, false>;
    launch(q_rows, pages_of(key_cache), arrays, static_cast<float*>(temp), p, max_kv_length, !all_many, !all_few, stream);
    return check_hip(hipGetLastError(), "attention_paged_weights launch");
}

}  // namespace
}  // namespace attention
}  // namespace lcpp_hip

using namespace lcpp_hip;

extern "C" {

size_t lcpp_hip_attention_paged_weights_temp_bytes(uint32_t requests, uint64_t q_tokens, uint64_t max_kv_length, uint32_t q_heads,
                                                   uint32_t kv_heads, uint32_t) {
    return kv_heads == 0 || attention::is_few(requests, q_tokens, q_heads / kv_heads) ? 0 : attention::Split(requests, q_tokens, max_kv_length, q_heads, kv_heads).bytes();
}

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
