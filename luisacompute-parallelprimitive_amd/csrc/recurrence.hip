// A gated linear recurrence over the sequences of a ragged batch, channel by channel, and its gradients:
//
//   h_t = exp(l_t) h_{t-1} + x_t,   h_0 an initial state or 0;
//   g_t = dh_t + c_{t+1},  c_t = exp(l_t) g_t,   dx_t = g_t,  dl_t = c_t h_{t-1},  dh_0 = c_1.
//
// States are f32; outputs are rounded once.  A state that remembers thousands of tokens adds up as many errors of exp(l): for
// small l the step is h + (exp(l) - 1) h + x with exp(l) - 1 from its series, whose error is relative to l.
//
// Memory bounds the large calls: 3 items a channel and token forwards, 5 backwards, each once, and 3% of what chunks hand on.
// 34,222 tokens of 4,096 channels in bf16: forwards 0.84 GB in 219 us, 3.8 TB/s, backwards 1.40 GB in 286, 4.9, where the library's copy
// reaches 6.0; in f32 twice the bytes in 304 and 482, 5.5 and 5.8.  A workgroup loads, waits for its state and stores, and two of them on a compute unit do not quite cover each
// other's waits (forwards without looking back, which is wrong, 183 us).  (One pass over the rows by a thread a channel took 27.8 ms
// for both.)  1,900 tokens of 770 channels: 14 us a direction, the latency of one chunk.  A wave has one sequence's channels: of 16 channels
// it uses 4 lanes, and 34,222 tokens take 45 us a direction for 3 MB, as those of 64 do.
#include "common.hpp"
#include "../../include/lcpp_hip.h"
#include "attention.hpp"

#include <initializer_list>

namespace lcpp_hip {
namespace recurrence {
namespace {

using attention::Bf16;
using attention::F16;
struct F32 {
    using Item = float;
};

template <typename T>
__device__ __forceinline__ float to_float(typename T::Item x) {
    return static_cast<float>(x);
}

// A number of 32 bits rounded to the items' type.  (In f16 a product or sum would be rounded to 16 bits in one step in one place and
// in two in another, as the compiler finds, and rows that are gone through twice would not come out the same.)
template <typename T>
__device__ __forceinline__ typename T::Item rounded(float x) {
    if constexpr (std::is_same_v<T, F16>) asm("" : "+v"(x));
    return static_cast<typename T::Item>(x);
}

constexpr float kSmall = 0.0625f;

// y -> exp(l) y + x, with what depends on l alone.
struct Decay {
    float factor;  // exp(l), or exp(l) - 1 where l is small
    bool small;
    bool keeps;    // l is above -infinity
    __device__ __forceinline__ explicit Decay(float l) {
        // (The first term left out is l^5 / 120, 1.3e-7 of l.)
        const float series = l * __builtin_fmaf(l, __builtin_fmaf(l, __builtin_fmaf(l, 1.f / 24.f, 1.f / 6.f), 0.5f), 1.f);
        small = __builtin_fabsf(l) < kSmall;
        factor = small ? series : attention::exp2_fast(l * attention::kLog2e);
        keeps = l > -INFINITY;
    }
    __device__ __forceinline__ float step(float y, float x) const { return __builtin_fmaf(factor, y, small ? y + x : x); }
    __device__ __forceinline__ float times(float y) const { return __builtin_fmaf(factor, y, small ? y : 0.f); }
    // The same of an infinite y too: any exp(l) above 0 leaves it what it is, where exp(l) - 1, or an exp(l) that is 0 in 32 bits,
    // makes NaN of it.  Rows in registers go without this and are gone through again where a NaN comes out, which stays to their end.
    // (Both directions of 34,222 tokens: 481 us, without any of it 470; with NaN looked for in the hand-over too 490.)
    __device__ __forceinline__ float step_any(float y, float x) const { return __builtin_isinf(y) && keeps ? y + x : step(y, x); }
    __device__ __forceinline__ float times_any(float y) const { return __builtin_isinf(y) && keeps ? y : times(y); }
};

struct Shape {
    int sequences;
    int64_t tokens;
    int channels;
    int num_states;
};

struct Steps {
    char* data;
    int64_t token_bytes;
    template <typename Item>
    __device__ __forceinline__ Item* at(int64_t token) const {
        return reinterpret_cast<Item*>(data + token * token_bytes);
    }
};

struct Span {
    int64_t begin, size;
};
__device__ __forceinline__ Span span_of(const int32_t* offsets, int sequence, int64_t tokens) {
    int64_t begin = offsets[sequence], end = offsets[sequence + 1];
    begin = begin < 0 ? 0 : begin > tokens ? tokens : begin;
    end = end < begin ? begin : end > tokens ? tokens : end;
    return {begin, end - begin};
}

// The row of the states that a sequence has; -1: none.
__device__ __forceinline__ int64_t state_of(const int32_t* rows, int sequence, int num_states) {
    const int row = rows != nullptr ? rows[sequence] : sequence;
    return row >= 0 && row < num_states ? row : -1;
}

// ---- chunks ------------------------------------------------------------------------------------------------------
// A chunk of a sequence is waves of kRows tokens; a lane has V neighbouring channels of a token, 8 bytes of them where the
// rows allow.  (The two directions of 34,222 tokens, measured before infinite states were kept, which added 11 us: eight waves of 16 rows
// 466 us, four waves 479, eight of 8 rows 515, sixteen of 8 rows 554.  Sequences of a few hundred rows alone would take 26 us for 31 with eight waves of 8.)  A chunk's effect on the state
// is h -> exp(L) h + B.  A workgroup reads its chunk into registers once, makes each wave's
// (L, B) and the chunk's, hands that on, gets the state that enters the chunk, and goes through its rows again with it.  The
// backward pass does the same towards the sequence's start, with c in the place of h.
//
// The state that enters a chunk is made from one that is known, the nearest, by the (L, B) of the chunks in between, in their order:
// it is the same sum whichever that was, so results do not depend on timing.  A workgroup that has polled for a chunk's (L, B) long
// enough makes it itself, from the rows: nothing has to run for another to end.
constexpr int kRows = 16;
constexpr uint32_t kNotYet = ~0u;  // a NaN that is never handed on

__device__ __forceinline__ uint32_t handed(float x) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, x);
    return bits == kNotYet ? 0x7FC00000u : bits;
}

// h -> exp(l) h + b.  With the sum of the l, not the product of the decays, a chunk's decay has no rounding of its own: where all
// tokens decay alike it would be the same one in every chunk, and add up.  (A memory of 10,000 tokens, all alike: 1.8e-5 off with
// products.)
struct Effect {
    float l, b;
    // (ANY: where b, or the state, may be infinite.)  This one, then another.
    template <bool ANY>
    __device__ __forceinline__ void then(Effect next) {
        b = next.of<ANY>(b);
        l += next.l;
    }
    // This one, then a row.
    template <bool BACK, bool ANY>
    __device__ __forceinline__ void row(float l_row, float x) {
        const Decay d(l_row);
        if constexpr (ANY) b = BACK ? d.times_any(x + b) : d.step_any(b, x);
        else b = BACK ? d.times(x + b) : d.step(b, x);
        l += l_row;
    }
    template <bool ANY>
    __device__ __forceinline__ float of(float h) const {
        return ANY ? Decay(l).step_any(h, b) : Decay(l).step(h, b);
    }
};

__device__ __forceinline__ uint64_t handed(Effect e) { return static_cast<uint64_t>(handed(e.b)) << 32 | handed(e.l); }

// What workgroups hand on, a word a channel of a chunk: (L, B), and the state that enters the chunk.
struct Handed {
    uint64_t* effects;
    uint32_t* states;
    int64_t stride;  // channels, rounded up
};

template <typename Item, int V>
struct alignas(sizeof(Item) * V) Items {
    Item at[V];
};

struct Inputs {
    Steps first;  // x, or dout
    Steps log_decay;
    Steps out;    // written forwards, read backwards
    Steps dx, dlog_decay;
    const int32_t* offsets;
    const float* initial;
    const float* dfinal;
    const int32_t* state_rows;
    float* last;  // final, or dinitial
};

// Rows [token, token + count) of an array as a wave reads and writes them: what lies past them, or is asked for at kNowhere, reads
// as zeros and is not written.  (Offsets are below 2^31, as strides are below 2^26 bytes.)
constexpr uint32_t kNowhere = 0x7FFFFFFF;
constexpr int kOnce = 2;  // (each row is read once and written once: they stay out of the caches, 466 us where 490 were taken then)

template <typename Vec>
struct Window {
    __amdgpu_buffer_rsrc_t rows;
    uint32_t token_bytes;
    __device__ __forceinline__ Window(const Steps& s, int64_t token, int count, int row_bytes)
        : rows(__builtin_amdgcn_make_buffer_rsrc(s.data + token * s.token_bytes, 0,
                                                 count > 0 ? (count - 1) * static_cast<int>(s.token_bytes) + row_bytes : 0, 0x00020000)),
          token_bytes(static_cast<uint32_t>(s.token_bytes)) {}
    __device__ __forceinline__ Vec load(int row, uint32_t at) const {
        const int offset = static_cast<int>(at + row * token_bytes);
        if constexpr (sizeof(Vec) == 8) return __builtin_bit_cast(Vec, __builtin_amdgcn_raw_buffer_load_b64(rows, offset, 0, kOnce));
        else if constexpr (sizeof(Vec) == 4) return __builtin_bit_cast(Vec, __builtin_amdgcn_raw_buffer_load_b32(rows, offset, 0, kOnce));
        else return __builtin_bit_cast(Vec, __builtin_amdgcn_raw_buffer_load_b16(rows, offset, 0, kOnce));
    }
    __device__ __forceinline__ void store(int row, uint32_t at, Vec x) const {
        const int offset = static_cast<int>(at + row * token_bytes);
        if constexpr (sizeof(Vec) == 8) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(attention::U32x2, x), rows, offset, 0, kOnce);
        else if constexpr (sizeof(Vec) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), rows, offset, 0, kOnce);
        else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, x), rows, offset, 0, kOnce);
    }
};

// A wave's rows of its channels; zeros, which are what is not there, leave a state as it is.
template <typename T, int V, bool BACK>
struct WaveRows {
    using Vec = Items<typename T::Item, V>;
    Vec x[kRows], l[kRows];
    __device__ __forceinline__ void load(const Window<Vec>& first, const Window<Vec>& log_decay, uint32_t at) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            x[r] = first.load(r, at);
            l[r] = log_decay.load(r, at);
        }
    }
    // Forgets what is known of the rows, so that nothing made of them for their effect is kept for the second time through them.
    __device__ __forceinline__ void forget() {
        using Word = std::conditional_t<sizeof(Vec) == 8, attention::U32x2, std::conditional_t<sizeof(Vec) == 4, uint32_t, uint16_t>>;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            Word a = __builtin_bit_cast(Word, x[r]), b = __builtin_bit_cast(Word, l[r]);
            asm volatile("" : "+v"(a), "+v"(b));
            x[r] = __builtin_bit_cast(Vec, a);
            l[r] = __builtin_bit_cast(Vec, b);
        }
    }
    __device__ __forceinline__ void effect(Effect (&e)[V], int count) const {
#pragma unroll
        for (int v = 0; v < V; ++v) e[v] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int r = BACK ? kRows - 1 - i : i;
            if (r < count)
#pragma unroll
                for (int v = 0; v < V; ++v) e[v].template row<BACK, false>(to_float<T>(l[r].at[v]), to_float<T>(x[r].at[v]));
            __builtin_amdgcn_sched_barrier(0);  // (a row at a time: all decays at once would take the registers)
        }
    }
    // The same where states may be infinite, from memory, row by row.
    __device__ __forceinline__ static void effect_any(Effect (&e)[V], int rows, const Window<Vec>& first, const Window<Vec>& log_decay, uint32_t at) {
#pragma unroll
        for (int v = 0; v < V; ++v) e[v] = {0.f, 0.f};
#pragma unroll 1
        for (int i = 0; i < rows; ++i) {
            const int r = BACK ? rows - 1 - i : i;
            const Vec x_row = first.load(r, at), l_row = log_decay.load(r, at);
#pragma unroll
            for (int v = 0; v < V; ++v) e[v].template row<BACK, true>(to_float<T>(l_row.at[v]), to_float<T>(x_row.at[v]));
        }
    }
    // Whether any of a wave's V values a lane is NaN.
    template <typename F>
    __device__ __forceinline__ static bool any_nan(F value) {
        bool found = false;
#pragma unroll
        for (int v = 0; v < V; ++v) found |= value(v) != value(v);
        return wave_ballot(found) != 0;
    }
};

// A chunk's place: chunk `index` of its sequence's, tokens [token, token + count).
struct Chunk {
    int sequence, index, chunks;
    int64_t begin;  // of the sequence
    int64_t size;
    template <int WAVES>
    __device__ __forceinline__ bool find(const int32_t* offsets, const Shape& p, int number) {
        constexpr int kChunk = WAVES * kRows;
        const attention::TilePlace place = attention::find_tile(offsets, p.sequences, 1, kChunk, number);
        if (place.sequence < 0) return false;
        const Span span = span_of(offsets, place.sequence, p.tokens);
        sequence = place.sequence;
        index = place.tile;
        begin = span.begin;
        size = span.size;
        chunks = static_cast<int>((span.size + kChunk - 1) / kChunk);
        return index < chunks || (index == 0 && size == 0);
    }
};

// What the owner of a chunk makes of it, the same way, for a channel.
template <typename T, bool BACK, int WAVES>
__device__ __forceinline__ Effect effect_of_chunk(const Inputs& in, int64_t token, int count, int channel) {
    using Item = typename T::Item;
    Effect all = {0.f, 0.f};
#pragma unroll 1
    for (int i = 0; i < WAVES; ++i) {
        const int w = BACK ? WAVES - 1 - i : i, rows = count - w * kRows < kRows ? count - w * kRows : kRows;
        Effect part = {0.f, 0.f};
#pragma unroll 1
        for (int k = 0; k < rows; ++k) {
            const int64_t t = token + w * kRows + (BACK ? rows - 1 - k : k);
            part.row<BACK, true>(to_float<T>(in.log_decay.template at<Item>(t)[channel]), to_float<T>(in.first.template at<Item>(t)[channel]));
        }
        all.then<true>(part);
    }
    return all;
}

// The state that enters chunk `number`, `before` chunks after the sequence's first one (the last one, backwards); a channel a lane.
template <typename T, bool BACK, int WAVES>
__device__ __forceinline__ float look_back(const Inputs& in, const Handed& h, const Chunk& chunk, int64_t number, int before, int channel,
                                           bool active, uint32_t patience) {
    constexpr int kChunk = WAVES * kRows, kAtOnce = 4;
    const int64_t step = BACK ? h.stride : -h.stride;  // to the chunk before
    const uint32_t* states = h.states + number * h.stride;
    const uint64_t* effects = h.effects + number * h.stride;
    const uint32_t lane_at = active ? channel : 0;
    // The nearest known state: of the chunk itself (0), or `back` before it.  (The first chunk's is there from the start.)
    int back = 0;
    uint32_t state = kNotYet;
    for (bool found = false; !found;) {
        uint32_t words[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) words[i] = atomic_load_agent(states + (back + i < before ? back + i : before) * step + lane_at);
        int nearest = before;
#pragma unroll
        for (int i = kAtOnce - 1; i >= 0; --i) {
            if (wave_ballot(active && words[i] == kNotYet) == 0) {
                found = true;
                nearest = back + i < before ? back + i : before;
                state = words[i];
            }
        }
        back = found ? nearest : back + kAtOnce < before ? back + kAtOnce : before;
    }
    float value = __builtin_bit_cast(float, state);
    // Then the chunks in between, as they come.
    for (; back > 0; back -= kAtOnce) {
        uint64_t words[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) words[i] = atomic_load_agent(effects + (back - i > 1 ? back - i : 1) * step + lane_at);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int at = back - i;
            if (at < 1) continue;
            for (uint32_t polls = 0; wave_ballot(active && words[i] == ~uint64_t{0}) != 0; ++polls) {
                if (polls < patience) {
                    __builtin_amdgcn_s_sleep(1);
                    words[i] = atomic_load_agent(effects + at * step + lane_at);
                    continue;
                }
                const int64_t row0 = static_cast<int64_t>(BACK ? chunk.index + at : chunk.index - at) * kChunk;
                const int count = chunk.size - row0 < kChunk ? static_cast<int>(chunk.size - row0) : kChunk;
                words[i] = handed(effect_of_chunk<T, BACK, WAVES>(in, chunk.begin + row0, count, active ? channel : 0));
                break;
            }
            const Effect e = {__builtin_bit_cast(float, static_cast<uint32_t>(words[i])),
                              __builtin_bit_cast(float, static_cast<uint32_t>(words[i] >> 32))};
            value = e.of<true>(value);
        }
    }
    return value;
}

// Short sequences: a lane walks its channels through a sequence, kWalkRows tokens at a time, the next ones on their way while it
// works on some.  256 states of 4,096 channels and a token each: 14.7 MB in 6 to 8 us, of which an empty launch takes 2 to 3.
constexpr int kWalkRows = 8;

template <typename T, int V, bool BACK>
struct WalkRows {
    using Vec = Items<typename T::Item, V>;
    Vec x[kWalkRows], l[kWalkRows], h[BACK ? kWalkRows : 1];
    // Tokens from `done` on (backwards, the sequence's last one first).
    __device__ __forceinline__ void load(const Inputs& in, const Span& span, int64_t done, int row_bytes, uint32_t at) {
        const int64_t left = span.size - done, token = BACK ? span.begin + left - kWalkRows : span.begin + done;
        const int some = left < kWalkRows ? static_cast<int>(left) : kWalkRows;
        // Backwards the last rows of the window are the sequence's next ones; a window that would begin before the sequence is short.
        const int skip = BACK && left < kWalkRows ? kWalkRows - (left > 0 ? static_cast<int>(left) : 0) : 0;
        const Window<Vec> first(in.first, token + skip, some, row_bytes), log_decay(in.log_decay, token + skip, some, row_bytes);
#pragma unroll
        for (int r = 0; r < kWalkRows; ++r) {
            const int row = BACK ? kWalkRows - 1 - r - skip : r;  // (negative: nowhere)
            const uint32_t from = BACK && row < 0 ? kNowhere : at;
            x[r] = first.load(BACK && row < 0 ? 0 : row, from);
            l[r] = log_decay.load(BACK && row < 0 ? 0 : row, from);
        }
        if constexpr (BACK) {
            const int late = token + skip == span.begin;
            const Window<Vec> out(in.out, token + skip - 1 + late, some - late, row_bytes);
#pragma unroll
            for (int r = 0; r < kWalkRows; ++r) {
                const int row = kWalkRows - 1 - r - skip - late;
                h[r] = out.load(row < 0 ? 0 : row, row < 0 ? kNowhere : at);
            }
        }
    }
};

template <typename T, int V, bool BACK>
__global__ __launch_bounds__(kWave) void recurrence_walk_kernel(Inputs in, Shape p, int first_sequence, int blocks) {
    using Item = typename T::Item;
    using Vec = Items<Item, V>;
    const int sequence = first_sequence + static_cast<int>(blockIdx.x / blocks);
    const int channel = (static_cast<int>(blockIdx.x % blocks) * kWave + static_cast<int>(threadIdx.x)) * V;
    const bool active = channel < p.channels;
    const Span span = span_of(in.offsets, sequence, p.tokens);
    const int64_t held = BACK ? sequence : state_of(in.state_rows, sequence, p.num_states);
    const int row_bytes = p.channels * static_cast<int>(sizeof(Item));
    const uint32_t at = active ? static_cast<uint32_t>(channel) * sizeof(Item) : kNowhere;
    WalkRows<T, V, BACK> even, odd;
    even.load(in, span, 0, row_bytes, at);
    const float* from = BACK ? in.dfinal : in.initial;
    float state[V], first[V];  // (backwards: the state before the first token)
#pragma unroll
    for (int v = 0; v < V; ++v) {
        state[v] = from != nullptr && held >= 0 && active ? from[held * p.channels + channel + v] : 0.f;
        first[v] = BACK && in.initial != nullptr && active ? in.initial[held * p.channels + channel + v] : 0.f;
    }
    const auto work = [&](const WalkRows<T, V, BACK>& rows, int64_t done) {
        const int64_t left = span.size - done;
        const int some = left < kWalkRows ? static_cast<int>(left) : kWalkRows;
        const int64_t token = BACK ? span.begin + left - some : span.begin + done;
        const Window<Vec> a(BACK ? in.dx : in.out, token, some, row_bytes), b(BACK ? in.dlog_decay : in.out, token, BACK ? some : 0, row_bytes);
#pragma unroll
        for (int r = 0; r < kWalkRows; ++r) {
            if (r >= some) continue;
            Vec g_row, l_row;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const Decay d(to_float<T>(rows.l[r].at[v]));
                const float input = to_float<T>(rows.x[r].at[v]);
                if constexpr (BACK) {
                    const float g = input + state[v];
                    state[v] = d.times_any(g);
                    const float before = r + 1 < left ? to_float<T>(rows.h[r].at[v]) : first[v];
                    g_row.at[v] = rounded<T>(g);
                    l_row.at[v] = rounded<T>(state[v] * before);
                } else {
                    state[v] = d.step_any(state[v], input);
                    g_row.at[v] = rounded<T>(state[v]);
                }
            }
            a.store(BACK ? some - 1 - r : r, at, g_row);
            if constexpr (BACK) b.store(some - 1 - r, at, l_row);
        }
    };
    for (int64_t done = 0; done < span.size; done += 2 * kWalkRows) {
        odd.load(in, span, done + kWalkRows, row_bytes, at);
        __builtin_amdgcn_sched_barrier(0);  // (sent before the rows in between are written, which they would wait for)
        work(even, done);
        if (done + kWalkRows >= span.size) break;
        even.load(in, span, done + 2 * kWalkRows, row_bytes, at);
        __builtin_amdgcn_sched_barrier(0);
        work(odd, done + kWalkRows);
    }
    if (in.last == nullptr || held < 0 || !active) return;
#pragma unroll
    for (int v = 0; v < V; ++v) in.last[held * p.channels + channel + v] = state[v];
}

// Before the chunks: no effect is there, and of the states that of each sequence's first chunk (the last one, backwards).
constexpr int kClearBlock = 256;

template <bool BACK, int WAVES>
__global__ __launch_bounds__(kClearBlock) void recurrence_clear_kernel(Inputs in, Handed h, Shape p, int first_number, int blocks) {
    const int number = first_number + static_cast<int>(blockIdx.x / blocks);
    const int channel = static_cast<int>(blockIdx.x % blocks) * kClearBlock + static_cast<int>(threadIdx.x);
    Chunk chunk;
    const bool there = chunk.find<WAVES>(in.offsets, p, number);
    if (!there || chunk.chunks <= 1 || channel >= p.channels) return;  // (a chunk alone hands nothing on)
    uint32_t state = kNotYet;
    if (chunk.index == (BACK ? chunk.chunks - 1 : 0)) {
        if constexpr (BACK) {
            state = in.dfinal != nullptr ? handed(in.dfinal[static_cast<int64_t>(chunk.sequence) * p.channels + channel]) : 0u;
        } else {
            const int64_t row = state_of(in.state_rows, chunk.sequence, p.num_states);
            state = in.initial != nullptr && row >= 0 ? handed(in.initial[row * p.channels + channel]) : 0u;
        }
    }
    h.states[number * h.stride + channel] = state;
    h.effects[number * h.stride + channel] = ~uint64_t{0};
}

template <typename T, int V, bool BACK, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, 4) void recurrence_kernel(Inputs in, Handed h, Shape p, int numbers, int first_ordinal, int blocks,
                                                                  uint32_t patience) {
    using Item = typename T::Item;
    using Vec = Items<Item, V>;
    constexpr int kChunk = WAVES * kRows, kTile = kWave * V;
    __shared__ __attribute__((aligned(16))) Effect parts[WAVES][kTile];
    __shared__ __attribute__((aligned(16))) float entering[kTile];
    // Chunks in the order that states go through them, all channels of one together.
    const int ordinal = first_ordinal + static_cast<int>(blockIdx.x / blocks), number = BACK ? numbers - 1 - ordinal : ordinal;
    Chunk chunk;
    if (!chunk.find<WAVES>(in.offsets, p, number)) return;
    const int lane = threadIdx.x % kWave, wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int own = (static_cast<int>(blockIdx.x % blocks) * kWave + lane) * V;
    const bool active = own < p.channels;
    const int64_t row0 = static_cast<int64_t>(chunk.index) * kChunk;
    const int count = chunk.size - row0 < kChunk ? static_cast<int>(chunk.size - row0) : kChunk;
    const int mine = count - wave * kRows;  // rows of this wave, if it has some
    const int64_t token = chunk.begin + row0 + wave * kRows;
    const int before = BACK ? chunk.chunks - 1 - chunk.index : chunk.index, after = chunk.chunks - 1 - before;
    const bool alone = chunk.chunks <= 1;

    WaveRows<T, V, BACK> rows;
    const int row_bytes = p.channels * static_cast<int>(sizeof(Item)), some = mine < kRows ? mine : kRows;
    const uint32_t at = active ? static_cast<uint32_t>(own) * sizeof(Item) : kNowhere;
    const auto rows_of = [&](const Steps& steps) { return Window<Vec>(steps, token, some, row_bytes); };
    rows.load(rows_of(in.first), rows_of(in.log_decay), at);
    if (!alone || WAVES > 1) {
        Effect effect[V];
        rows.effect(effect, mine);
        if (rows.any_nan([&](int v) { return effect[v].b; })) rows.effect_any(effect, some, rows_of(in.first), rows_of(in.log_decay), at);
#pragma unroll
        for (int v = 0; v < V; ++v) parts[wave][lane * V + v] = effect[v];
    }
    // Backwards: the states before each token, as they were stored.
    // (The window begins a row before the wave's, or where the sequence does: then it is read a row late.)
    Vec stored[BACK ? kRows : 1];
    const int late = BACK && token == chunk.begin;
    const Window<Vec> out(in.out, BACK ? token - 1 + late : token, some - late, row_bytes);
    if constexpr (BACK) {
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            if (r >= late) stored[r] = out.load(r - late, at);
    }
    // The states that enter the chunk, 64 channels a wave.
    const int64_t held = BACK ? chunk.sequence : state_of(in.state_rows, chunk.sequence, p.num_states);
    if constexpr (WAVES > 1) __syncthreads();
    else wave_lds_order();
    for (int group = wave; group < V; group += WAVES) {
        const int at = group * kWave + lane, target = own - lane * V + at;
        const bool there = target < p.channels;
        float state = 0.f;
        if (alone) {
            const float* from = BACK ? in.dfinal : in.initial;
            if (from != nullptr && held >= 0 && there) state = from[held * p.channels + target];
        } else {
            Effect all = {0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WAVES; ++w) all.then<true>(parts[BACK ? WAVES - 1 - w : w][at]);
            if (after > 0 && there) atomic_store_agent(h.effects + number * h.stride + target, handed(all));
            state = look_back<T, BACK, WAVES>(in, h, chunk, number, before, target, there, patience);
            if (after > 0 && there) atomic_store_agent(h.states + (BACK ? number - 1 : number + 1) * h.stride + target, handed(all.of<true>(state)));
        }
        entering[at] = there ? state : 0.f;  // (a lane without a channel may have found a word that was not there yet, a NaN)
    }
    if constexpr (WAVES > 1) __syncthreads();
    else wave_lds_order();
    float state[V];
    const auto enter = [&](auto any) {
        constexpr bool kAny = decltype(any)::value;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            state[v] = entering[lane * V + v];
            if constexpr (BACK) {
                for (int w = WAVES - 1; w > wave; --w) state[v] = parts[w][lane * V + v].template of<kAny>(state[v]);
            } else {
                for (int w = 0; w < wave; ++w) state[v] = parts[w][lane * V + v].template of<kAny>(state[v]);
            }
        }
    };
    // Row r of the wave with the state before it (backwards, after it); `h` is the stored state before a row.
    const Window<Vec> dx(in.dx, token, BACK ? some : 0, row_bytes), dlog_decay(in.dlog_decay, token, BACK ? some : 0, row_bytes);
    const auto work = [&](auto any, int r, const Vec& x, const Vec& l, const Vec& h_row) {
        constexpr bool kAny = decltype(any)::value;
        Vec row, l_row;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Decay d(to_float<T>(l.at[v]));
            if constexpr (BACK) {
                const float g = to_float<T>(x.at[v]) + state[v];
                state[v] = kAny ? d.times_any(g) : d.times(g);
                float h = to_float<T>(h_row.at[v]);
                if (r == 0 && late) h = in.initial != nullptr && active ? in.initial[static_cast<int64_t>(chunk.sequence) * p.channels + own + v] : 0.f;
                row.at[v] = rounded<T>(g);
                l_row.at[v] = rounded<T>(state[v] * h);
            } else {
                state[v] = kAny ? d.step_any(state[v], to_float<T>(x.at[v])) : d.step(state[v], to_float<T>(x.at[v]));
                row.at[v] = rounded<T>(state[v]);
            }
        }
        (BACK ? dx : out).store(r, at, row);
        if constexpr (BACK) dlog_decay.store(r, at, l_row);
    };
    enter(std::false_type{});
    rows.forget();
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = BACK ? kRows - 1 - i : i;
        __builtin_amdgcn_sched_barrier(0);
        if (r < mine) work(std::false_type{}, r, rows.x[r], rows.l[r], stored[BACK ? r : 0]);
    }
    if (rows.any_nan([&](int v) { return state[v]; })) {
        enter(std::true_type{});
        const Window<Vec> first = rows_of(in.first), log_decay = rows_of(in.log_decay);
#pragma unroll 1
        for (int i = 0; i < some; ++i) {
            const int r = BACK ? some - 1 - i : i;
            work(std::true_type{}, r, first.load(r, at), log_decay.load(r, at), BACK ? out.load(r < late ? 0 : r - late, at) : Vec{});
        }
    }
    // The last state: forwards of the wave that has the sequence's last token, backwards of the first.
    const bool ends = BACK ? chunk.index == 0 && wave == 0 : after <= 0 && (count == 0 ? wave == 0 : (count - 1) / kRows == wave);
    if (!ends || !active || in.last == nullptr) return;
    if (held < 0) return;
#pragma unroll
    for (int v = 0; v < V; ++v) in.last[held * p.channels + own + v] = state[v];
}

// ---- host side ---------------------------------------------------------------------------------------------------
// (A wave's rows lie within 2^30 bytes.)
constexpr int64_t kMostStride = int64_t{1} << 24;

constexpr uint64_t kWalkedEach = 2, kWalkedMore = 64;

// Waves of a chunk: one while sequences have no more than 64 tokens on average, else eight (64 sequences of 32 tokens of 4,096 channels:
// one 26 us, eight 34; of 100 tokens 62 and 54; 8 sequences of 1,000 tokens 94 and 52).
constexpr uint64_t kShortEach = 64;
constexpr int kLongWaves = 8;
bool short_sequences(uint64_t sequences, uint64_t tokens) { return tokens <= sequences * kShortEach; }

// Sequences of a token or two on average are walked: no chunk hands anything on, and there is one launch (4,096 channels, 256 sequences of
// one token 7 us, in chunks 17; of two 7.5 and 18).  The price is a batch of many short sequences and a long one, which a wave walks
// at 0.2 us a token: 255 of one token and one of 300 take 66 us, in chunks 37.
bool walked(uint64_t sequences, uint64_t tokens) { return tokens <= sequences * kWalkedEach + kWalkedMore; }

uint64_t numbers_of(uint64_t sequences, uint64_t tokens) {
    return tokens / (short_sequences(sequences, tokens) ? kRows : kRows * kLongWaves) + sequences;
}
// No sequence has two chunks where all tokens fit one.
bool handing(uint64_t sequences, uint64_t tokens) {
    return !walked(sequences, tokens) && tokens > static_cast<uint64_t>(short_sequences(sequences, tokens) ? kRows : kRows * kLongWaves);
}
uint64_t stride_of(uint64_t channels) { return align_up(channels, 64); }
size_t effects_bytes(uint64_t sequences, uint64_t tokens, uint64_t channels) {
    return align_up(numbers_of(sequences, tokens) * stride_of(channels) * sizeof(uint64_t), kViewAlign);
}
size_t needed_bytes(uint64_t sequences, uint64_t tokens, uint64_t channels) {
    if (sequences == 0 || !handing(sequences, tokens)) return 0;
    return effects_bytes(sequences, tokens, channels) +
           align_up(numbers_of(sequences, tokens) * stride_of(channels) * sizeof(uint32_t), kViewAlign);
}

template <typename T>
bool usable(const lcpp_hip_steps* s, uint32_t channels) {
    return s != nullptr && s->data != nullptr && reinterpret_cast<uintptr_t>(s->data) % sizeof(typename T::Item) == 0 &&
           s->token_stride >= static_cast<int64_t>(channels) && s->token_stride < kMostStride;
}
template <typename T>
Steps steps_of(const lcpp_hip_steps* s) {
    return {static_cast<char*>(s->data), s->token_stride * static_cast<int64_t>(sizeof(typename T::Item))};
}
int unusable(const char* what) {
    return set_error(kInvalidArgument, "%s: rows must be there and aligned to their items, at least their channels apart and less than 2^24 items", what);
}

int check_sizes(const char* what, uint32_t sequences, uint64_t tokens, uint32_t channels) {
    if (channels == 0 || channels >= kMostStride) return set_error(kInvalidArgument, "%s: no channels, or too many", what);
    if (tokens > 0x7FFFFFFFull) return set_error(kInvalidArgument, "%s: too many tokens", what);
    if (sequences > 0x7FFFFFFu) return set_error(kInvalidArgument, "%s: too many sequences", what);
    return kOk;
}

// Channels a lane: the most, up to 8 bytes of them, that divide the channels and that all rows are aligned to.
template <typename T>
int width_of(uint32_t channels, std::initializer_list<const lcpp_hip_steps*> rows) {
    uint64_t bits = channels;
    for (const lcpp_hip_steps* r : rows)
        bits |= static_cast<uint64_t>(r->token_stride) | reinterpret_cast<uintptr_t>(r->data) / sizeof(typename T::Item);
    constexpr int kMost = 8 / static_cast<int>(sizeof(typename T::Item));
    return bits % kMost == 0 ? kMost : bits % 2 == 0 ? 2 : 1;
}

// Whether rows of two arrays share an item, of arrays whose rows are equally far apart (others: whether their first rows do).
bool share(const Steps& a, const Steps& b, int64_t tokens, int64_t row_bytes) {
    const int64_t ahead = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.data) - reinterpret_cast<uintptr_t>(a.data));
    const int64_t stride = a.token_bytes;
    if (tokens == 1 || b.token_bytes != stride) return ahead < row_bytes && -ahead < row_bytes;
    int64_t rows = ahead / stride, past = ahead % stride;  // b's first row begins `past` bytes after a's row `rows`
    if (past < 0) {
        --rows;
        past += stride;
    }
    return (past < row_bytes && rows < tokens && -rows < tokens) || (stride - past < row_bytes && rows + 1 < tokens && -rows - 1 < tokens);
}

// A chunk's rows may be read again by the workgroups of later chunks: nothing is written where something is read.
template <bool BACK>
bool apart(const Inputs& in, const Shape& p, int64_t row_bytes) {
    if (p.tokens == 0) return true;
    for (const Steps& to : BACK ? std::initializer_list<Steps>{in.dx, in.dlog_decay} : std::initializer_list<Steps>{in.out}) {
        if (share(to, in.first, p.tokens, row_bytes) || share(to, in.log_decay, p.tokens, row_bytes)) return false;
        if (BACK && share(to, in.out, p.tokens, row_bytes)) return false;
    }
    return !BACK || !share(in.dx, in.dlog_decay, p.tokens, row_bytes);
}

// A launch holds fewer than 2^31 threads: units of `blocks` workgroups in as many launches as that takes, in their order (what a chunk
// waits for is in its own launch or an earlier one).
template <typename F>
void in_launches(uint64_t units, uint64_t blocks, uint64_t threads, F launch) {
    const uint64_t most = 0x7FFFFFFFull / (blocks * threads);
    for (uint64_t first = 0; first < units; first += most) {
        const uint64_t count = units - first < most ? units - first : most;
        launch(static_cast<int>(first), static_cast<unsigned>(count * blocks));
    }
}

template <typename T, int V, bool BACK, int WAVES>
int run(const char* what, const Inputs& in, const Handed& h, const Shape& p, bool hands, hipStream_t stream) {
    const int numbers = static_cast<int>(numbers_of(p.sequences, p.tokens));
    const int blocks = static_cast<int>(ceil_div(p.channels, kWave * V));
    if (walked(p.sequences, p.tokens)) {
        LaunchScope scope(what, stream);
        in_launches(p.sequences, blocks, kWave, [&](int first, unsigned grid) {
            recurrence_walk_kernel<T, V, BACK><<<grid, kWave, 0, stream>>>(in, p, first, blocks);
        });
        return check_hip(hipGetLastError(), what);
    }
    if (hands) {
        LaunchScope scope(BACK ? "recurrence_backward_clear" : "recurrence_clear", stream);
        const int parts = static_cast<int>(ceil_div(p.channels, kClearBlock));
        in_launches(numbers, parts, kClearBlock, [&](int first, unsigned grid) {
            recurrence_clear_kernel<BACK, WAVES><<<grid, kClearBlock, 0, stream>>>(in, h, p, first, parts);
        });
        if (int st = check_hip(hipGetLastError(), what); st != kOk) return st;
    }
    LaunchScope scope(what, stream);
    in_launches(numbers, blocks, WAVES * kWave, [&](int first, unsigned grid) {
        recurrence_kernel<T, V, BACK, WAVES><<<grid, WAVES * kWave, 0, stream>>>(in, h, p, numbers, first, blocks, lookback_spin_limit());
    });
    return check_hip(hipGetLastError(), what);
}

template <typename T, bool BACK>
int launch(const char* what, void* temp, size_t temp_bytes, const Inputs& in, const Shape& p, int width, hipStream_t stream) {
    const size_t needed = needed_bytes(p.sequences, p.tokens, p.channels);
    if (temp_bytes < needed || (needed && !temp)) return set_error(kTempTooSmall, "%s: temp storage too small", what);
    if (needed && reinterpret_cast<uintptr_t>(temp) % sizeof(uint64_t) != 0)
        return set_error(kInvalidArgument, "%s: temp storage must be 8-byte aligned", what);
    if (!apart<BACK>(in, p, static_cast<int64_t>(p.channels) * static_cast<int64_t>(sizeof(typename T::Item))))
        return set_error(kInvalidArgument, "%s: rows that are written share no memory with others", what);
    Handed h{static_cast<uint64_t*>(temp), nullptr, static_cast<int64_t>(stride_of(p.channels))};
    if (needed) h.states = reinterpret_cast<uint32_t*>(static_cast<char*>(temp) + effects_bytes(p.sequences, p.tokens, p.channels));
    const bool few = short_sequences(p.sequences, p.tokens);
    const auto choose = [&](auto v) {
        constexpr int kWide = decltype(v)::value;
        return few ? run<T, kWide, BACK, 1>(what, in, h, p, needed != 0, stream)
                   : run<T, kWide, BACK, kLongWaves>(what, in, h, p, needed != 0, stream);
    };
    if constexpr (sizeof(typename T::Item) == 2)
        if (width == 4) return choose(std::integral_constant<int, 4>{});
    return width == 2 ? choose(std::integral_constant<int, 2>{}) : choose(std::integral_constant<int, 1>{});
}

template <typename T>
int forward(void* temp, size_t temp_bytes, const lcpp_hip_steps* x, const lcpp_hip_steps* log_decay, const int32_t* offsets,
            const float* initial, const int32_t* state_rows, uint32_t num_states, const lcpp_hip_steps* out, float* final_states,
            uint32_t sequences, uint64_t tokens, uint32_t channels, void* stream_ptr) {
    const char* what = "recurrence";
    if (int st = check_sizes(what, sequences, tokens, channels); st != kOk) return st;
    if (num_states > 0x7FFFFFFFu) return set_error(kInvalidArgument, "%s: too many states", what);
    if (sequences == 0) return kOk;
    if (!offsets) return set_error(kInvalidArgument, "%s: null offsets", what);
    if (tokens && (!usable<T>(x, channels) || !usable<T>(log_decay, channels) || !usable<T>(out, channels))) return unusable(what);
    const Shape p{static_cast<int>(sequences), static_cast<int64_t>(tokens), static_cast<int>(channels), static_cast<int>(num_states)};
    Inputs in{};
    if (tokens) in = {steps_of<T>(x), steps_of<T>(log_decay), steps_of<T>(out)};
    in.offsets = offsets;
    in.initial = initial;
    in.state_rows = state_rows;
    in.last = final_states;
    const int width = tokens ? width_of<T>(channels, {x, log_decay, out}) : 1;
    return launch<T, false>(what, temp, temp_bytes, in, p, width, static_cast<hipStream_t>(stream_ptr));
}

template <typename T>
int backward(void* temp, size_t temp_bytes, const lcpp_hip_steps* log_decay, const lcpp_hip_steps* out, const lcpp_hip_steps* dout,
             const int32_t* offsets, const float* initial, const float* dfinal, const lcpp_hip_steps* dx,
             const lcpp_hip_steps* dlog_decay, float* dinitial, uint32_t sequences, uint64_t tokens, uint32_t channels, void* stream_ptr) {
    const char* what = "recurrence_backward";
    if (int st = check_sizes(what, sequences, tokens, channels); st != kOk) return st;
    if (sequences == 0) return kOk;
    if (!offsets) return set_error(kInvalidArgument, "%s: null offsets", what);
    if (tokens && (!usable<T>(log_decay, channels) || !usable<T>(out, channels) || !usable<T>(dout, channels) ||
                   !usable<T>(dx, channels) || !usable<T>(dlog_decay, channels)))
        return unusable(what);
    const Shape p{static_cast<int>(sequences), static_cast<int64_t>(tokens), static_cast<int>(channels), static_cast<int>(sequences)};
    Inputs in{};
    if (tokens) in = {steps_of<T>(dout), steps_of<T>(log_decay), steps_of<T>(out), steps_of<T>(dx), steps_of<T>(dlog_decay)};
    in.offsets = offsets;
    in.initial = initial;
    in.dfinal = dfinal;
    in.last = dinitial;
    const int width = tokens ? width_of<T>(channels, {log_decay, out, dout, dx, dlog_decay}) : 1;
    return launch<T, true>(what, temp, temp_bytes, in, p, width, static_cast<hipStream_t>(stream_ptr));
}

}  // namespace
}  // namespace recurrence
}  // namespace lcpp_hip

using namespace lcpp_hip;

extern "C" {

size_t lcpp_hip_recurrence_temp_bytes(uint32_t sequences, uint64_t tokens, uint32_t channels) {
    return recurrence::needed_bytes(sequences, tokens, channels);
}

#define LCPP_HIP_DEFINE_RECURRENCE(S, T)                                                                                      \
    int lcpp_hip_recurrence_##S(void* temp, size_t temp_bytes, const lcpp_hip_steps* x, const lcpp_hip_steps* log_decay,      \
                                const int32_t* offsets, const float* initial, const int32_t* state_rows, uint32_t num_states, \
                                const lcpp_hip_steps* out, float* final_states, uint32_t sequences, uint64_t tokens,          \
                                uint32_t channels, void* stream) {                                                            \
        return recurrence::forward<recurrence::T>(temp, temp_bytes, x, log_decay, offsets, initial, state_rows, num_states,   \
                                                  out, final_states, sequences, tokens, channels, stream);                    \
    }                                                                                                                         \
    int lcpp_hip_recurrence_backward_##S(                                                                                     \
        void* temp, size_t temp_bytes, const lcpp_hip_steps* log_decay, const lcpp_hip_steps* out, const lcpp_hip_steps* dout, \
        const int32_t* offsets, const float* initial, const float* dfinal, const lcpp_hip_steps* dx,                          \
        const lcpp_hip_steps* dlog_decay, float* dinitial, uint32_t sequences, uint64_t tokens, uint32_t channels,            \
        void* stream) {                                                                                                       \
        return recurrence::backward<recurrence::T>(temp, temp_bytes, log_decay, out, dout, offsets, initial, dfinal, dx,      \
                                                   dlog_decay, dinitial, sequences, tokens, channels, stream);                \
    }
LCPP_HIP_DEFINE_RECURRENCE(bf16, Bf16)
LCPP_HIP_DEFINE_RECURRENCE(f16, F16)
LCPP_HIP_DEFINE_RECURRENCE(f32, F32)
#undef LCPP_HIP_DEFINE_RECURRENCE

}  // extern "C"
