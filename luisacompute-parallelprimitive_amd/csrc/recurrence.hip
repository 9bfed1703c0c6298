// A gated linear recurrence over the sequences of a ragged batch, channel by channel, and its gradients:
//
//   h_t = exp(l_t) h_{t-1} + x_t,   h_0 an initial state or 0;
//   g_t = dh_t + c_{t+1},  c_t = exp(l_t) g_t,   dx_t = g_t,  dl_t = c_t h_{t-1},  dh_0 = c_1.
//
// States are f32; outputs are rounded once.  A state that remembers thousands of tokens adds up as many errors of exp(l): for
// small l the step is h + (exp(l) - 1) h + x with exp(l) - 1 from its series, whose error is relative to l.
#include "common.hpp"
#include "../../include/lcpp_hip.h"
#include "attention.hpp"

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

constexpr float kSmall = 0.0625f;

// y -> exp(l) y + x, with what depends on l alone.
struct Decay {
    float factor;  // exp(l), or exp(l) - 1 where l is small
    bool small;
    __device__ __forceinline__ explicit Decay(float l) {
        // (The first term left out is l^5 / 120, 1.3e-7 of l.)
        const float series = l * __builtin_fmaf(l, __builtin_fmaf(l, __builtin_fmaf(l, 1.f / 24.f, 1.f / 6.f), 0.5f), 1.f);
        small = __builtin_fabsf(l) < kSmall;
        factor = small ? series : attention::exp2_fast(l * attention::kLog2e);
    }
    __device__ __forceinline__ float step(float y, float x) const { return __builtin_fmaf(factor, y, small ? y + x : x); }
    __device__ __forceinline__ float times(float y) const { return __builtin_fmaf(factor, y, small ? y : 0.f); }
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

constexpr int kWalkBlock = 256;

// A thread walks a channel of a sequence.
template <typename T>
__global__ __launch_bounds__(kWalkBlock) void recurrence_walk_kernel(Steps x, Steps log_decay, const int32_t* __restrict__ offsets,
                                                                     const float* initial, const int32_t* __restrict__ rows, Steps out,
                                                                     float* final, Shape p) {
    using Item = typename T::Item;
    const int blocks = (p.channels + kWalkBlock - 1) / kWalkBlock, sequence = static_cast<int>(blockIdx.x / blocks);
    const int channel = static_cast<int>(blockIdx.x % blocks) * kWalkBlock + static_cast<int>(threadIdx.x);
    if (channel >= p.channels) return;
    const Span span = span_of(offsets, sequence, p.tokens);
    const int64_t row = state_of(rows, sequence, p.num_states);
    float h = initial != nullptr && row >= 0 ? initial[row * p.channels + channel] : 0.f;
    for (int64_t t = span.begin; t < span.begin + span.size; ++t) {
        h = Decay(to_float<T>(log_decay.at<Item>(t)[channel])).step(h, to_float<T>(x.at<Item>(t)[channel]));
        out.at<Item>(t)[channel] = static_cast<Item>(h);
    }
    if (final != nullptr && row >= 0) final[row * p.channels + channel] = h;
}

template <typename T>
__global__ __launch_bounds__(kWalkBlock) void recurrence_walk_back_kernel(Steps log_decay, Steps out, Steps dout,
                                                                          const int32_t* __restrict__ offsets,
                                                                          const float* __restrict__ initial,
                                                                          const float* __restrict__ dfinal, Steps dx, Steps dlog_decay,
                                                                          float* __restrict__ dinitial, Shape p) {
    using Item = typename T::Item;
    const int blocks = (p.channels + kWalkBlock - 1) / kWalkBlock, sequence = static_cast<int>(blockIdx.x / blocks);
    const int channel = static_cast<int>(blockIdx.x % blocks) * kWalkBlock + static_cast<int>(threadIdx.x);
    if (channel >= p.channels) return;
    const Span span = span_of(offsets, sequence, p.tokens);
    const int64_t state = static_cast<int64_t>(sequence) * p.channels + channel;
    float c = dfinal != nullptr ? dfinal[state] : 0.f;
    for (int64_t t = span.begin + span.size - 1; t >= span.begin; --t) {
        const float g = to_float<T>(dout.at<Item>(t)[channel]) + c;
        c = Decay(to_float<T>(log_decay.at<Item>(t)[channel])).times(g);
        const float before = t > span.begin ? to_float<T>(out.at<Item>(t - 1)[channel]) : initial != nullptr ? initial[state] : 0.f;
        dx.at<Item>(t)[channel] = static_cast<Item>(g);
        dlog_decay.at<Item>(t)[channel] = static_cast<Item>(c * before);
    }
    if (dinitial != nullptr) dinitial[state] = c;
}

// ---- host side ---------------------------------------------------------------------------------------------------
template <typename T>
bool usable(const lcpp_hip_steps* s, uint32_t channels) {
    return s != nullptr && s->data != nullptr && reinterpret_cast<uintptr_t>(s->data) % sizeof(typename T::Item) == 0 &&
           s->token_stride >= static_cast<int64_t>(channels) && s->token_stride <= (int64_t{1} << 40);
}
template <typename T>
Steps steps_of(const lcpp_hip_steps* s) {
    return {static_cast<char*>(s->data), s->token_stride * static_cast<int64_t>(sizeof(typename T::Item))};
}
int unusable(const char* what) {
    return set_error(kInvalidArgument, "%s: rows must be there and aligned to their items, at least their channels apart", what);
}

int check_sizes(const char* what, uint32_t sequences, uint64_t tokens, uint32_t channels) {
    if (channels == 0 || channels > 0x7FFFFFFu) return set_error(kInvalidArgument, "%s: no channels, or too many", what);
    if (ceil_div(channels, kWalkBlock) * sequences > 0x7FFFFFFFull / kWalkBlock)
        return set_error(kInvalidArgument, "%s: too many sequences of so many channels", what);
    if (tokens > 0x7FFFFFFFull) return set_error(kInvalidArgument, "%s: too many tokens", what);
    return kOk;
}

template <typename T>
int forward(void* temp, size_t temp_bytes, const lcpp_hip_steps* x, const lcpp_hip_steps* log_decay, const int32_t* offsets,
            const float* initial, const int32_t* state_rows, uint32_t num_states, const lcpp_hip_steps* out, float* final_states,
            uint32_t sequences, uint64_t tokens, uint32_t channels, void* stream_ptr) {
    const char* what = "recurrence";
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (int st = check_sizes(what, sequences, tokens, channels); st != kOk) return st;
    if (num_states > 0x7FFFFFFFu) return set_error(kInvalidArgument, "%s: too many states", what);
    if (sequences == 0) return kOk;
    if (!offsets) return set_error(kInvalidArgument, "%s: null offsets", what);
    if (tokens && (!usable<T>(x, channels) || !usable<T>(log_decay, channels) || !usable<T>(out, channels))) return unusable(what);
    const size_t needed = lcpp_hip_recurrence_temp_bytes(sequences, tokens, channels);
    if (temp_bytes < needed || (needed && !temp)) return set_error(kTempTooSmall, "%s: temp storage too small", what);
    const Shape p{static_cast<int>(sequences), static_cast<int64_t>(tokens), static_cast<int>(channels), static_cast<int>(num_states)};
    LaunchScope scope(what, stream);
    recurrence_walk_kernel<T><<<static_cast<unsigned>(ceil_div(channels, kWalkBlock) * sequences), kWalkBlock, 0, stream>>>(
        steps_of<T>(x), steps_of<T>(log_decay), offsets, initial, state_rows, steps_of<T>(out), final_states, p);
    return check_hip(hipGetLastError(), "recurrence launch");
}

template <typename T>
int backward(void* temp, size_t temp_bytes, const lcpp_hip_steps* log_decay, const lcpp_hip_steps* out, const lcpp_hip_steps* dout,
             const int32_t* offsets, const float* initial, const float* dfinal, const lcpp_hip_steps* dx,
             const lcpp_hip_steps* dlog_decay, float* dinitial, uint32_t sequences, uint64_t tokens, uint32_t channels, void* stream_ptr) {
    const char* what = "recurrence_backward";
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (int st = check_sizes(what, sequences, tokens, channels); st != kOk) return st;
    if (sequences == 0) return kOk;
    if (!offsets) return set_error(kInvalidArgument, "%s: null offsets", what);
    if (tokens && (!usable<T>(log_decay, channels) || !usable<T>(out, channels) || !usable<T>(dout, channels) ||
                   !usable<T>(dx, channels) || !usable<T>(dlog_decay, channels)))
        return unusable(what);
    const size_t needed = lcpp_hip_recurrence_temp_bytes(sequences, tokens, channels);
    if (temp_bytes < needed || (needed && !temp)) return set_error(kTempTooSmall, "%s: temp storage too small", what);
    const Shape p{static_cast<int>(sequences), static_cast<int64_t>(tokens), static_cast<int>(channels), static_cast<int>(sequences)};
    LaunchScope scope(what, stream);
    recurrence_walk_back_kernel<T><<<static_cast<unsigned>(ceil_div(channels, kWalkBlock) * sequences), kWalkBlock, 0, stream>>>(
        steps_of<T>(log_decay), steps_of<T>(out), steps_of<T>(dout), offsets, initial, dfinal, steps_of<T>(dx), steps_of<T>(dlog_decay),
        dinitial, p);
    return check_hip(hipGetLastError(), "recurrence_backward launch");
}

}  // namespace
}  // namespace recurrence
}  // namespace lcpp_hip

using namespace lcpp_hip;

extern "C" {

size_t lcpp_hip_recurrence_temp_bytes(uint32_t, uint64_t, uint32_t) { return 0; }

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
