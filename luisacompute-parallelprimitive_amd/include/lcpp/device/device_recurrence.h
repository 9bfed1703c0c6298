// DeviceRecurrence: a gated linear recurrence over the sequences of a ragged batch and its gradients (lcpp_hip_recurrence_*,
// lcpp_hip_recurrence_backward_*), in the shape of the other modules: create, a temp-storage query, and calls that check their
// views and record into a CommandList.  There is no reference counterpart; what the calls compute is documented in lcpp_hip.h.
#pragma once

#include <limits>
#include <type_traits>

#include "lcpp/device/device_attention.h"
#include "lcpp/runtime/core.h"

namespace luisa::parallel_primitive {

template <typename T>
concept RecurrenceItemT = AttentionItemT<T> || std::is_same_v<T, float>;

// [tokens][channels]; tokens `stride` items apart (0: packed).
template <RecurrenceItemT T>
struct RecurrenceRows {
    BufferView<T> view;
    size_t stride = 0;
    RecurrenceRows() = default;
    RecurrenceRows(BufferView<T> items, size_t token = 0) : view(items), stride(token) {}
};

class DeviceRecurrence : public LuisaModule {
  public:
    void create(Device& device) { create_module(device); }

    // Of both directions.
    [[nodiscard]] static size_t GetTempStorageBytes(uint sequences, size_t tokens, uint channels) {
        return lcpp_hip_recurrence_temp_bytes(sequences, tokens, channels);
    }

    // out[t] = exp(log_decay[t]) out[t - 1] + x[t] along each sequence, from the rows of `initial` [states][channels] to those of
    // `final`; either may be empty, and both may be the same view.  Sequence b's row is state_rows[b], or b where that is empty.
    // `out` shares no memory with x or log_decay (the command throws).
    template <RecurrenceItemT T>
    void Scan(CommandList& cmdlist, BufferView<uint> temp_storage, RecurrenceRows<T> x, RecurrenceRows<T> log_decay,
              BufferView<int32_t> offsets, RecurrenceRows<T> out, BufferView<float> initial, BufferView<float> final,
              BufferView<int32_t> state_rows, size_t tokens, uint channels) {
        const uint sequences = sequences_of(offsets, channels);
        auto xs = rows(x, tokens, channels), ls = rows(log_decay, tokens, channels), outs = rows(out, tokens, channels);
        const size_t states = (initial.size() ? initial.size() : final.size()) / channels;
        LCPP_ASSERT(initial.size() == 0 || final.size() == 0 || initial.size() == final.size(),
                    "DeviceRecurrence initial and final states differ in number.");
        LCPP_ASSERT(states <= static_cast<size_t>(std::numeric_limits<int32_t>::max()), "Too many states for DeviceRecurrence.");
        LCPP_ASSERT(state_rows.size() ? state_rows.size() >= sequences : states == 0 || states >= sequences,
                    "A DeviceRecurrence state view is too small.");
        check_temp(temp_storage, sequences, tokens, channels);
        cmdlist << [=](hipStream_t s) {
            auto* run = choose<T>(lcpp_hip_recurrence_bf16, lcpp_hip_recurrence_f16, lcpp_hip_recurrence_f32);
            luisa::detail::abi_check(run(temp_storage.data(), temp_storage.size_bytes(), &xs, &ls, offsets.data(), initial.data(),
                                         state_rows.data(), static_cast<uint>(states), &outs, final.data(), sequences, tokens, channels,
                                         detail::stream_ptr(s)),
                                     "DeviceRecurrence::Scan");
        };
    }

    // Gradients of Scan, from the out that it gave; states [sequences][channels], each view of them may be empty.
    // dx and dlog_decay share no memory with each other or with what is read (the command throws).
    template <RecurrenceItemT T>
    void ScanBackward(CommandList& cmdlist, BufferView<uint> temp_storage, RecurrenceRows<T> log_decay, RecurrenceRows<T> out,
                      RecurrenceRows<T> dout, BufferView<int32_t> offsets, BufferView<float> initial, BufferView<float> dfinal,
                      RecurrenceRows<T> dx, RecurrenceRows<T> dlog_decay, BufferView<float> dinitial, size_t tokens, uint channels) {
        const uint sequences = sequences_of(offsets, channels);
        auto ls = rows(log_decay, tokens, channels), outs = rows(out, tokens, channels), douts = rows(dout, tokens, channels);
        auto dxs = rows(dx, tokens, channels), dls = rows(dlog_decay, tokens, channels);
        for (const auto& states : {initial, dfinal, dinitial})
            LCPP_ASSERT(states.size() == 0 || states.size() >= static_cast<size_t>(sequences) * channels,
                        "A DeviceRecurrence state view is too small.");
        check_temp(temp_storage, sequences, tokens, channels);
        cmdlist << [=](hipStream_t s) {
            auto* run = choose<T>(lcpp_hip_recurrence_backward_bf16, lcpp_hip_recurrence_backward_f16, lcpp_hip_recurrence_backward_f32);
            luisa::detail::abi_check(run(temp_storage.data(), temp_storage.size_bytes(), &ls, &outs, &douts, offsets.data(), initial.data(),
                                         dfinal.data(), &dxs, &dls, dinitial.data(), sequences, tokens, channels, detail::stream_ptr(s)),
                                     "DeviceRecurrence::ScanBackward");
        };
    }

  private:
    template <typename T, typename F>
    static F* choose(F* bf16, F* f16, F* f32) {
        return std::is_same_v<T, bfloat16> ? bf16 : std::is_same_v<T, float16> ? f16 : f32;
    }
    [[nodiscard]] uint sequences_of(const BufferView<int32_t>& offsets, uint channels) const {
        LCPP_ASSERT(m_created, "DeviceRecurrence::create must be called before dispatch.");
        LCPP_ASSERT(offsets.size() > 0 && offsets.size() <= static_cast<size_t>(std::numeric_limits<int32_t>::max()),
                    "DeviceRecurrence offsets are empty, or too many.");
        LCPP_ASSERT(channels > 0, "DeviceRecurrence rows have no channels.");
        return static_cast<uint>(offsets.size() - 1);
    }
    static void check_temp(const BufferView<uint>& temp, uint sequences, size_t tokens, uint channels) {
        LCPP_ASSERT(temp.size_bytes() >= GetTempStorageBytes(sequences, tokens, channels),
                    "DeviceRecurrence temporary-storage view is too small.");
    }
    template <typename T>
    [[nodiscard]] static lcpp_hip_steps rows(const RecurrenceRows<T>& r, size_t tokens, uint channels) {
        const size_t stride = r.stride ? r.stride : channels;
        LCPP_ASSERT(stride >= channels && (tokens == 0 || r.view.size() >= (tokens - 1) * stride + channels),
                    "A DeviceRecurrence row view is too small.");
        return {r.view.data(), static_cast<int64_t>(stride)};
    }
};

}  // namespace luisa::parallel_primitive
