// The calls that keep a long request's memory bounded, as a C++ program would make them: rows turned and written into pages, their
// weights summed, a request cut and its rows moved, and a recurrence with its gradients.  Host checks against plain loops in double.
//
// Usage: long_request_test [--list] [case-substring]
#include <lcpp/parallel_primitive.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <numeric>
#include <string>
#include <vector>

using namespace luisa;
using namespace luisa::compute;
using namespace luisa::parallel_primitive;

namespace {

int g_failures = 0;
std::string g_current;

#define EXPECT(cond)                                                                               \
    do {                                                                                           \
        if (!(cond)) {                                                                             \
            ++g_failures;                                                                          \
            std::printf("  FAILED %s:%d in %s: %s\n", __FILE__, __LINE__, g_current.c_str(), #cond); \
        }                                                                                          \
    } while (0)

struct Env {
    Context context;
    Device device;
    Stream stream;
    DeviceAttention attention;
    DeviceRecurrence recurrence;
    Env() : device(context.create_device("hip")), stream(device.create_stream()) {
        attention.create(device);
        recurrence.create(device);
    }
    template <typename T>
    Buffer<T> upload(const std::vector<T>& host) {
        Buffer<T> b = device.create_buffer<T>(host.size());
        stream << b.copy_from(std::span<const T>(host)) << synchronize();
        return b;
    }
    template <typename T>
    std::vector<T> download(const Buffer<T>& b) {
        std::vector<T> host(b.size());
        stream << b.copy_to(std::span<T>(host)) << synchronize();
        return host;
    }
    void run(CommandList& c) { stream << c.commit() << synchronize(); }
};
Env* g_env = nullptr;

double value_of(bfloat16 x) {
    const uint32_t w = static_cast<uint32_t>(x.bits) << 16;
    float f;
    std::memcpy(&f, &w, 4);
    return f;
}

// Multiples of 1/64 in [-1, 1): exact in 16 bits.
double number(uint64_t seed, size_t i) {
    uint64_t z = (seed << 32) + (i + 1) * 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    return (static_cast<int>((z >> 33) % 128) - 64) / 64.0;
}
std::vector<bfloat16> items(size_t n, uint64_t seed) {
    std::vector<bfloat16> out(n);
    for (size_t i = 0; i < n; ++i) {
        const float f = static_cast<float>(number(seed, i));
        uint32_t w;
        std::memcpy(&w, &f, 4);
        out[i].bits = static_cast<uint16_t>(w >> 16);
    }
    return out;
}

constexpr uint kHeads = 4, kKvHeads = 2, kDim = 64, kPage = 8, kPages = 8;
constexpr size_t kTokens = 40;
const AttentionShape kShape{kHeads, kKvHeads, kDim, 0.f};
const PageShape kPageShape{kPage, kPages};

// One request of 40 tokens through its whole life: turned and written, weighed, cut to 20 keys, moved.
void case_request() {
    Env& e = *g_env;
    const auto q = items(kTokens * kHeads * kDim, 1), k = items(kTokens * kKvHeads * kDim, 2), v = items(kTokens * kKvHeads * kDim, 3);
    const std::vector<int32_t> pages{5, 0, 7, 2, 4};
    std::vector<int32_t> positions(kTokens), requests(kTokens, 0);
    std::vector<int64_t> slots(kTokens);
    for (size_t t = 0; t < kTokens; ++t) positions[t] = static_cast<int32_t>(t), slots[t] = pages[t / kPage] * kPage + t % kPage;
    const auto frequencies = DeviceAttention::RotaryFrequencies(kDim);
    auto dq = e.upload(q), dk = e.upload(k), dv = e.upload(v);
    auto keys = e.upload(items(size_t{kPages} * kPage * kKvHeads * kDim, 4)), values = e.upload(items(size_t{kPages} * kPage * kKvHeads * kDim, 5));
    auto q_out = e.upload(q), out = e.upload(q);
    auto dpositions = e.upload(positions), drequests = e.upload(requests), shifts = e.upload(std::vector<int32_t>{100});
    auto dslots = e.upload(slots);
    auto df = e.upload(frequencies);
    auto slot_positions = e.upload(std::vector<int32_t>(kPages * kPage, -1));
    auto table = e.upload(pages), offsets = e.upload(std::vector<int32_t>{0, kTokens}), lengths = e.upload(std::vector<int32_t>{kTokens});
    auto lse = e.upload(std::vector<float>(kHeads * kTokens)), sums = e.upload(std::vector<float>(kPages * kPage, -1.f));
    const size_t bytes = std::max(DeviceAttention::GetPagedTempStorageBytes(1, kTokens, kTokens, kShape),
                                  DeviceAttention::GetPagedWeightsTempStorageBytes(1, kTokens, kTokens, kShape));
    auto temp = e.device.create_buffer<uint>(std::max(bytes, DeviceAttention::GetEvictPlanTempStorageBytes(1, kTokens)) / 4 + 4);
    auto keep = e.upload(std::vector<int32_t>{20}), kept = e.upload(std::vector<int32_t>{-1}), ahead = e.upload(std::vector<int32_t>{-1});
    auto released = e.upload(std::vector<int32_t>(8, -1)), counts = e.upload(std::vector<int32_t>{-1, -1});
    auto from = e.upload(std::vector<int64_t>(20, -7)), to = e.upload(std::vector<int64_t>(20, -7));
    const BlockTable bt{table, 0, 0};

    CommandList c;
    e.attention.PagedWriteRotary<bfloat16>(c, dq.view(), dk.view(), dv.view(), {dpositions, drequests, shifts}, {df}, dslots, q_out.view(),
                                           keys.view(), values.view(), slot_positions, kShape, kPageShape);
    e.attention.Paged<bfloat16>(c, temp, q_out.view(), keys.view(), values.view(), bt, offsets, lengths, {}, out.view(), lse, kTokens,
                                kTokens, kShape, kPageShape);
    e.attention.PagedWeights<bfloat16>(c, temp, q_out.view(), keys.view(), bt, offsets, lengths, {}, {}, lse, {}, sums, kTokens, kTokens,
                                       kShape, kPageShape);
    e.run(c);
    const auto turned_q = e.download(q_out), turned_k = e.download(keys), stored_v = e.download(values);
    const auto at = e.download(slot_positions);
    // A turn rounds once: half a step of bf16, 2^-8, of at most the square root of two, and 2^-19 before.
    constexpr double kOff = 0.0056;
    double worst = 0;
    const auto turn = [&](const std::vector<bfloat16>& x, size_t row, size_t t, uint d) {
        const uint pair = d % (kDim / 2);
        const double angle = (t + 100.0) * frequencies[pair];
        const double a = value_of(x[row * kDim + pair]), b = value_of(x[row * kDim + pair + kDim / 2]);
        return d < kDim / 2 ? a * std::cos(angle) - b * std::sin(angle) : a * std::sin(angle) + b * std::cos(angle);
    };
    bool same = true;
    for (size_t t = 0; t < kTokens; ++t) {
        EXPECT(at[slots[t]] == static_cast<int32_t>(t) + 100);
        for (uint h = 0; h < kHeads; ++h)
            for (uint d = 0; d < kDim; ++d)
                worst = std::max(worst, std::abs(value_of(turned_q[(t * kHeads + h) * kDim + d]) - turn(q, t * kHeads + h, t, d)));
        for (uint h = 0; h < kKvHeads; ++h)
            for (uint d = 0; d < kDim; ++d) {
                const size_t stored = (slots[t] * kKvHeads + h) * kDim + d;
                worst = std::max(worst, std::abs(value_of(turned_k[stored]) - turn(k, t * kKvHeads + h, t, d)));
                same &= stored_v[stored].bits == v[(t * kKvHeads + h) * kDim + d].bits;
            }
    }
    EXPECT(worst <= kOff);
    EXPECT(same);
    EXPECT(std::count(at.begin(), at.end(), -1) == kPages * kPage - kTokens);

    // Weights from the turned rows as they are stored.
    std::vector<double> want(kTokens, 0.0);
    for (size_t i = 0; i < kTokens; ++i)
        for (uint h = 0; h < kHeads; ++h) {
            std::vector<double> s(i + 1);
            double total = 0;
            for (size_t j = 0; j <= i; ++j) {
                for (uint d = 0; d < kDim; ++d)
                    s[j] += value_of(turned_q[(i * kHeads + h) * kDim + d]) * value_of(turned_k[(slots[j] * kKvHeads + h / 2) * kDim + d]);
                total += std::exp(s[j] /= 8.0);
            }
            for (size_t j = 0; j <= i; ++j) want[j] += std::exp(s[j]) / total;
        }
    const auto weight = e.download(sums);
    worst = 0;
    for (size_t j = 0; j < kTokens; ++j) worst = std::max(worst, std::abs(weight[slots[j]] - want[j]) / want[j]);
    EXPECT(worst <= 1e-4);  // (scores and log-sums of at most 16 to 2^-18, and as much for the exponentials)

    CommandList d;
    e.attention.PageRelease(d, lengths, keep, kPage, bt, shifts, kept, ahead, released, counts);
    e.attention.EvictPlan(d, temp, sums, slot_positions, bt, lengths, kept, shifts, from, to, kTokens, kPageShape, ProtectedKeys{0, 4});
    e.attention.PagedMove<bfloat16>(d, from, to, keys.view(), values.view(), sums, slot_positions, kShape, kPageShape);
    e.run(d);
    EXPECT(e.download(kept)[0] == 20 && e.download(ahead)[0] == 120);
    const auto free_pages = e.download(released), number_of = e.download(counts);
    EXPECT(number_of[0] == 2 && number_of[1] == 20 && free_pages[0] == pages[3] && free_pages[1] == pages[4]);
    std::vector<size_t> order(kTokens);
    std::iota(order.begin(), order.end(), size_t{0});
    std::stable_sort(order.begin(), order.end(), [&](size_t a, size_t b) {
        const bool late_a = a >= kTokens - 4, late_b = b >= kTokens - 4;
        return late_a != late_b ? late_a : !late_a && weight[slots[a]] > weight[slots[b]];
    });
    std::vector<bool> stays(kTokens, false);
    for (size_t i = 0; i < 20; ++i) stays[order[i]] = true;
    std::vector<int64_t> sources, targets;
    for (size_t j = 0; j < kTokens; ++j)
        if (stays[j] != (j < 20)) (stays[j] ? sources : targets).push_back(slots[j]);
    sources.resize(20, -1), targets.resize(20, -1);
    EXPECT(e.download(from) == sources && e.download(to) == targets);
    const auto moved_k = e.download(keys);
    const auto moved_at = e.download(slot_positions);
    const auto moved_sums = e.download(sums);
    for (size_t i = 0; i < 20 && sources[i] >= 0; ++i) {
        EXPECT(moved_at[targets[i]] == at[sources[i]] && moved_sums[targets[i]] == weight[sources[i]]);
        EXPECT(std::memcmp(&moved_k[targets[i] * kKvHeads * kDim], &turned_k[sources[i] * kKvHeads * kDim], kKvHeads * kDim * 2) == 0);
    }
}

// The turn by the negative angles undoes the turn, in place.
void case_turn_back() {
    Env& e = *g_env;
    const auto q = items(kTokens * kHeads * kDim, 7), k = items(kTokens * kKvHeads * kDim, 8);
    std::vector<int32_t> positions(kTokens);
    for (size_t t = 0; t < kTokens; ++t) positions[t] = static_cast<int32_t>(1000 * t);
    auto dq = e.upload(q), dk = e.upload(k);
    auto dp = e.upload(positions);
    auto df = e.upload(DeviceAttention::RotaryFrequencies(kDim / 2, 10000.0, LCPP_HIP_ROTARY_LINEAR, 4.0));
    CommandList c;
    e.attention.Rotary<bfloat16>(c, dq.view(), dk.view(), {dp, {}, {}}, {df, true}, dq.view(), dk.view(), kShape);
    e.attention.Rotary<bfloat16>(c, dq.view(), dk.view(), {dp, {}, {}}, {df, true, true}, dq.view(), dk.view(), kShape);
    e.run(c);
    const auto back_q = e.download(dq), back_k = e.download(dk);
    double worst = 0;
    for (size_t i = 0; i < q.size(); ++i) worst = std::max(worst, std::abs(value_of(back_q[i]) - value_of(q[i])));
    for (size_t i = 0; i < k.size(); ++i) worst = std::max(worst, std::abs(value_of(back_k[i]) - value_of(k[i])));
    EXPECT(worst <= 3 * 0.0056);  // two roundings of each of a pair, which the second turn mixes
}

void case_recurrence() {
    Env& e = *g_env;
    constexpr uint kChannels = 70;
    const std::vector<int32_t> lengths{300, 1, 0, 45};
    std::vector<int32_t> offsets{0};
    for (int32_t n : lengths) offsets.push_back(offsets.back() + n);
    const size_t tokens = static_cast<size_t>(offsets.back());
    const auto floats = [&](size_t n, uint64_t seed) {
        std::vector<float> x(n);
        for (size_t i = 0; i < n; ++i) x[i] = static_cast<float>(number(seed, i));
        return x;
    };
    auto x = floats(tokens * kChannels, 1), l = floats(tokens * kChannels, 2), dout = floats(tokens * kChannels, 3);
    for (float& a : l) a = -std::abs(a) * 0.5f;
    const auto initial = floats(4 * kChannels, 4), dfinal = floats(4 * kChannels, 5);
    auto dx = e.upload(x), dl = e.upload(l), ddout = e.upload(dout), out = e.upload(x), gx = e.upload(x), gl = e.upload(x);
    auto di = e.upload(initial), df = e.upload(dfinal), final = e.upload(initial), gi = e.upload(initial);
    auto doff = e.upload(offsets);
    auto temp = e.device.create_buffer<uint>(DeviceRecurrence::GetTempStorageBytes(4, tokens, kChannels) / 4 + 4);
    CommandList c;
    e.recurrence.Scan<float>(c, temp, dx.view(), dl.view(), doff, out.view(), di, final, {}, tokens, kChannels);
    e.recurrence.ScanBackward<float>(c, temp, dl.view(), out.view(), ddout.view(), doff, di, df, gx.view(), gl.view(), gi, tokens, kChannels);
    e.run(c);
    const auto h = e.download(out), last = e.download(final), got_x = e.download(gx), got_l = e.download(gl), got_i = e.download(gi);
    // States of at most 300 steps of rounding of numbers below 300: 300 * 300 * 2^-23, twice over in their products.
    constexpr double kOff = 0.02;
    double worst = 0;
    for (size_t s = 0; s < lengths.size(); ++s)
        for (uint ch = 0; ch < kChannels; ++ch) {
            std::vector<double> state{initial[s * kChannels + ch]};
            for (int32_t t = offsets[s]; t < offsets[s + 1]; ++t) {
                state.push_back(std::exp(static_cast<double>(l[t * kChannels + ch])) * state.back() + x[t * kChannels + ch]);
                worst = std::max(worst, std::abs(h[t * kChannels + ch] - state.back()));
            }
            worst = std::max(worst, std::abs(last[s * kChannels + ch] - state.back()));
            double carry = dfinal[s * kChannels + ch];
            for (int32_t t = offsets[s + 1] - 1; t >= offsets[s]; --t) {
                const double g = dout[t * kChannels + ch] + carry;
                carry = std::exp(static_cast<double>(l[t * kChannels + ch])) * g;
                worst = std::max(worst, std::abs(got_x[t * kChannels + ch] - g));
                worst = std::max(worst, std::abs(got_l[t * kChannels + ch] - carry * state[t - offsets[s]]));
            }
            worst = std::max(worst, std::abs(got_i[s * kChannels + ch] - carry));
        }
    EXPECT(worst <= kOff);
}

struct Case {
    const char* name;
    void (*run)();
};
const Case kCases[] = {{"request", case_request}, {"turn_back", case_turn_back}, {"recurrence", case_recurrence}};

}  // namespace

int main(int argc, char** argv) {
    const std::string arg = argc > 1 ? argv[1] : "";
    if (arg == "--list") {
        for (const Case& c : kCases) std::printf("%s\n", c.name);
        return 0;
    }
    Env env;
    g_env = &env;
    int ran = 0;
    for (const Case& c : kCases) {
        if (!arg.empty() && std::string(c.name).find(arg) == std::string::npos) continue;
        g_current = c.name;
        std::printf("%s\n", c.name);
        std::fflush(stdout);
        c.run();
        ++ran;
    }
    std::printf("%d cases, %d failures\n", ran, g_failures);
    return g_failures == 0 ? 0 : 1;
}
