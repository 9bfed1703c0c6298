// DeviceAttention as a C++ program would call it: a step planned, written and attended to through pages, the same rows
// packed, their gradients, and what is refused when a command is recorded.  Host checks against plain loops in double.
//
// Usage: attention_test [--list] [case-substring]
#include <lcpp/parallel_primitive.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
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

template <typename F>
bool throws_error(F&& f) {
    try {
        f();
    } catch (const luisa::Error&) {
        return true;
    }
    return false;
}

struct Env {
    Context context;
    Device device;
    Stream stream;
    DeviceAttention attention;
    Env() : device(context.create_device("hip")), stream(device.create_stream()) { attention.create(device); }
};
Env* g_env = nullptr;

double value_of(bfloat16 x) {
    const uint32_t w = static_cast<uint32_t>(x.bits) << 16;
    float f;
    std::memcpy(&f, &w, 4);
    return f;
}

// Multiples of 1/64 in [-1, 1): exact in 16 bits.
std::vector<bfloat16> items(size_t n, uint64_t seed) {
    std::vector<bfloat16> out(n);
    for (size_t i = 0; i < n; ++i) {
        uint64_t z = (seed << 32) + (i + 1) * 0x9E3779B97F4A7C15ull;
        z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
        const float f = (static_cast<int>((z >> 33) % 128) - 64) / 64.f;
        uint32_t w;
        std::memcpy(&w, &f, 4);
        out[i].bits = static_cast<uint16_t>(w >> 16);
    }
    return out;
}

constexpr uint kHeads = 4, kKvHeads = 2, kDim = 64;
const AttentionShape kShape{kHeads, kKvHeads, kDim, 0.f};
// Products of 64 items of at most 1 with a scale of 1/8 and values of at most 1: weights are off by 2^-9 of themselves, and
// so is the result once rounded (2^-9 each of at most 1).
constexpr double kOff = 1.0 / 128;

struct Batch {
    std::vector<int32_t> lengths, offsets{0};
    std::vector<bfloat16> q, k, v;
    explicit Batch(std::vector<int32_t> n) : lengths(std::move(n)) {
        for (int32_t x : lengths) offsets.push_back(offsets.back() + x);
        q = items(tokens() * kHeads * kDim, 1), k = items(tokens() * kKvHeads * kDim, 2), v = items(tokens() * kKvHeads * kDim, 3);
    }
    size_t tokens() const { return static_cast<size_t>(offsets.back()); }
};

// Causal attention of one row.
void plain(const Batch& b, size_t sequence, int32_t row, uint head, std::vector<double>& out, double& lse) {
    const size_t first = static_cast<size_t>(b.offsets[sequence]), g = head / (kHeads / kKvHeads);
    std::vector<double> s(static_cast<size_t>(row) + 1);
    double top = -INFINITY, total = 0;
    for (size_t j = 0; j < s.size(); ++j) {
        for (uint d = 0; d < kDim; ++d)
            s[j] += value_of(b.q[((first + row) * kHeads + head) * kDim + d]) * value_of(b.k[((first + j) * kKvHeads + g) * kDim + d]);
        s[j] /= std::sqrt(static_cast<double>(kDim));
        top = std::max(top, s[j]);
    }
    for (double x : s) total += std::exp(x - top);
    lse = top + std::log(total);
    out.assign(kDim, 0.0);
    for (size_t j = 0; j < s.size(); ++j)
        for (uint d = 0; d < kDim; ++d) out[d] += std::exp(s[j] - lse) * value_of(b.v[((first + j) * kKvHeads + g) * kDim + d]);
}

void check_out(const Batch& b, const std::vector<bfloat16>& out, const std::vector<float>& lse) {
    std::vector<double> want;
    double worst = 0, worst_lse = 0, want_lse = 0;
    for (size_t s = 0; s < b.lengths.size(); ++s)
        for (int32_t i = 0; i < b.lengths[s]; ++i)
            for (uint h = 0; h < kHeads; ++h) {
                plain(b, s, i, h, want, want_lse);
                const size_t t = static_cast<size_t>(b.offsets[s] + i);
                for (uint d = 0; d < kDim; ++d) worst = std::max(worst, std::abs(value_of(out[(t * kHeads + h) * kDim + d]) - want[d]));
                worst_lse = std::max(worst_lse, std::abs(lse[h * b.tokens() + t] - want_lse));
            }
    EXPECT(worst <= kOff);
    EXPECT(worst_lse <= 1e-4);
}

template <typename T>
Buffer<T> upload(const std::vector<T>& host) {
    auto buffer = g_env->device.create_buffer<T>(host.size());
    g_env->stream << buffer.copy_from(host.data());
    return buffer;
}
template <typename T>
std::vector<T> download(const Buffer<T>& buffer) {
    std::vector<T> host(buffer.size());
    g_env->stream << buffer.copy_to(host.data()) << synchronize();
    return host;
}
Buffer<uint> temp_of(size_t bytes) { return g_env->device.create_buffer<uint>(bytes_to_uint_count(bytes)); }

void packed_forward() {
    auto& e = *g_env;
    const Batch b({5, 0, 1, 130, 64});
    auto q = upload(b.q), k = upload(b.k), v = upload(b.v);
    auto offsets = upload(b.offsets);
    auto out = e.device.create_buffer<bfloat16>(b.q.size());
    auto lse = e.device.create_buffer<float>(kHeads * b.tokens());
    auto temp = temp_of(DeviceAttention::GetPackedTempStorageBytes(5, b.tokens(), b.tokens(), kShape));
    CommandList cmd;
    e.attention.Packed<bfloat16>(cmd, temp, q.view(), k.view(), v.view(), offsets, offsets, out.view(), lse, b.tokens(), b.tokens(), kShape);
    e.stream << cmd.commit();
    check_out(b, download(out), download(lse));
}

void plan_write_and_paged() {
    auto& e = *g_env;
    const Batch b({7, 40, 1, 33});
    const uint page_size = 8, pages = 30, width = 6;
    auto q = upload(b.q), k = upload(b.k), v = upload(b.v);
    std::vector<int32_t> free_pages;
    for (uint i = 0; i < pages; ++i) free_pages.push_back(static_cast<int32_t>((i * 7 + 3) % pages));
    auto cached = upload(std::vector<int32_t>(4, 0)), fresh = upload(b.lengths), free = upload(free_pages);
    auto table = upload(std::vector<int32_t>(4 * width, -1));
    auto offsets = e.device.create_buffer<int32_t>(5), kv = e.device.create_buffer<int32_t>(4), counts = e.device.create_buffer<int32_t>(2);
    const size_t n = b.tokens();
    auto request = e.device.create_buffer<int32_t>(n), position = e.device.create_buffer<int32_t>(n);
    auto slot = e.device.create_buffer<int64_t>(n);
    auto key_cache = upload(items(size_t{pages} * page_size * kKvHeads * kDim, 9)), value_cache = upload(items(size_t{pages} * page_size * kKvHeads * kDim, 10));
    auto out = e.device.create_buffer<bfloat16>(b.q.size());
    auto lse = e.device.create_buffer<float>(kHeads * n);
    auto temp = temp_of(std::max(DeviceAttention::GetPagePlanTempStorageBytes(4), DeviceAttention::GetPagedTempStorageBytes(4, n, 40, kShape)));
    const PageShape page{page_size, pages};
    CommandList cmd;
    e.attention.PagePlan(cmd, temp, cached, fresh, page_size, free, {table, width, width}, offsets, kv, request, position, slot, counts);
    e.attention.PagedWrite<bfloat16>(cmd, k.view(), v.view(), slot, key_cache.view(), value_cache.view(), kShape, page);
    e.attention.Paged<bfloat16>(cmd, temp, q.view(), key_cache.view(), value_cache.view(), {table, 0, 0}, offsets, kv, {}, out.view(), lse, n, 40, kShape, page);
    e.stream << cmd.commit();
    check_out(b, download(out), download(lse));
    EXPECT(download(offsets) == b.offsets);
    EXPECT(download(counts) == (std::vector<int32_t>{static_cast<int32_t>(n), 1 + 5 + 1 + 5}));
    const auto slots = download(slot);
    EXPECT(slots[0] == int64_t{free_pages[0]} * page_size && slots[7] == int64_t{free_pages[1]} * page_size);
    EXPECT(slots[8 + 7] == int64_t{free_pages[2]} * page_size);
}

// Against the difference of sum(dout * out) along each input, in double.
void packed_gradients() {
    auto& e = *g_env;
    const Batch b({9, 21});
    const size_t n = b.tokens();
    auto q = upload(b.q), k = upload(b.k), v = upload(b.v);
    auto offsets = upload(b.offsets);
    const auto dout_host = items(b.q.size(), 4);
    auto dout = upload(dout_host);
    auto out = e.device.create_buffer<bfloat16>(b.q.size()), dq = e.device.create_buffer<bfloat16>(b.q.size());
    auto dk = e.device.create_buffer<bfloat16>(b.k.size()), dv = e.device.create_buffer<bfloat16>(b.k.size());
    auto lse = e.device.create_buffer<float>(kHeads * n);
    auto temp = temp_of(std::max(DeviceAttention::GetPackedTempStorageBytes(2, n, n, kShape),
                                 DeviceAttention::GetPackedBackwardTempStorageBytes(2, n, n, kShape)));
    CommandList cmd;
    e.attention.Packed<bfloat16>(cmd, temp, q.view(), k.view(), v.view(), offsets, offsets, out.view(), lse, n, n, kShape);
    e.attention.PackedBackward<bfloat16>(cmd, temp, q.view(), k.view(), v.view(), out.view(), lse, dout.view(), offsets, offsets,
                                         dq.view(), dk.view(), dv.view(), n, n, kShape);
    e.stream << cmd.commit();
    const auto got_q = download(dq), got_k = download(dk), got_v = download(dv);
    const auto loss = [&](const Batch& x) {
        std::vector<double> row;
        double sum = 0, l = 0;
        for (size_t s = 0; s < x.lengths.size(); ++s)
            for (int32_t i = 0; i < x.lengths[s]; ++i)
                for (uint h = 0; h < kHeads; ++h) {
                    plain(x, s, i, h, row, l);
                    for (uint d = 0; d < kDim; ++d)
                        sum += row[d] * value_of(dout_host[((static_cast<size_t>(x.offsets[s] + i)) * kHeads + h) * kDim + d]);
                }
        return sum;
    };
    // Single items moved by 1/8 each way: scores move by at most 1/64, so the difference is the derivative but for parts in
    // 10^4.  A key's weights over the rows of two heads add to at most 2 (1 + 1/2 + ... + 1/21) = 7.3; dP - delta is at most
    // about 8 and rounded with a part in 2^8, and delta carries at most 64 products' rounding, 2^-3: times the scale of 1/8
    // and items of at most 1 that is 0.03 + 0.11 of a gradient of a key, less of the others.
    const auto check = [&](std::vector<bfloat16> Batch::*member, const std::vector<bfloat16>& got, size_t at) {
        const auto moved = [&](float by) {
            Batch x = b;
            const float f = static_cast<float>(value_of((x.*member)[at])) + by;
            uint32_t w;
            std::memcpy(&w, &f, 4);
            (x.*member)[at].bits = static_cast<uint16_t>(w >> 16);
            return loss(x);
        };
        const double want = (moved(0.125f) - moved(-0.125f)) / 0.25;
        EXPECT(std::abs(value_of(got[at]) - want) <= 0.15 + 0.02 * std::abs(want));
    };
    for (size_t at : {size_t{0}, size_t{700}, b.q.size() - 3}) check(&Batch::q, got_q, at);
    for (size_t at : {size_t{5}, size_t{1400}, b.k.size() - 3}) check(&Batch::k, got_k, at);
    for (size_t at : {size_t{5}, size_t{1400}, b.v.size() - 3}) check(&Batch::v, got_v, at);
}

void refusals() {
    auto& e = *g_env;
    const size_t n = 4;
    auto q = e.device.create_buffer<bfloat16>(n * kHeads * kDim), k = e.device.create_buffer<bfloat16>(n * kKvHeads * kDim);
    auto offsets = upload(std::vector<int32_t>{0, 4});
    auto slots = upload(std::vector<int64_t>{0, 1, 2, 3});
    auto lse = e.device.create_buffer<float>(kHeads * n);
    CommandList cmd;
    const auto packed = [&](BufferView<bfloat16> rows, BufferView<int32_t> of, BufferView<float> l) {
        e.attention.Packed<bfloat16>(cmd, {}, rows, k.view(), k.view(), of, of, q.view(), l, n, n, kShape);
    };
    EXPECT(throws_error([&] { packed(q.view(0, n * kHeads * kDim - 8), offsets, lse); }));
    EXPECT(throws_error([&] { packed(q, {}, lse); }));
    EXPECT(throws_error([&] { packed(q, offsets, lse.view(0, 3)); }));
    EXPECT(throws_error([&] {
        e.attention.PackedBackward<bfloat16>(cmd, {}, q.view(), k.view(), k.view(), q.view(), lse, q.view(), offsets, offsets, q.view(),
                                             k.view(), k.view(), n, n, kShape);
    }));  // no temporary storage
    EXPECT(throws_error([&] {
        e.attention.PagedWrite<bfloat16>(cmd, k.view(), k.view(), slots, k.view(), k.view(), kShape, PageShape{8, 1});
    }));  // a cache of half a page
    DeviceAttention other;
    EXPECT(throws_error([&] {
        other.Packed<bfloat16>(cmd, {}, q.view(), k.view(), k.view(), offsets, offsets, q.view(), lse, n, n, kShape);
    }));  // not created
    EXPECT(cmd.empty());
    // What the library itself refuses comes with the command.
    CommandList odd;
    e.attention.Packed<bfloat16>(odd, {}, q.view(), k.view(), k.view(), offsets, offsets, q.view(), lse, n, n, {kHeads, kKvHeads, 60, 0.f});
    EXPECT(throws_error([&] { e.stream << odd.commit(); }));
}

struct Case {
    const char* name;
    std::function<void()> body;
};
const std::vector<Case>& cases() {
    static const std::vector<Case> all = {{"packed_forward", packed_forward},
                                          {"plan_write_and_paged", plan_write_and_paged},
                                          {"packed_gradients", packed_gradients},
                                          {"refusals", refusals}};
    return all;
}

}  // namespace

int main(int argc, char** argv) {
    const char* filter = nullptr;
    for (int i = 1; i < argc; ++i) {
        if (std::strcmp(argv[i], "--list") == 0) {
            for (const auto& c : cases()) std::printf("%s\n", c.name);
            return 0;
        }
        filter = argv[i];
    }
    Env env;
    g_env = &env;
    int run = 0;
    for (const auto& c : cases()) {
        if (filter && !std::strstr(c.name, filter)) continue;
        g_current = c.name;
        std::printf("case %s\n", c.name);
        std::fflush(stdout);
        const int before = g_failures;
        try {
            c.body();
        } catch (const std::exception& ex) {
            ++g_failures;
            std::printf("  FAILED %s: exception %s\n", c.name, ex.what());
        }
        std::printf("  %s\n", g_failures == before ? "ok" : "FAILED");
        std::fflush(stdout);
        ++run;
    }
    std::printf("%d cases, %d failures\n", run, g_failures);
    return g_failures == 0 && run > 0 ? 0 : 1;
}
