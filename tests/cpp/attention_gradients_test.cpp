// DeviceAttention's gradients, every item of dQ, dK and dV against the formulas in double, through packed views and through views into
// one fused buffer; and a check that what is compared would not pass if it were zero, negated, unscaled or exchanged.
//
// Usage: attention_gradients_test [--list | --host]
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

struct Env {
    Context context;
    Device device;
    Stream stream;
    DeviceAttention attention;
    Env() : device(context.create_device("hip")), stream(device.create_stream()) { attention.create(device); }
};
Env* g_env = nullptr;

// The two types: how a float becomes one (exactly, here) and back.
struct OfBfloat16 {
    using Item = bfloat16;
    static constexpr double kRoundoff = 1.0 / 256;
    static Item from(float f) {
        uint32_t w;
        std::memcpy(&w, &f, 4);
        return {static_cast<uint16_t>(w >> 16)};
    }
    static double value(Item x) {
        const uint32_t w = static_cast<uint32_t>(x.bits) << 16;
        float f;
        std::memcpy(&f, &w, 4);
        return f;
    }
};
struct OfFloat16 {
    using Item = float16;
    static constexpr double kRoundoff = 1.0 / 2048;
    static Item from(float f) {  // normal numbers or zero
        if (f == 0.f) return {0};
        int e;
        const float m = std::frexp(std::abs(f), &e);  // 0.5 <= m < 1
        return {static_cast<uint16_t>((f < 0 ? 0x8000u : 0u) | static_cast<uint32_t>(e + 14) << 10 | (static_cast<uint32_t>(m * 2048.f) & 1023u))};
    }
    static double value(Item x) {
        const int e = x.bits >> 10 & 31, m = x.bits & 1023;
        const double v = e == 31 ? (m ? NAN : INFINITY) : e ? std::ldexp(1024 + m, e - 25) : std::ldexp(m, -24);
        return x.bits & 0x8000 ? -v : v;
    }
};
constexpr uint16_t kUnwritten = 0x7FFF;  // NaN in both

constexpr uint kHeads = 4, kKvHeads = 2, kDim = 64, kGroup = kHeads / kKvHeads;
const AttentionShape kShape{kHeads, kKvHeads, kDim, 0.f};

// Multiples of `unit` in [-64, 64) of them: exact in 16 bits.
std::vector<float> numbers(size_t n, uint64_t seed, float unit) {
    std::vector<float> out(n);
    for (size_t i = 0; i < n; ++i) {
        uint64_t z = (seed << 32) + (i + 1) * 0x9E3779B97F4A7C15ull;
        z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
        out[i] = static_cast<float>(static_cast<int>((z >> 33) % 128) - 64) * unit;
    }
    return out;
}

struct Batch {
    std::vector<int32_t> offsets{0};
    std::vector<float> q, k, v, dout;
    std::vector<double> dq, dk, dv;  // by the formulas
    explicit Batch(const std::vector<int32_t>& lengths) {
        for (int32_t n : lengths) offsets.push_back(offsets.back() + n);
        const size_t of_q = tokens() * kHeads * kDim, of_k = tokens() * kKvHeads * kDim;
        q = numbers(of_q, 1, 1 / 32.f), k = numbers(of_k, 2, 1 / 32.f), v = numbers(of_k, 3, 1 / 32.f), dout = numbers(of_q, 4, 1 / 8.f);
        dq.assign(of_q, 0), dk.assign(of_k, 0), dv.assign(of_k, 0);
        for (size_t s = 0; s + 1 < offsets.size(); ++s)
            for (int32_t i = offsets[s]; i < offsets[s + 1]; ++i)
                for (uint h = 0; h < kHeads; ++h) row(offsets[s], i, h);
    }
    size_t tokens() const { return static_cast<size_t>(offsets.back()); }
    static double dot(const float* a, const float* b) {
        double sum = 0;
        for (uint d = 0; d < kDim; ++d) sum += double{a[d]} * b[d];
        return sum;
    }
    // A row's part of all gradients: keys first .. i are seen.
    void row(int32_t first, int32_t i, uint h) {
        const double scale = 1 / std::sqrt(double{kDim});
        const size_t n = static_cast<size_t>(i - first) + 1, at = (static_cast<size_t>(i) * kHeads + h) * kDim;
        const auto key = [&](size_t j) { return ((static_cast<size_t>(first) + j) * kKvHeads + h / kGroup) * kDim; };
        std::vector<double> p(n), dp(n);
        double total = 0, delta = 0;
        for (size_t j = 0; j < n; ++j) total += p[j] = std::exp(scale * dot(&q[at], &k[key(j)]));
        for (size_t j = 0; j < n; ++j) {
            p[j] /= total;
            dp[j] = dot(&dout[at], &v[key(j)]);
            delta += p[j] * dp[j];
        }
        for (size_t j = 0; j < n; ++j)
            for (uint d = 0; d < kDim; ++d) {
                const double ds = scale * p[j] * (dp[j] - delta);
                dq[at + d] += ds * k[key(j) + d];
                dk[key(j) + d] += ds * q[at + d];
                dv[key(j) + d] += p[j] * dout[at + d];
            }
    }
};

// The difference's size as a part of the wanted one's.
double apart(const std::vector<double>& got, const std::vector<double>& want) {
    double off = 0, size = 0;
    for (size_t i = 0; i < want.size(); ++i) off += (got[i] - want[i]) * (got[i] - want[i]), size += want[i] * want[i];
    return std::sqrt(off / size);
}

template <typename T>
Buffer<T> upload(const std::vector<T>& host) {
    auto buffer = g_env->device.create_buffer<T>(host.size());
    g_env->stream << buffer.copy_from(host.data()) << synchronize();
    return buffer;
}
template <typename T>
std::vector<T> download(const Buffer<T>& buffer) {
    std::vector<T> host(buffer.size());
    g_env->stream << buffer.copy_to(host.data()) << synchronize();
    return host;
}

// P, dS, the output behind rowsum(dO O) and the result are rounded to 16 bits: each by 0.41 of the unit roundoff in the
// root mean square, so by less than one of it together.
template <typename T>
void check(const char* name, const std::vector<double>& got, const std::vector<double>& want) {
    const double off = apart(got, want);
    std::printf("  %s: off by %.2e of its size, allowed %.2e\n", name, off, T::kRoundoff);
    EXPECT(off <= T::kRoundoff);
}

template <typename T>
void gradients(bool fused) {
    using Item = typename T::Item;
    auto& e = *g_env;
    const Batch b({9, 0, 150, 1, 70});
    const size_t n = b.tokens();
    const auto sequences = static_cast<uint>(b.offsets.size() - 1);
    const auto put = [](const std::vector<float>& x) {
        std::vector<Item> items;
        for (float f : x) items.push_back(T::from(f));
        return upload(items);
    };
    auto q = put(b.q), k = put(b.k), v = put(b.v), dout = put(b.dout);
    auto offsets = upload(b.offsets);
    auto out = e.device.create_buffer<Item>(b.q.size());
    auto lse = e.device.create_buffer<float>(kHeads * n);
    auto temp = e.device.create_buffer<uint>(
        bytes_to_uint_count(std::max({size_t{4}, DeviceAttention::GetPackedTempStorageBytes(sequences, n, n, kShape),
                                      DeviceAttention::GetPackedBackwardTempStorageBytes(sequences, n, n, kShape)})));
    // Separate and packed, or rows of one buffer: dq, dk and dv of a token side by side, then 8 items that are not theirs.
    const size_t width = fused ? (kHeads + 2 * kKvHeads) * kDim + 8 : 0;
    auto all = upload(std::vector<Item>(fused ? n * width : b.q.size() + 2 * b.k.size(), Item{kUnwritten}));
    const size_t at_k = fused ? kHeads * kDim : b.q.size(), at_v = at_k + (fused ? kKvHeads * kDim : b.k.size());
    const auto view = [&](size_t at, uint heads) {
        return fused ? AttentionRows<Item>(all.view(at, (n - 1) * width + heads * kDim), width, kDim)
                     : AttentionRows<Item>(all.view(at, n * heads * kDim));
    };
    CommandList cmd;
    e.attention.Packed<Item>(cmd, temp, q.view(), k.view(), v.view(), offsets, offsets, out.view(), lse, n, n, kShape);
    e.attention.PackedBackward<Item>(cmd, temp, q.view(), k.view(), v.view(), out.view(), lse, dout.view(), offsets, offsets,
                                     view(0, kHeads), view(at_k, kKvHeads), view(at_v, kKvHeads), n, n, kShape);
    e.stream << cmd.commit();
    const auto items = download(all);
    std::vector<bool> theirs(items.size(), false);
    const auto get = [&](size_t at, uint heads) {
        std::vector<double> x;
        for (size_t t = 0; t < n; ++t)
            for (size_t i = 0; i < heads * kDim; ++i) {
                const size_t place = at + t * (fused ? width : heads * kDim) + i;
                theirs[place] = true;
                x.push_back(T::value(items[place]));
            }
        return x;
    };
    check<T>("dq", get(0, kHeads), b.dq);
    check<T>("dk", get(at_k, kKvHeads), b.dk);
    check<T>("dv", get(at_v, kKvHeads), b.dv);
    bool kept = true;
    for (size_t i = 0; i < items.size(); ++i) kept &= theirs[i] || items[i].bits == kUnwritten;
    EXPECT(kept);
}

// What the comparison tells apart (on the host alone).
void comparison_rejects() {
    const Batch b({9, 0, 150, 1, 70});
    const auto times = [](std::vector<double> x, double f) {
        for (double& y : x) y *= f;
        return x;
    };
    for (const auto* want : {&b.dq, &b.dk, &b.dv}) {
        EXPECT(apart(*want, *want) == 0);
        for (double f : {0.0, -1.0, 8.0, 0.125, 0.99}) EXPECT(apart(times(*want, f), *want) > OfBfloat16::kRoundoff);
    }
    EXPECT(apart(b.dk, b.dv) > 0.5 && apart(b.dv, b.dk) > 0.5);
    EXPECT(!(apart(std::vector<double>(b.dq.size(), NAN), b.dq) <= 1));
    for (float f : {0.f, 1.f, -0.75f, 63 / 32.f, -8.f, 0.125f}) {
        EXPECT(OfFloat16::value(OfFloat16::from(f)) == f && OfBfloat16::value(OfBfloat16::from(f)) == f);
    }
}

struct Case {
    const char* name;
    std::function<void()> body;
};
const std::vector<Case>& cases() {
    static const std::vector<Case> all = {{"comparison_rejects", comparison_rejects},
                                          {"gradients_bf16", [] { gradients<OfBfloat16>(false); }},
                                          {"gradients_f16", [] { gradients<OfFloat16>(false); }},
                                          {"gradients_bf16_fused", [] { gradients<OfBfloat16>(true); }},
                                          {"gradients_f16_fused", [] { gradients<OfFloat16>(true); }}};
    return all;
}

}  // namespace

// The comparison's own case needs no device, and is all that runs with --host.
int main(int argc, char** argv) {
    const bool host = argc > 1 && std::strcmp(argv[1], "--host") == 0;
    if (argc > 1 && std::strcmp(argv[1], "--list") == 0) {
        for (const auto& c : cases()) std::printf("%s\n", c.name);
        return 0;
    }
    Env* env = host ? nullptr : new Env;
    g_env = env;
    int run = 0;
    for (const auto& c : cases()) {
        if (host && run == 1) break;
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
    delete env;
    return g_failures == 0 && run > 0 ? 0 : 1;
}
