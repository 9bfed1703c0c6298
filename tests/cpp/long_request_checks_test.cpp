// What the calls for rotary positions, eviction and the recurrence refuse when a command is recorded, on a machine without a GPU:
// views are made up and never looked at.
#include <lcpp/parallel_primitive.h>

#include <cstdio>
#include <cstring>
#include <string>

using namespace luisa;
using namespace luisa::compute;
using namespace luisa::parallel_primitive;

namespace {

int g_failures = 0;

template <typename T>
BufferView<T> made_up(size_t n) {
    return {reinterpret_cast<T*>(uintptr_t{1} << 20), n};
}

// Expects an error that says `words`, and nothing recorded; no words: recorded.
template <typename F>
void expect(const char* what, const char* words, F&& record) {
    CommandList cmd;
    std::string said;
    try {
        record(cmd);
    } catch (const luisa::Error& error) {
        said = error.what();
    }
    const bool ok = words ? std::strstr(said.c_str(), words) != nullptr && cmd.empty() : said.empty() && cmd.size() == 1;
    g_failures += !ok;
    std::printf("%s: %s\n", what, ok ? (words ? "refused" : "recorded") : ("FAILED, says " + said).c_str());
}

}  // namespace

int main() {
    const AttentionShape shape{4, 2, 64, 0.f};
    const size_t n = 8;
    const auto ints = [](size_t count) { return made_up<int32_t>(count); };
    const AttentionRows<float16> q(made_up<float16>(n * 4 * 64)), k(made_up<float16>(n * 2 * 64)), small(made_up<float16>(n * 2 * 64 - 1));
    const AttentionCache<float16> cache(made_up<float16>(2 * 16 * 2 * 64));
    const PageShape page{16, 2};
    const BlockTable table{ints(2), 0, 0};
    const RotaryPositions at{ints(n), {}, {}};
    const RotaryTurn turn{made_up<double>(32)};
    const auto temp = made_up<uint>(1 << 20);
    const auto lse = made_up<float>(n * 4), sums = made_up<float>(32);
    const auto slots = made_up<int64_t>(n), moves = made_up<int64_t>(6);
    DeviceAttention none, made;
    Context context;
    Device device = context.create_device("hip");
    made.create(device);

    expect("Rotary before create", "create", [&](CommandList& c) { none.Rotary(c, q, k, at, turn, q, k, shape); });
    expect("Rotary", nullptr, [&](CommandList& c) { made.Rotary(c, q, k, at, turn, q, k, shape); });
    expect("Rotary, small rows", "row view", [&](CommandList& c) { made.Rotary(c, q, small, at, turn, q, k, shape); });
    expect("Rotary, small output", "row view", [&](CommandList& c) { made.Rotary(c, q, k, at, turn, k, k, shape); });
    expect("Rotary, few requests", "request view",
           [&](CommandList& c) { made.Rotary(c, q, k, RotaryPositions{ints(n), ints(3), {}}, turn, q, k, shape); });
    expect("Rotary, shifts alone", "requests",
           [&](CommandList& c) { made.Rotary(c, q, k, RotaryPositions{ints(n), {}, ints(3)}, turn, q, k, shape); });
    expect("Rotary, many frequencies", "head size", [&](CommandList& c) { made.Rotary(c, q, k, at, RotaryTurn{made_up<double>(33)}, q, k, shape); });
    expect("Rotary, no frequencies", "head size", [&](CommandList& c) { made.Rotary(c, q, k, at, RotaryTurn{}, q, k, shape); });
    expect("PagedWriteRotary before create", "create",
           [&](CommandList& c) { none.PagedWriteRotary(c, q, k, k, at, turn, slots, q, cache, cache, ints(32), shape, page); });
    expect("PagedWriteRotary", nullptr,
           [&](CommandList& c) { made.PagedWriteRotary(c, q, k, k, at, turn, slots, q, cache, cache, {}, shape, page); });
    expect("PagedWriteRotary, few slots", "slot view", [&](CommandList& c) {
        made.PagedWriteRotary(c, q, k, k, at, turn, made_up<int64_t>(n - 1), q, cache, cache, {}, shape, page);
    });
    expect("PagedWriteRotary, few slot positions", "slot view",
           [&](CommandList& c) { made.PagedWriteRotary(c, q, k, k, at, turn, slots, q, cache, cache, ints(31), shape, page); });
    expect("PagedWriteRotary, small cache", "cache view",
           [&](CommandList& c) { made.PagedWriteRotary(c, q, k, k, at, turn, slots, q, cache, cache, {}, shape, PageShape{16, 3}); });
    expect("PagedWriteRotary, inverse", "forwards", [&](CommandList& c) {
        made.PagedWriteRotary(c, q, k, k, at, RotaryTurn{made_up<double>(32), false, true}, slots, q, cache, cache, {}, shape, page);
    });

    const auto weights = [&](DeviceAttention& m, CommandList& c, BufferView<float> l, BufferView<float> in, BufferView<float> out,
                             BufferView<int32_t> known, BufferView<uint64_t> tree) {
        m.PagedWeights(c, temp, q, cache, table, ints(2), ints(1), known, tree, l, in, out, n, 20, shape, page);
    };
    expect("PagedWeights before create", "create", [&](CommandList& c) { weights(none, c, lse, sums, sums, {}, {}); });
    expect("PagedWeights", nullptr, [&](CommandList& c) { weights(made, c, lse, {}, sums, {}, {}); });
    expect("PagedWeights, small lse", "lse", [&](CommandList& c) { weights(made, c, made_up<float>(31), sums, sums, {}, {}); });
    expect("PagedWeights, small sums", "slot view", [&](CommandList& c) { weights(made, c, lse, made_up<float>(31), sums, {}, {}); });
    expect("PagedWeights, no sums", "slot view", [&](CommandList& c) { weights(made, c, lse, sums, {}, {}, {}); });
    expect("PagedWeights, small tree", "tree", [&](CommandList& c) { weights(made, c, lse, sums, sums, {}, made_up<uint64_t>(n - 1)); });
    expect("PageRelease before create", "create",
           [&](CommandList& c) { none.PageRelease(c, ints(1), ints(1), 16, table, {}, ints(1), {}, ints(4), ints(2)); });
    expect("PageRelease", nullptr, [&](CommandList& c) { made.PageRelease(c, ints(1), ints(1), 16, table, {}, ints(1), {}, ints(4), ints(2)); });
    expect("PageRelease, few lengths", "length views",
           [&](CommandList& c) { made.PageRelease(c, ints(2), ints(1), 16, table, {}, ints(2), {}, ints(4), ints(2)); });
    expect("PageRelease, few counts", "count view",
           [&](CommandList& c) { made.PageRelease(c, ints(1), ints(1), 16, table, {}, ints(1), {}, ints(4), ints(1)); });
    const auto plan = [&](DeviceAttention& m, CommandList& c, BufferView<float> w, BufferView<int32_t> p, BufferView<int64_t> to) {
        m.EvictPlan(c, temp, w, p, table, ints(1), ints(1), {}, moves, to, 20, page, ProtectedKeys{1, 2});
    };
    expect("EvictPlan before create", "create", [&](CommandList& c) { plan(none, c, sums, ints(32), moves); });
    expect("EvictPlan", nullptr, [&](CommandList& c) { plan(made, c, sums, ints(32), moves); });
    expect("EvictPlan, small sums", "slot view", [&](CommandList& c) { plan(made, c, made_up<float>(31), ints(32), moves); });
    expect("EvictPlan, small positions", "slot view", [&](CommandList& c) { plan(made, c, sums, ints(31), moves); });
    expect("EvictPlan, uneven moves", "move views", [&](CommandList& c) { plan(made, c, sums, ints(32), slots); });
    expect("PagedMove before create", "create", [&](CommandList& c) { none.PagedMove(c, moves, moves, cache, cache, {}, {}, shape, page); });
    expect("PagedMove", nullptr, [&](CommandList& c) { made.PagedMove(c, moves, moves, cache, cache, sums, ints(32), shape, page); });
    expect("PagedMove, uneven moves", "move views", [&](CommandList& c) { made.PagedMove(c, moves, slots, cache, cache, {}, {}, shape, page); });
    expect("PagedMove, small sums", "slot view",
           [&](CommandList& c) { made.PagedMove(c, moves, moves, cache, cache, made_up<float>(3), {}, shape, page); });

    DeviceRecurrence raw, scan;
    scan.create(device);
    const RecurrenceRows<float> x(made_up<float>(9 * 10), 10), tight(made_up<float>(8 * 10), 10);
    const auto states = made_up<float>(2 * 10);
    const auto forward = [&](DeviceRecurrence& m, CommandList& c, RecurrenceRows<float> out, BufferView<float> from, BufferView<float> to,
                             BufferView<int32_t> rows) { m.Scan(c, temp, x, x, ints(3), out, from, to, rows, 9, 10); };
    expect("Scan before create", "create", [&](CommandList& c) { forward(raw, c, x, {}, {}, {}); });
    expect("Scan", nullptr, [&](CommandList& c) { forward(scan, c, x, states, states, {}); });
    expect("Scan, small rows", "row view", [&](CommandList& c) { forward(scan, c, tight, {}, {}, {}); });
    expect("Scan, few states", "state view", [&](CommandList& c) { forward(scan, c, x, made_up<float>(10), {}, {}); });
    expect("Scan, uneven states", "differ", [&](CommandList& c) { forward(scan, c, x, states, made_up<float>(30), {}); });
    expect("Scan, few state rows", "state view", [&](CommandList& c) { forward(scan, c, x, states, {}, ints(1)); });
    expect("Scan, no storage", "temporary", [&](CommandList& c) {
        scan.Scan(c, {}, RecurrenceRows<float>(made_up<float>(5000)), RecurrenceRows<float>(made_up<float>(5000)), ints(3),
                  RecurrenceRows<float>(made_up<float>(5000)), {}, {}, {}, 500, 10);
    });
    const auto backward = [&](DeviceRecurrence& m, CommandList& c, RecurrenceRows<float> dx, BufferView<float> from) {
        m.ScanBackward(c, temp, x, x, x, ints(3), from, {}, dx, x, {}, 9, 10);
    };
    expect("ScanBackward before create", "create", [&](CommandList& c) { backward(raw, c, x, {}); });
    expect("ScanBackward", nullptr, [&](CommandList& c) { backward(scan, c, x, states); });
    expect("ScanBackward, small rows", "row view", [&](CommandList& c) { backward(scan, c, tight, {}); });
    expect("ScanBackward, few states", "state view", [&](CommandList& c) { backward(scan, c, x, made_up<float>(10)); });
    std::printf("%d failures\n", g_failures);
    return g_failures == 0 ? 0 : 1;
}
