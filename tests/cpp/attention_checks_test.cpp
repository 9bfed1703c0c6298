// What DeviceAttention refuses when a command is recorded, on a machine without a GPU: views are made up and never looked at.
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

// Expects an error that says `words`, and nothing recorded.
template <typename F>
void refused(const char* what, const char* words, F&& record) {
    CommandList cmd;
    std::string said;
    try {
        record(cmd);
    } catch (const luisa::Error& error) {
        said = error.what();
    }
    const bool ok = std::strstr(said.c_str(), words) != nullptr && cmd.empty();
    g_failures += !ok;
    std::printf("%s: %s\n", what, ok ? "refused" : said.empty() ? "FAILED, recorded" : ("FAILED, says " + said).c_str());
}

}  // namespace

int main() {
    const AttentionShape shape{4, 2, 64, 0.f};
    const size_t n = 8;
    const AttentionRows<float16> q(made_up<float16>(n * 4 * 64)), k(made_up<float16>(n * 2 * 64));
    const AttentionCache<float16> cache(made_up<float16>(2 * 16 * 2 * 64));
    const PageShape page{16, 2};
    const auto ints = [](size_t count) { return made_up<int32_t>(count); };
    const auto temp = made_up<uint>(1 << 20);
    const auto lse = made_up<float>(n * 4);
    const auto slots = made_up<int64_t>(n);
    DeviceAttention none;  // not created
    refused("PagePlan before create", "create", [&](CommandList& c) {
        none.PagePlan(c, temp, ints(1), ints(1), 16, ints(2), {ints(2), 0, 0}, ints(2), ints(1), ints(n), ints(n), slots, ints(2));
    });
    refused("PagedWrite before create", "create", [&](CommandList& c) { none.PagedWrite(c, k, k, slots, cache, cache, shape, page); });
    refused("Packed before create", "create",
            [&](CommandList& c) { none.Packed(c, temp, q, k, k, ints(2), ints(2), q, lse, n, n, shape); });
    refused("PackedBackward before create", "create", [&](CommandList& c) {
        none.PackedBackward(c, temp, q, k, k, q, lse, q, ints(2), ints(2), q, k, k, n, n, shape);
    });
    refused("Paged before create", "create", [&](CommandList& c) {
        none.Paged(c, temp, q, cache, cache, {ints(2), 0, 0}, ints(2), ints(1), {}, q, lse, n, 20, shape, page);
    });
    std::printf("%d failures\n", g_failures);
    return g_failures == 0 ? 0 : 1;
}
