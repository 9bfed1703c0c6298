// DeviceAttention: attention over ragged batches and a paged cache (lcpp_hip_page_plan, lcpp_hip_paged_write_*,
// lcpp_hip_attention_packed_*, lcpp_hip_attention_paged_*), in the shape of the other modules: create, temp-storage
// queries, and calls that check their views and record into a CommandList.  There is no reference counterpart; what the
// calls compute is documented in lcpp_hip.h.
#pragma once

#include <cmath>
#include <limits>
#include <type_traits>

#include "lcpp/runtime/core.h"

namespace luisa::parallel_primitive {

// 16-bit floating point items, as bits.
struct bfloat16 {
    uint16_t bits;
};
struct float16 {
    uint16_t bits;
};

template <typename T>
concept AttentionItemT = std::is_same_v<T, bfloat16> || std::is_same_v<T, float16>;

// [tokens][heads][head_dim]; strides in items.  From a view alone: packed.
template <AttentionItemT T>
struct AttentionRows {
    BufferView<T> view;
    size_t token_stride = 0, head_stride = 0;  // 0 and 0: packed
    AttentionRows() = default;
    AttentionRows(BufferView<T> items) : view(items) {}
    AttentionRows(BufferView<T> items, size_t token, size_t head) : view(items), token_stride(token), head_stride(head) {}
};

// [pages][page_size][kv_heads][head_dim], the first three axes in any order; from a view alone: packed in this one.
template <AttentionItemT T>
struct AttentionCache {
    BufferView<T> view;
    size_t page_stride = 0, token_stride = 0, head_stride = 0;  // all 0: packed
    AttentionCache() = default;
    AttentionCache(BufferView<T> items) : view(items) {}
    AttentionCache(BufferView<T> items, size_t page, size_t token, size_t head)
        : view(items), page_stride(page), token_stride(token), head_stride(head) {}
};

struct AttentionShape {
    uint q_heads = 1, kv_heads = 1, head_dim = 64;
    float scale = 0.f;  // 0: 1 / sqrt(head_dim)
};

struct PageShape {
    uint page_size = 16, pages = 0;
};

// One request's pages a row; rows `stride` entries apart, of which `width` are used (0: the view's entries a request).
struct BlockTable {
    BufferView<int32_t> view;
    uint stride = 0, width = 0;
};

class DeviceAttention : public LuisaModule {
  public:
    void create(Device& device) { create_module(device); }

    [[nodiscard]] static size_t GetPagePlanTempStorageBytes(uint requests) { return lcpp_hip_page_plan_temp_bytes(requests); }
    [[nodiscard]] static size_t GetPackedTempStorageBytes(uint sequences, size_t q_tokens, size_t k_tokens, const AttentionShape& s) {
        return lcpp_hip_attention_packed_temp_bytes(sequences, q_tokens, k_tokens, s.q_heads, s.kv_heads, s.head_dim);
    }
    [[nodiscard]] static size_t GetPackedBackwardTempStorageBytes(uint sequences, size_t q_tokens, size_t k_tokens,
                                                                  const AttentionShape& s) {
        return lcpp_hip_attention_packed_backward_temp_bytes(sequences, q_tokens, k_tokens, s.q_heads, s.kv_heads, s.head_dim);
    }
    [[nodiscard]] static size_t GetPagedTempStorageBytes(uint requests, size_t q_tokens, size_t max_kv_length, const AttentionShape& s) {
        return lcpp_hip_attention_paged_temp_bytes(requests, q_tokens, max_kv_length, s.q_heads, s.kv_heads, s.head_dim);
    }

    // Offsets, lengths, and each new token's request, position and slot; token_slot's size is the capacity.
    void PagePlan(CommandList& cmdlist, BufferView<uint> temp_storage, BufferView<int32_t> cached_lengths,
                  BufferView<int32_t> new_lengths, uint page_size, BufferView<int32_t> free_pages, BlockTable table,
                  BufferView<int32_t> query_offsets, BufferView<int32_t> kv_lengths, BufferView<int32_t> token_request,
                  BufferView<int32_t> token_position, BufferView<int64_t> token_slot, BufferView<int32_t> counts) {
        const uint requests = count_of(cached_lengths.size(), "requests");
        const size_t tokens = token_slot.size();
        const uint num_free = count_of(free_pages.size(), "free pages");
        resolve(table, requests);
        LCPP_ASSERT(new_lengths.size() >= requests, "DeviceAttention new-length view is too small.");
        LCPP_ASSERT(query_offsets.size() > requests, "DeviceAttention query-offset view is too small.");
        LCPP_ASSERT(kv_lengths.size() >= requests, "DeviceAttention kv-length view is too small.");
        LCPP_ASSERT(token_request.size() >= tokens && token_position.size() >= tokens, "DeviceAttention token views are too small.");
        LCPP_ASSERT(counts.size() >= 2, "DeviceAttention count view is too small.");
        check_temp(temp_storage, GetPagePlanTempStorageBytes(requests));
        cmdlist << [=](hipStream_t s) {
            luisa::detail::abi_check(
                lcpp_hip_page_plan(temp_storage.data(), temp_storage.size_bytes(), cached_lengths.data(), new_lengths.data(), requests,
                                   page_size, free_pages.data(), num_free, table.view.data(), table.stride, table.width,
                                   query_offsets.data(), kv_lengths.data(), token_request.data(), token_position.data(),
                                   token_slot.data(), tokens, counts.data(), detail::stream_ptr(s)),
                "DeviceAttention::PagePlan");
        };
    }

    // Rows of key and value to slots[t] of the caches, a row for each slot.
    template <AttentionItemT T>
    void PagedWrite(CommandList& cmdlist, AttentionRows<T> key, AttentionRows<T> value, BufferView<int64_t> slots,
                    AttentionCache<T> key_cache, AttentionCache<T> value_cache, const AttentionShape& shape, PageShape page) {
        const size_t tokens = count_of(slots.size(), "tokens");
        auto k = rows(key, tokens, shape.kv_heads, shape.head_dim), v = rows(value, tokens, shape.kv_heads, shape.head_dim);
        auto kc = cache(key_cache, shape, page), vc = cache(value_cache, shape, page);
        cmdlist << [=](hipStream_t s) {
            auto* write = is_bf16<T> ? lcpp_hip_paged_write_bf16 : lcpp_hip_paged_write_f16;
            luisa::detail::abi_check(write(&k, &v, slots.data(), tokens, &kc, &vc, shape.kv_heads, shape.head_dim, page.page_size,
                                           page.pages, detail::stream_ptr(s)),
                                     "DeviceAttention::PagedWrite");
        };
    }

    // Rows of q to the keys of their sequence; offsets hold one entry more than there are sequences.  lse may be empty.
    template <AttentionItemT T>
    void Packed(CommandList& cmdlist, BufferView<uint> temp_storage, AttentionRows<T> q, AttentionRows<T> k, AttentionRows<T> v,
                BufferView<int32_t> q_offsets, BufferView<int32_t> k_offsets, AttentionRows<T> out, BufferView<float> lse,
                size_t q_tokens, size_t k_tokens, AttentionShape shape, bool causal = true) {
        const uint sequences = sequences_of(q_offsets, k_offsets);
        resolve(shape);
        auto qr = rows(q, q_tokens, shape.q_heads, shape.head_dim), kr = rows(k, k_tokens, shape.kv_heads, shape.head_dim);
        auto vr = rows(v, k_tokens, shape.kv_heads, shape.head_dim), outr = rows(out, q_tokens, shape.q_heads, shape.head_dim);
        LCPP_ASSERT(lse.size() == 0 || lse.size() >= q_tokens * shape.q_heads, "DeviceAttention lse view is too small.");
        check_temp(temp_storage, GetPackedTempStorageBytes(sequences, q_tokens, k_tokens, shape));
        cmdlist << [=](hipStream_t s) {
            auto* run = is_bf16<T> ? lcpp_hip_attention_packed_bf16 : lcpp_hip_attention_packed_f16;
            luisa::detail::abi_check(run(temp_storage.data(), temp_storage.size_bytes(), &qr, &kr, &vr, q_offsets.data(),
                                         k_offsets.data(), &outr, lse.data(), sequences, q_tokens, k_tokens, shape.q_heads,
                                         shape.kv_heads, shape.head_dim, shape.scale, causal, detail::stream_ptr(s)),
                                     "DeviceAttention::Packed");
        };
    }

    // Gradients of Packed, from the out and lse that it gave.
    template <AttentionItemT T>
    void PackedBackward(CommandList& cmdlist, BufferView<uint> temp_storage, AttentionRows<T> q, AttentionRows<T> k,
                        AttentionRows<T> v, AttentionRows<T> out, BufferView<float> lse, AttentionRows<T> dout,
                        BufferView<int32_t> q_offsets, BufferView<int32_t> k_offsets, AttentionRows<T> dq, AttentionRows<T> dk,
                        AttentionRows<T> dv, size_t q_tokens, size_t k_tokens, AttentionShape shape, bool causal = true) {
        const uint sequences = sequences_of(q_offsets, k_offsets);
        resolve(shape);
        const auto of_q = [&](const AttentionRows<T>& r) { return rows(r, q_tokens, shape.q_heads, shape.head_dim); };
        const auto of_k = [&](const AttentionRows<T>& r) { return rows(r, k_tokens, shape.kv_heads, shape.head_dim); };
        auto qr = of_q(q), outr = of_q(out), doutr = of_q(dout), dqr = of_q(dq);
        auto kr = of_k(k), vr = of_k(v), dkr = of_k(dk), dvr = of_k(dv);
        LCPP_ASSERT(lse.size() >= q_tokens * shape.q_heads, "DeviceAttention lse view is too small.");
        check_temp(temp_storage, GetPackedBackwardTempStorageBytes(sequences, q_tokens, k_tokens, shape));
        cmdlist << [=](hipStream_t s) {
            auto* run = is_bf16<T> ? lcpp_hip_attention_packed_backward_bf16 : lcpp_hip_attention_packed_backward_f16;
            luisa::detail::abi_check(run(temp_storage.data(), temp_storage.size_bytes(), &qr, &kr, &vr, &outr, lse.data(), &doutr,
                                         q_offsets.data(), k_offsets.data(), &dqr, &dkr, &dvr, sequences, q_tokens, k_tokens,
                                         shape.q_heads, shape.kv_heads, shape.head_dim, shape.scale, causal, detail::stream_ptr(s)),
                                     "DeviceAttention::PackedBackward");
        };
    }

    // New rows to their requests' pages; `tree` (a word a token) may be empty.
    template <AttentionItemT T>
    void Paged(CommandList& cmdlist, BufferView<uint> temp_storage, AttentionRows<T> q, AttentionCache<T> key_cache,
               AttentionCache<T> value_cache, BlockTable table, BufferView<int32_t> q_offsets, BufferView<int32_t> kv_lengths,
               BufferView<uint64_t> tree, AttentionRows<T> out, BufferView<float> lse, size_t q_tokens, size_t max_kv_length,
               AttentionShape shape, PageShape page) {
        const uint requests = count_of(kv_lengths.size(), "requests");
        resolve(shape);
        resolve(table, requests);
        auto qr = rows(q, q_tokens, shape.q_heads, shape.head_dim), outr = rows(out, q_tokens, shape.q_heads, shape.head_dim);
        auto kc = cache(key_cache, shape, page), vc = cache(value_cache, shape, page);
        LCPP_ASSERT(q_offsets.size() > requests, "DeviceAttention query-offset view is too small.");
        LCPP_ASSERT(tree.size() == 0 || tree.size() >= q_tokens, "DeviceAttention tree view is too small.");
        LCPP_ASSERT(lse.size() == 0 || lse.size() >= q_tokens * shape.q_heads, "DeviceAttention lse view is too small.");
        check_temp(temp_storage, GetPagedTempStorageBytes(requests, q_tokens, max_kv_length, shape));
        cmdlist << [=](hipStream_t s) {
            auto* run = is_bf16<T> ? lcpp_hip_attention_paged_bf16 : lcpp_hip_attention_paged_f16;
            luisa::detail::abi_check(run(temp_storage.data(), temp_storage.size_bytes(), &qr, &kc, &vc, table.view.data(),
                                         table.stride, table.width, q_offsets.data(), kv_lengths.data(), tree.data(), &outr,
                                         lse.data(), requests, q_tokens, max_kv_length, shape.q_heads, shape.kv_heads,
                                         shape.head_dim, page.page_size, page.pages, shape.scale, detail::stream_ptr(s)),
                                     "DeviceAttention::Paged");
        };
    }

  private:
    template <typename T>
    static constexpr bool is_bf16 = std::is_same_v<T, bfloat16>;

    [[nodiscard]] uint count_of(size_t n, const char* what) const {
        LCPP_ASSERT(m_created, "DeviceAttention::create must be called before dispatch.");
        LCPP_ASSERT(n <= static_cast<size_t>(std::numeric_limits<int32_t>::max()), string("Too many ") + what + " for DeviceAttention.");
        return static_cast<uint>(n);
    }
    [[nodiscard]] uint sequences_of(const BufferView<int32_t>& q_offsets, const BufferView<int32_t>& k_offsets) const {
        LCPP_ASSERT(q_offsets.size() > 0, "DeviceAttention query-offset view is empty.");
        LCPP_ASSERT(k_offsets.size() >= q_offsets.size(), "DeviceAttention key-offset view is too small.");
        return count_of(q_offsets.size() - 1, "sequences");
    }
    static void resolve(AttentionShape& shape) {
        if (shape.scale == 0.f && shape.head_dim > 0) shape.scale = 1.f / std::sqrt(static_cast<float>(shape.head_dim));
    }
    static void resolve(BlockTable& table, uint requests) {
        if (table.width == 0 && requests > 0)
            table.width = table.stride ? table.stride : static_cast<uint>(table.view.size() / requests);
        if (table.stride == 0) table.stride = table.width;
        LCPP_ASSERT(table.width <= table.stride, "A DeviceAttention block table's rows must hold their width.");
        LCPP_ASSERT(requests == 0 || table.view.size() >= static_cast<size_t>(requests - 1) * table.stride + table.width,
                    "DeviceAttention block-table view is too small.");
    }
    static void check_temp(const BufferView<uint>& temp, size_t bytes) {
        LCPP_ASSERT(temp.size_bytes() >= bytes, "DeviceAttention temporary-storage view is too small.");
    }
    // The last item that the strides reach lies inside the view.
    template <typename T>
    [[nodiscard]] static lcpp_hip_rows rows(const AttentionRows<T>& r, size_t tokens, size_t heads, size_t dim) {
        const bool packed = r.token_stride == 0 && r.head_stride == 0;
        const size_t token = packed ? heads * dim : r.token_stride, head = packed ? dim : r.head_stride;
        LCPP_ASSERT(tokens == 0 || heads == 0 || r.view.size() >= (tokens - 1) * token + (heads - 1) * head + dim,
                    "A DeviceAttention row view is too small.");
        return {r.view.data(), static_cast<int64_t>(token), static_cast<int64_t>(head)};
    }
    template <typename T>
    [[nodiscard]] static lcpp_hip_pages cache(const AttentionCache<T>& c, const AttentionShape& s, const PageShape& p) {
        const bool packed = c.page_stride == 0 && c.token_stride == 0 && c.head_stride == 0;
        const size_t head = packed ? s.head_dim : c.head_stride;
        const size_t token = packed ? static_cast<size_t>(s.kv_heads) * s.head_dim : c.token_stride;
        const size_t page = packed ? token * p.page_size : c.page_stride;
        LCPP_ASSERT(p.pages == 0 || p.page_size == 0 || s.kv_heads == 0 ||
                        c.view.size() >= (p.pages - size_t{1}) * page + (p.page_size - size_t{1}) * token +
                                             (s.kv_heads - size_t{1}) * head + s.head_dim,
                    "A DeviceAttention cache view is too small.");
        return {c.view.data(), static_cast<int64_t>(page), static_cast<int64_t>(token), static_cast<int64_t>(head)};
    }
};

}  // namespace luisa::parallel_primitive
