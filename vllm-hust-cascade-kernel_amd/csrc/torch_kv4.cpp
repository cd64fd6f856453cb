// torch_kv4.cpp - the ops over a 4-bit K/V cache on the C ABI (cascade_kernels.h), registered beside those of
// torch_ops.cpp under `npu`. Shapes decide everything on the host: no device->host copy, every
// launch on the current stream, so all four can be captured.
#include "torch_checks.h"

namespace cascade_amd {
namespace {

constexpr int64_t kHead = 128;

// A pool's kv heads.
int64_t check_pool(const char *op, const char *what, const at::Tensor &cache) {
    TORCH_CHECK(cache.scalar_type() == at::kByte && cache.dim() == 3 && cache.size(2) == CK_KV4_PAGE_BYTES &&
                    cache.is_contiguous(),
                op, ": ", what, " must be a contiguous uint8 (numBlocks, KVH, ", CK_KV4_PAGE_BYTES, ") pool");
    TORCH_CHECK(cache.size(1) > 0, op, ": ", what, " must have kv heads");
    return cache.size(1);
}

int64_t check_slots(const char *op, const at::Tensor &slots) {
    TORCH_CHECK(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.is_contiguous(), op,
                ": slots must be contiguous int64 (T,)");
    return slots.size(0);
}

void kv4_cache_write_impl(const at::Tensor &key, const at::Tensor &value, const at::Tensor &slots,
                          const at::Tensor &cache) {
    const char *op = "kv4_cache_write";
    const int dtype = check_type(op, "key", key);
    const int64_t kv_heads = check_pool(op, "cache", cache), tokens = check_slots(op, slots);
    int64_t strides[2][2];
    int n = 0;
    for (const at::Tensor *t : {&key, &value}) {
        TORCH_CHECK(t->dim() == 3 && t->size(0) == tokens && t->size(1) == kv_heads && t->size(2) == kHead, op,
                    ": key and value must be (T, KVH, 128) of the slots' tokens and the cache's kv heads");
        TORCH_CHECK(t->scalar_type() == key.scalar_type(), op, ": value must have key's dtype");
        TORCH_CHECK(tokens == 0 || t->stride(2) == 1, op, ": key and value must have unit stride in their last dim");
        // 16 bytes are moved at a time; strides of a dim of one element are not used
        for (int64_t d = 0; d < 2; ++d) {
            strides[n][d] = t->size(d) > 1 ? t->stride(d) : 0;
            TORCH_CHECK(strides[n][d] >= 0 && strides[n][d] % 8 == 0 && strides[n][d] <= (1 << 28), op,
                        ": key and value strides must be multiples of 8, at most 2^28");
        }
        ++n;
    }
    check_device(op, key, {&value, &slots, &cache});
    if (key.device().is_meta() || tokens == 0) return;
    c10::OptionalDeviceGuard guard(key.device());
    check_launch(ck_kv4_cache_write(key.data_ptr(), strides[0][0], strides[0][1], value.data_ptr(), strides[1][0],
                                    strides[1][1], slots.data_ptr<int64_t>(), cache.data_ptr(), cache.size(0), tokens,
                                    kv_heads, dtype, stream_of(key)),
                 op);
}

std::tuple<at::Tensor, at::Tensor> kv4_cache_read_impl(const at::Tensor &cache, const at::Tensor &slots,
                                                       c10::optional<at::ScalarType> dtype) {
    const char *op = "kv4_cache_read";
    const int64_t kv_heads = check_pool(op, "cache", cache), tokens = check_slots(op, slots);
    const at::ScalarType type = dtype.value_or(at::kBFloat16);
    TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf, op, ": dtype must be bf16 or fp16");
    check_device(op, cache, {&slots});
    auto key = at::empty({tokens, kv_heads, kHead}, cache.options().dtype(type));
    auto value = at::empty_like(key);
    if (cache.device().is_meta() || tokens == 0) return {key, value};
    c10::OptionalDeviceGuard guard(cache.device());
    check_launch(ck_kv4_cache_read(cache.data_ptr(), slots.data_ptr<int64_t>(), cache.size(0), tokens, kv_heads,
                                   type == at::kHalf ? CK_DTYPE_F16 : CK_DTYPE_BF16, key.data_ptr(), value.data_ptr(),
                                   stream_of(cache)),
                 op);
    return {key, value};
}

void check_heads(const char *op, int64_t heads, int64_t kv_heads) {
    TORCH_CHECK(heads % kv_heads == 0, op, ": query heads must be a multiple of the cache's kv heads");
}

std::tuple<at::Tensor, at::Tensor> kv4_decode_impl(const at::Tensor &query, const at::Tensor &cache,
                                                   const at::Tensor &block_table, const at::Tensor &actual_kv_seqlens,
                                                   double scale, int64_t q_seqlen_value) {
    const char *op = "kv4_decode";
    const int dtype = check_query(op, query, kHead);
    TORCH_CHECK(q_seqlen_value >= 1, op, ": q_seqlen_value must be >= 1");
    TORCH_CHECK(query.size(0) % q_seqlen_value == 0, op, ": query.size(0) must be a multiple of q_seqlen_value");
    const int64_t batch = query.size(0) / q_seqlen_value, heads = query.size(1);
    const int64_t kv_heads = check_pool(op, "cache", cache);
    check_heads(op, heads, kv_heads);
    check_table(op, "", block_table, actual_kv_seqlens, batch);
    check_scale(op, scale);
    check_device(op, query, {&cache, &block_table, &actual_kv_seqlens});
    auto out = at::empty_like(query);
    auto lse = at::empty({query.size(0) * heads}, query.options().dtype(at::kFloat));
    if (batch == 0 || query.device().is_meta()) return {out, lse};
    const int64_t cols = block_table.size(1);
    c10::OptionalDeviceGuard guard(query.device());
    int64_t ws_bytes = 0;
    check_launch(ck_kv4_decode_plan(batch, q_seqlen_value, heads, kv_heads, cols * kPageTokens, &ws_bytes), op);
    at::Tensor ws = at::empty({ws_bytes}, query.options().dtype(at::kByte));
    check_launch(ck_kv4_decode(query.data_ptr(), cache.data_ptr(), block_table.data_ptr<int32_t>(), cols,
                               actual_kv_seqlens.data_ptr<int64_t>(), batch, q_seqlen_value, heads, kv_heads,
                               cache.size(0), kPageTokens, dtype, static_cast<float>(scale), out.data_ptr(),
                               lse.data_ptr<float>(), ws.data_ptr(), ws_bytes, stream_of(query)),
                 op);
    return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> kv4_cascade_decode_impl(
    const at::Tensor &query, const at::Tensor &prefix_cache, const at::Tensor &prefix_block_table,
    const at::Tensor &prefix_kv_seqlens, const at::Tensor &suffix_cache, const at::Tensor &suffix_block_table,
    const at::Tensor &suffix_kv_seqlens, double scale) {
    const char *op = "kv4_cascade_decode";
    const int dtype = check_query(op, query, kHead);
    const int64_t batch = query.size(0), heads = query.size(1);
    const int64_t kv_heads = check_pool(op, "prefix_cache", prefix_cache);
    TORCH_CHECK(check_pool(op, "suffix_cache", suffix_cache) == kv_heads, op,
                ": prefix_cache and suffix_cache must have the same kv heads");
    check_heads(op, heads, kv_heads);
    check_table(op, "prefix ", prefix_block_table, prefix_kv_seqlens, 1);
    check_table(op, "suffix ", suffix_block_table, suffix_kv_seqlens, batch);
    check_scale(op, scale);
    check_device(op, query, {&prefix_cache, &prefix_block_table, &prefix_kv_seqlens, &suffix_cache, &suffix_block_table,
                             &suffix_kv_seqlens});
    auto out = at::empty_like(query);
    auto lse = at::empty({batch * heads}, query.options().dtype(at::kFloat));
    if (batch == 0 || query.device().is_meta()) return {out, lse};
    const int64_t pcols = prefix_block_table.size(1), scols = suffix_block_table.size(1);
    c10::OptionalDeviceGuard guard(query.device());
    int64_t ws_bytes = 0;
    check_launch(ck_kv4_cascade_decode_plan(batch, heads, kv_heads, pcols * kPageTokens, scols * kPageTokens, &ws_bytes),
                 op);
    at::Tensor ws = at::empty({ws_bytes}, query.options().dtype(at::kByte));
    check_launch(ck_kv4_cascade_decode(
                     query.data_ptr(), prefix_cache.data_ptr(), prefix_block_table.data_ptr<int32_t>(), pcols,
                     prefix_kv_seqlens.data_ptr<int64_t>(), prefix_cache.size(0), suffix_cache.data_ptr(),
                     suffix_block_table.data_ptr<int32_t>(), scols, suffix_kv_seqlens.data_ptr<int64_t>(),
                     suffix_cache.size(0), batch, heads, kv_heads, kPageTokens, dtype, static_cast<float>(scale),
                     out.data_ptr(), lse.data_ptr<float>(), ws.data_ptr(), ws_bytes, stream_of(query)),
                 op);
    return {out, lse};
}

}  // namespace
}  // namespace cascade_amd

TORCH_LIBRARY_FRAGMENT(npu, m) {
    m.def("kv4_cache_write(Tensor key, Tensor value, Tensor slots, Tensor(a!) cache) -> ()");
    m.def("kv4_cache_read(Tensor cache, Tensor slots, ScalarType? dtype=None) -> (Tensor, Tensor)");
    m.def("kv4_decode(Tensor query, Tensor cache, Tensor block_table, Tensor actual_kv_seqlens, float scale, "
          "int q_seqlen_value=1) -> (Tensor, Tensor)");
    m.def("kv4_cascade_decode(Tensor query, Tensor prefix_cache, Tensor prefix_block_table, Tensor prefix_kv_seqlens, "
          "Tensor suffix_cache, Tensor suffix_block_table, Tensor suffix_kv_seqlens, float scale) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(npu, CUDA, m) {
    m.impl("kv4_cache_write", TORCH_FN(cascade_amd::kv4_cache_write_impl));
    m.impl("kv4_cache_read", TORCH_FN(cascade_amd::kv4_cache_read_impl));
    m.impl("kv4_decode", TORCH_FN(cascade_amd::kv4_decode_impl));
    m.impl("kv4_cascade_decode", TORCH_FN(cascade_amd::kv4_cascade_decode_impl));
}

TORCH_LIBRARY_IMPL(npu, Meta, m) {
    m.impl("kv4_cache_write", TORCH_FN(cascade_amd::kv4_cache_write_impl));
    m.impl("kv4_cache_read", TORCH_FN(cascade_amd::kv4_cache_read_impl));
    m.impl("kv4_decode", TORCH_FN(cascade_amd::kv4_decode_impl));
    m.impl("kv4_cascade_decode", TORCH_FN(cascade_amd::kv4_cascade_decode_impl));
}
