// torch_latent.cpp - the latent-attention ops over the C ABI (cascade_kernels.h), registered
// beside those of torch_ops.cpp under `npu`. Shapes decide everything on the host: no
// device->host copy, every launch on the current stream, so all four can be captured.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cmath>
#include <tuple>

#include "cascade_kernels.h"

namespace cascade_amd {
namespace {

constexpr int64_t kLatent = 512, kRope = 64, kRow = kLatent + kRope, kHead = 128, kPageTokens = 128;

void *stream_of(const at::Tensor &t) {
    return reinterpret_cast<void *>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

void check_launch(int rc, const char *op) {
    TORCH_CHECK(rc == CK_OK, op, ": kernel launch failed: ", ck_error_string(rc), " (code ", rc, ")");
}

int check_type(const char *op, const char *what, const at::Tensor &t) {
    TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, op, ": ", what,
                " must be bf16 or fp16");
    return t.scalar_type() == at::kBFloat16 ? CK_DTYPE_BF16 : CK_DTYPE_F16;
}

void check_device(const char *op, const at::Tensor &first, std::initializer_list<const at::Tensor *> others) {
    TORCH_CHECK(first.device().is_cuda() || first.device().is_meta(), op, ": tensors must be on a HIP device");
    for (const at::Tensor *t : others)
        TORCH_CHECK(t->device() == first.device(), op, ": all tensors must be on the same HIP device");
}

void check_cache(const char *op, const char *what, const at::Tensor &cache, at::ScalarType type) {
    TORCH_CHECK(cache.dim() == 3 && cache.size(1) == kPageTokens && cache.size(2) == kRow && cache.is_contiguous(), op,
                ": ", what, " must be a contiguous (numBlocks, 128, 576) pool");
    TORCH_CHECK(cache.scalar_type() == type, op, ": ", what, " must have the dtype of the other operands");
}

void check_table(const char *op, const char *what, const at::Tensor &table, const at::Tensor &lens, int64_t batch) {
    TORCH_CHECK(table.scalar_type() == at::kInt && table.dim() == 2 && table.is_contiguous(), op, ": ", what,
                "block_table must be a contiguous int32 (B, cols)");
    TORCH_CHECK(lens.scalar_type() == at::kLong && lens.dim() == 1 && lens.is_contiguous(), op, ": ", what,
                "kv seqlens must be a contiguous int64 (B,)");
    TORCH_CHECK(table.size(0) == batch && lens.numel() == batch, op, ": ", what,
                "block_table rows and kv seqlens must have batch entries");
}

void check_scale(const char *op, double scale) {
    const float f = static_cast<float>(scale);
    // the kernels work with scale log2(e)
    TORCH_CHECK(f > 0.f && std::isfinite(f * 1.44269504f), op, ": scale must be > 0 and at most 2.3e38");
}

// q rows of `dim` elements; contiguous, its rows 16-byte aligned
int check_query(const char *op, const at::Tensor &query, int64_t dim) {
    TORCH_CHECK(query.dim() == 3 && query.size(2) == dim && query.is_contiguous(), op, ": query must be a contiguous (T, H, ",
                dim, ")");
    TORCH_CHECK(query.size(1) > 0, op, ": query must have heads");
    return check_type(op, "query", query);
}

void latent_cache_write_impl(const at::Tensor &kv, const at::Tensor &gamma, const at::Tensor &cos_sin,
                             const at::Tensor &positions, const at::Tensor &slots, const at::Tensor &cache, double eps,
                             bool interleaved) {
    const char *op = "latent_cache_write";
    const int dtype = check_type(op, "kv", kv);
    TORCH_CHECK(kv.dim() == 2 && kv.size(1) == kRow, op, ": kv must be (T, 576)");
    const int64_t tokens = kv.size(0), stride = tokens > 1 ? kv.stride(0) : kRow;
    TORCH_CHECK(tokens == 0 || (kv.stride(1) == 1 && stride >= kRow && stride % 8 == 0), op,
                ": kv must have unit column stride and a row stride >= 576 that is a multiple of 8");
    TORCH_CHECK(gamma.scalar_type() == kv.scalar_type() && gamma.dim() == 1 && gamma.size(0) == kLatent &&
                    gamma.is_contiguous(),
                op, ": gamma must be a contiguous (512,) of kv's dtype");
    TORCH_CHECK(cos_sin.scalar_type() == at::kFloat && cos_sin.dim() == 2 && cos_sin.size(1) == kRope &&
                    cos_sin.is_contiguous(),
                op, ": cos_sin must be a contiguous fp32 (positions, 64)");
    for (const at::Tensor *t : {&positions, &slots})
        TORCH_CHECK(t->scalar_type() == at::kLong && t->dim() == 1 && t->size(0) == tokens && t->is_contiguous(), op,
                    ": positions and slots must be contiguous int64 (T,)");
    check_cache(op, "cache", cache, kv.scalar_type());
    const float eps_f = static_cast<float>(eps);
    TORCH_CHECK(std::isfinite(eps_f) && eps_f > 0.f, op, ": eps must be finite and > 0");
    check_device(op, kv, {&gamma, &cos_sin, &positions, &slots, &cache});
    if (kv.device().is_meta() || tokens == 0) return;
    c10::OptionalDeviceGuard guard(kv.device());
    check_launch(ck_latent_cache_write(kv.data_ptr(), stride, gamma.data_ptr(), cos_sin.data_ptr<float>(),
                                       cos_sin.size(0), positions.data_ptr<int64_t>(), slots.data_ptr<int64_t>(),
                                       cache.data_ptr(), cache.size(0), tokens, dtype, eps_f, interleaved,
                                       stream_of(kv)),
                 op);
}

std::tuple<at::Tensor, at::Tensor> latent_decode_impl(const at::Tensor &query, const at::Tensor &cache,
                                                      const at::Tensor &block_table,
                                                      const at::Tensor &actual_kv_seqlens, double scale,
                                                      int64_t q_seqlen_value) {
    const char *op = "latent_decode";
    const int dtype = check_query(op, query, kRow);
    TORCH_CHECK(q_seqlen_value >= 1, op, ": q_seqlen_value must be >= 1");
    TORCH_CHECK(query.size(0) % q_seqlen_value == 0, op, ": query.size(0) must be a multiple of q_seqlen_value");
    const int64_t batch = query.size(0) / q_seqlen_value, heads = query.size(1);
    check_cache(op, "cache", cache, query.scalar_type());
    check_table(op, "", block_table, actual_kv_seqlens, batch);
    check_scale(op, scale);
    check_device(op, query, {&cache, &block_table, &actual_kv_seqlens});
    auto out = at::empty({query.size(0), heads, kLatent}, query.options());
    auto lse = at::empty({query.size(0) * heads}, query.options().dtype(at::kFloat));
    if (batch == 0 || query.device().is_meta()) return {out, lse};
    const int64_t cols = block_table.size(1);
    c10::OptionalDeviceGuard guard(query.device());
    int64_t ws_bytes = 0;
    check_launch(ck_latent_decode_plan(batch, q_seqlen_value, heads, cols * kPageTokens, &ws_bytes), op);
    at::Tensor ws = at::empty({ws_bytes}, query.options().dtype(at::kByte));
    check_launch(ck_latent_decode(query.data_ptr(), cache.data_ptr(), block_table.data_ptr<int32_t>(), cols,
                                  actual_kv_seqlens.data_ptr<int64_t>(), batch, q_seqlen_value, heads, cache.size(0),
                                  kPageTokens, dtype, static_cast<float>(scale), out.data_ptr(),
                                  lse.data_ptr<float>(), ws.data_ptr(), ws_bytes, stream_of(query)),
                 op);
    return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> latent_cascade_decode_impl(
    const at::Tensor &query, const at::Tensor &prefix_cache, const at::Tensor &prefix_block_table,
    const at::Tensor &prefix_kv_seqlens, const at::Tensor &suffix_cache, const at::Tensor &suffix_block_table,
    const at::Tensor &suffix_kv_seqlens, double scale) {
    const char *op = "latent_cascade_decode";
    const int dtype = check_query(op, query, kRow);
    const int64_t batch = query.size(0), heads = query.size(1);
    check_cache(op, "prefix_cache", prefix_cache, query.scalar_type());
    check_cache(op, "suffix_cache", suffix_cache, query.scalar_type());
    check_table(op, "prefix ", prefix_block_table, prefix_kv_seqlens, 1);
    check_table(op, "suffix ", suffix_block_table, suffix_kv_seqlens, batch);
    check_scale(op, scale);
    check_device(op, query, {&prefix_cache, &prefix_block_table, &prefix_kv_seqlens, &suffix_cache, &suffix_block_table,
                             &suffix_kv_seqlens});
    auto out = at::empty({batch, heads, kLatent}, query.options());
    auto lse = at::empty({batch * heads}, query.options().dtype(at::kFloat));
    if (batch == 0 || query.device().is_meta()) return {out, lse};
    const int64_t pcols = prefix_block_table.size(1), scols = suffix_block_table.size(1);
    c10::OptionalDeviceGuard guard(query.device());
    int64_t ws_bytes = 0;
    check_launch(ck_latent_cascade_decode_plan(batch, heads, pcols * kPageTokens, scols * kPageTokens, &ws_bytes), op);
    at::Tensor ws = at::empty({ws_bytes}, query.options().dtype(at::kByte));
    check_launch(ck_latent_cascade_decode(
                     query.data_ptr(), prefix_cache.data_ptr(), prefix_block_table.data_ptr<int32_t>(), pcols,
                     prefix_kv_seqlens.data_ptr<int64_t>(), prefix_cache.size(0), suffix_cache.data_ptr(),
                     suffix_block_table.data_ptr<int32_t>(), scols, suffix_kv_seqlens.data_ptr<int64_t>(),
                     suffix_cache.size(0), batch, heads, kPageTokens, dtype, static_cast<float>(scale), out.data_ptr(),
                     lse.data_ptr<float>(), ws.data_ptr(), ws_bytes, stream_of(query)),
                 op);
    return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> latent_prefill_impl(const at::Tensor &query, const at::Tensor &key,
                                                       const at::Tensor &key_rope, const at::Tensor &value,
                                                       const at::Tensor &actual_q_seqlens,
                                                       const at::Tensor &actual_kv_seqlens, double scale, bool causal) {
    const char *op = "latent_prefill";
    const int dtype = check_query(op, query, kHead + kRope);
    const int64_t tokens = query.size(0), heads = query.size(1);
    TORCH_CHECK(key.dim() == 3 && key.size(1) == heads && key.size(2) == kHead && key.sizes() == value.sizes(), op,
                ": key and value must be (S, H, 128)");
    const int64_t keys = key.size(0);
    TORCH_CHECK(key_rope.dim() == 2 && key_rope.size(0) == keys && key_rope.size(1) == kRope, op,
                ": key_rope must be (S, 64)");
    for (const at::Tensor *t : {&key, &key_rope, &value}) {
        TORCH_CHECK(t->scalar_type() == query.scalar_type(), op, ": key, key_rope and value must have query's dtype");
        TORCH_CHECK(keys == 0 || t->stride(-1) == 1, op, ": key, key_rope and value must have unit stride in their last dim");
        // 16 bytes are moved at a time; strides of a dim of one element are not used
        for (int64_t d = 0; d + 1 < t->dim(); ++d)
            TORCH_CHECK(t->size(d) <= 1 || (t->stride(d) >= 0 && t->stride(d) % 8 == 0 && t->stride(d) <= (1 << 24)), op,
                        ": key, key_rope and value strides must be multiples of 8, at most 2^24");
    }
    for (const at::Tensor *t : {&actual_q_seqlens, &actual_kv_seqlens})
        TORCH_CHECK(t->scalar_type() == at::kLong && t->dim() == 1 && t->is_contiguous(), op,
                    ": seqlens must be contiguous int64 (B,)");
    const int64_t batch = actual_q_seqlens.numel();
    TORCH_CHECK(actual_kv_seqlens.numel() == batch, op, ": seqlen tensors must have batch entries");
    check_scale(op, scale);
    check_device(op, query, {&key, &key_rope, &value, &actual_q_seqlens, &actual_kv_seqlens});
    auto out = at::empty({tokens, heads, kHead}, query.options());
    auto lse = at::empty({tokens * heads}, query.options().dtype(at::kFloat));
    if (tokens == 0 || query.device().is_meta()) return {out, lse};
    auto stride = [](const at::Tensor &t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; };
    c10::OptionalDeviceGuard guard(query.device());
    check_launch(ck_latent_prefill(query.data_ptr(), key.data_ptr(), stride(key, 0), stride(key, 1), key_rope.data_ptr(),
                                   stride(key_rope, 0), value.data_ptr(), stride(value, 0), stride(value, 1),
                                   actual_q_seqlens.data_ptr<int64_t>(), actual_kv_seqlens.data_ptr<int64_t>(), batch,
                                   tokens, keys, heads, dtype, static_cast<float>(scale), causal, out.data_ptr(),
                                   lse.data_ptr<float>(), stream_of(query)),
                 op);
    return {out, lse};
}

}  // namespace
}  // namespace cascade_amd

TORCH_LIBRARY_FRAGMENT(npu, m) {
    m.def("latent_cache_write(Tensor kv, Tensor gamma, Tensor cos_sin, Tensor positions, Tensor slots, "
          "Tensor(a!) cache, float eps=1e-6, bool interleaved=True) -> ()");
    m.def("latent_decode(Tensor query, Tensor cache, Tensor block_table, Tensor actual_kv_seqlens, float scale, "
          "int q_seqlen_value=1) -> (Tensor, Tensor)");
    m.def("latent_cascade_decode(Tensor query, Tensor prefix_cache, Tensor prefix_block_table, "
          "Tensor prefix_kv_seqlens, Tensor suffix_cache, Tensor suffix_block_table, Tensor suffix_kv_seqlens, "
          "float scale) -> (Tensor, Tensor)");
    m.def("latent_prefill(Tensor query, Tensor key, Tensor key_rope, Tensor value, Tensor actual_q_seqlens, "
          "Tensor actual_kv_seqlens, float scale, bool causal=True) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(npu, CUDA, m) {
    m.impl("latent_cache_write", TORCH_FN(cascade_amd::latent_cache_write_impl));
    m.impl("latent_decode", TORCH_FN(cascade_amd::latent_decode_impl));
    m.impl("latent_cascade_decode", TORCH_FN(cascade_amd::latent_cascade_decode_impl));
    m.impl("latent_prefill", TORCH_FN(cascade_amd::latent_prefill_impl));
}

TORCH_LIBRARY_IMPL(npu, Meta, m) {
    m.impl("latent_cache_write", TORCH_FN(cascade_amd::latent_cache_write_impl));
    m.impl("latent_decode", TORCH_FN(cascade_amd::latent_decode_impl));
    m.impl("latent_cascade_decode", TORCH_FN(cascade_amd::latent_cascade_decode_impl));
    m.impl("latent_prefill", TORCH_FN(cascade_amd::latent_prefill_impl));
}
