// torch_checks.h - what the torch-op layers of the paged attention families share: argument checks with
// their messages, and the stream of a call.
#pragma once

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cmath>
#include <initializer_list>
#include <tuple>

#include "cascade_kernels.h"

namespace cascade_amd {
namespace {

constexpr int64_t kPageTokens = 128;

inline void *stream_of(const at::Tensor &t) {
    return reinterpret_cast<void *>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

inline void check_launch(int rc, const char *op) {
    TORCH_CHECK(rc == CK_OK, op, ": kernel launch failed: ", ck_error_string(rc), " (code ", rc, ")");
}

inline int check_type(const char *op, const char *what, const at::Tensor &t) {
    TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, op, ": ", what,
                " must be bf16 or fp16");
    return t.scalar_type() == at::kBFloat16 ? CK_DTYPE_BF16 : CK_DTYPE_F16;
}

inline void check_device(const char *op, const at::Tensor &first, std::initializer_list<const at::Tensor *> others) {
    TORCH_CHECK(first.device().is_cuda() || first.device().is_meta(), op, ": tensors must be on a HIP device");
    for (const at::Tensor *t : others)
        TORCH_CHECK(t->device() == first.device(), op, ": all tensors must be on the same HIP device");
}

inline void check_table(const char *op, const char *what, const at::Tensor &table, const at::Tensor &lens, int64_t batch) {
    TORCH_CHECK(table.scalar_type() == at::kInt && table.dim() == 2 && table.is_contiguous(), op, ": ", what,
                "block_table must be a contiguous int32 (B, cols)");
    TORCH_CHECK(lens.scalar_type() == at::kLong && lens.dim() == 1 && lens.is_contiguous(), op, ": ", what,
                "kv seqlens must be a contiguous int64 (B,)");
    TORCH_CHECK(table.size(0) == batch && lens.numel() == batch, op, ": ", what,
                "block_table rows and kv seqlens must have batch entries");
}

inline void check_scale(const char *op, double scale) {
    const float f = static_cast<float>(scale);
    // the kernels work with scale log2(e)
    TORCH_CHECK(f > 0.f && std::isfinite(f * 1.44269504f), op, ": scale must be > 0 and at most 2.3e38");
}

// q rows of `dim` elements; contiguous, its rows 16-byte aligned
inline int check_query(const char *op, const at::Tensor &query, int64_t dim) {
    TORCH_CHECK(query.dim() == 3 && query.size(2) == dim && query.is_contiguous(), op, ": query must be a contiguous (T, H, ",
                dim, ")");
    TORCH_CHECK(query.size(1) > 0, op, ": query must have heads");
    return check_type(op, "query", query);
}

}  // namespace
}  // namespace cascade_amd
