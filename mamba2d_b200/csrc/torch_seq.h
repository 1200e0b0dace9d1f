// What the eager entry points of the sequence operators share: checks, pointers, streams.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "m2d_seq.h"

namespace m2d_entry {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline void check(int rc, const char* fn) { TORCH_CHECK(rc == M2D_OK, fn, " failed: ", m2d_strerror(rc), " (status ", rc, ")"); }
inline void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
inline int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? M2D_F32 : M2D_BF16; }
inline Tensor scratch(uint64_t bytes, const Tensor& like) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)); }
inline void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }

// Whether a call on these makes a node (one with a forward-mode tangent does: the node refuses it).
inline bool wants_grad(std::initializer_list<const Tensor*> inputs) {
    bool grad = false;
    for (const Tensor* t : inputs)
        if (t->defined()) grad = grad || (at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined();
    return grad;
}
// A wait between warps of an earlier launch that gave up (its results are NaN) surfaces at the next call.
inline void check_waits(const char* what) { TORCH_CHECK(!m2d_take_wait_failure(), what, ": a wait inside an earlier launch timed out; the results of that launch are invalid"); }
inline Tensor or_none(const optional<Tensor>& t) { return t ? *t : Tensor(); }
// neighbours along the last dimension
inline Tensor rows(const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
inline Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
// Tokens of each sequence of t (B, T, ...), as 32-bit integers.
inline Tensor token_counts(const char* what, const Tensor& lengths, const Tensor& t) {
    if (!lengths.defined()) return lengths;
    TORCH_CHECK(lengths.dim() == 1 && lengths.size(0) == t.size(0) && (lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong), what,
                ": lengths must be (B) integers, got ", lengths.sizes(), " ", lengths.scalar_type());
    TORCH_CHECK(lengths.device() == t.device(), what, ": lengths are on ", lengths.device(), ", expected ", t.device());
    return lengths.scalar_type() == at::kLong ? lengths.clamp(0, t.size(1)).to(at::kInt) : lengths;
}
inline void wrote(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace m2d_entry
