// What the entries of operators without a registration of TensorPlay's share:
// several result slots, index tensors, operands of one kind, axes that lie
// behind one another.
#pragma once

#include <initializer_list>

#include "tensor.h"

namespace tp_amd {

// Several results: every slot is written only once all of them exist.
template <typename Body>
int guarded_results(std::initializer_list<tp_amd_tensor*> slots, Body&& body) noexcept {
    return guarded([&] {
        for (tp_amd_tensor* s : slots) TP_AMD_CHECK(s != nullptr, "null result pointer");
        body();
    });
}

// The result slot of an output the caller did not ask for.
inline void set_undefined(tp_amd_tensor* r) {
    *r = tp_amd_tensor{};
    r->dtype = TP_AMD_UNDEFINED;
    r->device = -1;
}

inline bool index_tensor(const TensorRef& t, int device) {
    return on_device(t) && t.device == device && (t.dtype == TP_AMD_INT64 || t.dtype == TP_AMD_INT32);
}

// On ``like``'s device with its dtype.
inline bool same_kind(const TensorRef& t, const TensorRef& like) { return on_device(t) && t.device == like.device && t.dtype == like.dtype; }

// The first n axes of ``t`` as one index stepping by ``step``: false when
// they do not merge.  Axes without an element merge whatever their strides.
inline bool axes_merge(const TensorRef& t, int n, int64_t& step) {
    bool seen = false;
    int64_t next = 0;
    step = 0;
    for (int d = 0; d < n; ++d) {
        if (t.sizes[d] == 0) return true;
    }
    for (int d = n - 1; d >= 0; --d) {
        if (t.sizes[d] == 1) continue;
        if (seen && t.strides[d] != next) return false;
        if (!seen) step = t.strides[d];
        seen = true;
        next = t.strides[d] * t.sizes[d];
    }
    return true;
}

}  // namespace tp_amd
