// Checks shared by the operators on key / value caches.
#pragma once

#include <initializer_list>

#include "common.h"

namespace b200 {

// The innermost dimension is dense and every other pitch is a non-negative multiple of `multiple` elements; a tensor that is
// `written` shares no element between two indices by a pitch of zero.
bool kv_rows_fit(const TensorView& t, int64_t multiple, bool written);

// k / v: int8 [batch, kv heads, capacity, dim]; ks / vs: float32 [batch, kv heads, capacity].
diopiError_t kv_cache_check(const char* name, const TensorView& k, const TensorView& ks, const TensorView& v, const TensorView& vs, bool written);

// All tensors that are given lie on one device, the current one (kernels run there: another device's memory would be a fault).
diopiError_t one_device(const char* name, std::initializer_list<diopiConstTensorHandle_t> tensors);

}  // namespace b200
