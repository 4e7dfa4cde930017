// paged_device.h -- device helpers of the paged cache's kernels (gfx950).
#pragma once
#include "paged_internal.h"

namespace mkv {
namespace paged {

template <typename T>
using Vec8 = T __attribute__((ext_vector_type(8)));
template <typename T>
using Vec4 = T __attribute__((ext_vector_type(4)));

template <typename T>  // 16-byte aligned
__device__ inline Vec8<T> load8(const T* p) {
    return *(const Vec8<T>*)p;
}
template <typename T>
__device__ inline void store8(T* p, Vec8<T> x) {
    *(Vec8<T>*)p = x;
}

}  // namespace paged
}  // namespace mkv
