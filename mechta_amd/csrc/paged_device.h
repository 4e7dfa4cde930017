// paged_device.h -- device helpers of the paged cache's kernels (gfx950).
#pragma once
#include "paged_internal.h"

namespace mkv {
namespace paged {

template <typename T>
using Vec8 = T __attribute__((ext_vector_type(8)));

template <typename T>  // 16-byte aligned
__device__ inline Vec8<T> load8(const T* p) {
    return *(const Vec8<T>*)p;
}
template <typename T>
__device__ inline void store8(T* p, Vec8<T> x) {
    *(Vec8<T>*)p = x;
}

// What does not change while a kernel runs, read by all lanes alike, in the constant address space: by scalar loads. (By a
// vector load, as the compiler chose next to the direct loads' inline assembly, the wait for a page number was a wait for
// every copy on its way: a 4,096-token prompt, then 160 us with scalar loads, took 207 that way.)
template <typename T>
using Uniform = const __attribute__((address_space(4))) T*;
template <typename T>
__device__ inline Uniform<T> uniform(const T* p) {
    return (Uniform<T>)(uintptr_t)p;
}

}  // namespace paged
}  // namespace mkv
