// Shared by the kernels of expert layers and 4-bit products: element types, argument checks.
#pragma once

#include <math.h>

#include "../../include/h2o4gpu_experts.h"
#include "kmeans_common.h"

#define KM_API extern "C" __attribute__((visibility("default")))

namespace kmhip {

typedef __bf16 bfloat16_t;
typedef _Float16 float16_t;

template <typename T>
struct Tag {
  typedef T type;
};

// A number as a type, for lambdas that pick a kernel.
template <int N>
struct Int {
  static constexpr int value = N;
};

// f(Tag<T>()) for the element type a caller names, EARG for a number that is none.
template <typename F>
inline int with_type(int dtype, F f) {
  switch (dtype) {
    case H2O4GPU_EXPERTS_FLOAT32:
      return f(Tag<float>());
    case H2O4GPU_EXPERTS_BFLOAT16:
      return f(Tag<bfloat16_t>());
    case H2O4GPU_EXPERTS_FLOAT16:
      return f(Tag<float16_t>());
  }
  return H2O4GPU_KMEANS_EARG;
}

inline size_t type_size(int dtype) { return dtype == H2O4GPU_EXPERTS_FLOAT32 ? 4 : 2; }
inline bool known_type(int dtype) { return dtype >= H2O4GPU_EXPERTS_FLOAT32 && dtype <= H2O4GPU_EXPERTS_FLOAT16; }
inline bool aligned_to(const void *p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

inline int launched() {
  KM_HIP_TRY(hipGetLastError());
  return H2O4GPU_KMEANS_OK;
}

}  // namespace kmhip
