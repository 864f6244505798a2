// Row and vector helpers of the operators that stand next to the MoC layers
// (layer norm, causal convolution, selective scan).
#pragma once

#include <initializer_list>

#include "moc_common.h"

namespace moc {

// Element types of a storage dtype code.
template <int DT>
struct Elem;
template <>
struct Elem<DT_F32> {
  using type = float;
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};
template <>
struct Elem<DT_BF16> {
  using type = uint16_t;
  static __device__ __forceinline__ float up(uint16_t v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ uint16_t down(float v) { return f32_to_bf16(v); }
};

// V elements at p (aligned to their size together) as fp32.
template <int DT, int V>
__device__ __forceinline__ void load_vec(const void* p, int64_t i, float (&out)[V]) {
  using E = typename Elem<DT>::type;
  struct alignas(V * sizeof(E)) Pack {
    E e[V];
  };
  const Pack v = *reinterpret_cast<const Pack*>(static_cast<const E*>(p) + i);
#pragma unroll
  for (int k = 0; k < V; ++k) out[k] = Elem<DT>::up(v.e[k]);
}

template <int DT, int V>
__device__ __forceinline__ void store_vec(void* p, int64_t i, const float (&in)[V]) {
  using E = typename Elem<DT>::type;
  struct alignas(V * sizeof(E)) Pack {
    E e[V];
  };
  Pack v;
#pragma unroll
  for (int k = 0; k < V; ++k) v.e[k] = Elem<DT>::down(in[k]);
  *reinterpret_cast<Pack*>(static_cast<E*>(p) + i) = v;
}

// Whether every pointer is a multiple of `bytes` (a power of two).
inline bool aligned(std::initializer_list<const void*> ps, size_t bytes) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % bytes != 0) return false;
  return true;
}

// out[c] = sum over n rows of part[row][c] in a fixed order.  The columns are those of
// out0, then out1, then out2 (n0, n1, n2 of them, dtypes dt0..); a null output's are
// dropped.
struct ColumnSums {
  const float* part;
  int64_t n;
  int64_t n0, n1, n2;
  void *out0, *out1, *out2;
  int dt0, dt1, dt2;
};
void launch_column_sums(const ColumnSums& c, hipStream_t st);

}  // namespace moc
