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

// The first min(n, V) of V elements at p[i] as fp32, the others 0.  No alignment beyond an
// element's own is asked for: the hardware's wide loads and stores take any address, so
// that rows of odd lengths move in the same 16-byte pieces as aligned ones.
template <int DT, int V>
__device__ __forceinline__ void load_vec(const void* p, int64_t i, int64_t n, float (&out)[V]) {
  using E = typename Elem<DT>::type;
  struct __attribute__((packed, aligned(sizeof(E)))) Pack {
    E e[V];
  };
  const E* q = static_cast<const E*>(p) + i;
  if (n >= V) {
    const Pack v = *reinterpret_cast<const Pack*>(q);
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = Elem<DT>::up(v.e[k]);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = k < n ? Elem<DT>::up(q[k]) : 0.f;
  }
}

template <int DT, int V>
__device__ __forceinline__ void store_vec(void* p, int64_t i, int64_t n, const float (&in)[V]) {
  using E = typename Elem<DT>::type;
  struct __attribute__((packed, aligned(sizeof(E)))) Pack {
    E e[V];
  };
  E* q = static_cast<E*>(p) + i;
  if (n >= V) {
    Pack v;
#pragma unroll
    for (int k = 0; k < V; ++k) v.e[k] = Elem<DT>::down(in[k]);
    *reinterpret_cast<Pack*>(q) = v;
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < n) q[k] = Elem<DT>::down(in[k]);
  }
}

// The same on its way: loaded now, made fp32 when it is used (half the registers in bf16).
template <int DT, int V>
struct RawVec {
  typename Elem<DT>::type e[V];
  __device__ __forceinline__ void load(const void* p, int64_t i, int64_t n) {
    using E = typename Elem<DT>::type;
    struct __attribute__((packed, aligned(sizeof(E)))) Pack {
      E e[V];
    };
    const E* q = static_cast<const E*>(p) + i;
    if (n >= V) {
      const Pack v = *reinterpret_cast<const Pack*>(q);
      __builtin_memcpy(e, &v, sizeof(e));
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) e[k] = k < n ? q[k] : E(0);
    }
  }
  __device__ __forceinline__ void get(float (&out)[V]) const {
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = Elem<DT>::up(e[k]);
  }
};

// The same of a parameter of any dtype (null: every element `none`).
template <int V>
__device__ __forceinline__ void load_param(const void* p, int dt, int64_t i, int64_t n, float none, float (&out)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = none;
  } else if (dt == DT_F32) {
    load_vec<DT_F32, V>(p, i, n, out);
  } else if (dt == DT_BF16) {
    load_vec<DT_BF16, V>(p, i, n, out);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = k < n ? load_any(p, DT_F16, i + k) : 0.f;
  }
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
