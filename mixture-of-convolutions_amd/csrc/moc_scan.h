// Shared parts of the selective scan's kernels (moc_scan.hip, moc_scan_bwd.hip).
//
// Per head: u = softplus(dt + bias), h_t = exp(u_t A) h_{t-1} + u_t x_t (x) B_t,
// y_t = h_t C_t + D x_t, with h a [P, N] state (P: head_dim, N: state_dim).
//
// In chunks of kQ tokens of one sequence the recurrence is matrix products.  With s_t
// the running sum of u A within the chunk and h the state that enters it,
//   y_i    = sum_{j <= i} (C_i . B_j) exp(s_i - s_j) u_j x_j + exp(s_i) h C_i + D x_i
//   h'     = exp(s_last) h + sum_j exp(s_last - s_j) u_j x_j (x) B_j.
// A chunk never spans two sequences, so a sequence's values reach no other one.
//
// Matrix operands are bf16 planes: a bf16 tensor is one plane, an fp32 value three
// (v = p0 + p1 + p2 exactly: 24 bits of significand in three times 8), whose six
// products of at least 2^-16 relative weight give fp32's accuracy at 6/16 of the cost
// of the fp32 matrix instructions.  What the kernels form themselves (the decay-weighted
// tile, the state) enters a product with bf16 inputs in two planes: 2^-16 of it at most is
// lost, a 256th of what the result's own rounding loses.
#pragma once

#include <initializer_list>
#include <type_traits>

#include "moc_kernels.h"
#include "moc_rows.h"

namespace moc {
namespace scan {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kQ = 64;        // tokens of a chunk
constexpr int kTile = 64;     // channels of a head (P) and states (N) of a tile

// One operand of a 16 x 16 x 32 product: 8 consecutive contraction entries of a
// row, in NP planes.
template <int NP>
struct Frag {
  s16x8 v[NP];
};

template <int DT>
constexpr int kPlanes = DT == DT_BF16 ? 1 : 3;
// planes of an operand that a kernel formed, beside inputs of NP planes
template <int NP>
constexpr int kFormed = NP == 1 ? 2 : NP;

__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}

// c + a . b.  The products of the lower planes are summed by themselves and added
// once: each addition to c costs a rounding at c's size.
__device__ __forceinline__ f32x4 mm(const Frag<1>& a, const Frag<1>& b, f32x4 c) { return mfma(a.v[0], b.v[0], c); }
__device__ __forceinline__ f32x4 mm(const Frag<1>& a, const Frag<2>& b, f32x4 c) {
  return mfma(a.v[0], b.v[0], mfma(a.v[0], b.v[1], c));
}
__device__ __forceinline__ f32x4 mm(const Frag<2>& a, const Frag<1>& b, f32x4 c) {
  return mfma(a.v[0], b.v[0], mfma(a.v[1], b.v[0], c));
}
__device__ __forceinline__ f32x4 mm(const Frag<3>& a, const Frag<3>& b, f32x4 c) {
  f32x4 t = mfma(a.v[0], b.v[2], f32x4{0.f, 0.f, 0.f, 0.f});
  t = mfma(a.v[1], b.v[1], t);
  t = mfma(a.v[2], b.v[0], t);
  t = mfma(a.v[0], b.v[1], t);
  t = mfma(a.v[1], b.v[0], t);
  return mfma(a.v[0], b.v[0], c) + t;
}

// a0 . b0 + a1 . b1 with b in three planes, the low planes first
__device__ __forceinline__ f32x4 mm2(const Frag<1>& a0, const Frag<1>& a1, const Frag<3>& b0, const Frag<3>& b1) {
  f32x4 c = mfma(a0.v[0], b0.v[2], f32x4{0.f, 0.f, 0.f, 0.f});
  c = mfma(a1.v[0], b1.v[2], c);
  c = mfma(a0.v[0], b0.v[1], c);
  c = mfma(a1.v[0], b1.v[1], c);
  c = mfma(a0.v[0], b0.v[0], c);
  return mfma(a1.v[0], b1.v[0], c);
}
__device__ __forceinline__ f32x4 mm2(const Frag<3>& a0, const Frag<3>& a1, const Frag<3>& b0, const Frag<3>& b1) {
  return mm(a1, b1, mm(a0, b0, f32x4{0.f, 0.f, 0.f, 0.f}));
}

// Wait states between products made in a branch and the first use of their results behind
// it: the compiler has been seen to leave them out on a path around a branch's body.  Which
// places need it shows tests/test_wait_states.py, which follows every path of the assembly (as
// the code stands it finds none without these calls either; with other code around it may).
__device__ __forceinline__ void settle() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 7");
  __builtin_amdgcn_sched_barrier(0);
}

// Two fp32 rounded to bf16 in one dword, a in the low half (v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
__device__ __forceinline__ float lo_f(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_f(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// What the first of several planes of v is rounded from: values from 3.396e38 on, finite but
// an infinity in bf16, take bf16's largest, and the next plane the rest (so does an infinity:
// its second plane is the infinity).
__device__ __forceinline__ float below_top(float v) {
  constexpr float kTop = 0x1.fep127f;
  return __builtin_amdgcn_fmed3f(v, -kTop, kTop);
}

// Planes of 8 fp32 values: each plane is what the ones before it left, rounded to bf16
// (the differences are exact; those of an infinity are NaN, so what an infinity enters
// comes out as NaN where there are three planes).
template <int NP>
__device__ __forceinline__ Frag<NP> split(const float (&f)[8]) {
  u32x4 w[NP];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float a = f[2 * k], b = f[2 * k + 1];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint32_t v = p == 0 && NP > 1 ? pack2(below_top(a), below_top(b)) : pack2(a, b);
      w[p][k] = v;
      if (p + 1 < NP) a -= lo_f(v), b -= hi_f(v);
    }
  }
  Frag<NP> r;
#pragma unroll
  for (int p = 0; p < NP; ++p) r.v[p] = __builtin_bit_cast(s16x8, w[p]);
  return r;
}

// 4 fp32 values in planes `apart` elements from each other
template <int NP>
__device__ __forceinline__ void put_planes(uint16_t* q, int apart, f32x4 v) {
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    f32x4 c = v;
    if (k == 0 && NP > 1) c = f32x4{below_top(v[0]), below_top(v[1]), below_top(v[2]), below_top(v[3])};
    const u32x2 w{pack2(c[0], c[1]), pack2(c[2], c[3])};
    *reinterpret_cast<u32x2*>(q + k * apart) = w;
    if (k + 1 < NP) v -= f32x4{lo_f(w[0]), hi_f(w[0]), lo_f(w[1]), hi_f(w[1])};
  }
}

template <int NP>
__device__ __forceinline__ void join(const Frag<NP>& r, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const u32x4 top = __builtin_bit_cast(u32x4, r.v[NP - 1]);
    float a = lo_f(top[k]), b = hi_f(top[k]);
#pragma unroll
    for (int p = NP - 2; p >= 0; --p) {
      const u32x4 w = __builtin_bit_cast(u32x4, r.v[p]);
      a += lo_f(w[k]), b += hi_f(w[k]);
    }
    f[2 * k] = a, f[2 * k + 1] = b;
  }
}

// 8 elements as they lie in memory.
template <int DT>
struct Raw;
template <>
struct Raw<DT_BF16> {
  u32x4 w;
  __device__ __forceinline__ Frag<1> frag() const { return Frag<1>{{__builtin_bit_cast(s16x8, w)}}; }
  // bit 15 or 31 of a word: an exponent of all ones (an infinity or NaN)
  __device__ __forceinline__ uint32_t odd() const {
    uint32_t r = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) r |= ((w[k] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
    return r;
  }
};
template <>
struct Raw<DT_F32> {
  f32x4 lo, hi;
  __device__ __forceinline__ Frag<3> frag() const {
    const float f[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return split<3>(f);
  }
  __device__ __forceinline__ uint32_t odd() const {
    uint32_t r = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      r |= ((__float_as_uint(lo[k]) & 0x7f800000u) + 0x00800000u) |
           ((__float_as_uint(hi[k]) & 0x7f800000u) + 0x00800000u);
    return r & 0x80000000u;
  }
};

// Rows (tokens, or channels of a state) of a tensor from one of them on: element
// (row, col) lies at base + row * stride + col; rows from n on and columns from `cols` on
// read as 0 and are not written.  VEC: column counts and strides are multiples of it (8 for
// bf16, or 4; 0: any) and base is aligned to as many elements (16 bytes at most): accesses
// go through a buffer resource that ends behind row n - 1, whose range check makes the zeros
// without a branch (a lane whose columns are not there has an offset that no range reaches),
// and a lane's offset is the same for every chunk of a walk.
constexpr uint32_t kNowhere = 0x80000000u;
constexpr int64_t kMaxStride = int64_t(1) << 22;  // VEC: 64 rows stay below kNowhere

// 8 elements: all there or not (VEC 8, bf16), or two fours with a place of their own each
template <int VEC>
__device__ __forceinline__ void load8(Raw<DT_BF16>& v, __amdgpu_buffer_rsrc_t r, int lo, int hi, int s) {
  if constexpr (VEC == 8) {
    v.w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, lo, s, 0));
  } else {
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, lo, s, 0));
    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, hi, s, 0));
    v.w = u32x4{a[0], a[1], b[0], b[1]};
  }
}
template <int VEC>
__device__ __forceinline__ void load8(Raw<DT_F32>& v, __amdgpu_buffer_rsrc_t r, int lo, int hi, int s) {
  v.lo = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, lo, s, 0));
  v.hi = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, hi, s, 0));
}

template <int DT, int VEC>
struct Rows {
  static constexpr int E = DT == DT_BF16 ? 2 : 4;
  const char* base;
  int64_t stride;
  int n, cols;
  __device__ __forceinline__ Rows(const void* p, int64_t at, int64_t stride_, int n_, int cols_)
      : base(static_cast<const char*>(p) + at * E), stride(stride_), n(n_), cols(cols_) {}
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc() const {
    const int bytes = n > 0 ? ((n - 1) * static_cast<int>(stride) + cols) * E : 0;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, bytes, 0x00020000);
  }
  __device__ __forceinline__ int off(int row, int col) const {
    const uint32_t o = static_cast<uint32_t>(row * static_cast<int>(stride) + col) * E;
    return static_cast<int>(col < cols ? o : kNowhere);
  }
  // (row + more, col), `more` the same for every lane
  __device__ __forceinline__ Raw<DT> get8(int row, int col, int more = 0) const {
    Raw<DT> v;
    if constexpr (VEC != 0) {
      const int o = off(row, col), s = more * static_cast<int>(stride) * E;
      const auto r = rsrc();
      load8<VEC>(v, r, o, col + 4 < cols ? o + 4 * E : static_cast<int>(kNowhere), s);
    } else {
      row += more;
      const int have = row < n ? cols - col : 0;
      const int64_t at = row * stride + col;
      if constexpr (DT == DT_BF16) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + at;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a = 2 * k < have ? p[2 * k] : 0u, b = 2 * k + 1 < have ? p[2 * k + 1] : 0u;
          v.w[k] = a | (b << 16);
        }
      } else {
        const float* p = reinterpret_cast<const float*>(base) + at;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v.lo[k] = k < have ? p[k] : 0.f;
          v.hi[k] = 4 + k < have ? p[4 + k] : 0.f;
        }
      }
    }
    return v;
  }
  // 4 elements as fp32
  __device__ __forceinline__ f32x4 get4(int row, int col) const {
    f32x4 v;
    if constexpr (VEC != 0) {
      const int o = off(row, col);
      if constexpr (DT == DT_BF16) {
        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rsrc(), o, 0, 0));
        v = f32x4{lo_f(w[0]), hi_f(w[0]), lo_f(w[1]), hi_f(w[1])};
      } else {
        v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc(), o, 0, 0));
      }
    } else {
      const int have = row < n ? cols - col : 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = k < have ? load_any(base, DT, row * stride + col + k) : 0.f;
    }
    return v;
  }
  // (row + more, col), `more` the same for every lane
  __device__ __forceinline__ void put4(int row, int col, f32x4 v, int more = 0) const {
    if constexpr (VEC != 0) {
      const int o = off(row, col), s = more * static_cast<int>(stride) * E;
      if constexpr (DT == DT_BF16) {
        const u32x2 w{pack2(v[0], v[1]), pack2(v[2], v[3])};
        __builtin_amdgcn_raw_buffer_store_b64(w, rsrc(), o, s, 0);
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rsrc(), o, s, 0);
      }
    } else {
      row += more;
      const int have = row < n ? cols - col : 0;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < have) store_any(const_cast<char*>(base), DT, row * stride + col + k, v[k]);
    }
  }
  // 8 bf16 elements as they are, all or none of which are there
  __device__ __forceinline__ void put8(int row, int col, s16x8 v) const {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    if constexpr (VEC != 0) {
      __builtin_amdgcn_raw_buffer_store_b128(w, rsrc(), off(row, col), 0, 0);
    } else if (row < n && col < cols) {
      uint16_t* p = reinterpret_cast<uint16_t*>(const_cast<char*>(base)) + row * stride + col;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        p[2 * k] = static_cast<uint16_t>(w[k]);
        p[2 * k + 1] = static_cast<uint16_t>(w[k] >> 16);
      }
    }
  }
};

// States kept for the backward pass: [channels][kept_planes][kept_cols(N)] in the x dtype
// (fp32 as they are, for bf16 in the two planes in which they enter its products: 4 bytes a
// state in both), a row's states in the order
// in which the walks' lanes hold them: the 4 states of lane group g in the lower and the
// upper block of 16 of 32 states next to each other, so that a lane stores 8 at a time.
__host__ __device__ constexpr int64_t kept_cols(int64_t N) { return (N + 31) / 32 * 32; }
template <int DT>
constexpr int kKeptPlanes = DT == DT_BF16 ? 2 : 1;

// Rows at a place that moves by a uniform offset (a head's columns of a token, a head's rows
// of the states) under one buffer resource: `off` elements from base, row by row `stride`.
// `have`: how many of the elements asked for are there (at most 0: none).  VEC as in Rows.
template <int DT, int VEC>
struct Span {
  static constexpr int E = DT == DT_BF16 ? 2 : 4;
  const char* base;
  int stride, n;
  __device__ __forceinline__ Span(const void* p, int64_t at, int64_t stride_, int64_t n_)
      : base(static_cast<const char*>(p) + at * E), stride(static_cast<int>(stride_)), n(static_cast<int>(n_)) {}
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc() const {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, n * stride * E, 0x00020000);
  }
  __device__ __forceinline__ Raw<DT> get8(int row, int col, int have, int64_t off) const {
    Raw<DT> v;
    if constexpr (VEC != 0) {
      const int o = have > 0 ? (row * stride + col) * E : static_cast<int>(kNowhere);
      const int s = static_cast<int>(off) * E;
      load8<VEC>(v, rsrc(), o, have > 4 ? o + 4 * E : static_cast<int>(kNowhere), s);
    } else {
      if (row >= n) have = 0;
      const int64_t at = int64_t(row) * stride + col + off;
      if constexpr (DT == DT_BF16) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + at;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a = 2 * k < have ? p[2 * k] : 0u, b = 2 * k + 1 < have ? p[2 * k + 1] : 0u;
          v.w[k] = a | (b << 16);
        }
      } else {
        const float* p = reinterpret_cast<const float*>(base) + at;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v.lo[k] = k < have ? p[k] : 0.f;
          v.hi[k] = 4 + k < have ? p[4 + k] : 0.f;
        }
      }
    }
    return v;
  }
  __device__ __forceinline__ f32x4 get4(int row, int col, int have) const {
    f32x4 v;
    if constexpr (VEC != 0) {
      const int o = have > 0 ? (row * stride + col) * E : static_cast<int>(kNowhere);
      if constexpr (DT == DT_BF16) {
        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rsrc(), o, 0, 0));
        v = f32x4{lo_f(w[0]), hi_f(w[0]), lo_f(w[1]), hi_f(w[1])};
      } else {
        v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc(), o, 0, 0));
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = row < n && k < have ? load_any(base, DT, int64_t(row) * stride + col + k) : 0.f;
    }
    return v;
  }
  __device__ __forceinline__ void put4(int row, int col, int have, int64_t off, f32x4 v) const {
    if constexpr (VEC != 0) {
      const int o = have > 0 ? (row * stride + col) * E : static_cast<int>(kNowhere);
      const int s = static_cast<int>(off) * E;
      if constexpr (DT == DT_BF16) {
        const u32x2 w{pack2(v[0], v[1]), pack2(v[2], v[3])};
        __builtin_amdgcn_raw_buffer_store_b64(w, rsrc(), o, s, 0);
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rsrc(), o, s, 0);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (row < n && k < have)
          store_any(const_cast<char*>(base), DT, int64_t(row) * stride + col + k + off, v[k]);
    }
  }
};

// An LDS tile of bf16 planes, W = 64, 128 or 256 columns.  Blocks of 8 columns (16 bytes)
// of a row are permuted by an exclusive or with f(row), so that both kinds of operand
// reads meet every bank once (state_walk, which has no others, counts no conflicts; with the
// other accesses forward_walk counts 6.7 million cycles of them and backward_chunk 5.3, beside
// 3.8 and 10.9 million LDS instructions at 16384 bf16 tokens, 32 heads of 64 x 128).  A 16-byte read serves 16 lanes at a time: rows 0-3 and 12-15
// at block g with rows 4-11 at block g + 1, or the other way about (lanes 0-3, 12-15, 20-27,
// then the rest of 32), and their blocks must all differ (for W = 64, where two rows share
// the banks, those of rows of one parity).  A transposed read meets rows {0-3, 8-11} or
// {4-7, 12-15} at pairs of blocks, which f's bits but the lowest must keep apart.  With r the
// row's bits, (r2 ^ r3, r3) as f's low bits does both, r1 (and r0 for W > 64) above them.
//
// Offsets are (a lane's own) ^ (the column's part) + (the row block's part):
//   nat   row li, block g           (8 elements: column 8 g)
//   quad  row li, 4 elements        (column 4 g)
//   tr    row 8 g + L / 4, columns 4 (L % 4).. of a transposed read
template <int W>
struct Lane {
  int nat, quad, tr;
  static __device__ __forceinline__ int f(int row) {
    const int low = (((row >> 2 ^ row >> 3) & 1) << 1) | (row >> 3 & 1);
    return W == 64 ? ((row >> 1 & 1) << 2) | low : ((row & 1) << 3) | ((row >> 1 & 1) << 2) | low;
  }
  __device__ __forceinline__ Lane() {
    const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    nat = li * W + ((g ^ f(li)) << 3);
    quad = li * W + (((g >> 1) ^ f(li)) << 3) + 4 * (g & 1);
    const int row = 8 * g + (li >> 2);
    tr = row * W + ((((li & 3) >> 1) ^ f(row)) << 3) + 4 * (li & 1);
  }
  // In a loop: the compiler may not take the offsets formed from these for loop
  // invariants (it would hold all of them in registers, and spill).
  __device__ __forceinline__ void refresh() { asm volatile("" : "+v"(nat), "+v"(quad), "+v"(tr)); }
};

template <int NP, int W>
struct Tile {
  static constexpr int kPlane = 64 * W;  // elements
  static constexpr int kBytes = NP * kPlane * 2;
  uint16_t* p;
  // 8 elements of any row and column block
  __device__ __forceinline__ void put8(int row, int col, const Frag<NP>& r) const {
    uint16_t* q = p + row * W + (((col >> 3) ^ Lane<W>::f(row)) << 3);
#pragma unroll
    for (int k = 0; k < NP; ++k) *reinterpret_cast<s16x8*>(q + k * kPlane) = r.v[k];
  }
  // 8 kept states (block `col` / 8 of a row): lower and upper four
  __device__ __forceinline__ void put44(int row, int col, const Frag<NP>& r) const {
    const int c = (col & ~31) + ((col & 31) >> 1), x = Lane<W>::f(row) << 3;
    uint16_t *q = p + row * W + (c ^ x), *q2 = p + row * W + ((c + 16) ^ x);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      *reinterpret_cast<s16x4*>(q + k * kPlane) = __builtin_shufflevector(r.v[k], r.v[k], 0, 1, 2, 3);
      *reinterpret_cast<s16x4*>(q2 + k * kPlane) = __builtin_shufflevector(r.v[k], r.v[k], 4, 5, 6, 7);
    }
  }
  // row 16 rb + li, columns 32 ks + 8 g..
  __device__ __forceinline__ Frag<NP> get8(const Lane<W>& l, int rb, int ks) const {
    const uint16_t* q = p + (l.nat ^ (32 * ks)) + 16 * rb * W;
    Frag<NP> r;
#pragma unroll
    for (int k = 0; k < NP; ++k) r.v[k] = *reinterpret_cast<const s16x8*>(q + k * kPlane);
    return r;
  }
  // row 16 rb + li, columns 32 ks + 4 g.. and 32 ks + 16 + 4 g..
  __device__ __forceinline__ Frag<NP> get44(const Lane<W>& l, int rb, int ks) const {
    const uint16_t *q = p + (l.quad ^ (32 * ks)) + 16 * rb * W, *q2 = p + (l.quad ^ (32 * ks + 16)) + 16 * rb * W;
    Frag<NP> r;
#pragma unroll
    for (int k = 0; k < NP; ++k)
      r.v[k] = __builtin_shufflevector(*reinterpret_cast<const s16x4*>(q + k * kPlane),
                                       *reinterpret_cast<const s16x4*>(q2 + k * kPlane), 0, 1, 2, 3, 4, 5, 6, 7);
    return r;
  }
  // row 16 rb + li, columns 16 cb + 4 g..: 4 fp32 values split over the planes
  __device__ __forceinline__ void put4(const Lane<W>& l, int rb, int cb, f32x4 v) const {
    uint16_t* q = p + (l.quad ^ (16 * cb)) + 16 * rb * W;
    put_planes<NP>(q, kPlane, v);
  }
  __device__ __forceinline__ f32x4 get4(const Lane<W>& l, int rb, int cb) const {
    const uint16_t* q = p + (l.quad ^ (16 * cb)) + 16 * rb * W;
    f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = NP - 1; k >= 0; --k) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(q + k * kPlane);
      v += f32x4{lo_f(w[0]), hi_f(w[0]), lo_f(w[1]), hi_f(w[1])};
    }
    return v;
  }
  // one element as fp32
  __device__ __forceinline__ float at(int row, int col) const {
    const uint16_t* q = p + row * W + (((col >> 3) ^ Lane<W>::f(row)) << 3) + (col & 7);
    float v = 0.f;
#pragma unroll
    for (int k = NP - 1; k >= 0; --k) v += bf16_to_f32(q[k * kPlane]);
    return v;
  }
  // A transposed operand: entry k of lane (li, g) is element [32 ks + 8 g + k][16 cb + li].
  // Two ds_read_b64_tr_b16 a plane: lane i of a 16-lane group gets element i % 4 of the
  // 8-byte rows read by lanes i / 4 + {0, 4, 8, 12}, so lane L reads row L / 4 of four,
  // columns 4 (L % 4)..; the next four rows differ in one bit of f (two blocks).
  __device__ __forceinline__ Frag<NP> tr8(const Lane<W>& l, int ks, int cb) const {
    const int o = l.tr ^ (16 * cb);
    const uint16_t *q = p + o + 32 * ks * W, *q2 = p + (o ^ 16) + (32 * ks + 4) * W;
    Frag<NP> r;
#pragma unroll
    for (int k = 0; k < NP; ++k)
      r.v[k] = __builtin_shufflevector(tr(q + k * kPlane), tr(q2 + k * kPlane), 0, 1, 2, 3, 4, 5, 6, 7);
    return r;
  }
  static __device__ __forceinline__ s16x4 tr(const uint16_t* q) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(const_cast<uint16_t*>(q)));
  }
};

// The blocks of 16 x 16 on and below the diagonal of a 64 x 64 tile, row by row of blocks, a
// block's rows 32 bytes each: 10 KB for two planes, where a whole tile's 16 would leave room
// for two workgroups a CU in place of three.  (A 16-byte read's 16 lanes, see Lane, meet rows
// 0-3 and 12-15 of one half of a block's columns and 4-11 of the other: every bank once.)
template <int NP>
struct Lower {
  static constexpr int kPlane = 10 * 256;  // elements
  static constexpr int kBytes = NP * kPlane * 2;
  uint16_t* p;
  static __device__ __forceinline__ constexpr int block(int ib, int jb) { return (ib * (ib + 1) / 2 + jb) * 256; }
  // row 16 ib + li, columns 16 jb + 4 g..
  __device__ __forceinline__ void put4(int li, int g, int ib, int jb, f32x4 v) const {
    uint16_t* q = p + block(ib, jb) + 16 * li + 4 * g;
    put_planes<NP>(q, kPlane, v);
  }
  // row 16 ib + li, columns 32 ks + 8 g.. (2 ks <= ib; 0 right of the diagonal's block)
  __device__ __forceinline__ Frag<NP> get8(int li, int g, int ib, int ks) const {
    const uint16_t* q = p + block(ib, 2 * ks) + 16 * li + 8 * (g & 1) + 256 * (g >> 1);
    Frag<NP> r;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      u32x4 w = *reinterpret_cast<const u32x4*>(q + k * kPlane);
      if (2 * ks == ib) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = g < 2 ? w[e] : 0u;
      }
      r.v[k] = __builtin_bit_cast(s16x8, w);
    }
    return r;
  }
  // element (i, j), j <= i, as fp32
  __device__ __forceinline__ float at(int i, int j) const {
    const uint16_t* q = p + block(i >> 4, j >> 4) + 16 * (i & 15) + (j & 15);
    float v = 0.f;
#pragma unroll
    for (int k = NP - 1; k >= 0; --k) v += bf16_to_f32(q[k * kPlane]);
    return v;
  }
};

// 64 rows of a tensor on their way to an LDS tile of W columns: loads first (all in
// flight), the tile once the last chunk's readers are done.
template <int DT, int VEC, int W, int THREADS>
struct Staged {
  static constexpr int kLoads = 8 * W / THREADS;  // vectors of 8 of a thread
  Raw<DT> v[kLoads];
  __device__ __forceinline__ void load(const Rows<DT, VEC>& src) {
#pragma unroll
    for (int k = 0; k < kLoads; ++k) v[k] = src.get8(row(0), col(k), k * (THREADS / (W / 8)));
  }
  // rows 0..rows of a span at `off`, `cols` columns of them
  __device__ __forceinline__ void load(const Span<DT, VEC>& src, int rows, int cols, int64_t off) {
    constexpr int kStep = THREADS / (W / 8);
    // (without a resource's range check the span's own end is checked here, for every step)
    if (VEC == 0 && rows > src.n) rows = src.n;
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      v[k] = src.get8(row(0), col(k), row(0) + k * kStep < rows ? cols - col(k) : 0, off + int64_t(k) * kStep * src.stride);
  }
  template <int NP>
  __device__ __forceinline__ void put(const Tile<NP, W>& t) const {
#pragma unroll
    for (int k = 0; k < kLoads; ++k) t.put8(row(k), col(k), v[k].frag());
  }
  __device__ __forceinline__ uint32_t odd() const {
    uint32_t r = 0;
#pragma unroll
    for (int k = 0; k < kLoads; ++k) r |= v[k].odd();
    return r;
  }
  static __device__ __forceinline__ int row(int k) { return threadIdx.x / (W / 8) + k * (THREADS / (W / 8)); }
  static __device__ __forceinline__ int col(int) { return threadIdx.x % (W / 8) * 8; }
};

// 64 rows of kept states on their way to an LDS tile of W columns.
template <int DT, int VEC, int W, int THREADS>
struct KeptStates {
  static constexpr int PL = kKeptPlanes<DT>, NP = kFormed<kPlanes<DT>>;
  Staged<DT, VEC, W, THREADS> s[PL];
  static constexpr int kLoads = Staged<DT, VEC, W, THREADS>::kLoads;
  // `rows` rows of a span at `off`, `cols` columns of a plane's NK
  __device__ __forceinline__ void load(const Span<DT, VEC>& src, int rows, int cols, int64_t off, int NK) {
#pragma unroll
    for (int p = 0; p < PL; ++p) s[p].load(src, rows, cols, off + p * NK);
  }
  __device__ __forceinline__ Frag<NP> frag(int k) const {
    if constexpr (PL == 1) {
      return s[0].v[k].frag();
    } else {
      return Frag<2>{{s[0].v[k].frag().v[0], s[1].v[k].frag().v[0]}};
    }
  }
  __device__ __forceinline__ void get(int k, float (&f)[8]) const {
    if constexpr (PL == 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = s[0].v[k].lo[e], f[4 + e] = s[0].v[k].hi[e];
    } else {
      join(frag(k), f);
    }
  }
  __device__ __forceinline__ void put(const Tile<NP, W>& t) const {
#pragma unroll
    for (int k = 0; k < kLoads; ++k) t.put44(s[0].row(k), s[0].col(k), frag(k));
  }
};

// The factors of a chunk's decays.  For tokens of two blocks of 16, i's after j's,
//   exp(s_i - s_j) = a_i exp(start of i's block - end of j's block) b_j
// with a_i = exp(s_i - start) and b_j = exp(end - s_j): one exponential a token instead of one
// a pair (a at a block's last token is the whole block's); within a block the pair's own.
struct Decays {
  float* a;    // exp(s - its block's start)
  float* b;    // exp(its block's end - s)
  float* e;    // exp(s)
  float* f;    // exp(s_last - s)
  float* w;    // u f: a token's weight in the state behind the chunk
  float* u;
  double* s;
  static constexpr int kBytes = kQ * (6 * 4 + 8);
  __device__ __forceinline__ explicit Decays(char* p) {
    s = reinterpret_cast<double*>(p);
    a = reinterpret_cast<float*>(s + kQ);
    b = a + kQ;
    e = b + kQ;
    f = e + kQ;
    w = f + kQ;
    u = w + kQ;
  }
  // every wave: lane t with token t's u and s; wave w makes a part of them
  __device__ __forceinline__ void put(int wave, double sv, float uv) const {
    int t = threadIdx.x & 63;
    asm volatile("" : "+v"(t));  // (no address of these is kept over a walk)
    auto ex = [](double d) { return __builtin_amdgcn_exp2f(static_cast<float>(d)); };
    if (wave == 0) {
      const double before = __shfl(sv, (t & 48) > 0 ? (t & 48) - 1 : 0);
      a[t] = ex(t < 16 ? sv : sv - before);
      s[t] = sv;
    } else if (wave == 1) {
      b[t] = ex(__shfl(sv, t | 15) - sv);
    } else if (wave == 2) {
      e[t] = ex(sv);
      u[t] = uv;
    } else {
      const float fv = ex(__shfl(sv, 63) - sv);
      f[t] = fv;
      w[t] = uv * fv;
    }
  }
  // exp(start of block ib - end of block jb), jb < ib
  __device__ __forceinline__ float between(int ib, int jb) const {
    float v = 1.f;
    if (jb < 1 && ib > 1) v *= a[31];
    if (jb < 2 && ib > 2) v *= a[47];
    return v;
  }
};

// a[at + lane] for the uniform place `at` of an array (no 64-bit address a lane)
__device__ __forceinline__ double lane_of(const double* a, int64_t at, int lane) {
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<double*>(a + at), 0, kQ * 8, 0x00020000);
  return __builtin_bit_cast(double, __builtin_amdgcn_raw_buffer_load_b64(r, lane * 8, 0, 0));
}
__device__ __forceinline__ float lane_of(const float* a, int64_t at, int lane) {
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a + at), 0, kQ * 4, 0x00020000);
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, lane * 4, 0, 0));
}

// Sequences as [edge(m), edge(m + 1)), m < count: the batch's rows, or the packed axis
// cut at 0, every cu entry and n_tokens (what lies outside the cu entries is a sequence
// of its own, as in the convolutions).  cu entries are clamped to the token axis.
//
// A chunk's number is floor(edge / kQ) + m + its place in the sequence: numbers of
// one sequence are consecutive, those of two never meet (a sequence of n tokens has
// ceil(n / kQ) chunks, and floor((e + n) / kQ) + 1 >= floor(e / kQ) + ceil(n / kQ)), and
// no table has to be made on the device.  Segments (a multiple of kQ tokens) likewise.
//
// States are kept under numbers of their own, which do not grow with the sequences.  What
// enters piece k of a sequence that began without a state has the slot floor(edge / q) + k - 1
// (k >= 1; in reverse floor(edge / q) + k, k before the last): ceil(n / q) - 1 of them a
// sequence, and floor((e + n) / q) >= floor(e / q) + ceil(n / q) - 1, so that they are
// distinct and below floor(n_tokens / q).
struct Seqs {
  SeqLayout l;
  int64_t count;
  __device__ __forceinline__ int64_t edge(int64_t m) const {
    if (l.cu == nullptr) return m * l.seq_len;
    if (m == 0) return 0;
    if (m > l.n_seqs + 1) return l.n_tokens;
    const int64_t v = l.cu_at(m - 1);
    return v < 0 ? 0 : (v > l.n_tokens ? l.n_tokens : v);
  }
  __device__ __forceinline__ int64_t base(int64_t m, int64_t q) const {
    return l.cu == nullptr ? m * ((l.seq_len + q - 1) / q) : edge(m) / q + m;
  }
  // sequence and place of piece `id` (pieces of q tokens); false: no such piece
  __device__ __forceinline__ bool find(int64_t id, int64_t q, int64_t& m, int64_t& k) const {
    if (l.cu == nullptr) {
      const int64_t per = (l.seq_len + q - 1) / q;
      m = id / per;
      k = id - m * per;
      return true;
    }
    int64_t a = 0, b = count - 1;
    while (a < b) {
      const int64_t c = (a + b + 1) >> 1;
      if (base(c, q) <= id) a = c; else b = c - 1;
    }
    m = a;
    k = id - base(a, q);
    return k >= 0 && edge(a) + k * q < edge(a + 1);
  }
};
// what piece k's slot is
__device__ __forceinline__ int64_t slot_of(const Seqs& s, int64_t m, int64_t k, int64_t q, bool rev) {
  return s.edge(m) / q + k - (rev ? 0 : 1);
}
inline int64_t pieces(const Seqs& s, int64_t q) {
  return s.l.cu == nullptr ? s.count * ((s.l.seq_len + q - 1) / q) : s.l.n_tokens / q + s.count;
}

// Everything the kernels share.
struct Args {
  Scan p;
  Seqs seqs;
  int64_t chunks;   // chunk numbers
  int64_t seg;      // tokens of a segment
  float* u;         // [H][chunks][kQ] softplus(dt + bias), 0 behind a sequence's end
  double* s;        // [H][chunks][kQ] running sum of u A log2(e) within the chunk
  float* par;       // [H][2] A and D (or 0)
  int vec;          // VEC of everything that the kernels load and store
};

// Chunk `id`: false where there is none.
struct Chunk {
  int64_t m, t0, id;
  int64_t h, dh;   // places of the kept state before it and of the gradient behind it
  int n;           // tokens
  bool first, last;
};
// The same of any chunk.  A fixed-length sequence may begin and end with a state, so its chunks
// keep one each, under their own numbers.
__device__ __forceinline__ int64_t kept_at(const Args& a, int64_t m, int64_t k, int64_t id, bool rev) {
  return a.seqs.l.cu == nullptr ? id : slot_of(a.seqs, m, k, kQ, rev);
}
inline int64_t kept_states(const Args& a) { return a.seqs.l.cu == nullptr ? a.chunks : a.p.seq.n_tokens / kQ; }
__device__ __forceinline__ bool chunk_at(const Args& a, int64_t id, Chunk& c) {
  int64_t k;
  if (!a.seqs.find(id, kQ, c.m, k)) return false;
  const int64_t lo = a.seqs.edge(c.m), hi = a.seqs.edge(c.m + 1);
  c.id = id;
  c.h = kept_at(a, c.m, k, id, false);
  c.dh = kept_at(a, c.m, k, id, true);
  c.t0 = lo + k * kQ;
  c.n = static_cast<int>(hi - c.t0 < kQ ? hi - c.t0 : kQ);
  c.first = k == 0;
  c.last = c.t0 + c.n == hi;
  return true;
}

Args make_args(const Scan& p, void* prep);
void align(Args& a, std::initializer_list<const void*> of_x, std::initializer_list<const void*> others);
// f with a.vec as a constant
template <int DT, typename F>
void with_vec(const Args& a, F&& f) {
  if constexpr (DT == DT_BF16) {
    if (a.vec == 8) return f(std::integral_constant<int, 8>{});
  }
  if (a.vec == 4) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 0>{});
}
size_t prep_bytes(const Scan& p);
// tokens of a segment: see moc_scan.hip
int64_t segment(const Scan& p);
void launch_prep(const Args& a, hipStream_t st);

// Walks of the state over a sequence's chunks (moc_scan.hip).  rev == false: the state
// h from x and B; rev == true: its gradient from dy (in x's place) and C (in B's).
struct Walk {
  const void* x;        // [tokens][H][P], x_stride apart
  const void* b;        // [tokens][G][N]
  int64_t x_stride, b_stride;
  const float* start;   // [sequences][H][P][N] or null: state at the walk's start
  float* end;           // the same or null: state at its end
  float* seg_state;     // [n_tokens / seg][H][P][N]: state that enters each segment but a first one
  double* seg_decay;    // [n_tokens / seg][H]: log2 of the decay of the segment before it
  void* kept;           // [kept_states][H][P] rows of kept states or null: state before each chunk
};
size_t walk_bytes(const Args& a);   // seg_state and seg_decay
void carve_walk(const Args& a, void* workspace, Walk& w);
// segments' states, then (kept or end wanted) the walk itself
void launch_segments(const Args& a, const Walk& w, bool rev, hipStream_t st);
void launch_reverse(const Args& a, const Walk& w, hipStream_t st);

}  // namespace scan
}  // namespace moc
