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
// of the fp32 matrix instructions.
#pragma once

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
constexpr int kRow = 64 + 8;  // elements of an LDS tile's row (the pad spreads rows over banks)
constexpr float kLog2e = 1.4426950408889634f;

// One operand of a 16 x 16 x 32 product: 8 consecutive contraction entries of a
// row, in NP planes.
template <int NP>
struct Frag {
  s16x8 v[NP];
};

template <int DT>
constexpr int kPlanes = DT == DT_BF16 ? 1 : 3;

__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}

// c += a . b, small products first
__device__ __forceinline__ f32x4 mm(const Frag<1>& a, const Frag<1>& b, f32x4 c) { return mfma(a.v[0], b.v[0], c); }
__device__ __forceinline__ f32x4 mm(const Frag<1>& a, const Frag<3>& b, f32x4 c) {
  c = mfma(a.v[0], b.v[2], c);
  c = mfma(a.v[0], b.v[1], c);
  return mfma(a.v[0], b.v[0], c);
}
__device__ __forceinline__ f32x4 mm(const Frag<3>& a, const Frag<3>& b, f32x4 c) {
  c = mfma(a.v[0], b.v[2], c);
  c = mfma(a.v[1], b.v[1], c);
  c = mfma(a.v[2], b.v[0], c);
  c = mfma(a.v[0], b.v[1], c);
  c = mfma(a.v[1], b.v[0], c);
  return mfma(a.v[0], b.v[0], c);
}

// Planes of 8 fp32 values: each plane is what is left, rounded to bf16 (the
// differences are exact).
template <int NP>
__device__ __forceinline__ Frag<NP> split(const float (&f)[8]) {
  Frag<NP> r;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float rest = f[k];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint16_t b = f32_to_bf16(rest);
      r.v[p][k] = static_cast<short>(b);
      if (p + 1 < NP) {
        // (an infinity's difference with itself would be NaN in the next planes)
        const float d = rest - bf16_to_f32(b);
        rest = (__float_as_uint(f[k]) & 0x7f800000u) == 0x7f800000u ? 0.f : d;
      }
    }
  }
  return r;
}

template <int NP>
__device__ __forceinline__ void join(const Frag<NP>& r, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float v = bf16_to_f32(static_cast<uint16_t>(r.v[NP - 1][k]));
#pragma unroll
    for (int p = NP - 2; p >= 0; --p) v += bf16_to_f32(static_cast<uint16_t>(r.v[p][k]));
    f[k] = v;
  }
}

// 8 elements at p, the first `valid` of them real (the others 0); vec: p is aligned
// to 16 bytes where valid == 8.
template <int DT>
__device__ __forceinline__ Frag<kPlanes<DT>> load8(const void* base, int64_t at, int valid, bool vec) {
  if constexpr (DT == DT_BF16) {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    Frag<1> r;
    if (vec && valid >= 8) {
      r.v[0] = *reinterpret_cast<const s16x8*>(p);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) r.v[0][k] = k < valid ? static_cast<short>(p[k]) : short(0);
    }
    return r;
  } else {
    const float* p = static_cast<const float*>(base) + at;
    float f[8];
    if (vec && valid >= 8) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = a[k], f[4 + k] = b[k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = k < valid ? p[k] : 0.f;
    }
    return split<3>(f);
  }
}

// 4 elements as fp32, likewise (vec: aligned to 4 elements).
template <int DT>
__device__ __forceinline__ f32x4 load4(const void* base, int64_t at, int valid, bool vec) {
  f32x4 r;
  if (vec && valid >= 4) {
    float f[4];
    load_vec<DT, 4>(base, at, f);
    r = f32x4{f[0], f[1], f[2], f[3]};
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = k < valid ? load_any(base, DT, at + k) : 0.f;
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void store4(void* base, int64_t at, int valid, bool vec, f32x4 v) {
  if (vec && valid >= 4) {
    const float f[4] = {v[0], v[1], v[2], v[3]};
    store_vec<DT, 4>(base, at, f);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < valid) store_any(base, DT, at + k, v[k]);
  }
}

// An LDS tile of bf16 planes: rows of `stride` elements.
template <int NP>
struct Tile {
  uint16_t* p;
  int stride, plane;  // elements
  __device__ __forceinline__ void put8(int row, int col, const Frag<NP>& r) const {
#pragma unroll
    for (int k = 0; k < NP; ++k) *reinterpret_cast<s16x8*>(p + k * plane + row * stride + col) = r.v[k];
  }
  __device__ __forceinline__ Frag<NP> get8(int row, int col) const {
    Frag<NP> r;
#pragma unroll
    for (int k = 0; k < NP; ++k) r.v[k] = *reinterpret_cast<const s16x8*>(p + k * plane + row * stride + col);
    return r;
  }
  // 4 values (fp32) split over the planes
  __device__ __forceinline__ void put4(int row, int col, f32x4 v) const {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      s16x4 b;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint16_t h = f32_to_bf16(v[e]);
        b[e] = static_cast<short>(h);
        if (k + 1 < NP)
          v[e] = (__float_as_uint(v[e]) & 0x7f800000u) == 0x7f800000u ? 0.f : v[e] - bf16_to_f32(h);
      }
      *reinterpret_cast<s16x4*>(p + k * plane + row * stride + col) = b;
    }
  }
  __device__ __forceinline__ f32x4 get4(int row, int col) const {
    f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = NP - 1; k >= 0; --k) {
      const s16x4 b = *reinterpret_cast<const s16x4*>(p + k * plane + row * stride + col);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += bf16_to_f32(static_cast<uint16_t>(b[e]));
    }
    return v;
  }
  // A transposed operand: entry k of lane (i, g) (i = lane % 16, g = lane / 16) is
  // element [row0 + 8 g + k][col0 + i].  Two ds_read_b64_tr_b16 a plane: lane i of a
  // 16-lane group gets element i % 4 of the 8-byte rows read by lanes i / 4 + {0, 4,
  // 8, 12}, so lane L reads row L / 4 of four, columns 4 (L % 4)...
  __device__ __forceinline__ Frag<NP> tr8(int row0, int col0, int lane) const {
    const int L = lane & 15, at = (row0 + 8 * (lane >> 4) + (L >> 2)) * stride + col0 + 4 * (L & 3);
    Frag<NP> r;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const uint16_t* q = p + k * plane + at;
      const s16x4 a = tr(q), b = tr(q + 4 * stride);
      r.v[k] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return r;
  }
  static __device__ __forceinline__ s16x4 tr(const uint16_t* q) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(const_cast<uint16_t*>(q)));
  }
};

// Sequences as [edge(m), edge(m + 1)), m < count: the batch's rows, or the packed axis
// cut at 0, every cu entry and n_tokens (what lies outside the cu entries is a sequence
// of its own, as in the convolutions).  cu entries are clamped to the token axis.
//
// A chunk's number is floor(edge / kQ) + m + its place in the sequence: numbers of
// one sequence are consecutive, those of two never meet (a sequence of n tokens has
// ceil(n / kQ) chunks, and floor((e + n) / kQ) + 1 >= floor(e / kQ) + ceil(n / kQ)), and
// no table has to be made on the device.  Segments (a multiple of kQ tokens) likewise.
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
  bool vec_x, vec_b, vec_c, vec_h, vec_y;  // 16-byte loads of x, B, C, states, y-like
};

// Chunk `id`: false where there is none.
struct Chunk {
  int64_t m, t0, id;
  int n;           // tokens
  bool first, last;
};
__device__ __forceinline__ bool chunk_at(const Args& a, int64_t id, Chunk& c) {
  int64_t k;
  if (!a.seqs.find(id, kQ, c.m, k)) return false;
  const int64_t lo = a.seqs.edge(c.m), hi = a.seqs.edge(c.m + 1);
  c.id = id;
  c.t0 = lo + k * kQ;
  c.n = static_cast<int>(hi - c.t0 < kQ ? hi - c.t0 : kQ);
  c.first = k == 0;
  c.last = c.t0 + c.n == hi;
  return true;
}

Args make_args(const Scan& p, void* prep);
size_t prep_bytes(const Scan& p);
// tokens of a segment: see moc_scan.hip
int64_t segment(const Scan& p, bool backward);
void launch_prep(const Args& a, hipStream_t st);

// Walks of the state over a sequence's chunks (moc_scan.hip).  rev == false: the state
// h from x and B; rev == true: its gradient from dy (in x's place) and C (in B's).
struct Walk {
  const void* x;        // [tokens][H][P], x_stride apart
  const void* b;        // [tokens][G][N]
  int64_t x_stride, b_stride;
  bool vec_x, vec_b;
  const float* start;   // [sequences][H][P][N] or null: state at the walk's start
  float* end;           // the same or null: state at its end
  float* seg_state;     // [segments][H][P][N]: state at each segment's start
  double* seg_decay;    // [segments][H]: log2 of a segment's decay
  void* kept;           // [chunks][H][P][N] in the x dtype or null: state before each chunk
};
size_t walk_bytes(const Args& a);   // seg_state and seg_decay
void carve_walk(const Args& a, void* workspace, Walk& w);
// segments' states, then (kept or end wanted) the walk itself
void launch_segments(const Args& a, const Walk& w, bool rev, hipStream_t st);
void launch_reverse(const Args& a, const Walk& w, hipStream_t st);

}  // namespace scan
}  // namespace moc
