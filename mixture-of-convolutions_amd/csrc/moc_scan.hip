// Selective scan: step lengths, forward, walks of the state, single tokens (gfx950).
// The mathematics and the operand planes are in moc_scan.h.
//
// The forward moves x and y once and is bound by memory at 64 channels and 128 states
// a head (5 x 64 x 128 operations beside 256 bytes a token and head), so the [P, N] state
// never leaves the registers of the waves that walk a sequence: a wave owns 16 channels
// of a head and all states (N / 16 result blocks), which makes the state's decay, its
// product with C and its update wave-private; the waves of a workgroup share the
// chunk's (C B^T o decays) tile in LDS, a quarter of its rows each.
//
// A batch of few heads and sequences would leave most CUs idle, so sequences are
// cut into segments: every segment's own state is formed first (state_walk, no output),
// a pass over segments joins them (join_segments), then every segment is walked with the
// state that enters it.
#include <type_traits>

#include "moc_scan.h"

namespace moc {
namespace scan {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// u and s of every chunk and head.  Lanes are tokens for the running sum (in 64 bits:
// s_i - s_j is formed from it, where a 32-bit sum of tens would lose the differences of
// neighbours), heads for the loads.
__global__ __launch_bounds__(kThreads) void prep_kernel(Args a) {
  __shared__ float raw[16][kQ + 1];
  Chunk c;
  if (!chunk_at(a, blockIdx.x, c)) return;
  const int h0 = blockIdx.y * 16;
  for (int k = threadIdx.x; k < 16 * kQ; k += kThreads) {
    const int t = k >> 4, h = h0 + (k & 15);
    if (t < c.n && h < a.p.H) raw[k & 15][t] = load_any(a.p.dt, a.p.x_dt, (c.t0 + t) * a.p.dt_stride + h);
  }
  __syncthreads();
  const int t = threadIdx.x & 63;
  for (int k = threadIdx.x >> 6; k < 16 && h0 + k < a.p.H; k += 4) {
    const int h = h0 + k;
    float u = 0.f;
    if (t < c.n) {
      u = raw[k][t] + (a.p.bias == nullptr ? 0.f : load_any(a.p.bias, a.p.bias_dt, h));
      if (a.p.softplus) u = fmaxf(u, 0.f) + log1pf(expf(-fabsf(u)));
    }
    double s = static_cast<double>(u) * load_any(a.p.A, a.p.a_dt, h) * 1.4426950408889634074;
    if (t >= c.n) s = 0.0;  // (also where A is not finite)
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double o = __shfl_up(s, d);
      if (t >= d) s += o;
    }
    const int64_t at = (int64_t(h) * a.chunks + c.id) * kQ + t;
    a.u[at] = u;
    a.s[at] = s;
  }
}

// ---------------------------------------------------------------------------
// rows t0.. of a [tokens][..] tensor to an LDS tile of 64 NT columns; n rows and
// `cols` columns are real, the others 0.  Returns whether a value is not finite.
template <int DT, int NT>
__device__ __forceinline__ bool stage(const Tile<kPlanes<DT>>& tile, const void* src, int64_t t0, int64_t stride,
                                      int64_t col0, int n, int cols, bool vec) {
  bool odd = false;
#pragma unroll
  for (int k = 0; k < 2 * NT; ++k) {
    const int at = threadIdx.x + k * kThreads, row = at / (8 * NT), col = (at % (8 * NT)) * 8;
    const int valid = row < n ? cols - col : 0;
    const Frag<kPlanes<DT>> f = load8<DT>(src, (t0 + row) * stride + col0 + col, valid, vec);
#pragma unroll
    for (int e = 0; e < 8; ++e) odd |= (f.v[0][e] & 0x7f80) == 0x7f80;
    tile.put8(row, col, f);
  }
  return odd;
}

// acc (n = 16 nb + 4 g + r rows, channel column) from / to a [P][N] state
template <int NB, int DT>
__device__ __forceinline__ void load_state(const void* src, int64_t at, int p, int P, int N, int g, bool vec,
                                           f32x4 (&acc)[NB]) {
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int n = 16 * nb + 4 * g;
    acc[nb] = load4<DT>(src, at + int64_t(p) * N + n, p < P ? N - n : 0, vec);
  }
}
template <int NB, int DT>
__device__ __forceinline__ void store_state(void* dst, int64_t at, int p, int P, int N, int g, bool vec,
                                            const f32x4 (&acc)[NB]) {
  if (p >= P) return;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int n = 16 * nb + 4 * g;
    store4<DT>(dst, at + int64_t(p) * N + n, N - n, vec, acc[nb]);
  }
}

// 8 products of a transposed x operand and the weights w[row0 + 8 g ..] as three planes
template <int NP>
__device__ __forceinline__ Frag<3> weighted(const Frag<NP>& x, const float* w) {
  float f[8];
  join(x, f);
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] *= w[k];
  return split<3>(f);
}

// acc = decay acc + sum over the chunk's tokens of (w x) (x) b
template <int NP, int NB>
__device__ __forceinline__ void update_state(const Tile<NP>& bt, const Frag<3> (&uf)[2], float decay, int lane,
                                             f32x4 (&acc)[NB]) {
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    f32x4 v = acc[nb] * decay;
    v = mm(bt.tr8(0, 16 * nb, lane), uf[0], v);
    acc[nb] = mm(bt.tr8(32, 16 * nb, lane), uf[1], v);
  }
}

// The state over one segment's chunks, forwards (REV false) or backwards.  LOCAL: from
// zero, for segments that another one follows, to seg_state and seg_decay; else from the
// state that enters the segment, kept before each chunk.
template <int DT, int NT, bool REV, bool LOCAL>
__global__ __launch_bounds__(kThreads) void state_walk(Args a, Walk w) {
  constexpr int NP = kPlanes<DT>, NB = 4 * NT, NS = 64 * NT + 8;
  extern __shared__ char smem[];
  const Tile<NP> bt{reinterpret_cast<uint16_t*>(smem), NS, kQ * NS};
  const Tile<NP> xt{bt.p + NP * kQ * NS, kRow, kQ * kRow};
  float* wj = reinterpret_cast<float*>(xt.p + NP * kQ * kRow);
  const int lane = threadIdx.x & 63, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int P = static_cast<int>(a.p.P), N = static_cast<int>(a.p.N);
  const int ptiles = (P + kTile - 1) / kTile;
  const int h = blockIdx.y / ptiles, p0 = (blockIdx.y % ptiles) * kTile, p = p0 + 16 * wave + (lane & 15);
  int64_t m, j;
  if (!a.seqs.find(blockIdx.x, a.seg, m, j)) return;
  const int64_t lo = a.seqs.edge(m), hi = a.seqs.edge(m + 1);
  const int64_t t0 = lo + j * a.seg, t1 = t0 + a.seg < hi ? t0 + a.seg : hi;
  const bool at_start = REV ? t1 == hi : j == 0, at_end = REV ? j == 0 : t1 == hi;
  if (LOCAL && at_end) return;
  const int64_t n_chunks = (t1 - t0 + kQ - 1) / kQ, c0 = a.seqs.base(m, kQ) + j * (a.seg / kQ);
  const int64_t state = ((LOCAL || !at_start ? int64_t(blockIdx.x) : m) * a.p.H + h) * P * N;
  const bool active = p0 + 16 * wave < P;
  f32x4 acc[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) acc[nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float* from = LOCAL ? nullptr : (at_start ? w.start : w.seg_state);
  if (from != nullptr) load_state<NB, DT_F32>(from, state, p, P, N, g, a.vec_h, acc);
  double total = 0.0;
  for (int64_t k = 0; k < n_chunks; ++k) {
    const int64_t i = REV ? n_chunks - 1 - k : k, id = c0 + i, t = t0 + i * kQ;
    const int n = static_cast<int>(t1 - t < kQ ? t1 - t : kQ);
    if (!LOCAL && w.kept != nullptr && !(k == 0 && from == nullptr))
      store_state<NB, DT>(w.kept, (id * a.p.H + h) * P * N, p, P, N, g, a.vec_h, acc);
    const int64_t at = (int64_t(h) * a.chunks + id) * kQ;
    const double last = a.s[at + kQ - 1];
    total += last;
    if (threadIdx.x < kQ) {
      const double s = a.s[at + threadIdx.x];
      wj[threadIdx.x] = REV ? __builtin_amdgcn_exp2f(static_cast<float>(s))
                            : a.u[at + threadIdx.x] * __builtin_amdgcn_exp2f(static_cast<float>(last - s));
    }
    stage<DT, 1>(xt, w.x, t, w.x_stride, int64_t(h) * P + p0, n, P - p0 < kTile ? P - p0 : kTile, w.vec_x);
    stage<DT, NT>(bt, w.b, t, w.b_stride, int64_t(h / (a.p.H / a.p.G)) * N, n, N, w.vec_b);
    __syncthreads();
    if (active) {
      const Frag<3> uf[2] = {weighted(xt.tr8(0, 16 * wave, lane), wj + 8 * g),
                             weighted(xt.tr8(32, 16 * wave, lane), wj + 32 + 8 * g)};
      update_state<NP, NB>(bt, uf, __builtin_amdgcn_exp2f(static_cast<float>(last)), lane, acc);
    }
    __syncthreads();
  }
  if (LOCAL) {
    store_state<NB, DT_F32>(w.seg_state, state, p, P, N, g, a.vec_h, acc);
    if (threadIdx.x == 0 && p0 == 0) w.seg_decay[int64_t(blockIdx.x) * a.p.H + h] = total;
  } else if (at_end && w.end != nullptr) {
    store_state<NB, DT_F32>(w.end, (m * a.p.H + h) * P * N, p, P, N, g, a.vec_h, acc);
  }
}

// seg_state: from each segment's own state to the state that enters it.
template <bool REV>
__global__ __launch_bounds__(kThreads) void join_segments(Args a, Walk w) {
  const int64_t pn = a.p.P * a.p.N, per = a.p.H * pn;
  const int64_t e = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (e >= per) return;
  const int64_t h = e / pn;
  for (int64_t m = blockIdx.y; m < a.seqs.count; m += gridDim.y) {
    const int64_t n = (a.seqs.edge(m + 1) - a.seqs.edge(m) + a.seg - 1) / a.seg;
    if (n <= 1) continue;
    const int64_t s0 = a.seqs.base(m, a.seg);
    float cur = w.start == nullptr ? 0.f : w.start[m * per + e];
    for (int64_t k = 0; k < n; ++k) {
      const int64_t id = s0 + (REV ? n - 1 - k : k);
      if (k + 1 < n) {
        const float own = w.seg_state[id * per + e];
        const float decay = __builtin_amdgcn_exp2f(static_cast<float>(w.seg_decay[id * a.p.H + h]));
        w.seg_state[id * per + e] = cur;
        cur = decay * cur + own;
      } else {
        w.seg_state[id * per + e] = cur;
      }
    }
  }
}

// ---------------------------------------------------------------------------
template <int DT, int NT>
__global__ __launch_bounds__(kThreads) void forward_walk(Args a, Walk w, void* __restrict__ y) {
  constexpr int NP = kPlanes<DT>, NB = 4 * NT, NS = 64 * NT + 8;
  constexpr bool kCInLds = DT == DT_BF16;  // (three planes of it beside B's would not fit)
  extern __shared__ char smem[];
  const Tile<NP> bt{reinterpret_cast<uint16_t*>(smem), NS, kQ * NS};
  const Tile<NP> ct{bt.p + NP * kQ * NS, NS, kQ * NS};
  const Tile<NP> xt{ct.p + (kCInLds ? NP * kQ * NS : 0), kRow, kQ * kRow};
  const Tile<NP> mt{xt.p + NP * kQ * kRow, kRow, kQ * kRow};
  double* ss = reinterpret_cast<double*>(mt.p + NP * kQ * kRow);
  float* us = reinterpret_cast<float*>(ss + kQ);
  float* wj = us + kQ;
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int P = static_cast<int>(a.p.P), N = static_cast<int>(a.p.N);
  const int ptiles = (P + kTile - 1) / kTile;
  const int h = blockIdx.y / ptiles, p0 = (blockIdx.y % ptiles) * kTile, p = p0 + 16 * wave + li;
  int64_t m, j;
  if (!a.seqs.find(blockIdx.x, a.seg, m, j)) return;
  const int64_t lo = a.seqs.edge(m), hi = a.seqs.edge(m + 1);
  const int64_t t0 = lo + j * a.seg, t1 = t0 + a.seg < hi ? t0 + a.seg : hi;
  const int64_t n_chunks = (t1 - t0 + kQ - 1) / kQ, c0 = a.seqs.base(m, kQ) + j * (a.seg / kQ);
  const bool active = p0 + 16 * wave < P;
  const int cols = P - p0 < kTile ? P - p0 : kTile;
  const int64_t group = int64_t(h / (a.p.H / a.p.G)) * N;
  const float skip = a.p.D == nullptr ? 0.f : load_any(a.p.D, a.p.d_dt, h);
  f32x4 acc[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) acc[nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float* from = j == 0 ? w.start : w.seg_state;
  if (from != nullptr)
    load_state<NB, DT_F32>(from, ((j == 0 ? m : int64_t(blockIdx.x)) * a.p.H + h) * P * N, p, P, N, g, a.vec_h, acc);
  // the block right of the diagonal that a 32-token product step reads (no wave writes it)
  if ((wave & 1) == 0) mt.put4(16 * wave + li, 16 * wave + 16 + 4 * g, f32x4{0.f, 0.f, 0.f, 0.f});
  for (int64_t k = 0; k < n_chunks; ++k) {
    const int64_t id = c0 + k, t = t0 + k * kQ;
    const int n = static_cast<int>(t1 - t < kQ ? t1 - t : kQ);
    const int64_t at = (int64_t(h) * a.chunks + id) * kQ;
    const double last = a.s[at + kQ - 1];
    if (threadIdx.x < kQ) {
      const double s = a.s[at + threadIdx.x];
      const float u = a.u[at + threadIdx.x];
      ss[threadIdx.x] = s;
      us[threadIdx.x] = u;
      wj[threadIdx.x] = u * __builtin_amdgcn_exp2f(static_cast<float>(last - s));
    }
    const bool odd = stage<DT, 1>(xt, a.p.x, t, a.p.x_stride, int64_t(h) * P + p0, n, cols, a.vec_x);
    stage<DT, NT>(bt, a.p.B, t, a.p.b_stride, group, n, N, a.vec_b);
    if (kCInLds) stage<DT, NT>(ct, a.p.C, t, a.p.c_stride, group, n, N, a.vec_c);
    const bool bad = __syncthreads_or(odd);
    // rows i = 16 wave + li of M, as M^T[j][i] blocks: 4 neighbouring j a lane
    {
      const int i = 16 * wave + li;
      f32x4 gm[4];
#pragma unroll
      for (int jb = 0; jb < 4; ++jb) gm[jb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 2 * NT; ++ks) {
        const int col = 32 * ks + 8 * g;
        const Frag<NP> cf = kCInLds ? ct.get8(i, col)
                                    : load8<DT>(a.p.C, (t + i) * a.p.c_stride + group + col, i < n ? N - col : 0,
                                                a.vec_c);
#pragma unroll
        for (int jb = 0; jb < 4; ++jb)
          if (jb <= wave) gm[jb] = mm(bt.get8(16 * jb + li, col), cf, gm[jb]);
      }
      const double si = ss[i];
#pragma unroll
      for (int jb = 0; jb < 4; ++jb) {
        if (jb > wave) continue;
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int jj = 16 * jb + 4 * g + r;
          v[r] = jj <= i ? gm[jb][r] * (__builtin_amdgcn_exp2f(static_cast<float>(si - ss[jj])) * us[jj]) : 0.f;
        }
        mt.put4(i, 16 * jb + 4 * g, v);
      }
    }
    if (w.kept != nullptr && !(k == 0 && from == nullptr))
      store_state<NB, DT>(w.kept, (id * a.p.H + h) * P * N, p, P, N, g, a.vec_h, acc);
    f32x4 ya[4];
#pragma unroll
    for (int ib = 0; ib < 4; ++ib) ya[ib] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (active) {
      // h C: the state's registers are the operand, whose entry e of lane group g is state
      // 32 ks + 16 (e / 4) + 4 g + e % 4; C's entries are read in the same order
#pragma unroll
      for (int ks = 0; ks < 2 * NT; ++ks) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = acc[2 * ks + e / 4][e % 4];
        const Frag<NP> hf = split<NP>(f);
#pragma unroll
        for (int ib = 0; ib < 4; ++ib) {
          const int i = 16 * ib + li, col = 32 * ks + 4 * g;
          Frag<NP> cf;
          if (kCInLds) {
#pragma unroll
            for (int q = 0; q < NP; ++q) {
              const uint16_t* s = ct.p + q * ct.plane + i * NS + col;
              cf.v[q] = __builtin_shufflevector(*reinterpret_cast<const s16x4*>(s),
                                                *reinterpret_cast<const s16x4*>(s + 16), 0, 1, 2, 3, 4, 5, 6, 7);
            }
          } else {
            const int64_t src = (t + i) * a.p.c_stride + group + col;
            const f32x4 c_lo = load4<DT>(a.p.C, src, i < n ? N - col : 0, a.vec_c);
            const f32x4 c_hi = load4<DT>(a.p.C, src + 16, i < n ? N - col - 16 : 0, a.vec_c);
            const float cv[8] = {c_lo[0], c_lo[1], c_lo[2], c_lo[3], c_hi[0], c_hi[1], c_hi[2], c_hi[3]};
            cf = split<NP>(cv);
          }
          ya[ib] = mm(hf, cf, ya[ib]);
        }
      }
#pragma unroll
      for (int ib = 0; ib < 4; ++ib) ya[ib] *= __builtin_amdgcn_exp2f(static_cast<float>(ss[16 * ib + li]));
    }
    __syncthreads();  // M is whole
    if (active) {
      const Frag<NP> xf[2] = {xt.tr8(0, 16 * wave, lane), xt.tr8(32, 16 * wave, lane)};
      Frag<NP> xm[2] = {xf[0], xf[1]};
      if (bad) {
        // 0 x_j of a later token's infinity or NaN would reach the rows before it: those
        // products are left out here and made one by one below
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if ((xf[ks].v[0][e] & 0x7f80) == 0x7f80)
#pragma unroll
              for (int q = 0; q < NP; ++q) xm[ks].v[q][e] = 0;
      }
#pragma unroll
      for (int ib = 0; ib < 4; ++ib) {
        const int i = 16 * ib + li;
        ya[ib] = mm(xm[0], mt.get8(i, 8 * g), ya[ib]);
        if (ib >= 2) ya[ib] = mm(xm[1], mt.get8(i, 32 + 8 * g), ya[ib]);
        const f32x4 xi = xt.get4(i, 16 * wave + 4 * g);
        if (bad) {
          for (int jj = 0; jj <= i; ++jj) {
            const f32x4 xj = xt.get4(jj, 16 * wave + 4 * g);
            float mij = 0.f;
#pragma unroll
            for (int q = 0; q < NP; ++q) mij += bf16_to_f32(mt.p[q * mt.plane + i * kRow + jj]);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if ((__float_as_uint(xj[r]) & 0x7f800000u) == 0x7f800000u) ya[ib][r] += mij * xj[r];
          }
        }
        if (a.p.D != nullptr) ya[ib] += skip * xi;
        if (i < n)
          store4<DT>(y, ((t + i) * a.p.H + h) * P + p0 + 16 * wave + 4 * g, cols - 16 * wave - 4 * g, a.vec_y, ya[ib]);
      }
      const Frag<3> uf[2] = {weighted(xf[0], wj + 8 * g), weighted(xf[1], wj + 32 + 8 * g)};
      update_state<NP, NB>(bt, uf, __builtin_amdgcn_exp2f(static_cast<float>(last)), lane, acc);
    }
    __syncthreads();  // the tiles are free
  }
  if (t1 == hi && w.end != nullptr)
    store_state<NB, DT_F32>(w.end, (m * a.p.H + h) * P * N, p, P, N, g, a.vec_h, acc);
}

// ---------------------------------------------------------------------------
// One token per sequence: reads and writes the fp32 state once (memory bound: 8 bytes a
// state beside one product each for h and y).  LPR lanes hold a channel's N states, 4
// each (or fewer, one by one, where N or an address does not allow vectors).
template <int LPR>
__global__ __launch_bounds__(kThreads) void step_kernel(Scan p, float* __restrict__ state, void* __restrict__ y,
                                                        bool vec) {
  const int64_t bh = int64_t(blockIdx.x);
  const int64_t b = bh / p.H, h = bh - b * p.H;
  const int lane = threadIdx.x % LPR, n = lane * 4;
  const int P = static_cast<int>(p.P), N = static_cast<int>(p.N);
  float u = load_any(p.dt, p.x_dt, b * p.dt_stride + h) + (p.bias == nullptr ? 0.f : load_any(p.bias, p.bias_dt, h));
  if (p.softplus) u = fmaxf(u, 0.f) + log1pf(expf(-fabsf(u)));
  const float decay = expf(u * load_any(p.A, p.a_dt, h));
  const float skip = p.D == nullptr ? 0.f : load_any(p.D, p.d_dt, h);
  const int64_t grp = h / (p.H / p.G) * N;
  float bv[4], cv[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    bv[k] = n + k < N ? u * load_any(p.B, p.x_dt, b * p.b_stride + grp + n + k) : 0.f;
    cv[k] = n + k < N ? load_any(p.C, p.x_dt, b * p.c_stride + grp + n + k) : 0.f;
  }
  for (int c0 = blockIdx.y * (kThreads / LPR); c0 < P; c0 += gridDim.y * (kThreads / LPR)) {
    const int c = c0 + threadIdx.x / LPR;
    const bool live = c < P;
    const float x = live ? load_any(p.x, p.x_dt, b * p.x_stride + h * P + c) : 0.f;
    const int64_t at = (bh * P + c) * N + n;
    f32x4 v = load4<DT_F32>(state, at, live ? N - n : 0, vec);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (n + k < N) {
        v[k] = decay * v[k] + x * bv[k];
        s += v[k] * cv[k];
      }
    }
    if (live) store4<DT_F32>(state, at, N - n, vec, v);
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) s += __shfl_xor(s, d);
    if (live && lane == 0) {
      if (p.D != nullptr) s += skip * x;
      store_any(y, p.x_dt, bh * P + c, s);
    }
  }
}

int n_tiles(int64_t N) { return N <= 64 ? 1 : (N <= 128 ? 2 : 4); }

template <typename F>
void with_types(const Scan& p, F&& f) {
  const int nt = n_tiles(p.N);
#define MOC_SCAN_CASE(DT, NT) \
  if (p.x_dt == DT && nt == NT) return f(std::integral_constant<int, DT>{}, std::integral_constant<int, NT>{});
  MOC_SCAN_CASE(DT_BF16, 1) MOC_SCAN_CASE(DT_BF16, 2) MOC_SCAN_CASE(DT_BF16, 4)
  MOC_SCAN_CASE(DT_F32, 1) MOC_SCAN_CASE(DT_F32, 2) MOC_SCAN_CASE(DT_F32, 4)
#undef MOC_SCAN_CASE
}

size_t up(size_t v) { return (v + 255) / 256 * 256; }

// A kernel whose LDS passes 64 KB says so first.
template <typename K>
void allow_lds(K* kernel, size_t bytes) {
  if (bytes > 65536)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(bytes));
}

template <bool REV, bool LOCAL>
void run_walk(const Args& a, const Walk& w, hipStream_t st) {
  with_types(a.p, [&](auto DT, auto NT) {
    constexpr int np = kPlanes<DT.value>;
    const size_t lds = size_t(np) * kQ * (64 * NT.value + 8 + kRow) * 2 + kQ * 4;
    auto* k = state_walk<DT.value, NT.value, REV, LOCAL>;
    allow_lds(k, lds);
    const dim3 grid(static_cast<unsigned>(pieces(a.seqs, a.seg)),
                    static_cast<unsigned>(a.p.H * ((a.p.P + kTile - 1) / kTile)));
    hipLaunchKernelGGL(k, grid, dim3(kThreads), static_cast<unsigned>(lds), st, a, w);
  });
}

bool segmented(const Args& a) { return a.seg < (a.seqs.l.cu == nullptr ? a.seqs.l.seq_len : a.seqs.l.n_tokens); }

}  // namespace

size_t prep_bytes(const Scan& p) {
  Args a = make_args(p, nullptr);
  const size_t n = size_t(p.H) * a.chunks * kQ;
  return up(n * 4) + up(n * 8);
}

// Segments: a walk's workgroups are heads x segments, and about 1024 of them (four a CU)
// fill the card; a segment has 256 tokens at least, as every one but the last is
// walked twice.
int64_t segment(const Scan& p, bool) {
  const int64_t n = p.seq.n_tokens, heads = p.H * ((p.P + kTile - 1) / kTile);
  const int64_t longest = p.seq.cu == nullptr ? p.seq.seq_len : n;
  const int64_t want = (1024 + heads - 1) / heads;  // segments of the whole token axis
  int64_t seg = (n + want - 1) / want;
  seg = (seg + kQ - 1) / kQ * kQ;
  if (seg < 256) seg = 256;
  const int64_t whole = (longest + kQ - 1) / kQ * kQ;
  return seg < whole ? seg : whole;
}

Args make_args(const Scan& p, void* prep) {
  Args a{};
  a.p = p;
  a.seqs.l = p.seq;
  a.seqs.count = p.seq.cu == nullptr ? p.seq.n_tokens / p.seq.seq_len : p.seq.n_seqs + 2;
  a.chunks = pieces(a.seqs, kQ);
  a.seg = segment(p, false);
  const size_t n = size_t(p.H) * a.chunks * kQ;
  a.u = static_cast<float*>(prep);
  a.s = reinterpret_cast<double*>(static_cast<char*>(prep) + up(n * 4));
  a.vec_x = p.P % 8 == 0 && p.x_stride % 8 == 0 && aligned({p.x}, 16);
  a.vec_b = p.N % 8 == 0 && p.b_stride % 8 == 0 && aligned({p.B}, 16);
  a.vec_c = p.N % 8 == 0 && p.c_stride % 8 == 0 && aligned({p.C}, 16);
  a.vec_h = p.N % 8 == 0;
  a.vec_y = p.P % 4 == 0;
  return a;
}

void launch_prep(const Args& a, hipStream_t st) {
  hipLaunchKernelGGL(prep_kernel, dim3(static_cast<unsigned>(a.chunks), static_cast<unsigned>((a.p.H + 15) / 16)),
                     dim3(kThreads), 0, st, a);
}

size_t walk_bytes(const Args& a) {
  if (!segmented(a)) return 0;
  const size_t n = size_t(pieces(a.seqs, a.seg)) * a.p.H;
  return up(n * a.p.P * a.p.N * 4) + up(n * 8);
}

void carve_walk(const Args& a, void* workspace, Walk& w) {
  if (!segmented(a)) return;
  const size_t n = size_t(pieces(a.seqs, a.seg)) * a.p.H;
  w.seg_state = static_cast<float*>(workspace);
  w.seg_decay = reinterpret_cast<double*>(static_cast<char*>(workspace) + up(n * a.p.P * a.p.N * 4));
}

void launch_segments(const Args& a, const Walk& w, bool rev, hipStream_t st) {
  if (!segmented(a)) return;
  const int64_t per = a.p.H * a.p.P * a.p.N;
  const dim3 grid(static_cast<unsigned>((per + kThreads - 1) / kThreads),
                  static_cast<unsigned>(a.seqs.count < 65535 ? a.seqs.count : 65535));
  if (rev) {
    run_walk<true, true>(a, w, st);
    hipLaunchKernelGGL(join_segments<true>, grid, dim3(kThreads), 0, st, a, w);
  } else {
    run_walk<false, true>(a, w, st);
    hipLaunchKernelGGL(join_segments<false>, grid, dim3(kThreads), 0, st, a, w);
  }
}

void launch_reverse(const Args& a, const Walk& w, hipStream_t st) { run_walk<true, false>(a, w, st); }

}  // namespace scan

using namespace scan;

size_t scan_saved_bytes(const Scan& p) {
  const Args a = make_args(p, nullptr);
  return prep_bytes(p) + size_t(a.chunks) * p.H * p.P * p.N * (p.x_dt == DT_BF16 ? 2 : 4);
}

size_t scan_forward_workspace(const Scan& p, bool saved) {
  return walk_bytes(make_args(p, nullptr)) + (saved ? 0 : prep_bytes(p));
}

void scan_forward(const Scan& p, void* y, const float* init, float* fin, void* saved, void* workspace,
                  hipStream_t st) {
  char* ws = static_cast<char*>(workspace);
  Args a = make_args(p, saved != nullptr ? saved : ws);
  a.vec_y = a.vec_y && aligned({y}, 16);
  a.vec_h = a.vec_h && aligned({init, fin}, 16);
  Walk w{};
  w.x = p.x;
  w.b = p.B;
  w.x_stride = p.x_stride;
  w.b_stride = p.b_stride;
  w.vec_x = a.vec_x;
  w.vec_b = a.vec_b;
  w.start = init;
  w.end = fin;
  w.kept = saved != nullptr ? static_cast<char*>(saved) + prep_bytes(p) : nullptr;
  carve_walk(a, saved != nullptr ? ws : ws + prep_bytes(p), w);
  launch_prep(a, st);
  launch_segments(a, w, false, st);
  with_types(p, [&](auto DT, auto NT) {
    constexpr int np = kPlanes<DT.value>;
    constexpr int wide = DT.value == DT_BF16 ? 2 : 1;  // B, and C where it is staged
    const size_t lds = size_t(np) * kQ * (wide * (64 * NT.value + 8) + 2 * kRow) * 2 + kQ * 16;
    auto* k = forward_walk<DT.value, NT.value>;
    allow_lds(k, lds);
    const dim3 grid(static_cast<unsigned>(pieces(a.seqs, a.seg)),
                    static_cast<unsigned>(p.H * ((p.P + kTile - 1) / kTile)));
    hipLaunchKernelGGL(k, grid, dim3(kThreads), static_cast<unsigned>(lds), st, a, w, y);
  });
}

void scan_update(const Scan& p, float* state, void* y, int64_t n_seqs, hipStream_t st) {
  const bool vec = p.N % 4 == 0 && aligned({state}, 16);
  int lpr = 4;
  while (lpr * 4 < p.N) lpr *= 2;
  const int64_t bh = n_seqs * p.H;
  // a head's channels over more workgroups where there are few heads
  const int64_t per = (p.P + kThreads / lpr - 1) / (kThreads / lpr);
  int64_t gy = bh >= 1024 ? 1 : (1024 + bh - 1) / bh;
  if (gy > per) gy = per;
  const dim3 grid(static_cast<unsigned>(bh), static_cast<unsigned>(gy));
  auto go = [&](auto L) {
    hipLaunchKernelGGL(step_kernel<L.value>, grid, dim3(kThreads), 0, st, p, state, y, vec);
  };
  if (lpr == 4) go(std::integral_constant<int, 4>{});
  else if (lpr == 8) go(std::integral_constant<int, 8>{});
  else if (lpr == 16) go(std::integral_constant<int, 16>{});
  else if (lpr == 32) go(std::integral_constant<int, 32>{});
  else go(std::integral_constant<int, 64>{});
}

}  // namespace moc
