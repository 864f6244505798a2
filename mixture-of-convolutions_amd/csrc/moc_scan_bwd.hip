// Selective scan: backward (gfx950).
//
// With h the state that enters a chunk, dh the gradient of the state that leaves it,
// L_ij = exp(s_i - s_j) for j <= i (else 0), e_i = exp(s_i), f_j = exp(s_last - s_j),
// G_ij = C_i . B_j and V_ij = dy_i . x_j, one head at a time:
//   dx_j = u_j (sum_i G_ij L_ij dy_i + f_j dh B_j) + D dy_j
//   dC_i = sum_j (V L u)_ij B_j + e_i h^T dy_i            (summed over a group's heads)
//   dB_j = sum_i (V L u)_ij C_i + u_j f_j dh^T x_j        (likewise)
//   dh'  = exp(s_last) dh + sum_i e_i dy_i (x) C_i        (the walk, moc_scan.hip)
// and with W = G L V (each pair's part of du_j), K_j = sum_{i>j} W_ij,
// R_i = sum_{j<i} u_j W_ij, q_i = e_i C_i . h^T dy_i, g_j = f_j B_j . dh^T x_j and
// z = exp(s_last) <h, dh>, the gradient of a_t = u_t A is what crosses token t:
//   da_t = sum_{i>=t} (R_i - u_i K_i + q_i) + sum_{j<t} u_j g_j + z
//   du_t = K_t + W_tt + g_t + A da_t,  ddt_t = du_t sigmoid = du_t (1 - exp(-u_t)).
// R and K are sums of the same fp32 products, so that what cancels between them
// cancels to fp32's accuracy.
//
// One workgroup takes a chunk, a group and some of the group's heads: G is formed
// once for all of them, and dB, dC stay in its registers over its heads (a sum over
// heads through memory would move N fp32 values a token and head, more than x).  h and
// dh come from memory in the x dtype (2 P N / kQ elements a token and head, as many as
// x at 64 x 128): for bf16 one rounding of a matrix operand, as C and B have.
#include <type_traits>

#include "moc_scan.h"

namespace moc {
namespace scan {
namespace {

constexpr int kThreads = 256;

struct Back {
  const void* dy;       // [tokens][H][P] contiguous
  const void* h;        // [chunks][H][P][N], x dtype: state before each chunk
  const void* dh;       // the same: gradient of the state behind each chunk
  bool has_init, has_dfin;
  void *dx, *ddt, *dB, *dC;
  float* part;          // [chunks][3 H]: dA, dD, ddt_bias
  float *dB_part, *dC_part;  // [subs][tokens][G][N] or null (one sub: dB, dC directly)
  int subs, per_sub;    // parts of a group's heads, heads of a part
  bool vec_dy, vec_dx, vec_h;
};

__device__ __forceinline__ f32x4 zero4() { return f32x4{0.f, 0.f, 0.f, 0.f}; }

// sum over lanes i % 16 (column sums of a result block)
__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) v += __shfl_xor(v, m);
  return v;
}
// sum over lane groups (row sums)
__device__ __forceinline__ float sum_groups(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float sum64(float v) { return sum_groups(sum16(v)); }

template <int DT, int NT>
__global__ __launch_bounds__(kThreads, 2) void backward_chunk(Args a, Back b) {
  constexpr int NP = kPlanes<DT>;
  constexpr int kPlane = kQ * kRow, kTileBytes = NP * kPlane * 2;
  extern __shared__ char smem[];
  auto tile = [&](int k) { return Tile<NP>{reinterpret_cast<uint16_t*>(smem + k * kTileBytes), kRow, kPlane}; };
  const Tile<NP> xt = tile(0), yt = tile(1), ht = tile(2), dt = tile(3), mt = tile(4);
  double* ss = reinterpret_cast<double*>(smem + 5 * kTileBytes);
  double* scan_s = ss + kQ;
  float* us = reinterpret_cast<float*>(scan_s + kQ);
  float* Kp = us + kQ;       // [4][64] column sums by row block
  float* Rv = Kp + 4 * kQ;   // row sums
  float* dg = Rv + kQ;       // diagonal
  float* qp = dg + kQ;       // [4][64] q by state slice
  float* gp = qp + 4 * kQ;   // [4][64] g by state slice
  float* zp = gp + 4 * kQ;   // [4] z by wave, [4] <x, dy> by wave
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int H = static_cast<int>(a.p.H), P = static_cast<int>(a.p.P), G = static_cast<int>(a.p.G),
            N = static_cast<int>(a.p.N);
  const int grp = blockIdx.y / b.subs, sub = blockIdx.y % b.subs, hpg = H / G;
  const int h_lo = grp * hpg + sub * b.per_sub;
  const int h_hi = (sub + 1) * b.per_sub < hpg ? h_lo + b.per_sub : (grp + 1) * hpg;
  Chunk c;
  if (!chunk_at(a, blockIdx.x, c)) {
    // no such chunk: its rows of the sums over chunks are 0
    for (int k = threadIdx.x; k < 3 * (h_hi - h_lo); k += kThreads)
      b.part[int64_t(blockIdx.x) * 3 * H + (k % 3) * H + h_lo + k / 3] = 0.f;
    return;
  }
  const int n = c.n;
  const bool use_h = !c.first || b.has_init, use_dh = !c.last || b.has_dfin;
  const int64_t gcol = int64_t(grp) * N;
  const int i = 16 * wave + li;  // this lane's row i of G, V (result column)

  // G^T blocks [j][i] of row block `wave`
  f32x4 gm[4], ds[4];
#pragma unroll
  for (int jb = 0; jb < 4; ++jb) gm[jb] = ds[jb] = zero4();
#pragma unroll
  for (int ks = 0; ks < 2 * NT; ++ks) {
    const int col = 32 * ks + 8 * g;
    const Frag<NP> cf = load8<DT>(a.p.C, (c.t0 + i) * a.p.c_stride + gcol + col, i < n ? N - col : 0, a.vec_c);
#pragma unroll
    for (int jb = 0; jb < 4; ++jb) {
      if (jb > wave) continue;
      const int j = 16 * jb + li;
      gm[jb] = mm(load8<DT>(a.p.B, (c.t0 + j) * a.p.b_stride + gcol + col, j < n ? N - col : 0, a.vec_b), cf, gm[jb]);
    }
  }
  // dB^T, dC^T blocks: states 64 nt + 16 wave + 4 g + r, tokens 16 q + li
  f32x4 dBa[NT][4], dCa[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int q = 0; q < 4; ++q) dBa[nt][q] = dCa[nt][q] = zero4();
  const int ptiles = (P + kTile - 1) / kTile;

  for (int h = h_lo; h < h_hi; ++h) {
    const int64_t at = (int64_t(h) * a.chunks + c.id) * kQ;
    const float skip = a.p.D == nullptr ? 0.f : load_any(a.p.D, a.p.d_dt, h);
    __syncthreads();  // (the last head's readers are done)
    if (threadIdx.x < kQ) {
      ss[threadIdx.x] = a.s[at + threadIdx.x];
      us[threadIdx.x] = a.u[at + threadIdx.x];
    }
    float qa[4] = {0.f, 0.f, 0.f, 0.f}, ga[4] = {0.f, 0.f, 0.f, 0.f}, ka[4][4], ra = 0.f, da = 0.f;
#pragma unroll
    for (int jb = 0; jb < 4; ++jb)
#pragma unroll
      for (int r = 0; r < 4; ++r) ka[jb][r] = 0.f;
    float za = 0.f, xy = 0.f;
    for (int pt = 0; pt < ptiles; ++pt) {
      const int p0 = pt * kTile, cols = P - p0 < kTile ? P - p0 : kTile;
      if (pt > 0) __syncthreads();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int w = threadIdx.x + k * kThreads, row = w >> 3, col = (w & 7) * 8;
        const int valid = row < n ? cols - col : 0;
        const Frag<NP> fx = load8<DT>(a.p.x, (c.t0 + row) * a.p.x_stride + int64_t(h) * P + p0 + col, valid, a.vec_x);
        const Frag<NP> fy = load8<DT>(b.dy, ((c.t0 + row) * H + h) * P + p0 + col, valid, b.vec_dy);
        float vx[8], vy[8];
        join(fx, vx);
        join(fy, vy);
#pragma unroll
        for (int e = 0; e < 8; ++e) xy += vx[e] * vy[e];
        xt.put8(row, col, fx);
        yt.put8(row, col, fy);
      }
      __syncthreads();
      // V^T, then W and what of it goes where
      f32x4 vm[4];
#pragma unroll
      for (int jb = 0; jb < 4; ++jb) vm[jb] = zero4();
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const Frag<NP> yf = yt.get8(i, 32 * ks + 8 * g);
#pragma unroll
        for (int jb = 0; jb < 4; ++jb)
          if (jb <= wave) vm[jb] = mm(xt.get8(16 * jb + li, 32 * ks + 8 * g), yf, vm[jb]);
      }
      const double si = ss[i];
#pragma unroll
      for (int jb = 0; jb < 4; ++jb) {
        if (jb > wave) continue;
        f32x4 gl;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = 16 * jb + 4 * g + r;
          const float L = j <= i ? __builtin_amdgcn_exp2f(static_cast<float>(si - ss[j])) : 0.f;
          const float u = us[j];
          gl[r] = j <= i ? gm[jb][r] * L : 0.f;
          const float wv = j <= i ? gl[r] * vm[jb][r] : 0.f;
          ds[jb][r] += j <= i ? vm[jb][r] * (L * u) : 0.f;
          if (j == i) {
            da += wv;
          } else {
            ka[jb][r] += wv;
            ra += u * wv;
          }
        }
        if (pt == 0) mt.put4(i, 16 * jb + 4 * g, gl);
      }
      if (pt == 0 && (wave & 1) == 0) mt.put4(i, 16 * wave + 16 + 4 * g, zero4());
      __syncthreads();
      // dx^T[p][j]: channels p0 + 16 wave + 4 g + r, tokens 16 q + li
      const bool active = 16 * wave < cols;
      f32x4 x1[4], x2[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) x1[q] = x2[q] = zero4();
      if (active) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const Frag<NP> yf = yt.tr8(32 * ks, 16 * wave, lane);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (32 * ks + 31 >= 16 * q) x1[q] = mm(yf, mt.tr8(32 * ks, 16 * q, lane), x1[q]);
        }
      }
      if (use_h || use_dh) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (nt * 64 >= N) continue;
          __syncthreads();  // (the last state tile's readers)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int w = threadIdx.x + k * kThreads, row = w >> 3, col = nt * 64 + (w & 7) * 8;
            const int valid = row < cols ? N - col : 0;
            const int64_t src = ((c.id * H + h) * P + p0 + row) * N + col;
            const Frag<NP> fh = load8<DT>(b.h, src, use_h ? valid : 0, b.vec_h);
            const Frag<NP> fd = load8<DT>(b.dh, src, use_dh ? valid : 0, b.vec_h);
            float vh[8], vd[8];
            join(fh, vh);
            join(fd, vd);
#pragma unroll
            for (int e = 0; e < 8; ++e) za += vh[e] * vd[e];
            ht.put8(row, (w & 7) * 8, fh);
            dt.put8(row, (w & 7) * 8, fd);
          }
          __syncthreads();
          if (active && use_dh) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
              const int col = nt * 64 + 32 * ks + 8 * g;
              const Frag<NP> df = dt.get8(16 * wave + li, 32 * ks + 8 * g);
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int j = 16 * q + li;
                x2[q] = mm(df, load8<DT>(a.p.B, (c.t0 + j) * a.p.b_stride + gcol + col, j < n ? N - col : 0, a.vec_b),
                           x2[q]);
              }
            }
          }
          // states 64 nt + 16 wave + ...: h^T dy and dh^T x
          const int sc = nt * 64 + 16 * wave + 4 * g;
          if (nt * 64 + 16 * wave < N) {
            Frag<NP> hf[2], df[2];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
              hf[ks] = ht.tr8(32 * ks, 16 * wave, lane);
              df[ks] = dt.tr8(32 * ks, 16 * wave, lane);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int t = 16 * q + li;
              const float st = static_cast<float>(ss[t]);
              if (use_h) {
                f32x4 v = mm(hf[0], yt.get8(t, 8 * g), zero4());
                v = mm(hf[1], yt.get8(t, 32 + 8 * g), v);
                v *= __builtin_amdgcn_exp2f(st);
                dCa[nt][q] += v;
                const f32x4 cv = load4<DT>(a.p.C, (c.t0 + t) * a.p.c_stride + gcol + sc, t < n ? N - sc : 0, a.vec_c);
                qa[q] += v[0] * cv[0] + v[1] * cv[1] + v[2] * cv[2] + v[3] * cv[3];
              }
              if (use_dh) {
                f32x4 v = mm(df[0], xt.get8(t, 8 * g), zero4());
                v = mm(df[1], xt.get8(t, 32 + 8 * g), v);
                v *= __builtin_amdgcn_exp2f(static_cast<float>(ss[kQ - 1] - ss[t]));
                dBa[nt][q] += v * us[t];
                const f32x4 bv = load4<DT>(a.p.B, (c.t0 + t) * a.p.b_stride + gcol + sc, t < n ? N - sc : 0, a.vec_b);
                ga[q] += v[0] * bv[0] + v[1] * bv[1] + v[2] * bv[2] + v[3] * bv[3];
              }
            }
          }
        }
      }
      if (active && b.dx != nullptr) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int j = 16 * q + li;
          const float f = __builtin_amdgcn_exp2f(static_cast<float>(ss[kQ - 1] - ss[j]));
          f32x4 v = us[j] * (x1[q] + f * x2[q]);
          if (a.p.D != nullptr) v += skip * yt.get4(j, 16 * wave + 4 * g);
          if (j < n)
            store4<DT>(b.dx, ((c.t0 + j) * H + h) * P + p0 + 16 * wave + 4 * g, cols - 16 * wave - 4 * g, b.vec_dx, v);
        }
      }
    }
    // the head's sums over channels and states
#pragma unroll
    for (int jb = 0; jb < 4; ++jb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = sum16(ka[jb][r]);
        if (li == 0) Kp[wave * kQ + 16 * jb + 4 * g + r] = v;
      }
    ra = sum_groups(ra);
    da = sum_groups(da);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float v = sum_groups(qa[q]), v2 = sum_groups(ga[q]);
      if (g == 0) qp[wave * kQ + 16 * q + li] = v, gp[wave * kQ + 16 * q + li] = v2;
    }
    if (g == 0) Rv[i] = ra, dg[i] = da;
    za = sum64(za);
    xy = sum64(xy);
    if (lane == 0) zp[wave] = za, zp[4 + wave] = xy;
    __syncthreads();
    if (wave == 0) {
      const int t = lane;
      const float K = (Kp[t] + Kp[kQ + t]) + (Kp[2 * kQ + t] + Kp[3 * kQ + t]);
      const float q = (qp[t] + qp[kQ + t]) + (qp[2 * kQ + t] + qp[3 * kQ + t]);
      const float gt = (gp[t] + gp[kQ + t]) + (gp[2 * kQ + t] + gp[3 * kQ + t]);
      const float u = us[t];
      const float z = ((zp[0] + zp[1]) + (zp[2] + zp[3])) * __builtin_amdgcn_exp2f(static_cast<float>(ss[kQ - 1]));
      // suffix sums of one part, prefix sums (before t) of the other, in 64 bits
      double suf = static_cast<double>(Rv[t]) - static_cast<double>(u) * K + q;
      double pre = static_cast<double>(u) * gt;
      const double own = pre;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_down(suf, d), o2 = __shfl_up(pre, d);
        if (t + d < 64) suf += o;
        if (t >= d) pre += o2;
      }
      const float dat = static_cast<float>(suf + (pre - own) + z);
      const float A = load_any(a.p.A, a.p.a_dt, h);
      float du = K + dg[t] + gt + A * dat;
      if (a.p.softplus) du *= -expm1f(-u);
      const bool real = t < n;
      if (real && b.ddt != nullptr) store_any(b.ddt, DT, (c.t0 + t) * H + h, du);
      const float sA = sum64(real ? u * dat : 0.f), sb = sum64(real ? du : 0.f);
      if (lane == 0) {
        float* out = b.part + int64_t(blockIdx.x) * 3 * H + h;
        out[0] = sA;
        out[H] = (zp[4] + zp[5]) + (zp[6] + zp[7]);
        out[2 * H] = sb;
      }
    }
  }
  // what the chunk's own tokens give of dB and dC, summed over the heads
  __syncthreads();
#pragma unroll
  for (int jb = 0; jb < 4; ++jb)
    if (jb <= wave) mt.put4(i, 16 * jb + 4 * g, ds[jb]);
  if ((wave & 1) == 0) mt.put4(i, 16 * wave + 16 + 4 * g, zero4());
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (nt * 64 >= N) continue;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int w = threadIdx.x + k * kThreads, row = w >> 3, col = nt * 64 + (w & 7) * 8;
      const int valid = row < n ? N - col : 0;
      xt.put8(row, (w & 7) * 8, load8<DT>(a.p.B, (c.t0 + row) * a.p.b_stride + gcol + col, valid, a.vec_b));
      yt.put8(row, (w & 7) * 8, load8<DT>(a.p.C, (c.t0 + row) * a.p.c_stride + gcol + col, valid, a.vec_c));
    }
    __syncthreads();
    const int sc = nt * 64 + 16 * wave + 4 * g;
    if (nt * 64 + 16 * wave >= N) continue;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const Frag<NP> bf = xt.tr8(32 * ks, 16 * wave, lane), cf = yt.tr8(32 * ks, 16 * wave, lane);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        // dC_i: j <= i; dB_j: i >= j
        if (32 * ks < 16 * q + 16) dCa[nt][q] = mm(bf, mt.get8(16 * q + li, 32 * ks + 8 * g), dCa[nt][q]);
        if (32 * ks + 31 >= 16 * q) dBa[nt][q] = mm(cf, mt.tr8(32 * ks, 16 * q, lane), dBa[nt][q]);
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int t = 16 * q + li;
      if (t >= n) continue;
      const int64_t dst = ((c.t0 + t) * G + grp) * N + sc;
      if (b.subs == 1) {
        store4<DT>(b.dB, dst, N - sc, b.vec_h, dBa[nt][q]);
        store4<DT>(b.dC, dst, N - sc, b.vec_h, dCa[nt][q]);
      } else {
        const int64_t all = a.p.seq.n_tokens * int64_t(G) * N;
        store4<DT_F32>(b.dB_part, sub * all + dst, N - sc, b.vec_h, dBa[nt][q]);
        store4<DT_F32>(b.dC_part, sub * all + dst, N - sc, b.vec_h, dCa[nt][q]);
      }
    }
  }
}

// dB, dC from the parts of a group's heads, in order
__global__ __launch_bounds__(kThreads) void sum_subs(const float* __restrict__ pb, const float* __restrict__ pc,
                                                     int subs, int64_t n, void* dB, void* dC, int dt) {
  for (int64_t k = int64_t(blockIdx.x) * kThreads + threadIdx.x; k < n; k += int64_t(gridDim.x) * kThreads) {
    float vb = pb[k], vc = pc[k];
    for (int s = 1; s < subs; ++s) vb += pb[s * n + k], vc += pc[s * n + k];
    store_any(dB, dt, k, vb);
    store_any(dC, dt, k, vc);
  }
}

size_t up(size_t v) { return (v + 255) / 256 * 256; }

// Parts of a group's heads: about 1024 workgroups (four a CU) where the heads give
// them; each part adds 8 N bytes a token and group to the traffic.
int64_t subs_of(const Args& a) {
  const int64_t wgs = a.chunks * a.p.G, hpg = a.p.H / a.p.G;
  int64_t s = (1024 + wgs - 1) / wgs;
  if (s > hpg) s = hpg;
  const int64_t per = (hpg + s - 1) / s;
  return (hpg + per - 1) / per;
}

struct Bytes {
  size_t walk, dh, part, sub;
  size_t all() const { return walk + dh + part + 2 * sub; }
};
Bytes bytes_of(const Args& a) {
  Bytes r;
  r.walk = walk_bytes(a);
  r.dh = up(size_t(a.chunks) * a.p.H * a.p.P * a.p.N * (a.p.x_dt == DT_BF16 ? 2 : 4));
  r.part = up(size_t(a.chunks) * 3 * a.p.H * 4);
  const int64_t s = subs_of(a);
  r.sub = s == 1 ? 0 : up(size_t(s) * a.p.seq.n_tokens * a.p.G * a.p.N * 4);
  return r;
}

}  // namespace
}  // namespace scan

using namespace scan;

size_t scan_backward_workspace(const Scan& p) { return bytes_of(make_args(p, nullptr)).all(); }

void scan_backward(const Scan& p, const void* dy, bool has_init, const float* dfin, const void* saved,
                   const ScanGrads& g, void* workspace, hipStream_t st) {
  Args a = make_args(p, const_cast<void*>(saved));
  const Bytes n = bytes_of(a);
  char* ws = static_cast<char*>(workspace);
  a.vec_h = a.vec_h && aligned({dfin, g.dinit}, 16);
  Walk w{};
  w.x = dy;
  w.b = p.C;
  w.x_stride = p.H * p.P;
  w.b_stride = p.c_stride;
  w.vec_x = p.P % 8 == 0 && aligned({dy}, 16);
  w.vec_b = a.vec_c;
  w.start = dfin;
  w.end = g.dinit;
  w.kept = ws + n.walk;
  carve_walk(a, ws, w);
  launch_segments(a, w, true, st);
  launch_reverse(a, w, st);

  Back b{};
  b.dy = dy;
  b.h = static_cast<const char*>(saved) + prep_bytes(p);
  b.dh = w.kept;
  b.has_init = has_init;
  b.has_dfin = dfin != nullptr;
  b.dx = g.dx;
  b.ddt = g.ddt;
  b.dB = g.dB;
  b.dC = g.dC;
  b.part = reinterpret_cast<float*>(ws + n.walk + n.dh);
  b.subs = static_cast<int>(subs_of(a));
  const int64_t hpg = p.H / p.G;
  b.per_sub = static_cast<int>((hpg + b.subs - 1) / b.subs);
  b.dB_part = reinterpret_cast<float*>(ws + n.walk + n.dh + n.part);
  b.dC_part = reinterpret_cast<float*>(ws + n.walk + n.dh + n.part + n.sub);
  b.vec_dy = w.vec_x;
  b.vec_dx = p.P % 4 == 0 && aligned({g.dx}, 16);
  b.vec_h = p.N % 8 == 0 && aligned({g.dB, g.dC}, 16);
  auto go = [&](auto DT, auto NT) {
    constexpr int np = kPlanes<DT.value>;
    const size_t lds = size_t(np) * 5 * kQ * kRow * 2 + kQ * (2 * 8 + 15 * 4) + 64;
    auto* k = backward_chunk<DT.value, NT.value>;
    if (lds > 65536)
      (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(lds));
    hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(a.chunks), static_cast<unsigned>(p.G * b.subs)), dim3(kThreads),
                       static_cast<unsigned>(lds), st, a, b);
  };
  using BF = std::integral_constant<int, DT_BF16>;
  using F = std::integral_constant<int, DT_F32>;
  auto nt = [&](auto DT) {
    if (p.N <= 64) go(DT, std::integral_constant<int, 1>{});
    else if (p.N <= 128) go(DT, std::integral_constant<int, 2>{});
    else go(DT, std::integral_constant<int, 4>{});
  };
  if (p.x_dt == DT_BF16) nt(BF{});
  else nt(F{});
  if (b.subs > 1) {
    const int64_t all = p.seq.n_tokens * p.G * p.N;
    const int64_t wgs = (all + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(sum_subs, dim3(static_cast<unsigned>(wgs < 8192 ? wgs : 8192)), dim3(kThreads), 0, st,
                       b.dB_part, b.dC_part, b.subs, all, g.dB, g.dC, p.x_dt);
  }
  // [dA | dD | ddt_bias]
  launch_column_sums({b.part, a.chunks, p.H, p.H, p.H, g.dA, g.dD, g.dbias, p.a_dt, p.d_dt, p.bias_dt}, st);
}

}  // namespace moc
