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
// dh come from memory in 4 bytes a state (2 P N / kQ states a token and head: at 64 x 128
// eight times a bf16 x), for bf16 in two planes: in one they would move half as much, but each
// pair's product in dA, a sum over all tokens, would be off by 0.001 and more.
//
// 16384 bf16 tokens, 32 heads of 64 x 128: 255 us back to back for 740 MB (2.9 TB/s; 67 us more
// where the next head's loads were waited for early, by reloads of spilled addresses, by loads of
// A, C and D behind them and by moves of their registers).  One workgroup of 8 waves fits a CU
// (254 registers, 134 KB), and the phases of a head, parted by three barriers, overlap little:
// vector instructions issue for a third of the time, LDS reads take as much.
#include <type_traits>

#include "moc_scan.h"

namespace moc {
namespace scan {
namespace {

constexpr int kThreads = 256;

struct Back {
  const void* dy;       // [tokens][H][P] contiguous
  const void* h;        // [kept_states][H][P] rows of kept states: state before each chunk
  const void* dh;       // the same: gradient of the state behind each chunk
  bool has_init, has_dfin;
  void *dx, *ddt, *dB, *dC;
  float* part;          // [chunks][3 H]: dA, dD, ddt_bias
  float *dB_part, *dC_part;  // [subs][tokens][G][N] or null (one sub: dB, dC directly)
  int subs, per_sub;    // parts of a group's heads, heads of a part
};

__device__ __forceinline__ f32x4 zero4() { return f32x4{0.f, 0.f, 0.f, 0.f}; }

// v of the lane N places on in its group of 16
template <int N>
__device__ __forceinline__ float rotate(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, true));
}
template <int N>
__device__ __forceinline__ double rotate(double v) {
  const uint64_t w = __double_as_longlong(v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(w), 0x120 + N, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(w >> 32), 0x120 + N, 0xf, 0xf, true);
  return __longlong_as_double((static_cast<uint64_t>(hi) << 32) | lo);
}
// sum over lanes i % 16 (column sums of a result block)
template <typename T>
__device__ __forceinline__ T sum16(T v) {
  v += rotate<8>(v);
  v += rotate<4>(v);
  v += rotate<2>(v);
  return v + rotate<1>(v);
}
// sum over lane groups (row sums)
template <typename T>
__device__ __forceinline__ T sum_groups(T v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
template <typename T>
__device__ __forceinline__ T sum64(T v) {
  return sum_groups(sum16(v));
}

// sum of the products of two vectors' elements
template <typename Acc>
__device__ __forceinline__ Acc dot(const Raw<DT_BF16>& a, const Raw<DT_BF16>& b) {
  Acc s = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) s += lo_f(a.w[k]) * lo_f(b.w[k]) + hi_f(a.w[k]) * hi_f(b.w[k]);
  return s;
}
template <typename Acc>
__device__ __forceinline__ Acc dot(const float (&a)[8], const float (&b)[8]) {
  Acc s = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) s += static_cast<Acc>(a[k]) * b[k];
  return s;
}
template <typename Acc>
__device__ __forceinline__ Acc dot(const Raw<DT_F32>& a, const Raw<DT_F32>& b) {
  Acc s = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) s += static_cast<Acc>(a.lo[k]) * b.lo[k] + static_cast<Acc>(a.hi[k]) * b.hi[k];
  return s;
}

// LDS of backward_chunk, at most 135 KB.
template <int DT, int NT>
struct Layout {
  static constexpr int NP = kPlanes<DT>, MP = kFormed<NP>;
  // B and C whole in LDS (bf16: loads return in order, so that one of B or C behind the next
  // head's would wait for those, 296 -> 277 us at 16384 tokens, 32 heads, 64 x 128; three
  // planes leave no room)
  static constexpr bool kInLds = DT == DT_BF16;
  static constexpr int WB = 64 * NT;
  // state tiles of 64 at a time: two where B and C leave room for them, or one
  static constexpr int TW = DT == DT_BF16 && NT <= 2 ? NT : 1, W = 64 * TW;
  using Acc = typename std::conditional<DT == DT_BF16, float, double>::type;
  static constexpr int kSums = (4 + 2 + 4 + 4 + 1) * kQ;  // Acc values
  static constexpr int kBytes = 2 * Tile<NP, 64>::kBytes + Tile<MP, 64>::kBytes + 2 * Tile<MP, W>::kBytes +
                                (kInLds ? 2 * Tile<NP, WB>::kBytes : 0) + Decays::kBytes +
                                kSums * static_cast<int>(sizeof(Acc));
  static constexpr int kWaves = 2;  // a SIMD: one workgroup a CU (with more, registers spill)
};

// (the lanes' offsets in tiles of two widths: the same object where the widths are one)
template <bool SAME, typename T, typename U>
__device__ __forceinline__ decltype(auto) same_or_own(U& u) {
  if constexpr (SAME) return (u);
  else return T();
}

constexpr int kHalves = 2;
constexpr int kBack = 256 * kHalves;  // threads of backward_chunk

// Wave w: row / channel / state slice w % 4, and of the column blocks of a result (tokens
// 16 q.., 16 jb..) those of parity w / 4.  For fp32 the sums that da is formed from are
// kept in 64 bits (Acc): da is one number for a whole chunk to a large part (z, and the
// sums over the tokens behind), so that its rounding does not average out over tokens.
template <int DT, int NT, int VEC>
__global__ __launch_bounds__(kBack, (Layout<DT, NT>::kWaves)) void backward_chunk(Args a, Back b) {
  using LY = Layout<DT, NT>;
  using Acc = typename LY::Acc;
  constexpr int NP = LY::NP, MP = LY::MP, TW = LY::TW, W = LY::W, WB = LY::WB, Q = 4 / kHalves;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const Tile<NP, 64> xt{reinterpret_cast<uint16_t*>(smem)}, yt{reinterpret_cast<uint16_t*>(smem + xt.kBytes)};
  char* rest = smem + 2 * xt.kBytes;
  const Tile<MP, 64> mt{reinterpret_cast<uint16_t*>(rest)};
  rest += mt.kBytes;
  const Tile<MP, W> ht{reinterpret_cast<uint16_t*>(rest)}, dt{reinterpret_cast<uint16_t*>(rest + ht.kBytes)};
  rest += 2 * ht.kBytes;
  const Tile<NP, WB> bt{reinterpret_cast<uint16_t*>(rest)}, ct{reinterpret_cast<uint16_t*>(rest + bt.kBytes)};
  rest += LY::kInLds ? 2 * bt.kBytes : 0;
  const Decays dec(rest);
  Acc* Kp = reinterpret_cast<Acc*>(rest + Decays::kBytes);  // [4][64] column sums by row block
  Acc* Rv = Kp + 4 * kQ;                                    // [2][64] row sums by half
  Acc* qp = Rv + 2 * kQ;                                    // [4][64] q by state slice
  Acc* gp = qp + 4 * kQ;                                    // [4][64] g by channel slice
  Acc* dg = gp + 4 * kQ;                                    // [64] the diagonal
  __shared__ Acc zp[2][4 * kHalves];                        // z, <x, dy> by wave
  Lane<64> lx;
  Lane<W> lw;
  typename std::conditional<W == WB, Lane<W>&, Lane<WB>>::type lb(same_or_own<W == WB, Lane<WB>>(lw));
  const int lane = threadIdx.x & 63;
  int li = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = wid & 3, half = wid >> 2;
  const int H = static_cast<int>(a.p.H), P = static_cast<int>(a.p.P), G = static_cast<int>(a.p.G),
            N = static_cast<int>(a.p.N), NK = static_cast<int>(kept_cols(N)), NR = kKeptPlanes<DT> * NK;
  const int grp = blockIdx.y / b.subs, sub = blockIdx.y % b.subs, hpg = H / G;
  const int h_lo = grp * hpg + sub * b.per_sub;
  const int h_hi = (sub + 1) * b.per_sub < hpg ? h_lo + b.per_sub : (grp + 1) * hpg;
  Chunk c;
  if (!chunk_at(a, blockIdx.x, c)) {
    // no such chunk: its rows of the sums over chunks are 0
    for (int k = threadIdx.x; k < 3 * (h_hi - h_lo); k += kBack)
      b.part[int64_t(blockIdx.x) * 3 * H + (k % 3) * H + h_lo + k / 3] = 0.f;
    return;
  }
  const int n = c.n, ptiles = (P + kTile - 1) / kTile, ntiles = (N + 63) / 64;
  const bool use_h = !c.first || b.has_init, use_dh = !c.last || b.has_dfin;
  const int64_t gcol = int64_t(grp) * N;
  const Span<DT, VEC> brow(a.p.B, c.t0 * a.p.b_stride + gcol, a.p.b_stride, n);
  const Span<DT, VEC> crow(a.p.C, c.t0 * a.p.c_stride + gcol, a.p.c_stride, n);
  const Span<DT, VEC> xrow(a.p.x, c.t0 * a.p.x_stride, a.p.x_stride, n);
  const Span<DT, VEC> yrow(b.dy, c.t0 * H * P, int64_t(H) * P, n);
  const Span<DT, VEC> orow(b.dx, c.t0 * H * P, int64_t(H) * P, n);
  const Span<DT, VEC> hrow(b.h, c.h * H * P * NR, NR, int64_t(H) * P);
  const Span<DT, VEC> drow(b.dh, c.dh * H * P * NR, NR, int64_t(H) * P);
  auto blk = [&](int k) { return k * kHalves + half; };  // this wave's column blocks

  // the loads of a head's (and channel tile's) tensors, ahead of their use
  Staged<DT, VEC, 64, kBack> sx, sy;
  KeptStates<DT, VEC, W, kBack> sh, sd;
  double sv = 0.0;
  float uv = 0.f, rate_v = 0.f, skip_v = 0.f;
  auto width = [&](int pt) { return P - pt * kTile < kTile ? P - pt * kTile : kTile; };
  auto fetch_states = [&](int h, int pt, int nt) {
    const int64_t off = (int64_t(h) * P + pt * kTile) * NR + nt * 64;
    sh.load(hrow, use_h ? width(pt) : 0, NK - nt * 64, off, NK);
    sd.load(drow, use_dh ? width(pt) : 0, NK - nt * 64, off, NK);
  };
  // (one place in the code with no branch in it, or the compiler loads to other registers and
  // waits to move the values over; behind the last head nothing is loaded)
  auto fetch = [&](int h, int pt) {
    const bool more = h < h_hi;
    const int at = more ? h : h_lo, off = at * P + pt * kTile, w = more ? width(pt) : 0;
    sx.load(xrow, kQ, w, off);
    sy.load(yrow, kQ, w, off);
    const int64_t soff = int64_t(off) * NR;
    sh.load(hrow, use_h ? w : 0, NK, soff, NK);
    sd.load(drow, use_dh ? w : 0, NK, soff, NK);
    const int64_t tok = (int64_t(at) * a.chunks + c.id) * kQ;
    sv = lane_of(a.s, tok, lane);
    uv = lane_of(a.u, tok, lane);
    rate_v = lane_of(a.par, 2 * at, 0);
    skip_v = lane_of(a.par, 2 * at, 1);
  };
  fetch(h_lo, 0);

  // G^T blocks [j][i] of row block `wave` (above the diagonal too: no branch parts the code)
  f32x4 gm[Q], ds[Q];
#pragma unroll
  for (int k = 0; k < Q; ++k) gm[k] = ds[k] = zero4();
  if (LY::kInLds) {
    Staged<DT, VEC, WB, kBack> sb;
    sb.load(brow, kQ, N, 0);
    sb.put(bt);
    sb.load(crow, kQ, N, 0);
    sb.put(ct);
  }
#pragma unroll
  for (int ks = 0; ks < 2 * NT; ++ks) {
    const int col = 32 * ks + 8 * g;
    const Frag<NP> cf = crow.get8(16 * wave + li, col, N - col, 0).frag();
#pragma unroll
    for (int k = 0; k < Q; ++k) gm[k] = mm(brow.get8(16 * blk(k) + li, col, N - col, 0).frag(), cf, gm[k]);
  }
  // dB^T, dC^T blocks: states 64 nt + 16 wave + 4 g + r, tokens 16 blk + li
  f32x4 dBa[NT][Q], dCa[NT][Q];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < Q; ++k) dBa[nt][k] = dCa[nt][k] = zero4();

#pragma unroll 1
  for (int h = h_lo; h < h_hi; ++h) {
    const float rate = rate_v, skip = skip_v;
    Acc qa[Q], ga[Q], ka[Q][4], ra = 0, da = 0, za = 0, xy = 0;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      qa[k] = ga[k] = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) ka[k][r] = 0;
    }
#pragma unroll 1
    for (int pt = 0; pt < ptiles; ++pt) {
      lx.refresh(), lw.refresh();
      // (lane masks and addresses are formed anew: kept over the heads, they fill the registers
      // and spill, and a reload waits for every load ahead)
      asm volatile("" : "+v"(li), "+v"(g));
      const int i = 16 * wave + li, rel = i - 4 * g - 16 * half;  // this lane's row i of G, V (result column)
      if (pt > 0) __syncthreads();  // (the last tile's readers; a head's last barrier is behind them too)
#pragma unroll
      for (int k = 0; k < sx.kLoads; ++k) xy += dot<Acc>(sx.v[k], sy.v[k]);
      if (pt == 0) dec.put(wave, sv, uv);  // (both halves write the same)
      sx.put(xt);
      sy.put(yt);
      auto put_states = [&]() {
#pragma unroll
        for (int k = 0; k < sh.kLoads; ++k) {
          float hv[8], dv[8];
          sh.get(k, hv);
          sd.get(k, dv);
          za += dot<Acc>(hv, dv);
        }
        sh.put(ht);
        sd.put(dt);
      };
      if (use_h || use_dh) put_states();
      __syncthreads();
      // V^T, then W and what of it goes where
      {
        f32x4 vm[Q];
#pragma unroll
        for (int k = 0; k < Q; ++k) vm[k] = zero4();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const Frag<NP> yf = yt.get8(lx, wave, ks);
#pragma unroll
          for (int k = 0; k < Q; ++k) vm[k] = mm(xt.get8(lx, blk(k), ks), yf, vm[k]);
        }
        const double si = dec.s[i];
#pragma unroll
        for (int k = 0; k < Q; ++k) {
          const int j0 = 16 * blk(k) + 4 * g;
          const f32x4 u = *reinterpret_cast<const f32x4*>(dec.u + j0);
          f32x4 gl;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool in = rel >= 16 * kHalves * k + r, diag = rel == 16 * kHalves * k + r;
            const float L = __builtin_amdgcn_exp2f(static_cast<float>(si - dec.s[j0 + r]));
            const float gv = gm[k][r] * L, vv = vm[k][r] * (L * u[r]), wv = gv * vm[k][r];
            gl[r] = in ? gv : 0.f;
            ds[k][r] += in ? vv : 0.f;
            da += diag ? wv : 0.f;
            const float below = in && !diag ? wv : 0.f;
            ka[k][r] += below;
            ra += static_cast<Acc>(u[r]) * below;
          }
          if (pt == 0) mt.put4(lx, wave, blk(k), gl);
        }
      }
      // dx^T[p][j]: channels 64 pt + 16 wave + 4 g + r, tokens 16 blk + li; the state's part first
      f32x4 xa[Q];
#pragma unroll
      for (int k = 0; k < Q; ++k) xa[k] = zero4();
#pragma unroll
      for (int nt0 = 0; nt0 < NT; nt0 += TW) {
        if (TW < NT && nt0 >= ntiles) continue;
        if (nt0 > 0 && (use_h || use_dh)) {
          __syncthreads();  // (the last state tile's readers)
          put_states();
          __syncthreads();
        }
        if (TW < NT && nt0 + TW < ntiles) {
          fetch_states(h, pt, nt0 + TW);
        } else {
          const bool same = pt + 1 < ptiles;
          fetch(same ? h : h + 1, same ? pt + 1 : 0);
        }
        if (!use_h && !use_dh) continue;
#pragma unroll
        for (int ks = 0; ks < 2 * TW; ++ks) {
          const Frag<MP> df = dt.get8(lw, wave, ks);
#pragma unroll
          for (int k = 0; k < Q; ++k) {
            const int col = 64 * nt0 + 32 * ks + 8 * g;
            const Frag<NP> bf = LY::kInLds ? bt.get8(lb, blk(k), 2 * nt0 + ks)
                                            : brow.get8(16 * blk(k) + li, col, N - col, 0).frag();
            xa[k] = mm(df, bf, xa[k]);
          }
        }
        // states 64 nt + 16 wave + ...: h^T dy and dh^T x
#pragma unroll
        for (int tw = 0; tw < TW; ++tw) {
          const int nt = nt0 + tw, sc = 64 * nt + 16 * wave + 4 * g;
          const Frag<MP> h0 = ht.tr8(lw, 0, 4 * tw + wave), h1 = ht.tr8(lw, 1, 4 * tw + wave);
#pragma unroll
          for (int k = 0; k < Q; ++k) {
            const f32x4 v = mm(h1, yt.get8(lx, blk(k), 1), mm(h0, yt.get8(lx, blk(k), 0), zero4()));
            const f32x4 cv = LY::kInLds ? ct.get4(lb, blk(k), 4 * nt + wave)
                                        : crow.get4(16 * blk(k) + li, sc, N - sc);
            dCa[nt][k] += dec.e[16 * blk(k) + li] * v;
#pragma unroll
            for (int r = 0; r < 4; ++r) qa[k] += static_cast<Acc>(v[r]) * cv[r];
          }
          const Frag<MP> d0 = dt.tr8(lw, 0, 4 * tw + wave), d1 = dt.tr8(lw, 1, 4 * tw + wave);
#pragma unroll
          for (int k = 0; k < Q; ++k) {
            const f32x4 v = mm(d1, xt.get8(lx, blk(k), 1), mm(d0, xt.get8(lx, blk(k), 0), zero4()));
            dBa[nt][k] += dec.w[16 * blk(k) + li] * v;
          }
        }
      }
      settle();
#pragma unroll
      for (int k = 0; k < Q; ++k) {
        const f32x4 xv = xt.get4(lx, blk(k), wave);
#pragma unroll
        for (int r = 0; r < 4; ++r) ga[k] += static_cast<Acc>(xv[r]) * xa[k][r];
        xa[k] *= dec.f[16 * blk(k) + li];
      }
      __syncthreads();  // M is whole
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const Frag<NP> yf = yt.tr8(lx, ks, wave);
#pragma unroll
        for (int k = 0; k < Q; ++k) xa[k] = mm(yf, mt.tr8(lx, ks, blk(k)), xa[k]);
      }
#pragma unroll
      for (int k = 0; k < Q; ++k) {
        const int col = 16 * wave + 4 * g;
        const f32x4 v = dec.u[16 * blk(k) + li] * xa[k] + skip * yt.get4(lx, blk(k), wave);
        orow.put4(16 * blk(k) + li, col, width(pt) - col, h * P + pt * kTile, v);
      }
    }
    // the head's sums over channels and states
    asm volatile("" : "+v"(li), "+v"(g));
    const int i = 16 * wave + li;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const Acc v = sum16(ka[k][r]);
        if (li == 0) Kp[wave * kQ + 16 * blk(k) + 4 * g + r] = v;
      }
      const Acc v = sum_groups(qa[k]), v2 = sum_groups(ga[k]);
      if (g == 0) qp[wave * kQ + 16 * blk(k) + li] = v, gp[wave * kQ + 16 * blk(k) + li] = v2;
    }
    ra = sum_groups(ra);
    da = sum_groups(da);
    if (g == 0) {
      Rv[half * kQ + i] = ra;
      if (half == wave % kHalves) dg[i] = da;
    }
    za = sum64(za);
    xy = sum64(xy);
    if (lane == 0) zp[0][wid] = za, zp[1][wid] = xy;
    const float u = dec.u[lane], e = dec.e[lane], f = dec.f[lane], e_last = dec.e[kQ - 1];
    __syncthreads();  // the sums are whole, every tile and factor has been read
    if (wid == (h & 7)) {  // (each head another wave's: the others go on)
      int t = lane;
      asm volatile("" : "+v"(t));
      auto four = [&](const Acc* p) { return (p[t] + p[kQ + t]) + (p[2 * kQ + t] + p[3 * kQ + t]); };
      const Acc K = four(Kp), q = e * four(qp), gt = f * four(gp);
      Acc z = 0, xd = 0;
#pragma unroll
      for (int k = 0; k < 4 * kHalves; ++k) z += zp[0][k], xd += zp[1][k];
      // suffix sums of one part, prefix sums (before t) of the other, in 64 bits
      double suf = static_cast<double>(Rv[t] + Rv[kQ + t]) - static_cast<double>(u) * K + q;
      double pre = static_cast<double>(u) * gt;
      const double own = pre;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_down(suf, d), o2 = __shfl_up(pre, d);
        if (t + d < 64) suf += o;
        if (t >= d) pre += o2;
      }
      const double dat = suf + (pre - own) + static_cast<double>(z) * e_last;
      double du = K + dg[t] + gt + rate * dat;
      if (a.p.softplus) du *= -expm1f(-u);
      const bool real = t < n;
      if (real) store_any(b.ddt, DT, (c.t0 + t) * H + h, static_cast<float>(du));
      const double sA = sum64(real ? u * dat : 0.0), sb = sum64(real ? du : 0.0);
      if (lane == 0) {
        float* out = b.part + int64_t(blockIdx.x) * 3 * H + h;
        out[0] = static_cast<float>(sA);
        out[H] = static_cast<float>(xd);
        out[2 * H] = static_cast<float>(sb);
      }
    }
  }
  // what the chunk's own tokens give of dB and dC, summed over the heads, where M was
  const Tile<MP, 64>& st = mt;
#pragma unroll
  for (int k = 0; k < Q; ++k) st.put4(lx, wave, blk(k), ds[k]);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (nt >= ntiles) continue;
    lx.refresh();
    __syncthreads();
    sx.load(brow, kQ, N - 64 * nt, 64 * nt);
    sy.load(crow, kQ, N - 64 * nt, 64 * nt);
    sx.put(xt);
    sy.put(yt);
    __syncthreads();
    const int sc = 64 * nt + 16 * wave + 4 * g;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const Frag<NP> bf = xt.tr8(lx, ks, wave), cf = yt.tr8(lx, ks, wave);
#pragma unroll
      for (int k = 0; k < Q; ++k) {
        dCa[nt][k] = mm(bf, st.get8(lx, blk(k), ks), dCa[nt][k]);
        dBa[nt][k] = mm(cf, st.tr8(lx, ks, blk(k)), dBa[nt][k]);
      }
    }
    const int64_t at = (c.t0 * G + grp) * N, all = a.p.seq.n_tokens * int64_t(G) * N * sub;
    settle();
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      const int t = 16 * blk(k) + li;
      if (b.subs == 1) {
        Span<DT, VEC>(b.dB, at, int64_t(G) * N, n).put4(t, sc, N - sc, 0, dBa[nt][k]);
        Span<DT, VEC>(b.dC, at, int64_t(G) * N, n).put4(t, sc, N - sc, 0, dCa[nt][k]);
      } else {
        Span<DT_F32, VEC>(b.dB_part, all + at, int64_t(G) * N, n).put4(t, sc, N - sc, 0, dBa[nt][k]);
        Span<DT_F32, VEC>(b.dC_part, all + at, int64_t(G) * N, n).put4(t, sc, N - sc, 0, dCa[nt][k]);
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

// Parts of a group's heads.  A CU holds one workgroup, so that the time goes with the rounds
// of 256 of them: each takes a part's heads and, measured in heads (8 us for bf16 at 64 x
// 128, more for fp32), 1.25 (fp32: 0.75) for what is done once a workgroup.  More than one
// part also costs the launch that adds them and their way through memory.  The whole backward
// in us with 1 / 2 / 4 / 8 parts: bf16 16384 tokens, 32 heads of 64 x 128, one group 378 / 405 /
// 434 / 485 (1 is taken); 8000 tokens, 40 heads, 4 groups 266 / 312 / 362 / 397 (1); 2 x 2048, 16
// heads 142 / 101 / 81 / 94 (4); 300 tokens, 32 heads 217 / 124 / 78 / 56 (32: 48); fp32 2 x 2048,
// 16 heads 337 / 217 / 157 / 173 (4).  Costs are those of heads of 64 x 128: with small heads the
// rule can miss the best, 3 x 3000 tokens, 10 heads of 40 x 24, 2 groups by 12% (fp32 135 / 120 /
// 119 / 133, 5 parts are taken: 133) and 9% (bf16 86 / 79 / 79 / 89, 1 is taken).
int64_t subs_of(const Args& a) {
  const int64_t wgs = a.chunks * a.p.G, hpg = a.p.H / a.p.G;
  const bool bf = a.p.x_dt == DT_BF16;
  const double once = bf ? 1.25 : 0.75, launch = bf ? 0.5 : 0.3, way = (bf ? 1.8e-5 : 0.8e-5) * a.p.N;
  int64_t best = 1;
  double least = 0.0;
  for (int64_t s = 1; s <= hpg && s <= 64; ++s) {
    const int64_t per = (hpg + s - 1) / s, parts = (hpg + per - 1) / per;
    if (parts != s) continue;
    const double cost = static_cast<double>((wgs * s + 255) / 256) * (static_cast<double>(per) + once) +
                        (s > 1 ? launch + way * static_cast<double>(wgs * s) : 0.0);
    if (s == 1 || cost < least) best = s, least = cost;
  }
  return best;
}

struct Bytes {
  size_t walk, dh, part, sub;
  size_t all() const { return walk + dh + part + 2 * sub; }
};
Bytes bytes_of(const Args& a) {
  Bytes r;
  r.walk = walk_bytes(a);
  r.dh = up(size_t(kept_states(a)) * a.p.H * a.p.P * kept_cols(a.p.N) * 4);
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
  align(a, {dy, g.dx, g.dB, g.dC}, {dfin, saved, workspace, g.dinit});
  Walk w{};
  w.x = dy;
  w.b = p.C;
  w.x_stride = p.H * p.P;
  w.b_stride = p.c_stride;
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
  auto go = [&](auto DT, auto NT, auto VEC) {
    constexpr size_t lds = Layout<DT.value, NT.value>::kBytes;
    auto* k = backward_chunk<DT.value, NT.value, VEC.value>;
    if (lds > 65536)
      (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(lds));
    hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(a.chunks), static_cast<unsigned>(p.G * b.subs)), dim3(kBack),
                       static_cast<unsigned>(lds), st, a, b);
  };
  using BF = std::integral_constant<int, DT_BF16>;
  using F = std::integral_constant<int, DT_F32>;
  auto nt = [&](auto DT) {
    auto with = [&](auto NT) { with_vec<DT.value>(a, [&](auto VEC) { go(DT, NT, VEC); }); };
    if (p.N <= 64) with(std::integral_constant<int, 1>{});
    else if (p.N <= 128) with(std::integral_constant<int, 2>{});
    else with(std::integral_constant<int, 4>{});
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
