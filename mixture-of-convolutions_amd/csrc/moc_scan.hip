// Selective scan: step lengths, forward, walks of the state, single tokens (gfx950).
// The mathematics and the operand planes are in moc_scan.h.
//
// x and y are moved once (256 bytes a token and head of 64 bf16 channels, beside 5 x 64 x 128
// operations for 128 states), and the [P, N] state never leaves the registers of the waves
// that walk a sequence: a wave owns 16 channels of a head and all states (N / 16 result
// blocks), which makes the state's decay, its product with C and its update wave-private;
// the waves of a workgroup share the chunk's (C B^T o decays) tile in LDS, its blocks on and
// below the diagonal dealt out 2, 2, 3 and 3.
//
// 16384 bf16 tokens, 32 heads of 64 x 128, in 24 segments: forward_walk 89 us, 133 with the
// states kept for the backward (268 MB, which alone take memory 53); state_walk 39 (the reverse
// one, which keeps as much, 99), join 12, prep 7.  x and y alone would take memory 27 us: what
// bounds the walk without kept states is LDS (its reads fill about half of the time) and
// vector instructions (a third), which the barriers of a chunk keep apart.  An address kept
// in a register over a walk is dear: one that spills is reloaded behind the next chunk's
// loads and waits for them (138 -> 114 us without, when that was changed).
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

template <int V>
using Int = std::integral_constant<int, V>;

constexpr int kPrepHeads = 8;  // of a workgroup: two a wave

// v of the lane N below in its group of 16 (0 where there is none)
template <int N>
__device__ __forceinline__ double row_below(double v) {
  const uint64_t w = __double_as_longlong(v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(w), 0x110 + N, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(w >> 32), 0x110 + N, 0xf, 0xf, true);
  return __longlong_as_double((static_cast<uint64_t>(hi) << 32) | lo);
}

// ---------------------------------------------------------------------------
// u and s of every chunk and head.  Lanes are tokens for the running sum (in 64 bits:
// s_i - s_j is formed from it, where a 32-bit sum of tens would lose the differences of
// neighbours), heads for the loads.
__global__ __launch_bounds__(kThreads) void prep_kernel(Args a) {
  __shared__ float raw[kPrepHeads][kQ + 1];
  const int h0 = blockIdx.y * kPrepHeads;
  if (blockIdx.x == 0 && threadIdx.x < kPrepHeads && h0 + threadIdx.x < a.p.H) {
    const int64_t h = h0 + threadIdx.x;
    a.par[2 * h] = load_any(a.p.A, a.p.a_dt, h);
    a.par[2 * h + 1] = a.p.D == nullptr ? 0.f : load_any(a.p.D, a.p.d_dt, h);
  }
  Chunk c;
  if (!chunk_at(a, blockIdx.x, c)) return;
  for (int k = threadIdx.x; k < kPrepHeads * kQ; k += kThreads) {
    const int t = k / kPrepHeads, q = k % kPrepHeads;
    if (t < c.n && h0 + q < a.p.H) raw[q][t] = load_any(a.p.dt, a.p.x_dt, (c.t0 + t) * a.p.dt_stride + h0 + q);
  }
  __syncthreads();
  const int t = threadIdx.x & 63;
  for (int k = threadIdx.x >> 6; k < kPrepHeads && h0 + k < a.p.H; k += 4) {
    const int h = h0 + k;
    float u = 0.f;
    if (t < c.n) {
      u = raw[k][t] + (a.p.bias == nullptr ? 0.f : load_any(a.p.bias, a.p.bias_dt, h));
      if (a.p.softplus) u = fmaxf(u, 0.f) + log1pf(expf(-fabsf(u)));
    }
    double s = static_cast<double>(u) * load_any(a.p.A, a.p.a_dt, h) * 1.4426950408889634074;
    if (t >= c.n) s = 0.0;  // (also where A is not finite)
    // running sum: within groups of 16 lanes by row operations, then the groups before
    s += row_below<1>(s);
    s += row_below<2>(s);
    s += row_below<4>(s);
    s += row_below<8>(s);
    const double e0 = __shfl(s, 15), e1 = __shfl(s, 31), e2 = __shfl(s, 47);
    const int g = t >> 4;
    s += g == 0 ? 0.0 : (g == 1 ? e0 : (g == 2 ? e0 + e1 : (e0 + e1) + e2));
    const int64_t at = (int64_t(h) * a.chunks + c.id) * kQ + t;
    a.u[at] = u;
    a.s[at] = s;
  }
}

// ---------------------------------------------------------------------------
// acc: states 16 nb + 4 g + r of one channel, from / to a [P][N] state's rows
template <int NB, int DT, int VEC>
__device__ __forceinline__ void load_state(const Rows<DT, VEC>& src, int row, f32x4 (&acc)[NB]) {
  const int n0 = 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) acc[nb] = src.get4(row, 16 * nb + n0);
}
template <int NB, int DT, int VEC>
__device__ __forceinline__ void store_state(const Rows<DT, VEC>& dst, int row, const f32x4 (&acc)[NB]) {
  int n0 = 4 * ((threadIdx.x & 63) >> 4);
  // (the blocks' offsets are formed here each time: kept over a walk, they push others to
  // memory, whose reloads wait for every load ahead)
  asm volatile("" : "+v"(n0));
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) dst.put4(row, 16 * nb + n0, acc[nb]);
}

// The kept states of one head's channels from p0 on, `cols` of them, at place `at`.
template <int DT, int VEC>
__device__ __forceinline__ Rows<DT, VEC> kept_rows(const Args& a, void* kept, int64_t at, int h, int p0, int cols, int NK) {
  const int row = kKeptPlanes<DT> * NK;
  return Rows<DT, VEC>(kept, ((at * a.p.H + h) * a.p.P + p0) * row, row, cols, row);
}
// acc to a row of them
template <int NB, int DT, int VEC>
__device__ __forceinline__ void keep_state(const Rows<DT, VEC>& dst, int row, int NK, const f32x4 (&acc)[NB]) {
  int g8 = 8 * ((threadIdx.x & 63) >> 4);
  asm volatile("" : "+v"(g8));
#pragma unroll
  for (int nb = 0; nb < NB; nb += 2) {
    const int col = 16 * nb + g8;
    if constexpr (DT == DT_BF16) {
      const float f[8] = {acc[nb][0],     acc[nb][1],     acc[nb][2],     acc[nb][3],
                          acc[nb + 1][0], acc[nb + 1][1], acc[nb + 1][2], acc[nb + 1][3]};
      const Frag<2> v = split<2>(f);
#pragma unroll
      for (int p = 0; p < 2; ++p)
        if (16 * nb < NK) dst.put8(row, col + p * NK, v.v[p]);
    } else {
      dst.put4(row, col, acc[nb]);
      dst.put4(row, col + 4, acc[nb + 1]);
    }
  }
}

// 8 products of a transposed x operand and the tokens' weights w[0..8) as three planes
template <int NP>
__device__ __forceinline__ Frag<3> weighted(const Frag<NP>& x, const float* w) {
  float f[8];
  join(x, f);
  const f32x4 lo = *reinterpret_cast<const f32x4*>(w), hi = *reinterpret_cast<const f32x4*>(w + 4);
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] *= lo[k], f[4 + k] *= hi[k];
  return split<3>(f);
}

// acc = decay acc + sum over the chunk's tokens of (w x) (x) b, the sum by itself first:
// the state's own rounding is one a chunk, not one a product step
template <int NP, int W, int NB>
__device__ __forceinline__ void update_state(const Tile<NP, W>& bt, const Lane<W>& l, const Frag<3> (&uf)[2],
                                             float decay, f32x4 (&acc)[NB]) {
  // one block's operands ahead of its products, no more: left to itself the compiler reads
  // every block's first and spills them
  Frag<NP> b0 = bt.tr8(l, 0, 0), b1 = bt.tr8(l, 1, 0);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const Frag<NP> c0 = b0, c1 = b1;
    if (nb + 1 < NB) b0 = bt.tr8(l, 0, nb + 1), b1 = bt.tr8(l, 1, nb + 1);
    acc[nb] = acc[nb] * decay + mm2(c0, c1, uf[0], uf[1]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The segment of a walk's workgroup.
struct Segment {
  int64_t m, t0, c0;   // sequence, first token, first chunk
  int64_t kept;        // place of its first chunk's kept state (in reverse: gradient)
  int64_t enters;      // slot of the state that enters it (in reverse: from behind)
  int n, chunks;       // tokens, chunks
  bool first, last;    // of its sequence
};
template <bool REV>
__device__ __forceinline__ bool segment_at(const Args& a, int64_t id, Segment& s) {
  int64_t j;
  if (!a.seqs.find(id, a.seg, s.m, j)) return false;
  const int64_t lo = a.seqs.edge(s.m), hi = a.seqs.edge(s.m + 1);
  s.t0 = lo + j * a.seg;
  s.n = static_cast<int>(hi - s.t0 < a.seg ? hi - s.t0 : a.seg);
  s.chunks = (s.n + kQ - 1) / kQ;
  const int64_t k = j * (a.seg / kQ);
  s.c0 = a.seqs.base(s.m, kQ) + k;
  s.kept = kept_at(a, s.m, k, s.c0, REV);
  s.enters = slot_of(a.seqs, s.m, j, a.seg, REV);
  s.first = j == 0;
  s.last = s.t0 + s.n == hi;
  return true;
}

// Workgroups of 256 threads (waves a SIMD) that `lds` bytes each leave room for on a CU, at
// most `most`: the registers are bounded by what that many waves can have.
constexpr int waves_for(int lds, int most) { return 160 * 1024 / lds < most ? 160 * 1024 / lds : most; }

template <int DT, int NT>
constexpr int kWalkLds = kPlanes<DT> * kQ * (64 * NT + 64) * 2 + kQ * 4;
// (B, and C where it is staged)
template <int DT, int NT>
constexpr int kForwardLds =
    kPlanes<DT> * kQ * ((DT == DT_BF16 ? 2 : 1) * 64 * NT + 64) * 2 + Lower<kFormed<kPlanes<DT>>>::kBytes +
    Decays::kBytes + 16;

// The state over one segment's chunks, forwards (REV false) or backwards.  LOCAL: from
// zero, for segments that another one follows, to that one's seg_state and seg_decay; else from
// the state that enters the segment, kept before each chunk.
template <int DT, int NT, int VEC, bool REV, bool LOCAL>
__global__ __launch_bounds__(kThreads, waves_for(kWalkLds<DT, NT>, NT == 1 ? 4 : (NT == 2 ? 3 : 2))) void state_walk(Args a, Walk w) {
  constexpr int NP = kPlanes<DT>, NB = 4 * NT, W = 64 * NT;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const Tile<NP, W> bt{reinterpret_cast<uint16_t*>(smem)};
  const Tile<NP, 64> xt{reinterpret_cast<uint16_t*>(smem + bt.kBytes)};
  float* wj = reinterpret_cast<float*>(smem + bt.kBytes + xt.kBytes);
  Lane<W> lw;
  Lane<64> lx;
  const int lane = threadIdx.x & 63, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int P = static_cast<int>(a.p.P), N = static_cast<int>(a.p.N), NK = static_cast<int>(kept_cols(N));
  const int ptiles = (P + kTile - 1) / kTile;
  const int h = blockIdx.y / ptiles, p0 = (blockIdx.y % ptiles) * kTile, cols = P - p0 < kTile ? P - p0 : kTile;
  Segment s;
  if (!segment_at<REV>(a, blockIdx.x, s)) return;
  const bool at_start = REV ? s.last : s.first, at_end = REV ? s.first : s.last;
  if (LOCAL && at_end) return;
  const int row = 16 * wave + (lane & 15);  // this lane's channel, from p0 on
  const bool active = 16 * wave < cols;
  auto state = [&](const void* p, int64_t at) {
    return Rows<DT_F32, VEC>(p, ((at * a.p.H + h) * P + p0) * N, N, cols, N);
  };
  f32x4 acc[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) acc[nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float* from = LOCAL ? nullptr : (at_start ? w.start : w.seg_state);
  if (from != nullptr) load_state<NB>(state(from, at_start ? s.m : s.enters), row, acc);
  const int64_t at = (int64_t(h) * a.chunks + s.c0) * kQ;
  const int64_t xcol = int64_t(h) * P + p0, bcol = int64_t(h / (a.p.H / a.p.G)) * N;
  Staged<DT, VEC, 64, kThreads> sx;
  Staged<DT, VEC, W, kThreads> sb;
  double sv;
  float uv = 0.f;
  auto fetch = [&](int i) {
    const int64_t t = s.t0 + int64_t(i) * kQ;
    const int n = s.n - i * kQ < kQ ? s.n - i * kQ : kQ;
    sx.load(Rows<DT, VEC>(w.x, t * w.x_stride + xcol, w.x_stride, n, cols));
    sb.load(Rows<DT, VEC>(w.b, t * w.b_stride + bcol, w.b_stride, n, N));
    sv = lane_of(a.s, at + i * kQ, lane);
    if (!REV) uv = lane_of(a.u, at + i * kQ, lane);
  };
  double total = 0.0;
  fetch(REV ? s.chunks - 1 : 0);
#pragma unroll 1
  for (int k = 0; k < s.chunks; ++k) {
    lw.refresh(), lx.refresh();
    const int i = REV ? s.chunks - 1 - k : k;
    if (!LOCAL && w.kept != nullptr && !(k == 0 && from == nullptr))
      keep_state<NB>(kept_rows<DT, VEC>(a, w.kept, s.kept + i, h, p0, cols, NK), row, NK, acc);
    sx.put(xt);
    sb.put(bt);
    const double last = __shfl(sv, 63);
    total += last;
    const float decay = __builtin_amdgcn_exp2f(static_cast<float>(last));
    if (wave == 0)
      wj[lane] = REV ? __builtin_amdgcn_exp2f(static_cast<float>(sv))
                     : uv * __builtin_amdgcn_exp2f(static_cast<float>(last - sv));
    __syncthreads();
    if (k + 1 < s.chunks) fetch(REV ? i - 1 : i + 1);
    if (active) {
      const Frag<3> uf[2] = {weighted(xt.tr8(lx, 0, wave), wj + 8 * g),
                             weighted(xt.tr8(lx, 1, wave), wj + 32 + 8 * g)};
      update_state(bt, lw, uf, decay, acc);
    }
    __syncthreads();
  }
  if (LOCAL) {
    const int64_t next = REV ? s.enters - 1 : s.enters + 1;
    store_state<NB>(state(w.seg_state, next), row, acc);
    if (threadIdx.x == 0 && p0 == 0) w.seg_decay[next * a.p.H + h] = total;
  } else if (at_end && w.end != nullptr) {
    store_state<NB>(state(w.end, s.m), row, acc);
  }
}

// seg_state: from what the segment before leaves by itself to the state that enters, one
// element a thread.  Bound by memory (24 segments of 32 heads, 64 x 128: 50 MB in 13 us).
template <bool REV>
__global__ __launch_bounds__(kThreads) void join_segments(Args a, Walk w) {
  const int64_t pn = a.p.P * a.p.N, per = a.p.H * pn;
  const int64_t e = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (e >= per) return;
  const int64_t h = e / pn;
  for (int64_t m = blockIdx.y; m < a.seqs.count; m += gridDim.y) {
    const int64_t n = (a.seqs.edge(m + 1) - a.seqs.edge(m) + a.seg - 1) / a.seg;
    if (n <= 1) continue;
    const int64_t s0 = a.seqs.edge(m) / a.seg;
    float cur = w.start == nullptr ? 0.f : w.start[m * per + e];
    for (int64_t k = 0; k + 1 < n; ++k) {
      const int64_t at = s0 + (REV ? n - 2 - k : k);
      const float decay = __builtin_amdgcn_exp2f(static_cast<float>(w.seg_decay[at * a.p.H + h]));
      cur = decay * cur + w.seg_state[at * per + e];
      w.seg_state[at * per + e] = cur;
    }
  }
}

// ---------------------------------------------------------------------------
// KEEP: w.kept is filled (a form of its own: the others would spill more for code they skip)
template <int DT, int NT, int VEC, bool KEEP>
__global__ __launch_bounds__(kThreads, waves_for(kForwardLds<DT, NT>, 3)) void forward_walk(Args a, Walk w, void* y) {
  constexpr int NP = kPlanes<DT>, MP = kFormed<NP>, NB = 4 * NT, W = 64 * NT;
  constexpr bool kCInLds = DT == DT_BF16;  // (three planes of it beside B's would not fit)
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const Tile<NP, W> bt{reinterpret_cast<uint16_t*>(smem)};
  const Tile<NP, W> ct{reinterpret_cast<uint16_t*>(smem + bt.kBytes)};
  const Tile<NP, 64> xt{reinterpret_cast<uint16_t*>(smem + (kCInLds ? 2 : 1) * bt.kBytes)};
  const Lower<MP> mt{xt.p + xt.kBytes / 2};
  const Decays dec(reinterpret_cast<char*>(mt.p + mt.kBytes / 2));
  int* odd = reinterpret_cast<int*>(reinterpret_cast<char*>(dec.s) + Decays::kBytes);  // [2], by chunk parity
  Lane<W> lw;
  Lane<64> lx;
  const int lane = threadIdx.x & 63;
  int li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int P = static_cast<int>(a.p.P), N = static_cast<int>(a.p.N), NK = static_cast<int>(kept_cols(N));
  const int ptiles = (P + kTile - 1) / kTile;
  const int h = blockIdx.y / ptiles, p0 = (blockIdx.y % ptiles) * kTile, cols = P - p0 < kTile ? P - p0 : kTile;
  Segment s;
  if (!segment_at<false>(a, blockIdx.x, s)) return;
  const int row = 16 * wave + li;  // this lane's channel of the state, from p0 on
  const bool active = 16 * wave < cols;
  const float skip = a.p.D == nullptr ? 0.f : load_any(a.p.D, a.p.d_dt, h);
  auto state = [&](const void* p, int64_t at) {
    return Rows<DT_F32, VEC>(p, ((at * a.p.H + h) * P + p0) * N, N, cols, N);
  };
  f32x4 acc[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) acc[nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float* from = s.first ? w.start : w.seg_state;
  if (from != nullptr) load_state<NB>(state(from, s.first ? s.m : s.enters), row, acc);
  if (threadIdx.x < 2) odd[threadIdx.x] = 0;
  const int64_t at = (int64_t(h) * a.chunks + s.c0) * kQ;
  const int64_t xcol = int64_t(h) * P + p0, bcol = int64_t(h / (a.p.H / a.p.G)) * N;
  Staged<DT, VEC, 64, kThreads> sx;
  Staged<DT, VEC, W, kThreads> sb, sc;
  double sv;
  float uv;
  auto tokens = [&](int k) { return s.n - k * kQ < kQ ? s.n - k * kQ : kQ; };
  auto c_rows = [&](int k) {
    return Rows<DT, VEC>(a.p.C, (s.t0 + int64_t(k) * kQ) * a.p.c_stride + bcol, a.p.c_stride, tokens(k), N);
  };
  auto fetch = [&](int k) {
    const int64_t t = s.t0 + int64_t(k) * kQ;
    sx.load(Rows<DT, VEC>(a.p.x, t * a.p.x_stride + xcol, a.p.x_stride, tokens(k), cols));
    sb.load(Rows<DT, VEC>(a.p.B, t * a.p.b_stride + bcol, a.p.b_stride, tokens(k), N));
    if (kCInLds) sc.load(c_rows(k));
    sv = lane_of(a.s, at + k * kQ, lane);
    uv = lane_of(a.u, at + k * kQ, lane);
  };
  fetch(0);
  __syncthreads();  // odd is 0
#pragma unroll 1
  for (int k = 0; k < s.chunks; ++k) {
    lw.refresh(), lx.refresh();
    asm volatile("" : "+v"(li), "+v"(g));  // (nor are addresses in the factors kept from chunk to chunk)
    const int n = tokens(k);
    sx.put(xt);
    sb.put(bt);
    if (kCInLds) sc.put(ct);
    dec.put(wave, sv, uv);
    if (sx.odd() != 0) odd[k & 1] = 1;
    __syncthreads();
    const bool bad = odd[k & 1] != 0;
    // blocks of M, as M^T[j][i]: 4 neighbouring j a lane.  The ten on and below the diagonal
    // are 2, 2, 3 and 3 a wave; a wave's own code each, so that no branch parts its reads
    const Rows<DT, VEC> crow = c_rows(k);
    auto m_blocks = [&](auto... pair) {
      constexpr int kPairs = sizeof...(pair);
      constexpr int ib[] = {pair.value / 4 ...}, jb[] = {pair.value % 4 ...};
      f32x4 gm[kPairs];
#pragma unroll
      for (int q = 0; q < kPairs; ++q) gm[q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 2 * NT; ++ks) {
        Frag<NP> cf;
#pragma unroll
        for (int q = 0; q < kPairs; ++q) {
          if (q == 0 || ib[q] != ib[q > 0 ? q - 1 : 0])
            cf = kCInLds ? ct.get8(lw, ib[q], ks) : crow.get8(li, 32 * ks + 8 * g, 16 * ib[q]).frag();
          gm[q] = mm(bt.get8(lw, jb[q], ks), cf, gm[q]);
        }
      }
#pragma unroll
      for (int q = 0; q < kPairs; ++q) {
        const f32x4 u = *reinterpret_cast<const f32x4*>(dec.u + 16 * jb[q] + 4 * g);
        f32x4 v;
        if (jb[q] < ib[q]) {
          const float af = dec.a[16 * ib[q] + li] * dec.between(ib[q], jb[q]);
          const f32x4 b = *reinterpret_cast<const f32x4*>(dec.b + 16 * jb[q] + 4 * g);
          v = gm[q] * ((af * b) * u);
        } else {
          const double si = dec.s[16 * ib[q] + li];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float e = __builtin_amdgcn_exp2f(static_cast<float>(si - dec.s[16 * jb[q] + 4 * g + r])) * u[r];
            const float m = gm[q][r] * e;
            v[r] = 4 * g + r <= li ? m : 0.f;
          }
        }
        mt.put4(li, g, ib[q], jb[q], v);
      }
    };
    // (a pair is 4 i + j, in blocks)
    if (wave == 0) m_blocks(Int<0>{}, Int<12>{});
    else if (wave == 1) m_blocks(Int<4>{}, Int<5>{});
    else if (wave == 2) m_blocks(Int<8>{}, Int<9>{}, Int<10>{});
    else m_blocks(Int<13>{}, Int<14>{}, Int<15>{});
    const bool keep = KEEP && !(k == 0 && from == nullptr);
    const Rows<DT, VEC> kept = kept_rows<DT, VEC>(a, w.kept, s.kept + k, h, p0, cols, NK);
    if (DT == DT_F32 && keep) keep_state<NB>(kept, row, NK, acc);
    if (k + 1 < s.chunks) fetch(k + 1);
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
        const Frag<MP> hf = split<MP>(f);
        if (DT == DT_BF16 && keep && 32 * ks < NK) {
          kept.put8(row, 32 * ks + 8 * g, hf.v[0]);
          kept.put8(row, NK + 32 * ks + 8 * g, hf.v[1]);
        }
#pragma unroll
        for (int ib = 0; ib < 4; ++ib) {
          Frag<NP> cf;
          if (kCInLds) {
            cf = ct.get44(lw, ib, ks);
          } else {
            const f32x4 lo = crow.get4(16 * ib + li, 32 * ks + 4 * g), hi = crow.get4(16 * ib + li, 32 * ks + 16 + 4 * g);
            const float cv[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            cf = split<NP>(cv);
          }
          ya[ib] = mm(hf, cf, ya[ib]);
        }
      }
#pragma unroll
      for (int ib = 0; ib < 4; ++ib) ya[ib] *= dec.e[16 * ib + li];
    }
    __syncthreads();  // M is whole, odd has been read
    if (threadIdx.x == 0) odd[k & 1] = 0;
    if (active) {
      const Frag<NP> xf[2] = {xt.tr8(lx, 0, wave), xt.tr8(lx, 1, wave)};
      Frag<NP> xm[2] = {xf[0], xf[1]};
      if (bad) {
        // 0 x_j of a later token's infinity or NaN would reach the rows before it: those
        // products are left out here and added to y one by one below
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if ((xf[ks].v[NP - 1][e] & 0x7f80) == 0x7f80)  // (of the last plane: see below_top)
#pragma unroll
              for (int q = 0; q < NP; ++q) xm[ks].v[q][e] = 0;
      }
      const Rows<DT, VEC> yrow(y, ((s.t0 + int64_t(k) * kQ) * a.p.H + h) * P + p0, a.p.H * P, n, cols);
#pragma unroll
      for (int ib = 0; ib < 4; ++ib) {
        ya[ib] = mm(xm[0], mt.get8(li, g, ib, 0), ya[ib]);
        if (ib >= 2) ya[ib] = mm(xm[1], mt.get8(li, g, ib, 1), ya[ib]);
        // (without D skip is 0: no branch between a product and the first use of its result,
        // whose wait states the compiler has been seen to leave out on the path around a body)
        ya[ib] += skip * xt.get4(lx, ib, wave);
        yrow.put4(li, 16 * wave + 4 * g, ya[ib], 16 * ib);
      }
      if (bad) {
#pragma unroll 1
        for (int ib = 0; ib < 4; ++ib) {
          const int i = 16 * ib + li, col = 16 * wave + 4 * g;
          f32x4 v = yrow.get4(i, col);
#pragma unroll 1
          for (int jj = 0; jj <= i; ++jj)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float xj = xt.at(jj, col + r);
              if (!(fabsf(xj) < INFINITY)) v[r] += mt.at(i, jj) * xj;
            }
          yrow.put4(i, col, v);
        }
      }
      const Frag<3> uf[2] = {weighted(xf[0], dec.w + 8 * g), weighted(xf[1], dec.w + 32 + 8 * g)};
      update_state(bt, lw, uf, dec.e[kQ - 1], acc);
    }
    __syncthreads();  // the tiles are free
  }
  if (s.last && w.end != nullptr) store_state<NB>(state(w.end, s.m), row, acc);
}

// ---------------------------------------------------------------------------
// One token per sequence: reads and writes the fp32 state once (memory bound: 8 bytes a
// state beside one product each for h and y; 256 sequences of 32 heads, 64 x 128: 537 MB in
// 111 us, 4.8 TB/s).  LPR lanes hold a channel's N states, 4 each (or fewer, one by one,
// where N or an address does not allow vectors).
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
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    if (vec && live && n < N) {
      v = *reinterpret_cast<const f32x4*>(state + at);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (live && n + k < N) v[k] = state[at + k];
    }
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (n + k < N) {
        v[k] = decay * v[k] + x * bv[k];
        s += v[k] * cv[k];
      }
    }
    if (vec && live && n < N) {
      *reinterpret_cast<f32x4*>(state + at) = v;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (live && n + k < N) state[at + k] = v[k];
    }
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
void with_types(const Args& a, F&& f) {
  const int nt = n_tiles(a.p.N);
#define MOC_SCAN_CASE(DT, NT) \
  if (a.p.x_dt == DT && nt == NT) { \
    with_vec<DT>(a, [&](auto VEC) { f(Int<DT>{}, Int<NT>{}, VEC); }); \
    return; \
  }
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
  with_types(a, [&](auto DT, auto NT, auto VEC) {
    constexpr size_t lds = kWalkLds<DT.value, NT.value>;
    auto* k = state_walk<DT.value, NT.value, VEC.value, REV, LOCAL>;
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
  return up(n * 4) + up(n * 8) + up(size_t(p.H) * 8);
}

// Segments: a walk's workgroups are heads x segments, and 768 of them are on the card at
// a time (three a CU, what registers and LDS allow): at most one round of them where
// sequences are cut, as a second one would run with the card part empty (16384 tokens, 32
// heads of 64 x 128, forward: 133 us with 768, 142 with 512, 138 with 1024, with the backward
// 585, 590, 624).
//
// Cutting halves a walk's length at the price of a second walk, without output, and the
// joining.  In units of one workgroup's time for a chunk, alone on its CU (3 us for bf16, 7
// to 11 for fp32), a walk of q chunks takes q f, f = 1/4 + 3/4 of the workgroups a CU (at
// least 1), the first walk half of that, and launches and joining 4 (bf16) or 1.3 (fp32).
// The least of whole sequences, segments from 256 and segments from 128 tokens on is taken
// (us, forward, whole / 256 / 128: bf16 8 x 777 tokens, 24 heads of 64 x 64: 44 / 51 / 50; 2 x
// 2000, 16 heads of 64 x 128: 121 / 46 / 48; 16 x 1000, 8 heads of 64 x 128: 66 / 56 / 57; fp32 8
// x 600, 12 heads of 64 x 64: 79 / 68 / 49).  A packed axis counts as one sequence, whatever
// its longest: 16384 tokens in 256 sequences take 355 us forward where 64 take 160.
int64_t segment(const Scan& p) {
  const int64_t n = p.seq.n_tokens, heads = p.H * ((p.P + kTile - 1) / kTile);
  const bool packed = p.seq.cu != nullptr;
  const int64_t longest = packed ? n : p.seq.seq_len, seqs = packed ? 1 : n / longest;
  const int64_t whole = (longest + kQ - 1) / kQ * kQ;
  int64_t want = 768 / heads;  // segments of the whole token axis
  if (want < 1) want = 1;
  if (!packed) want = want < seqs ? seqs : want / seqs * seqs;  // the same number in every sequence
  const int64_t even = ((n + want - 1) / want + kQ - 1) / kQ * kQ;
  auto cost = [&](int64_t seg) {
    const double wgs = static_cast<double>(heads * seqs * ((longest + seg - 1) / seg));
    const double f = 0.25 + 0.75 * wgs / 256.0;
    const double walk = static_cast<double>(seg / kQ) * (f < 1.0 ? 1.0 : f);
    return seg >= whole ? walk : 1.5 * walk + (p.x_dt == DT_BF16 ? 4.0 : 1.3);
  };
  int64_t best = whole;
  for (int64_t least : {256, 128}) {
    const int64_t seg = even < least ? least : even;
    if (seg < whole && cost(seg) < cost(best)) best = seg;
  }
  return best;
}

// a.vec for tensors of the x type and others (16 bytes) at these addresses
void align(Args& a, std::initializer_list<const void*> of_x, std::initializer_list<const void*> others) {
  const int size = a.p.x_dt == DT_BF16 ? 2 : 4;
  if (a.vec == 8 && !aligned(of_x, 8 * size)) a.vec = 4;
  if (!aligned(of_x, 4 * size) || !aligned(others, 16)) a.vec = 0;
}

Args make_args(const Scan& p, void* prep) {
  Args a{};
  a.p = p;
  a.seqs.l = p.seq;
  a.seqs.count = p.seq.cu == nullptr ? p.seq.n_tokens / p.seq.seq_len : p.seq.n_seqs + 2;
  a.chunks = pieces(a.seqs, kQ);
  a.seg = segment(p);
  const size_t n = size_t(p.H) * a.chunks * kQ;
  a.u = static_cast<float*>(prep);
  a.s = reinterpret_cast<double*>(static_cast<char*>(prep) + up(n * 4));
  a.par = reinterpret_cast<float*>(static_cast<char*>(prep) + up(n * 4) + up(n * 8));
  // (a chunk's states lie under one buffer resource)
  const bool small = p.H * p.P * kept_cols(p.N) * 4 < int64_t(kNowhere) - 16;
  for (int v : {8, 4}) {
    bool ok = small && a.vec == 0 && (v == 4 || p.x_dt == DT_BF16);
    for (int64_t k : {p.P, p.N}) ok = ok && k % v == 0;
    for (int64_t st : {p.x_stride, p.b_stride, p.c_stride, p.H * p.P, p.G * p.N}) ok = ok && st % v == 0 && st < kMaxStride;
    if (ok) a.vec = v;
  }
  align(a, {p.x, p.B, p.C}, {});
  return a;
}

void launch_prep(const Args& a, hipStream_t st) {
  hipLaunchKernelGGL(prep_kernel, dim3(static_cast<unsigned>(a.chunks), static_cast<unsigned>((a.p.H + kPrepHeads - 1) / kPrepHeads)),
                     dim3(kThreads), 0, st, a);
}

size_t walk_bytes(const Args& a) {
  if (!segmented(a)) return 0;
  const size_t n = size_t(a.p.seq.n_tokens / a.seg) * a.p.H;
  return up(n * a.p.P * a.p.N * 4) + up(n * 8);
}

void carve_walk(const Args& a, void* workspace, Walk& w) {
  if (!segmented(a)) return;
  const size_t n = size_t(a.p.seq.n_tokens / a.seg) * a.p.H;
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
  return prep_bytes(p) + size_t(kept_states(a)) * p.H * p.P * kept_cols(p.N) * 4;
}

size_t scan_forward_workspace(const Scan& p, bool saved) {
  return walk_bytes(make_args(p, nullptr)) + (saved ? 0 : prep_bytes(p));
}

void scan_forward(const Scan& p, void* y, const float* init, float* fin, void* saved, void* workspace,
                  hipStream_t st) {
  char* ws = static_cast<char*>(workspace);
  Args a = make_args(p, saved != nullptr ? saved : ws);
  align(a, {y}, {init, fin, saved, workspace});
  Walk w{};
  w.x = p.x;
  w.b = p.B;
  w.x_stride = p.x_stride;
  w.b_stride = p.b_stride;
  w.start = init;
  w.end = fin;
  w.kept = saved != nullptr ? static_cast<char*>(saved) + prep_bytes(p) : nullptr;
  carve_walk(a, saved != nullptr ? ws : ws + prep_bytes(p), w);
  launch_prep(a, st);
  launch_segments(a, w, false, st);
  with_types(a, [&](auto DT, auto NT, auto VEC) {
    constexpr size_t lds = kForwardLds<DT.value, NT.value>;
    auto* k = w.kept != nullptr ? forward_walk<DT.value, NT.value, VEC.value, true>
                                : forward_walk<DT.value, NT.value, VEC.value, false>;
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
