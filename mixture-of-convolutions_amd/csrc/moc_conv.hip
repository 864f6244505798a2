// Short causal convolution, one kernel per channel for every token (gfx950).
//
//   P[t,d] = bias[d] + sum_s w[s,d] x[t-(S-1-s),d],   y = silu(P) or P
//   g = dy silu'(P) (or dy), dx[t] = sum_k w[S-1-k] g[t+k],
//   dw[s] = sum_t g[t] x[t-(S-1-s)], dbias = sum_t g[t]
// (x taken as 0, or from the cache, before a sequence's first token; g as 0 behind its
// last).
//
// Bound by memory: 2 S products a channel and token beside 2 elements moved.  A wave
// owns 64 V neighbouring channels and walks a strip of rows, the last S rows of x in
// registers, so that x is read once but for the S - 1 rows before each strip; what a
// row belongs to is the same for all its lanes, so sequence ends are wave-uniform
// branches.  The backward forms P again (x is read anyway), keeps the last S rows of g
// too, and the sums of dw and dbias of its strip; a workgroup's four strips are added in
// LDS, the workgroups' rows by column_sums in a fixed order.  All arithmetic is fp32,
// results are rounded once.
//
// 16384 bf16 tokens of 2048 channels, 4 taps: forward 35 us (3.8 TB/s of x and y), backward
// 55 (3.6 TB/s of x, dy and dx), sums 4; a step of 8 rows 3.4 us, a launch.
#include <type_traits>

#include "moc_kernels.h"
#include "moc_rows.h"

namespace moc {
namespace {

constexpr int kWaves = 4;
constexpr int kAhead = 4;  // rows that the forward loads together

struct ConvArgs {
  const void* x;
  const void* w;      // [S, D]
  const void* bias;   // [D] or null
  const void* cache;  // [B, D, S] in the x dtype or null
  void* y;
  void* fin;          // [B, D, S] or null
  const void* dy;
  void* dx;
  float* part;        // [workgroups][(S + 1) D]
  SeqLayout seq;
  int64_t D;
  int w_dt, b_dt, act, rows;  // rows: tokens of a strip
};

// x[t - k] for k = 1..S-1 of a row at position pos of its sequence [lo, ..):
// win[S-1-k]; rows before the sequence come from the cache or are 0.
template <int DT, int S, int V>
__device__ __forceinline__ void history(const ConvArgs& a, int64_t t, int64_t lo, int64_t c, float (&win)[S][V]) {
#pragma unroll
  for (int k = 1; k < S; ++k) {
    const int64_t u = t - k;
    if (u >= lo) {
      load_vec<DT, V>(a.x, u * a.D + c, a.D - c, win[S - 1 - k]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float v = 0.f;
        if (a.cache != nullptr && c + i < a.D)  // fixed length: sequence lo / seq_len, slot S - (lo - u)
          v = load_any(a.cache, DT, ((lo / a.seq.seq_len) * a.D + c + i) * S + (S - (lo - u)));
        win[S - 1 - k][i] = v;
      }
    }
  }
}

template <int DT, int S, int V>
__global__ __launch_bounds__(64 * kWaves) void conv_fwd(ConvArgs a) {
  const int64_t c = (int64_t(blockIdx.x) * 64 + (threadIdx.x & 63)) * V;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r0 = (int64_t(blockIdx.y) * kWaves + wave) * a.rows;
  const int64_t n = a.seq.n_tokens;
  if (r0 >= n || c >= a.D) return;
  const int64_t r1 = r0 + a.rows < n ? r0 + a.rows : n;
  float w[S][V], b[V], win[S][V];
#pragma unroll
  for (int s = 0; s < S; ++s) load_param<V>(a.w, a.w_dt, s * a.D + c, a.D - c, 0.f, w[s]);
  load_param<V>(a.bias, a.b_dt, c, a.D - c, 0.f, b);
  int64_t lo, hi;
  a.seq.bounds(r0, lo, hi);
  history<DT, S, V>(a, r0, lo, c, win);
  const int64_t left = a.D - c;
  auto row = [&](int64_t t) {  // win[S - 1] holds x[t]
    float p[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[i] = b[i];
#pragma unroll
      for (int s = 0; s < S; ++s) p[i] += w[s][i] * win[s][i];
      if (a.act) p[i] *= sigmoid_f(p[i]);
    }
    store_vec<DT, V>(a.y, t * a.D + c, left, p);
    if (a.fin != nullptr && hi - t <= S) {  // slots of the last S rows (fixed length)
      const int64_t q = lo / a.seq.seq_len;
      for (int i = 0; i < V && i < left; ++i) {
        const int64_t at = (q * a.D + c + i) * S;
        store_any(a.fin, DT, at + S - (hi - t), win[S - 1][i]);
        // a sequence shorter than the state: its first row also writes the older slots
        if (t == lo)
          for (int64_t s = 0; s < S - (hi - lo); ++s)
            store_any(a.fin, DT, at + s, a.cache == nullptr ? 0.f : load_any(a.cache, DT, at + s + (hi - lo)));
      }
    }
#pragma unroll
    for (int s = 0; s + 1 < S; ++s)
#pragma unroll
      for (int i = 0; i < V; ++i) win[s][i] = win[s + 1][i];
  };
  int64_t t = r0;
  while (t < r1) {
    if (t >= hi) {
      a.seq.bounds(t, lo, hi);
      history<DT, S, V>(a, t, lo, c, win);
    }
    const int64_t end = hi < r1 ? hi : r1;
    // kAhead rows' loads in flight at a time
    for (; t + kAhead <= end; t += kAhead) {
      RawVec<DT, V> x[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) x[k].load(a.x, (t + k) * a.D + c, left);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        x[k].get(win[S - 1]);
        row(t + k);
      }
    }
    for (; t < end; ++t) {
      load_vec<DT, V>(a.x, t * a.D + c, left, win[S - 1]);
      row(t);
    }
  }
}

template <int DT, int S, int V, int AHEAD>
__global__ __launch_bounds__(64 * kWaves) void conv_bwd(ConvArgs a) {
  __shared__ float lds[kWaves - 1][64 * V];
  const int64_t c = (int64_t(blockIdx.x) * 64 + (threadIdx.x & 63)) * V;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r0 = (int64_t(blockIdx.y) * kWaves + wave) * a.rows;
  const int64_t n = a.seq.n_tokens;
  const int64_t r1 = r0 + a.rows < n ? r0 + a.rows : n;
  float dw[S][V], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    db[i] = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s) dw[s][i] = 0.f;
  }
  if (r0 < n && c < a.D) {
    float w[S][V], b[V], win[S][V], acc[S][V];  // acc[k]: dx of row u - k so far
#pragma unroll
    for (int s = 0; s < S; ++s) load_param<V>(a.w, a.w_dt, s * a.D + c, a.D - c, 0.f, w[s]);
    load_param<V>(a.bias, a.b_dt, c, a.D - c, 0.f, b);
#pragma unroll
    for (int k = 0; k < S; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[k][i] = 0.f;
    int64_t lo, hi;
    a.seq.bounds(r0, lo, hi);
    history<DT, S, V>(a, r0, lo, c, win);
    const int64_t left = a.D - c;
    // g of row u (dy read into g, x into win[S - 1]), its part of the sums where the row is
    // this strip's own, and of the gradients of the rows it reaches back to
    auto row = [&](int64_t u, float (&g)[V]) {
      if (a.act) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float p = b[i];
#pragma unroll
          for (int s = 0; s < S; ++s) p += w[s][i] * win[s][i];
          const float sg = sigmoid_f(p);
          g[i] *= sg * (1.f + p * (1.f - sg));
        }
      }
      if (u < r1) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          db[i] += g[i];
#pragma unroll
          for (int s = 0; s < S; ++s) dw[s][i] += g[i] * win[s][i];
        }
      }
      const int64_t back = u - lo;  // rows of the same sequence before u
#pragma unroll
      for (int k = 0; k < S; ++k) {
        if (k <= back) {
#pragma unroll
          for (int i = 0; i < V; ++i) acc[k][i] += w[S - 1 - k][i] * g[i];
        }
      }
#pragma unroll
      for (int s = 0; s + 1 < S; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) win[s][i] = win[s + 1][i];
    };
    auto emit = [&](int64_t u) {  // dx of row u - (S - 1) is whole
      const int64_t t = u - (S - 1);
      if (t >= r0 && t < r1 && a.dx != nullptr) store_vec<DT, V>(a.dx, t * a.D + c, left, acc[S - 1]);
#pragma unroll
      for (int k = S - 1; k > 0; --k)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[k][i] = acc[k - 1][i];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[0][i] = 0.f;
    };
    // rows u < r1 are this strip's; the S - 1 rows behind them only reach back into it
    int64_t u = r0;
    while (u < r1 + S - 1) {
      if (u < n && u >= hi) {
        a.seq.bounds(u, lo, hi);
        history<DT, S, V>(a, u, lo, c, win);
      }
      auto one = [&]() {
        float g[V];
        load_vec<DT, V>(a.x, u * a.D + c, left, win[S - 1]);
        load_vec<DT, V>(a.dy, u * a.D + c, left, g);
        row(u, g);
      };
      if (u >= r1) {
        if (u < n && lo < r1) one();
        emit(u);
        ++u;
        continue;
      }
      const int64_t end = hi < r1 ? hi : r1;
      for (; u + AHEAD <= end; u += AHEAD) {
        RawVec<DT, V> x[AHEAD], dy[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          x[k].load(a.x, (u + k) * a.D + c, left);
          dy[k].load(a.dy, (u + k) * a.D + c, left);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          float g[V];
          x[k].get(win[S - 1]);
          dy[k].get(g);
          row(u + k, g);
          emit(u + k);
        }
      }
      for (; u < end; ++u) {
        one();
        emit(u);
      }
    }
  }
  if (a.part == nullptr) return;
  float* out = a.part + int64_t(blockIdx.y) * (S + 1) * a.D;
  const int at = (threadIdx.x & 63) * V;
#pragma unroll
  for (int s = 0; s <= S; ++s) {
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = s < S ? dw[s < S ? s : 0][i] : db[i];
    if (wave > 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) lds[wave - 1][at + i] = v[i];
    }
    __syncthreads();
    if (wave == 0 && c < a.D) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c + i < a.D) out[s * a.D + c + i] = ((v[i] + lds[0][at + i]) + lds[1][at + i]) + lds[2][at + i];
    }
    __syncthreads();
  }
}

// One token per sequence, in place on the cache (element strides cb, cd, cs): slot s
// takes slot s + 1, the last slot the token; y from the new cache.
template <int DT, int S>
__global__ __launch_bounds__(256) void conv_step(const void* __restrict__ x, const void* __restrict__ w,
                                                 const void* __restrict__ bias, void* __restrict__ cache, int64_t cb,
                                                 int64_t cd, int64_t cs, void* __restrict__ y, int64_t B, int64_t D,
                                                 int w_dt, int b_dt, int act) {
  const int64_t n = B * D;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    const int64_t q = i / D, d = i - q * D;
    const int64_t at = q * cb + d * cd;
    float win[S];
#pragma unroll
    for (int s = 0; s + 1 < S; ++s) win[s] = load_any(cache, DT, at + (s + 1) * cs);
    win[S - 1] = load_any(x, DT, i);
    float p = bias == nullptr ? 0.f : load_any(bias, b_dt, d);
#pragma unroll
    for (int s = 0; s < S; ++s) p += load_any(w, w_dt, s * D + d) * win[s];
    if (act) p *= sigmoid_f(p);
    store_any(y, DT, i, p);
#pragma unroll
    for (int s = 0; s < S; ++s) store_any(cache, DT, at + s * cs, win[s]);
  }
}

template <int V>
using Int = std::integral_constant<int, V>;

template <int DT, typename F>
void with_taps(int64_t S, F&& f) {
  switch (S) {
#define MOC_CONV_S(SS) \
  case SS: return f(Int<DT>{}, Int<SS>{});
    MOC_CONV_S(1) MOC_CONV_S(2) MOC_CONV_S(3) MOC_CONV_S(4) MOC_CONV_S(5) MOC_CONV_S(6) MOC_CONV_S(7) MOC_CONV_S(8)
    MOC_CONV_S(9) MOC_CONV_S(10) MOC_CONV_S(11) MOC_CONV_S(12) MOC_CONV_S(13) MOC_CONV_S(14) MOC_CONV_S(15)
    MOC_CONV_S(16)
#undef MOC_CONV_S
    default: return;
  }
}
template <typename F>
void with_shape(int dt, int64_t S, F&& f) {
  if (dt == DT_BF16) with_taps<DT_BF16>(S, f);
  else with_taps<DT_F32>(S, f);
}

// Channels of a lane: 16 bytes of them, fewer where S rows of them in fp32 (twice, and
// the weights and their sums, in the backward) would not stay in registers.
constexpr int vec(int dt, int64_t S, bool backward) {
  const int v = dt == DT_BF16 ? 8 : 4, most = backward ? (S <= 2 ? 8 : (S <= 8 ? 4 : 2)) : (S <= 8 ? 8 : 4);
  return v < most ? v : most;
}

// Rows that the backward loads together: four, so that more loads are in flight and the windows
// move less often, or two where up to 6 taps' rows end within a lane's vector, whose loads one
// by one are too much code four times over.  Us with two / four, at 2, 3, 4, 6 and 8 taps: bf16
// 16384 x 2048 54/52, 47/45, 53/50, 66/60, 77/74 (12 taps 117/108), 8192 x 2048 34/34, 30/29,
// 33/32, 41/40, 50/49, fp32 16384 x 2048 103/93, 106/93, 111/98, 117/104, 128/111; odd rows:
// bf16 6000 x 1130 26/36, 25/31, 29/36, 48/55, 69/69, 24000 x 1130 67/97, 61/71, 65/77, 96/113,
// 134/130, fp32 6000 x 1130 23/24, 25/29, 28/33, 42/42, 53/52.  Four loses at 16384 x 4096 with
// 3 and 4 taps: 91/111, 96/117 (2, 6 and 8 taps: 142/136, 147/129, 166/151).
constexpr int ahead(int64_t S, bool odd) { return odd && S <= 6 ? 2 : 4; }

// Rows of a strip: as many as still leave about 2048 waves (two a SIMD), 4 to 64.
int strip(int64_t tokens, int64_t D, int v) {
  const int64_t across = (D + 64 * v - 1) / (64 * v);
  int r = 4;
  while (r < 64 && across * (tokens / (2 * r)) >= 2048) r *= 2;
  // (a grid's second axis holds 65535 workgroups)
  while ((tokens + kWaves * r - 1) / (kWaves * r) > 65535) r *= 2;
  return r;
}

int64_t strip_groups(int64_t tokens, int r) { return (tokens + kWaves * r - 1) / (kWaves * r); }

ConvArgs args(const Conv& p, const void* x, const void* w, const void* bias) {
  ConvArgs a{};
  a.x = x;
  a.w = w;
  a.bias = bias;
  a.seq = p.seq;
  a.D = p.D;
  a.w_dt = p.w_dt;
  a.b_dt = p.b_dt;
  a.act = p.activation;
  return a;
}

}  // namespace

size_t conv_backward_workspace(const Conv& p) {
  return size_t(strip_groups(p.seq.n_tokens, strip(p.seq.n_tokens, p.D, vec(p.x_dt, p.S, true)))) * (p.S + 1) * p.D *
         sizeof(float);
}

void conv_forward(const Conv& p, const void* x, const void* w, const void* bias, const void* cache, void* y, void* fin,
                  hipStream_t st) {
  ConvArgs a = args(p, x, w, bias);
  a.cache = cache;
  a.y = y;
  a.fin = fin;
  const int v = vec(p.x_dt, p.S, false);
  a.rows = strip(p.seq.n_tokens, p.D, v);
  const dim3 grid(static_cast<unsigned>((p.D + 64 * v - 1) / (64 * v)),
                  static_cast<unsigned>(strip_groups(p.seq.n_tokens, a.rows)));
  with_shape(p.x_dt, p.S, [&](auto DT, auto S) {
    hipLaunchKernelGGL((conv_fwd<DT.value, S.value, vec(DT.value, S.value, false)>), grid, dim3(64 * kWaves), 0, st, a);
  });
}

void conv_backward(const Conv& p, const void* x, const void* w, const void* bias, const void* dy, void* dx, void* dw,
                   void* dbias, void* workspace, hipStream_t st) {
  ConvArgs a = args(p, x, w, bias);
  a.dy = dy;
  a.dx = dx;
  const bool sums = dw != nullptr || dbias != nullptr;
  a.part = sums ? static_cast<float*>(workspace) : nullptr;
  const int v = vec(p.x_dt, p.S, true);
  a.rows = strip(p.seq.n_tokens, p.D, v);
  const int64_t groups = strip_groups(p.seq.n_tokens, a.rows);
  const dim3 grid(static_cast<unsigned>((p.D + 64 * v - 1) / (64 * v)), static_cast<unsigned>(groups));
  const bool odd = p.D % v != 0;
  with_shape(p.x_dt, p.S, [&](auto DT, auto S) {
    constexpr int V = vec(DT.value, S.value, true);
    auto* k = odd ? conv_bwd<DT.value, S.value, V, ahead(S.value, true)> : conv_bwd<DT.value, S.value, V, ahead(S.value, false)>;
    hipLaunchKernelGGL(k, grid, dim3(64 * kWaves), 0, st, a);
  });
  if (sums) launch_column_sums({a.part, groups, p.S * p.D, p.D, 0, dw, dbias, nullptr, p.w_dt, p.b_dt, 0}, st);
}

void conv_update(const void* x, const void* w, const void* bias, void* cache, int64_t cb, int64_t cd, int64_t cs,
                 void* y, int64_t B, int64_t D, int64_t S, int x_dt, int w_dt, int b_dt, int act, hipStream_t st) {
  const int64_t n = (B * D + 255) / 256;
  const dim3 grid(static_cast<unsigned>(n < (1 << 22) ? n : (1 << 22)));
  with_shape(x_dt, S, [&](auto DT, auto SS) {
    hipLaunchKernelGGL((conv_step<DT.value, SS.value>), grid, dim3(256), 0, st, x, w, bias, cache, cb, cd, cs, y, B, D,
                       w_dt, b_dt, act);
  });
}

}  // namespace moc
