// Layer norm over the last axis, forward and backward (gfx950).
//
//   mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
//   xh = (x - mean) rstd, y = xh w + b
//   g = dy w, dx = rstd (g - sum(g)/D - xh sum(g xh)/D)
//   dw = sum_rows dy xh, db = sum_rows dy
//
// Bound by memory: x is read once and y written once; the backward reads x and dy
// and writes dx.  So a row stays in registers: TPR lanes (16, 64, or the workgroup)
// hold NV vectors of V elements each, the mean is summed first and the squares of
// x - mean after it, from the registers (no sum of squares that a far mean would
// cancel).  Statistics and sums are fp32; y, dx, dw, db are rounded once.
//
// The weight's gradient is a sum over rows while a row is spread over lanes: a lane
// keeps dw and db of its own columns while its workgroup walks rows, and only
// workgroups' sums go through memory, kParts rows of them, added in a fixed order.
#include <initializer_list>
#include <type_traits>

#include "moc_kernels.h"
#include "moc_rows.h"

namespace moc {
namespace {

constexpr int kThreads = 256;

// Sum over the TPR lanes of a row (all of them get it).  `buf`: 4 floats, used by a
// row of a whole workgroup only.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* buf) {
#pragma unroll
  for (int m = 1; m < (TPR < 64 ? TPR : 64); m <<= 1) v += __shfl_xor(v, m);
  if (TPR > 64) {
    __syncthreads();  // (buf's last readers are done)
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (buf[0] + buf[1]) + (buf[2] + buf[3]);
  }
  return v;
}

// w / b of V columns, in any dtype.
template <int V>
__device__ __forceinline__ void load_param(const void* p, int dt, int64_t i, float none, float (&out)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) out[k] = p == nullptr ? none : load_any(p, dt, i + k);
}

template <int DT, int V, int NV, int TPR>
__global__ __launch_bounds__(kThreads) void norm_fwd(const void* __restrict__ x, const void* __restrict__ w,
                                                     const void* __restrict__ b, void* __restrict__ y,
                                                     float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                     int64_t rows, int D, int w_dt, int b_dt, float eps) {
  __shared__ float buf[4];
  const int lane = threadIdx.x % TPR;
  constexpr int RPW = kThreads / TPR;
  const float inv = 1.0f / static_cast<float>(D);
  // (every lane runs every round: a row of a whole workgroup has barriers in it)
  for (int64_t r0 = int64_t(blockIdx.x) * RPW; r0 < rows; r0 += int64_t(gridDim.x) * RPW) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool live = row < rows;
    const int64_t base = row * D;
    float v[NV][V];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      if (live && c < D) {
        load_vec<DT, V>(x, base + c, v[i]);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[i][k] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < V; ++k) s += v[i][k];
    }
    const float mean = row_sum<TPR>(s, buf) * inv;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * TPR + lane) * V < D) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          v[i][k] -= mean;
          s += v[i][k] * v[i][k];
        }
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(s, buf) * inv + eps);
    if (!live) continue;
    if (mean_out != nullptr && lane == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      if (c >= D) continue;
      float wv[V], bv[V];
      load_param<V>(w, w_dt, c, 1.f, wv);
      load_param<V>(b, b_dt, c, 0.f, bv);
#pragma unroll
      for (int k = 0; k < V; ++k) v[i][k] = v[i][k] * rstd * wv[k] + bv[k];
      store_vec<DT, V>(y, base + c, v[i]);
    }
  }
}

// Workgroup wg walks rows (wg + i * gridDim) * RPW + its row group; part[wg] = [dw | db].
template <int DT, int V, int NV, int TPR, bool SUMS>
__global__ __launch_bounds__(kThreads) void norm_bwd(const void* __restrict__ x, const void* __restrict__ w,
                                                     const void* __restrict__ dy, const float* __restrict__ mean_in,
                                                     const float* __restrict__ rstd_in, void* __restrict__ dx,
                                                     float* __restrict__ part, int64_t rows, int D, int w_dt) {
  extern __shared__ float lds[];  // TPR < 256: [2][D] sums of the workgroup's row groups
  __shared__ float buf[4];
  constexpr int RPW = kThreads / TPR;
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.0f / static_cast<float>(D);
  float dw[NV][V], db[NV][V], wv[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * V;
#pragma unroll
    for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = wv[i][k] = 0.f;
    if (c < D) load_param<V>(w, w_dt, c, 1.f, wv[i]);
  }
  // (every lane runs every round: a row of a whole workgroup has barriers in it)
  for (int64_t r0 = int64_t(blockIdx.x) * RPW; r0 < rows; r0 += int64_t(gridDim.x) * RPW) {
    const int64_t row = r0 + group;
    const bool live = row < rows;
    const int64_t base = row * D;
    const float mean = live ? mean_in[row] : 0.f, rstd = live ? rstd_in[row] : 0.f;
    float xh[NV][V], g[NV][V];
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      if (live && c < D) {
        load_vec<DT, V>(x, base + c, xh[i]);
        load_vec<DT, V>(dy, base + c, g[i]);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) xh[i][k] = mean, g[i][k] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        xh[i][k] = (xh[i][k] - mean) * rstd;
        if (SUMS) {
          dw[i][k] += g[i][k] * xh[i][k];
          db[i][k] += g[i][k];
        }
        g[i][k] *= wv[i][k];
        s0 += g[i][k];
        s1 += g[i][k] * xh[i][k];
      }
    }
    if (dx == nullptr) continue;
    s0 = row_sum<TPR>(s0, buf) * inv;
    s1 = row_sum<TPR>(s1, buf) * inv;
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      if (c >= D) continue;
#pragma unroll
      for (int k = 0; k < V; ++k) g[i][k] = rstd * (g[i][k] - s0 - xh[i][k] * s1);
      store_vec<DT, V>(dx, base + c, g[i]);
    }
  }
  if (!SUMS) return;
  float* out = part + int64_t(blockIdx.x) * 2 * D;
  if (TPR == kThreads) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      if (c < D) {
#pragma unroll
        for (int k = 0; k < V; ++k) out[c + k] = dw[i][k], out[D + c + k] = db[i][k];
      }
    }
    return;
  }
  for (int q = 0; q < RPW; ++q) {  // row groups in order
    if (group == q) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * V;
        if (c < D) {
#pragma unroll
          for (int k = 0; k < V; ++k) {
            lds[c + k] = (q == 0 ? 0.f : lds[c + k]) + dw[i][k];
            lds[D + c + k] = (q == 0 ? 0.f : lds[D + c + k]) + db[i][k];
          }
        }
      }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < 2 * D; c += kThreads) out[c] = lds[c];
}

// Rows too long for a workgroup's registers: the row is read again for each sum.
template <int DT>
__global__ __launch_bounds__(kThreads) void norm_fwd_long(const void* __restrict__ x, const void* __restrict__ w,
                                                          const void* __restrict__ b, void* __restrict__ y,
                                                          float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                          int64_t rows, int64_t D, int w_dt, int b_dt, float eps) {
  __shared__ float buf[4];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t base = row * D;
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < D; c += kThreads) s += load_any(x, DT, base + c);
    const float mean = row_sum<kThreads>(s, buf) / static_cast<float>(D);
    s = 0.f;
    for (int64_t c = threadIdx.x; c < D; c += kThreads) {
      const float d = load_any(x, DT, base + c) - mean;
      s += d * d;
    }
    const float rstd = 1.0f / sqrtf(row_sum<kThreads>(s, buf) / static_cast<float>(D) + eps);
    if (mean_out != nullptr && threadIdx.x == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    for (int64_t c = threadIdx.x; c < D; c += kThreads) {
      const float wv = w == nullptr ? 1.f : load_any(w, w_dt, c);
      const float bv = b == nullptr ? 0.f : load_any(b, b_dt, c);
      store_any(y, DT, base + c, (load_any(x, DT, base + c) - mean) * rstd * wv + bv);
    }
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void norm_dx_long(const void* __restrict__ x, const void* __restrict__ w,
                                                         const void* __restrict__ dy,
                                                         const float* __restrict__ mean_in,
                                                         const float* __restrict__ rstd_in, void* __restrict__ dx,
                                                         int64_t rows, int64_t D, int w_dt) {
  __shared__ float buf[4];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t base = row * D;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float s0 = 0.f, s1 = 0.f;
    for (int64_t c = threadIdx.x; c < D; c += kThreads) {
      const float g = load_any(dy, DT, base + c) * (w == nullptr ? 1.f : load_any(w, w_dt, c));
      s0 += g;
      s1 += g * (load_any(x, DT, base + c) - mean) * rstd;
    }
    s0 = row_sum<kThreads>(s0, buf) / static_cast<float>(D);
    s1 = row_sum<kThreads>(s1, buf) / static_cast<float>(D);
    for (int64_t c = threadIdx.x; c < D; c += kThreads) {
      const float g = load_any(dy, DT, base + c) * (w == nullptr ? 1.f : load_any(w, w_dt, c));
      store_any(dx, DT, base + c, rstd * (g - s0 - (load_any(x, DT, base + c) - mean) * rstd * s1));
    }
  }
}

// part[blockIdx.y] = [dw | db] of rows blockIdx.y, + gridDim.y, ...; a column per lane.
template <int DT>
__global__ __launch_bounds__(kThreads) void norm_sums_long(const void* __restrict__ x, const void* __restrict__ dy,
                                                           const float* __restrict__ mean_in,
                                                           const float* __restrict__ rstd_in,
                                                           float* __restrict__ part, int64_t rows, int64_t D) {
  const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= D) return;
  float dw = 0.f, db = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float g = load_any(dy, DT, r * D + c);
    dw += g * (load_any(x, DT, r * D + c) - mean_in[r]) * rstd_in[r];
    db += g;
  }
  part[int64_t(blockIdx.y) * 2 * D + c] = dw;
  part[int64_t(blockIdx.y) * 2 * D + D + c] = db;
}

// How a row is spread: TPR lanes of NV vectors of V elements.
struct Plan {
  int v, nv, tpr;  // nv 0: the long kernels
};

// V: 16-byte vectors where rows and tensors allow them, pairs of bf16 or single
// elements otherwise.  Lanes: a row of up to 16 vectors takes 16 lanes (four rows a
// wave, where a wave a row would leave most lanes idle), up to 4 vectors a lane a
// wave, more the workgroup.
Plan plan(int64_t D, int dt, bool al16, bool al4) {
  const int full = dt == DT_BF16 ? 8 : 4;
  int v = 1;
  if (D % full == 0 && al16) v = full;
  else if (dt == DT_BF16 && D % 2 == 0 && al4) v = 2;
  const int most = v == 1 ? 32 : (v == 2 ? 16 : (v == 4 ? 8 : 4));  // vectors a lane holds
  const int64_t n = (D + v - 1) / v;
  if (n <= 16) return {v, 1, 16};
  for (int tpr : {64, 256}) {
    const int64_t nv = (n + tpr - 1) / tpr;
    if (nv <= most) {
      int r = 1;
      while (r < nv) r <<= 1;
      return {v, r, tpr};
    }
  }
  return {v, 0, 256};
}

template <typename F>
void with_plan(const Plan& p, int dt, F&& f) {
#define MOC_NORM_CASE(DT, V, NV, TPR) \
  if (dt == DT && p.v == V && p.nv == NV && p.tpr == TPR) \
    return f(std::integral_constant<int, DT>{}, std::integral_constant<int, V>{}, std::integral_constant<int, NV>{}, \
             std::integral_constant<int, TPR>{});
#define MOC_NORM_WIDE(DT, V, NV) MOC_NORM_CASE(DT, V, NV, 64) MOC_NORM_CASE(DT, V, NV, 256)
  MOC_NORM_CASE(DT_BF16, 8, 1, 16) MOC_NORM_CASE(DT_BF16, 2, 1, 16) MOC_NORM_CASE(DT_BF16, 1, 1, 16)
  MOC_NORM_CASE(DT_F32, 4, 1, 16) MOC_NORM_CASE(DT_F32, 1, 1, 16)
  MOC_NORM_WIDE(DT_BF16, 8, 1) MOC_NORM_WIDE(DT_BF16, 8, 2) MOC_NORM_WIDE(DT_BF16, 8, 4)
  MOC_NORM_WIDE(DT_BF16, 2, 1) MOC_NORM_WIDE(DT_BF16, 2, 2) MOC_NORM_WIDE(DT_BF16, 2, 4)
  MOC_NORM_WIDE(DT_BF16, 2, 8) MOC_NORM_WIDE(DT_BF16, 2, 16)
  MOC_NORM_WIDE(DT_BF16, 1, 1) MOC_NORM_WIDE(DT_BF16, 1, 2) MOC_NORM_WIDE(DT_BF16, 1, 4)
  MOC_NORM_WIDE(DT_BF16, 1, 8) MOC_NORM_WIDE(DT_BF16, 1, 16) MOC_NORM_WIDE(DT_BF16, 1, 32)
  MOC_NORM_WIDE(DT_F32, 4, 1) MOC_NORM_WIDE(DT_F32, 4, 2) MOC_NORM_WIDE(DT_F32, 4, 4) MOC_NORM_WIDE(DT_F32, 4, 8)
  MOC_NORM_WIDE(DT_F32, 1, 1) MOC_NORM_WIDE(DT_F32, 1, 2) MOC_NORM_WIDE(DT_F32, 1, 4)
  MOC_NORM_WIDE(DT_F32, 1, 8) MOC_NORM_WIDE(DT_F32, 1, 16) MOC_NORM_WIDE(DT_F32, 1, 32)
#undef MOC_NORM_WIDE
#undef MOC_NORM_CASE
}

// Workgroups of a kernel that walks rows (a grid's threads are counted in 32 bits).
unsigned grid(int64_t n) { return static_cast<unsigned>(n < (1 << 22) ? n : (1 << 22)); }

// Workgroups of the backward, and rows of partial sums: two a CU, or what the rows
// give.
constexpr int64_t kParts = 512;

int64_t parts(int64_t rows) { return rows < kParts ? rows : kParts; }

__global__ __launch_bounds__(1024) void column_sums(ColumnSums a) {
  __shared__ float s[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int64_t cols = a.n0 + a.n1 + a.n2, c = int64_t(blockIdx.x) * 32 + cx;
  float v = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int64_t r = ry; r < a.n; r += 32) v += a.part[r * cols + c];
  }
  s[ry][cx] = v;
  __syncthreads();
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) {
    if (ry < m) s[ry][cx] += s[ry + m][cx];
    __syncthreads();
  }
  if (ry != 0 || c >= cols) return;
  if (c < a.n0) {
    if (a.out0 != nullptr) store_any(a.out0, a.dt0, c, s[0][cx]);
  } else if (c < a.n0 + a.n1) {
    if (a.out1 != nullptr) store_any(a.out1, a.dt1, c - a.n0, s[0][cx]);
  } else if (a.out2 != nullptr) {
    store_any(a.out2, a.dt2, c - a.n0 - a.n1, s[0][cx]);
  }
}

}  // namespace

void launch_column_sums(const ColumnSums& c, hipStream_t st) {
  const int64_t cols = c.n0 + c.n1 + c.n2;
  hipLaunchKernelGGL(column_sums, dim3(static_cast<unsigned>((cols + 31) / 32)), dim3(1024), 0, st, c);
}

size_t norm_backward_workspace(int64_t rows, int64_t D) { return size_t(parts(rows)) * 2 * D * sizeof(float); }

void norm_forward(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows,
                  int64_t D, int dt, int w_dt, int b_dt, float eps, hipStream_t st) {
  const Plan p = plan(D, dt, aligned({x, y}, 16), aligned({x, y}, 4));
  if (p.nv == 0) {
    auto* k = dt == DT_BF16 ? norm_fwd_long<DT_BF16> : norm_fwd_long<DT_F32>;
    hipLaunchKernelGGL(k, dim3(grid(rows)), dim3(kThreads), 0, st, x, w, b, y, mean, rstd, rows, D, w_dt, b_dt, eps);
    return;
  }
  with_plan(p, dt, [&](auto DT, auto V, auto NV, auto TPR) {
    constexpr int rpw = kThreads / TPR.value;
    hipLaunchKernelGGL((norm_fwd<DT.value, V.value, NV.value, TPR.value>),
                       dim3(grid((rows + rpw - 1) / rpw)), dim3(kThreads), 0, st, x, w, b, y, mean, rstd, rows,
                       static_cast<int>(D), w_dt, b_dt, eps);
  });
}

void norm_backward(const void* x, const void* w, const void* dy, const float* mean, const float* rstd, void* dx,
                   void* dw, void* db, int64_t rows, int64_t D, int dt, int w_dt, int b_dt, void* workspace,
                   hipStream_t st) {
  const Plan p = plan(D, dt, aligned({x, dy, dx}, 16), aligned({x, dy, dx}, 4));
  float* part = static_cast<float*>(workspace);
  const bool sums = dw != nullptr || db != nullptr;
  int64_t n = parts(rows);
  if (p.nv == 0) {
    if (dx != nullptr) {
      auto* k = dt == DT_BF16 ? norm_dx_long<DT_BF16> : norm_dx_long<DT_F32>;
      hipLaunchKernelGGL(k, dim3(grid(rows)), dim3(kThreads), 0, st, x, w, dy, mean, rstd, dx, rows, D, w_dt);
    }
    if (sums) {
      if (n > 64) n = 64;
      auto* k = dt == DT_BF16 ? norm_sums_long<DT_BF16> : norm_sums_long<DT_F32>;
      hipLaunchKernelGGL(k, dim3(static_cast<unsigned>((D + kThreads - 1) / kThreads), static_cast<unsigned>(n)),
                         dim3(kThreads), 0, st, x, dy, mean, rstd, part, rows, D);
    }
  } else {
    with_plan(p, dt, [&](auto DT, auto V, auto NV, auto TPR) {
      constexpr int rpw = kThreads / TPR.value;
      const int64_t wgs = (rows + rpw - 1) / rpw;
      if (wgs < n) n = wgs;
      const size_t lds = TPR.value == kThreads ? 0 : size_t(2 * D) * sizeof(float);
      auto* k = sums ? norm_bwd<DT.value, V.value, NV.value, TPR.value, true>
                     : norm_bwd<DT.value, V.value, NV.value, TPR.value, false>;
      hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(n)), dim3(kThreads), sums ? lds : 0, st, x, w, dy, mean, rstd,
                         dx, part, rows, static_cast<int>(D), w_dt);
    });
  }
  if (sums) launch_column_sums({part, n, D, D, 0, dw, db, nullptr, w_dt, b_dt, 0}, st);
}

}  // namespace moc
