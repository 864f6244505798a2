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
//
// 16384 bf16 rows of 2048: forward 27.5 us (4.9 TB/s), backward 44 (4.6 TB/s of x, dy and
// dx), sums 4: the rate of a large copy.  5001 fp32 rows of 1131, an odd length: 15 and 25.
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

// A row's NV vectors of a lane; TAIL: the last one may end behind the row.
template <int DT, int V, int NV, int TPR, bool TAIL>
struct Row {
  RawVec<DT, V> r[NV];
  __device__ __forceinline__ void load(const void* p, int64_t row, int D, int lane, bool live) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      const int n = live ? D - c : 0;
      if (TAIL) {
        r[i].load(p, row * D + c, n);
      } else if (n > 0) {
        r[i].load(p, row * D + c, V);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) r[i].e[k] = 0;
      }
    }
  }
};

// Rows are walked a grid apart with the weights in registers and the next row's loads in
// flight: a workgroup a row would read w and b, twice a bf16 row's bytes, for each of them.
template <int DT, int V, int NV, int TPR, bool TAIL>
__global__ __launch_bounds__(kThreads) void norm_fwd(const void* __restrict__ x, const void* __restrict__ w,
                                                     const void* __restrict__ b, void* __restrict__ y,
                                                     float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                     int64_t rows, int D, int w_dt, int b_dt, float eps) {
  __shared__ float buf[4];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  constexpr int RPW = kThreads / TPR;
  const float inv = 1.0f / static_cast<float>(D);
  const int64_t step = int64_t(gridDim.x) * RPW;
  int64_t row = int64_t(blockIdx.x) * RPW + group;
  Row<DT, V, NV, TPR, TAIL> next;
  next.load(x, row, D, lane, row < rows);
  float wv[NV][V], bv[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * V;
    if (c < D) {
      load_param<V>(w, w_dt, c, TAIL ? D - c : V, 1.f, wv[i]);
      load_param<V>(b, b_dt, c, TAIL ? D - c : V, 0.f, bv[i]);
    }
  }
  // (every lane runs every round: a row of a whole workgroup has barriers in it)
  for (; row - group < rows; row += step) {
    const bool live = row < rows;
    float v[NV][V];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      next.r[i].get(v[i]);
#pragma unroll
      for (int k = 0; k < V; ++k) s += v[i][k];
    }
    next.load(x, row + step, D, lane, row + step < rows);
    // (a true quotient: a mean of equal elements is that element)
    const float mean = row_sum<TPR>(s, buf) / static_cast<float>(D);
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int have = D - (i * TPR + lane) * V;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        v[i][k] = (TAIL ? k < have : have > 0) ? v[i][k] - mean : 0.f;
        s += v[i][k] * v[i][k];
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
#pragma unroll
      for (int k = 0; k < V; ++k) v[i][k] = v[i][k] * rstd * wv[i][k] + bv[i][k];
      store_vec<DT, V>(y, row * D + c, TAIL ? D - c : V, v[i]);
    }
  }
}

// part[blockIdx.x] = [dw | db] of the workgroup's rows.
template <int DT, int V, int NV, int TPR, bool TAIL, bool SUMS>
__global__ __launch_bounds__(kThreads) void norm_bwd(const void* __restrict__ x, const void* __restrict__ w,
                                                     const void* __restrict__ dy, const float* __restrict__ mean_in,
                                                     const float* __restrict__ rstd_in, void* __restrict__ dx,
                                                     float* __restrict__ part, int64_t rows, int D, int w_dt) {
  extern __shared__ float lds[];  // TPR < 256: [2][D] sums of the workgroup's row groups
  __shared__ float buf[4];
  constexpr int RPW = kThreads / TPR;
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.0f / static_cast<float>(D);
  const int64_t step = int64_t(gridDim.x) * RPW;
  int64_t row = int64_t(blockIdx.x) * RPW + group;
  Row<DT, V, NV, TPR, TAIL> nx, ng;
  float mean_n = 0.f, rstd_n = 0.f;
  auto fetch = [&](int64_t r) {
    const bool live = r < rows;
    nx.load(x, r, D, lane, live);
    ng.load(dy, r, D, lane, live);
    mean_n = live ? mean_in[r] : 0.f;
    rstd_n = live ? rstd_in[r] : 0.f;
  };
  fetch(row);
  float dw[NV][V], db[NV][V], wv[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * V;
#pragma unroll
    for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = wv[i][k] = 0.f;
    if (c < D) load_param<V>(w, w_dt, c, TAIL ? D - c : V, 1.f, wv[i]);
  }
  // (every lane runs every round: a row of a whole workgroup has barriers in it)
  for (; row - group < rows; row += step) {
    const float mean = mean_n, rstd = rstd_n;
    float xh[NV][V], g[NV][V];
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      nx.r[i].get(xh[i]);
      ng.r[i].get(g[i]);
    }
    fetch(row + step);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        // (past the row's end, or the last row, x reads as 0 and g too: it adds nothing)
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
    if (row >= rows) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      if (c >= D) continue;
#pragma unroll
      for (int k = 0; k < V; ++k) g[i][k] = rstd * (g[i][k] - s0 - xh[i][k] * s1);
      store_vec<DT, V>(dx, row * D + c, TAIL ? D - c : V, g[i]);
    }
  }
  if (!SUMS) return;
  float* out = part + int64_t(blockIdx.x) * 2 * D;
  float* to = TPR == kThreads ? out : lds;
  for (int q = 0; q < RPW; ++q) {  // row groups in order
    if (group == q) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * V;
        if (c >= D) continue;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          if (TAIL && c + k >= D) continue;
          to[c + k] = q == 0 ? dw[i][k] : to[c + k] + dw[i][k];
          to[D + c + k] = q == 0 ? db[i][k] : to[D + c + k] + db[i][k];
        }
      }
    }
    if (TPR < kThreads) __syncthreads();
  }
  if (TPR < kThreads)
    for (int c = threadIdx.x; c < 2 * D; c += kThreads) out[c] = lds[c];
}

// Rows too long for a workgroup's registers (past 16384 bf16 or 8192 fp32 elements, wider than
// any stream that the layers next to it are run on): the row is read again for each sum, an
// element a lane and load.  2048 rows of 16392 bf16 elements 110 us forward and 247 with the
// backward, where 16384 take 49 and 154; of 8196 fp32 elements 46 and 130, of 8192 22 and 79.
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

template <int V>
using Int = std::integral_constant<int, V>;

// How a row is spread: TPR lanes of NV vectors of 16 bytes.
struct Plan {
  int nv, tpr;  // nv 0: the long kernels
};

// A row of up to 16 vectors takes 16 lanes (four rows a wave, where a wave a row would
// leave most lanes idle), up to 4 vectors a lane a wave, more of it the workgroup, whose
// sums have two barriers each.  16384 bf16 rows of 2048 (4 vectors a lane): a wave 28 us
// forward and 45 backward, the workgroup 31 and 60; 5001 fp32 rows of 1131, 5 vectors a
// lane in a wave: 18 and 38 us, the workgroup 15 and 25.
Plan plan(int64_t D, int dt) {
  const int v = dt == DT_BF16 ? 8 : 4;
  const int64_t n = (D + v - 1) / v;
  if (n <= 16) return {1, 16};
  const int tpr = n <= 4 * 64 ? 64 : 256;
  const int64_t nv = (n + tpr - 1) / tpr;
  return {nv <= 1 ? 1 : (nv <= 2 ? 2 : (nv <= 4 ? 4 : (nv <= 8 ? 8 : 0))), tpr};
}

template <typename F>
void with_plan(const Plan& p, int dt, int64_t D, F&& f) {
#define MOC_NORM_CASE(DT, V, NV, TPR) \
  if (dt == DT && p.nv == NV && p.tpr == TPR) { \
    if (D % V == 0) f(Int<DT>{}, Int<V>{}, Int<NV>{}, Int<TPR>{}, std::false_type{}); \
    else f(Int<DT>{}, Int<V>{}, Int<NV>{}, Int<TPR>{}, std::true_type{}); \
    return; \
  }
#define MOC_NORM_TYPE(DT, V) \
  MOC_NORM_CASE(DT, V, 1, 16) MOC_NORM_CASE(DT, V, 1, 64) MOC_NORM_CASE(DT, V, 2, 64) MOC_NORM_CASE(DT, V, 4, 64) \
  MOC_NORM_CASE(DT, V, 2, 256) MOC_NORM_CASE(DT, V, 4, 256) MOC_NORM_CASE(DT, V, 8, 256)
  MOC_NORM_TYPE(DT_BF16, 8) MOC_NORM_TYPE(DT_F32, 4)
#undef MOC_NORM_TYPE
#undef MOC_NORM_CASE
}

// Workgroups of the forward: four a CU, or what the rows give; of the long kernels: a row
// each, as long as a grid counts them.
constexpr int64_t kWalkers = 1024;
unsigned grid(int64_t n, int64_t most) { return static_cast<unsigned>(n < most ? n : most); }

// Workgroups of the backward, and rows of partial sums: two a CU, or what the rows
// give; of the long kernels 64 (a column a lane, so that the columns fill the card).
constexpr int64_t kParts = 512, kPartsLong = 64;

int64_t parts(int64_t rows, int64_t D, int dt) {
  const int64_t most = plan(D, dt).nv == 0 ? kPartsLong : kParts;
  return rows < most ? rows : most;
}

__global__ __launch_bounds__(1024) void column_sums(ColumnSums a) {
  __shared__ float s[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int64_t cols = a.n0 + a.n1 + a.n2;
  for (int64_t c0 = int64_t(blockIdx.x) * 32; c0 < cols; c0 += int64_t(gridDim.x) * 32) {
    const int64_t c = c0 + cx;
    float v = 0.f;
    if (c < cols) {
#pragma unroll 4
      for (int64_t r = ry; r < a.n; r += 32) v += a.part[r * cols + c];
    }
    __syncthreads();  // (the last columns have been read)
    s[ry][cx] = v;
    __syncthreads();
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
      if (ry < m) s[ry][cx] += s[ry + m][cx];
      __syncthreads();
    }
    if (ry != 0 || c >= cols) continue;
    if (c < a.n0) {
      if (a.out0 != nullptr) store_any(a.out0, a.dt0, c, s[0][cx]);
    } else if (c < a.n0 + a.n1) {
      if (a.out1 != nullptr) store_any(a.out1, a.dt1, c - a.n0, s[0][cx]);
    } else if (a.out2 != nullptr) {
      store_any(a.out2, a.dt2, c - a.n0 - a.n1, s[0][cx]);
    }
  }
}

}  // namespace

void launch_column_sums(const ColumnSums& c, hipStream_t st) {
  const int64_t cols = c.n0 + c.n1 + c.n2;
  // (a grid counts threads in 32 bits: 2^27 columns would pass it)
  hipLaunchKernelGGL(column_sums, dim3(grid((cols + 31) / 32, 1 << 16)), dim3(1024), 0, st, c);
}

size_t norm_backward_workspace(int64_t rows, int64_t D) {
  // (for either type: fp32's rows end in the long kernels first)
  return size_t(parts(rows, D, DT_BF16)) * 2 * D * sizeof(float);
}

void norm_forward(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows,
                  int64_t D, int dt, int w_dt, int b_dt, float eps, hipStream_t st) {
  const Plan p = plan(D, dt);
  if (p.nv == 0) {
    auto* k = dt == DT_BF16 ? norm_fwd_long<DT_BF16> : norm_fwd_long<DT_F32>;
    hipLaunchKernelGGL(k, dim3(grid(rows, 1 << 22)), dim3(kThreads), 0, st, x, w, b, y, mean, rstd, rows, D, w_dt, b_dt, eps);
    return;
  }
  with_plan(p, dt, D, [&](auto DT, auto V, auto NV, auto TPR, auto TAIL) {
    constexpr int rpw = kThreads / TPR.value;
    hipLaunchKernelGGL((norm_fwd<DT.value, V.value, NV.value, TPR.value, TAIL.value>),
                       dim3(grid((rows + rpw - 1) / rpw, kWalkers)), dim3(kThreads), 0, st, x, w, b, y, mean, rstd, rows,
                       static_cast<int>(D), w_dt, b_dt, eps);
  });
}

void norm_backward(const void* x, const void* w, const void* dy, const float* mean, const float* rstd, void* dx,
                   void* dw, void* db, int64_t rows, int64_t D, int dt, int w_dt, int b_dt, void* workspace,
                   hipStream_t st) {
  const Plan p = plan(D, dt);
  float* part = static_cast<float*>(workspace);
  const bool sums = dw != nullptr || db != nullptr;
  int64_t n = parts(rows, D, dt);
  if (p.nv == 0) {
    if (dx != nullptr) {
      auto* k = dt == DT_BF16 ? norm_dx_long<DT_BF16> : norm_dx_long<DT_F32>;
      hipLaunchKernelGGL(k, dim3(grid(rows, 1 << 22)), dim3(kThreads), 0, st, x, w, dy, mean, rstd, dx, rows, D, w_dt);
    }
    if (sums) {
      auto* k = dt == DT_BF16 ? norm_sums_long<DT_BF16> : norm_sums_long<DT_F32>;
      hipLaunchKernelGGL(k, dim3(static_cast<unsigned>((D + kThreads - 1) / kThreads), static_cast<unsigned>(n)),
                         dim3(kThreads), 0, st, x, dy, mean, rstd, part, rows, D);
    }
  } else {
    with_plan(p, dt, D, [&](auto DT, auto V, auto NV, auto TPR, auto TAIL) {
      constexpr int rpw = kThreads / TPR.value;
      const int64_t wgs = (rows + rpw - 1) / rpw;
      if (wgs < n) n = wgs;
      const size_t lds = TPR.value == kThreads ? 0 : size_t(2 * D) * sizeof(float);
      auto* k = sums ? norm_bwd<DT.value, V.value, NV.value, TPR.value, TAIL.value, true>
                     : norm_bwd<DT.value, V.value, NV.value, TPR.value, TAIL.value, false>;
      hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(n)), dim3(kThreads), sums ? lds : 0, st, x, w, dy, mean, rstd,
                         dx, part, rows, static_cast<int>(D), w_dt);
    });
  }
  if (sums) launch_column_sums({part, n, D, D, 0, dw, db, nullptr, w_dt, b_dt, 0}, st);
}

}  // namespace moc
