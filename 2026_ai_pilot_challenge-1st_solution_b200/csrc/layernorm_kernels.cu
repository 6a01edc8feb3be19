// layernorm_kernels.cu -- layer norm over the last axis, forward and backward.
//
// Forward, per row:  mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), y = (x - mu) r w + b.
// Backward, per row: with xh = (x - mu) r and g = dy w,
//   dx = r (g - mean(g) - xh mean(g xh)),   dw = sum over rows of dy xh,   db = sum over rows of dy.
//
// Both passes are bound by HBM: a row is read once into registers and everything is computed from
// there (the variance from the centred values, so that a mean far from zero costs no digits).
// `lanes` threads share a row -- a power of two, the fewest whose registers hold it -- so narrow
// rows share a warp and wide rows take a block.  Blocks are persistent: weights stay in registers
// over all rows of a block, the next row is loaded while the current one is reduced, and in the
// backward pass so do the columns' partial sums of dw and db, which leave the block once, to be
// added up by k_ln_wgrad in a fixed order (no atomics: the same inputs give the same gradients).
// Sums, statistics and partial sums are fp32; values are rounded once, when stored.
#include "typed.cuh"

namespace f16 {
namespace ln {

constexpr int BLOCK = 256;          // threads of a block whose rows take a warp or less
constexpr int MAX_LANES = 512;     // threads of a row: 128 registers each
constexpr int E = 16;               // most values of a row in one thread
constexpr int WIDE = 1024;          // threads of a block on a row too wide for registers

struct Weights {
  const void* w;
  const void* b;
  int dtype;
};

__device__ __forceinline__ float load_as_f32(const void* p, int dtype, int64_t i) {
  if (dtype == F16_DTYPE_FP32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == F16_DTYPE_BF16) return to_f32(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return to_f32(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_from_f32(void* p, int dtype, int64_t i, float v) {
  if (dtype == F16_DTYPE_FP32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == F16_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
  else reinterpret_cast<__half*>(p)[i] = from_f32<__half>(v);
}

// Sum over the `lanes` threads of a row (xor shuffles: every thread gets the same bits).  Rows wider
// than a warp take the whole block and `red`; consecutive calls alternate its halves, so one barrier
// a call is enough.
__device__ __forceinline__ float row_sum(float v, int lanes, float (*red)[32], int& half) {
  const int w = lanes < 32 ? lanes : 32;
  for (int o = w >> 1; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if (lanes > 32) {
    float* r = red[half];
    half ^= 1;
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    const int n = lanes >> 5, l = threadIdx.x & 31;
    v = l < n ? r[l] : 0.0f;
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  }
  return v;
}

template <typename T, int V, int NV>
__device__ __forceinline__ void load_row(Vec<T, V> (&v)[NV], const T* row, bool live, int lane, int lanes, int cols) {
#pragma unroll
  for (int j = 0; j < NV; j++) {
    const int c = (j * lanes + lane) * V;
    if (live && c < cols) {
      v[j] = load_vec_nc<T, V>(row + c);
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) v[j].e[k] = from_f32<T>(0.0f);
    }
  }
}

template <typename T, int V, int NV>
__global__ void __launch_bounds__(MAX_LANES)
    k_ln_fwd(const T* __restrict__ x, int64_t ldx, int64_t rows, int cols, Weights wb, float eps, T* __restrict__ y,
             int64_t ldy, float* __restrict__ mean, float* __restrict__ rstd, int lanes) {
  __shared__ float red[2][32];
  int half = 0;
  const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, per = blockDim.x / lanes;
  const int64_t step = (int64_t)gridDim.x * per;
  float w[NV][V], b[NV][V];
#pragma unroll
  for (int j = 0; j < NV; j++)
#pragma unroll
    for (int k = 0; k < V; k++) {
      const int c = (j * lanes + lane) * V + k;
      w[j][k] = wb.w && c < cols ? load_as_f32(wb.w, wb.dtype, c) : 1.0f;
      b[j][k] = wb.b && c < cols ? load_as_f32(wb.b, wb.dtype, c) : 0.0f;
    }
  Vec<T, V> next[NV];
  int64_t r0 = (int64_t)blockIdx.x * per;
  load_row<T, V, NV>(next, x + (r0 + group) * ldx, r0 + group < rows, lane, lanes, cols);
  const float inv = 1.0f / (float)cols;
  for (; r0 < rows; r0 += step) {
    const int64_t row = r0 + group;
    const bool live = row < rows;
    float v[NV][V], s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int k = 0; k < V; k++) {
        v[j][k] = to_f32(next[j].e[k]);
        s += v[j][k];
      }
    load_row<T, V, NV>(next, x + (row + step) * ldx, row + step < rows, lane, lanes, cols);
    const float mu = row_sum(s, lanes, red, half) * inv;
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int k = 0; k < V; k++) {
        v[j][k] -= mu;
        if ((j * lanes + lane) * V < cols) q = fmaf(v[j][k], v[j][k], q);
      }
    const float r = 1.0f / sqrtf(row_sum(q, lanes, red, half) * inv + eps);
    if (!live) continue;
    if (lane == 0 && mean) {
      mean[row] = mu;
      rstd[row] = r;
    }
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int c = (j * lanes + lane) * V;
      Vec<T, V> o;
#pragma unroll
      for (int k = 0; k < V; k++) o.e[k] = from_f32<T>(fmaf(v[j][k] * r, w[j][k], b[j][k]));
      if (c < cols) store_vec<T, V>(y + row * ldy + c, o);
    }
  }
}

// Backward of the rows of one block, and its columns' sums part[block][0][cols] (dw) and
// part[block][1][cols] (db).  dx or part may be null.
template <typename T, int V, int NV>
__global__ void __launch_bounds__(MAX_LANES)
    k_ln_bwd(const T* __restrict__ dy, int64_t ldg, const T* __restrict__ x, int64_t ldx, int64_t rows, int cols,
             Weights wb, const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
             int64_t ldd, float* __restrict__ part, int lanes) {
  __shared__ float red[2][32];
  extern __shared__ float col_sum[];            // 2 cols floats where several rows share the block
  int half = 0;
  const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, per = blockDim.x / lanes;
  const int64_t step = (int64_t)gridDim.x * per;
  float w[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
  for (int j = 0; j < NV; j++)
#pragma unroll
    for (int k = 0; k < V; k++) {
      const int c = (j * lanes + lane) * V + k;
      w[j][k] = wb.w && c < cols ? load_as_f32(wb.w, wb.dtype, c) : 1.0f;
      aw[j][k] = ab[j][k] = 0.0f;
    }
  Vec<T, V> nx[NV], ng[NV];
  float nmu = 0.0f, nr = 0.0f;
  int64_t r0 = (int64_t)blockIdx.x * per;
  const auto fetch = [&](int64_t row) {
    const bool live = row < rows;
    load_row<T, V, NV>(nx, x + row * ldx, live, lane, lanes, cols);
    load_row<T, V, NV>(ng, dy + row * ldg, live, lane, lanes, cols);
    nmu = live ? mean[row] : 0.0f;
    nr = live ? rstd[row] : 0.0f;
  };
  fetch(r0 + group);
  const float inv = 1.0f / (float)cols;
  for (; r0 < rows; r0 += step) {
    const int64_t row = r0 + group;
    const bool live = row < rows;
    const float mu = nmu, r = nr;
    Vec<T, V> cx[NV], cg[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
      cx[j] = nx[j];
      cg[j] = ng[j];
    }
    fetch(row + step);
    float s1 = 0.0f, s2 = 0.0f;
    if (live) {
#pragma unroll
      for (int j = 0; j < NV; j++)
        if ((j * lanes + lane) * V < cols) {
#pragma unroll
          for (int k = 0; k < V; k++) {
            const float xh = (to_f32(cx[j].e[k]) - mu) * r, d = to_f32(cg[j].e[k]), g = d * w[j][k];
            s1 += g;
            s2 = fmaf(g, xh, s2);
            aw[j][k] = fmaf(d, xh, aw[j][k]);
            ab[j][k] += d;
          }
        }
    }
    if (!dx) continue;
    const float m1 = row_sum(s1, lanes, red, half) * inv, m2 = row_sum(s2, lanes, red, half) * inv;
    if (!live) continue;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int c = (j * lanes + lane) * V;
      Vec<T, V> o;
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float xh = (to_f32(cx[j].e[k]) - mu) * r, g = to_f32(cg[j].e[k]) * w[j][k];
        o.e[k] = from_f32<T>(r * (g - m1 - xh * m2));
      }
      if (c < cols) store_vec<T, V>(dx + row * ldd + c, o);
    }
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * cols;
  if (per == 1) {
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int k = 0; k < V; k++) {
        const int c = (j * lanes + lane) * V + k;
        if (c < cols) {
          out[c] = aw[j][k];
          out[cols + c] = ab[j][k];
        }
      }
    return;
  }
  // rows of one warp first (shuffles), then the warps in turn
#pragma unroll
  for (int j = 0; j < NV; j++)
#pragma unroll
    for (int k = 0; k < V; k++)
      for (int o = 16; o >= lanes; o >>= 1) {
        aw[j][k] += __shfl_xor_sync(~0u, aw[j][k], o);
        ab[j][k] += __shfl_xor_sync(~0u, ab[j][k], o);
      }
  for (int turn = 0; turn < (int)(blockDim.x >> 5); turn++) {
    if ((int)(threadIdx.x >> 5) == turn && (int)(threadIdx.x & 31) < lanes) {
#pragma unroll
      for (int j = 0; j < NV; j++)
#pragma unroll
        for (int k = 0; k < V; k++) {
          const int c = (j * lanes + lane) * V + k;
          if (c < cols) {
            col_sum[c] = turn ? col_sum[c] + aw[j][k] : aw[j][k];
            col_sum[cols + c] = turn ? col_sum[cols + c] + ab[j][k] : ab[j][k];
          }
        }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < 2 * cols; c += blockDim.x) out[c] = col_sum[c];
}

// Rows too wide for a block's registers: a block a row, read again for each of the three passes (the
// second and third hit L2).
template <typename T>
__global__ void __launch_bounds__(WIDE)
    k_ln_fwd_wide(const T* __restrict__ x, int64_t ldx, int64_t rows, int cols, Weights wb, float eps,
                  T* __restrict__ y, int64_t ldy, float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float red[2][32];
  int half = 0;
  const float inv = 1.0f / (float)cols;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s = 0.0f, q = 0.0f;
    for (int c = threadIdx.x; c < cols; c += WIDE) s += to_f32(xr[c]);
    const float mu = row_sum(s, WIDE, red, half) * inv;
    for (int c = threadIdx.x; c < cols; c += WIDE) {
      const float d = to_f32(xr[c]) - mu;
      q = fmaf(d, d, q);
    }
    const float r = 1.0f / sqrtf(row_sum(q, WIDE, red, half) * inv + eps);
    if (threadIdx.x == 0 && mean) {
      mean[row] = mu;
      rstd[row] = r;
    }
    for (int c = threadIdx.x; c < cols; c += WIDE) {
      const float w = wb.w ? load_as_f32(wb.w, wb.dtype, c) : 1.0f, b = wb.b ? load_as_f32(wb.b, wb.dtype, c) : 0.0f;
      y[row * ldy + c] = from_f32<T>(fmaf((to_f32(xr[c]) - mu) * r, w, b));
    }
  }
}

// Its backward: every thread keeps its columns' sums in the block's row of `part`.
template <typename T>
__global__ void __launch_bounds__(WIDE)
    k_ln_bwd_wide(const T* __restrict__ dy, int64_t ldg, const T* __restrict__ x, int64_t ldx, int64_t rows, int cols,
                  Weights wb, const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
                  int64_t ldd, float* part) {
  __shared__ float red[2][32];
  int half = 0;
  const float inv = 1.0f / (float)cols;
  float* out = part ? part + (int64_t)blockIdx.x * 2 * cols : nullptr;
  bool first = true;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, first = false) {
    const float mu = mean[row], r = rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < cols; c += WIDE) {
      const float d = to_f32(dy[row * ldg + c]), xh = (to_f32(x[row * ldx + c]) - mu) * r;
      const float g = wb.w ? d * load_as_f32(wb.w, wb.dtype, c) : d;
      s1 += g;
      s2 = fmaf(g, xh, s2);
      if (out) {
        out[c] = first ? d * xh : fmaf(d, xh, out[c]);
        out[cols + c] = first ? d : out[cols + c] + d;
      }
    }
    if (!dx) continue;
    const float m1 = row_sum(s1, WIDE, red, half) * inv, m2 = row_sum(s2, WIDE, red, half) * inv;
    for (int c = threadIdx.x; c < cols; c += WIDE) {
      const float xh = (to_f32(x[row * ldx + c]) - mu) * r;
      const float g = to_f32(dy[row * ldg + c]) * (wb.w ? load_as_f32(wb.w, wb.dtype, c) : 1.0f);
      dx[row * ldd + c] = from_f32<T>(r * (g - m1 - xh * m2));
    }
  }
}

// dw and db from the blocks' partial sums: 32 columns a block, 32 threads a column, in a fixed order.
__global__ void __launch_bounds__(1024) k_ln_wgrad(const float* __restrict__ part, int nblk, int cols, void* dw, void* db,
                                                   int dtype) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float v = 0.0f;
  if (c < 2 * cols)
    for (int r = threadIdx.y; r < nblk; r += 32) v += part[(int64_t)r * 2 * cols + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = s[threadIdx.x][threadIdx.y];
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && col < 2 * cols) {
    if (col < cols) {
      if (dw) store_from_f32(dw, dtype, col, v);
    } else if (db) {
      store_from_f32(db, dtype, col - cols, v);
    }
  }
}

// How a row is spread: V values a load, NV loads and `lanes` threads a row; nv 0: the wide kernels.
struct Plan {
  int v, nv, lanes, threads;
};

inline int pow2_up(int n) {
  int p = 1;
  while (p < n) p <<= 1;
  return p;
}

inline Plan plan_for(int cols, int v) {
  Plan p;
  p.v = v;
  const int vecs = (cols + v - 1) / v;
  // one value a load: 8 of them, so that a warp's request covers 32 neighbours before a row is
  // spread over more of a thread's registers
  const int most = v == 1 ? 8 : E / v;
  p.lanes = pow2_up((vecs + most - 1) / most);
  if (p.lanes > MAX_LANES) {
    p.lanes = MAX_LANES;
    p.nv = pow2_up((vecs + MAX_LANES - 1) / MAX_LANES);
    if (p.nv * v > E) p.nv = 0;
  } else {
    p.nv = pow2_up((vecs + p.lanes - 1) / p.lanes);
  }
  p.threads = p.lanes > 32 ? p.lanes : BLOCK;
  return p;
}

// Widest vector (in values of `size` bytes) that every row start allows: 16 bytes, two values, one.
inline int vec_for(int cols, int size, const void* const* ptrs, const int64_t* lds, int n) {
  const int widths[2] = {16 / size, 2};
  for (int w : widths) {
    bool ok = cols % w == 0;
    for (int i = 0; i < n && ok; i++) ok = !ptrs[i] || (aligned(ptrs[i], (uintptr_t)w * size) && lds[i] % w == 0);
    if (ok) return w;
  }
  return 1;
}

inline int64_t grid_rows(int64_t rows, const Plan& p, int warps_per_sm) {
  const int64_t per = p.threads / p.lanes, need = (rows + per - 1) / per;
  int64_t most = (int64_t)sm_count() * (warps_per_sm * 32 / p.threads > 0 ? warps_per_sm * 32 / p.threads : 1);
  return need < most ? need : most;
}

constexpr int FWD_WARPS = 32, BWD_WARPS = 16;    // persistent warps per SM

template <typename T>
int forward(const T* x, int64_t rows, int cols, int64_t ldx, Weights wb, float eps, T* y, int64_t ldy, float* mean,
            float* rstd, cudaStream_t st) {
  const void* ptrs[2] = {x, y};
  const int64_t lds[2] = {ldx, ldy};
  const Plan p = plan_for(cols, vec_for(cols, sizeof(T), ptrs, lds, 2));
  if (!p.nv) {
    const int64_t grid = rows < 2 * sm_count() ? rows : 2 * sm_count();
    k_ln_fwd_wide<T><<<(unsigned)grid, WIDE, 0, st>>>(x, ldx, rows, cols, wb, eps, y, ldy, mean, rstd);
    return launch_status();
  }
  const unsigned grid = (unsigned)grid_rows(rows, p, FWD_WARPS);
  const auto go = [&](auto k) {
    k<<<grid, p.threads, 0, st>>>(x, ldx, rows, cols, wb, eps, y, ldy, mean, rstd, p.lanes);
  };
  constexpr int VW = 16 / sizeof(T);
  if (p.v == VW) {
    if (p.nv == 1) go(k_ln_fwd<T, VW, 1>);
    else if (p.nv == 2) go(k_ln_fwd<T, VW, 2>);
    else if constexpr (VW == 4) go(k_ln_fwd<T, VW, 4>);
  } else if (p.v == 2) {
    if (p.nv == 1) go(k_ln_fwd<T, 2, 1>);
    else if (p.nv == 2) go(k_ln_fwd<T, 2, 2>);
    else if (p.nv == 4) go(k_ln_fwd<T, 2, 4>);
    else go(k_ln_fwd<T, 2, 8>);
  } else {
    if (p.nv == 1) go(k_ln_fwd<T, 1, 1>);
    else if (p.nv == 2) go(k_ln_fwd<T, 1, 2>);
    else if (p.nv == 4) go(k_ln_fwd<T, 1, 4>);
    else if (p.nv == 8) go(k_ln_fwd<T, 1, 8>);
    else go(k_ln_fwd<T, 1, 16>);
  }
  return launch_status();
}

template <typename T>
int backward(const T* dy, int64_t ldg, const T* x, int64_t ldx, int64_t rows, int cols, Weights wb, const float* mean,
             const float* rstd, T* dx, int64_t ldd, float* part, int64_t part_floats, void* dw, void* db,
             cudaStream_t st) {
  const void* ptrs[3] = {dy, x, dx};
  const int64_t lds[3] = {ldg, ldx, ldd};
  const Plan p = plan_for(cols, vec_for(cols, sizeof(T), ptrs, lds, 3));
  int64_t grid = p.nv ? grid_rows(rows, p, BWD_WARPS) : (rows < sm_count() ? rows : sm_count());
  if (part && grid > part_floats / (2 * (int64_t)cols)) grid = part_floats / (2 * (int64_t)cols);
  if (grid < 1) return F16_ERR_ARG;
  if (!p.nv) {
    k_ln_bwd_wide<T><<<(unsigned)grid, WIDE, 0, st>>>(dy, ldg, x, ldx, rows, cols, wb, mean, rstd, dx, ldd, part);
  } else {
    const size_t smem = part && p.threads > p.lanes ? 2 * (size_t)cols * sizeof(float) : 0;
    const auto go = [&](auto k) {
      k<<<(unsigned)grid, p.threads, smem, st>>>(dy, ldg, x, ldx, rows, cols, wb, mean, rstd, dx, ldd, part, p.lanes);
    };
    constexpr int VW = 16 / sizeof(T);
    if (p.v == VW) {
      if (p.nv == 1) go(k_ln_bwd<T, VW, 1>);
      else if (p.nv == 2) go(k_ln_bwd<T, VW, 2>);
      else if constexpr (VW == 4) go(k_ln_bwd<T, VW, 4>);
    } else if (p.v == 2) {
      if (p.nv == 1) go(k_ln_bwd<T, 2, 1>);
      else if (p.nv == 2) go(k_ln_bwd<T, 2, 2>);
      else if (p.nv == 4) go(k_ln_bwd<T, 2, 4>);
      else go(k_ln_bwd<T, 2, 8>);
    } else {
      if (p.nv == 1) go(k_ln_bwd<T, 1, 1>);
      else if (p.nv == 2) go(k_ln_bwd<T, 1, 2>);
      else if (p.nv == 4) go(k_ln_bwd<T, 1, 4>);
      else if (p.nv == 8) go(k_ln_bwd<T, 1, 8>);
      else go(k_ln_bwd<T, 1, 16>);
    }
  }
  const int rc = launch_status();
  if (rc != F16_OK || !part) return rc;
  k_ln_wgrad<<<(unsigned)((2 * (int64_t)cols + 31) / 32), dim3(32, 32), 0, st>>>(part, (int)grid, cols, dw, db, wb.dtype);
  return launch_status();
}

inline bool is_dtype(int t) { return t == F16_DTYPE_BF16 || t == F16_DTYPE_FP16 || t == F16_DTYPE_FP32; }
inline int size_of(int t) { return t == F16_DTYPE_FP32 ? 4 : 2; }

}  // namespace ln
}  // namespace f16

using namespace f16;

extern "C" int f16_layer_norm_fwd(const void* x, int64_t rows, int cols, int64_t ldx, int dtype, const void* weight,
                                  const void* bias, int wdtype, double eps, void* y, int64_t ldy, float* mean,
                                  float* rstd, f16_stream_t stream) {
  if (!x || !y || rows <= 0 || cols <= 0 || ldx < 0 || ldy < cols || !ln::is_dtype(dtype) || !ln::is_dtype(wdtype) ||
      !mean != !rstd || !(eps >= 0.0))
    return F16_ERR_ARG;
  if (!aligned(x, ln::size_of(dtype)) || !aligned(y, ln::size_of(dtype)) || !aligned(weight, ln::size_of(wdtype)) ||
      !aligned(bias, ln::size_of(wdtype)))
    return F16_ERR_ALIGN;
  const ln::Weights wb = {weight, bias, wdtype};
  const cudaStream_t st = cu_stream(stream);
  if (dtype == F16_DTYPE_FP32)
    return ln::forward((const float*)x, rows, cols, ldx, wb, (float)eps, (float*)y, ldy, mean, rstd, st);
  if (dtype == F16_DTYPE_BF16)
    return ln::forward((const __nv_bfloat16*)x, rows, cols, ldx, wb, (float)eps, (__nv_bfloat16*)y, ldy, mean, rstd, st);
  return ln::forward((const __half*)x, rows, cols, ldx, wb, (float)eps, (__half*)y, ldy, mean, rstd, st);
}

extern "C" int64_t f16_layer_norm_scratch_floats(int64_t rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  // no block has less than one row, no SM more backward blocks than its warps allow
  const int64_t most = (int64_t)sm_count() * (ln::BWD_WARPS / 2);
  return 2 * (int64_t)cols * (rows < most ? rows : most);
}

extern "C" int f16_layer_norm_bwd(const void* dy, int64_t ldg, const void* x, int64_t ldx, int64_t rows, int cols,
                                  int dtype, const void* weight, int wdtype, const float* mean, const float* rstd,
                                  void* dx, int64_t ldd, void* dweight, void* dbias, float* scratch,
                                  int64_t scratch_floats, f16_stream_t stream) {
  if (!dy || !x || !mean || !rstd || rows <= 0 || cols <= 0 || ldg < 0 || ldx < 0 || (dx && ldd < cols) ||
      !ln::is_dtype(dtype) || !ln::is_dtype(wdtype))
    return F16_ERR_ARG;
  const bool sums = dweight || dbias;
  if (!dx && !sums) return F16_OK;
  if (sums && (!scratch || scratch_floats < 2 * (int64_t)cols)) return F16_ERR_ARG;
  const int size = ln::size_of(dtype);
  if (!aligned(dy, size) || !aligned(x, size) || !aligned(dx, size) || !aligned(weight, ln::size_of(wdtype)))
    return F16_ERR_ALIGN;
  const ln::Weights wb = {weight, nullptr, wdtype};
  float* part = sums ? scratch : nullptr;
  const cudaStream_t st = cu_stream(stream);
  if (dtype == F16_DTYPE_FP32)
    return ln::backward((const float*)dy, ldg, (const float*)x, ldx, rows, cols, wb, mean, rstd, (float*)dx, ldd, part,
                        scratch_floats, dweight, dbias, st);
  if (dtype == F16_DTYPE_BF16)
    return ln::backward((const __nv_bfloat16*)dy, ldg, (const __nv_bfloat16*)x, ldx, rows, cols, wb, mean, rstd,
                        (__nv_bfloat16*)dx, ldd, part, scratch_floats, dweight, dbias, st);
  return ln::backward((const __half*)dy, ldg, (const __half*)x, ldx, rows, cols, wb, mean, rstd, (__half*)dx, ldd, part,
                      scratch_floats, dweight, dbias, st);
}
