// layernorm_kernels.cu -- layer norm over the last axis, forward and backward.
//
// Forward, per row:  mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), y = (x - mu) r w + b.
// Backward, per row: with xh = (x - mu) r and g = dy w,
//   dx = r (g - mean(g) - xh mean(g xh)),   dw = sum over rows of dy xh,   db = sum over rows of dy.
//
// Both passes are bound by HBM: a row is read once into registers and everything is computed from
// there.  The mean is kept in two parts, so that one far above the spread costs no digits and rows of one value
// give the bias (512 fp32 columns of 1e4 + N(0, 1) were off by 1e-3 with one rounded mean):
//  * fp32 rows: the sum is rounded many times; what the mean is off by is the mean of the centred values, summed
//    beside their squares and taken out of them (16,384 x 4,096 forward 94 us, 91 without);
//  * 16-bit rows: where the mean lies far above the spread all values are of one binade or two, and 2^13 fp16 or 2^16
//    bf16 ones of a binade add up exactly in fp32 (a block's last addition keeps its error, the wide kernel adds
//    its threads' sums of CHAIN values in fp64), so the remainder of the division is all there is to know: no second sum.
// `lanes` threads share a row -- a power of two up to a warp, whole warps beyond, the fewest whose registers
// hold it -- so narrow rows share a warp and wide rows take a block.  Blocks are persistent: weights stay in registers
// over all rows of a block, the next row is loaded while the current one is reduced, and in the
// backward pass so do the columns' partial sums of dw and db, which leave the block once, to be
// added up by k_ln_wgrad in a fixed order (no atomics: the same inputs give the same gradients).
// Sums, statistics and partial sums are fp32 (a thread's sum over its rows is one chain of additions: 221 of
// them at 524,288 x 512); values are rounded once, when stored.
//
// Rows of a warp or less: sums of products are made of products rounded by themselves (pairs of values are multiplied by adding a
// zero that the assembler does not know to be one; it would fuse the product with the sum after it): what
// cancels in the formulas then cancels in fp32 -- a row of one value has no gradient, of two values hardly one.
//
// Measured on a B200 whose copy makes 6.55 TB/s, with a cold L2 (forward / backward / k_ln_wgrad, us, and the
// share of that rate): 524,288 x 512 fp32 354 / 521 / 4 (93%, 94%); 16,384 x 4,096 bf16 46 / 80 / 4 (88%, 77%);
// 100,003 x 215 fp16, in loads of 2 bytes, 30 / 42 / 3 (44%, 47%); 128 x 184 fp32, forward alone, 3.4.
#include "typed.cuh"

namespace f16 {
namespace ln {

constexpr int BLOCK = 256;          // threads of a block whose rows take a warp or less
constexpr int MAX_LANES = 512, FWD_LANES = 768;      // threads of a row, at most: see most_of
// Most values of a row in one thread.  16-byte loads take so many; with narrower ones a thread takes 8, of rows
// up to 16 values 4 (500,000 x 33 fp16, forward + backward: 8 a thread 107 us, 4 149 us;
// 300,000 x 15 bf16: 29 and 28 us), and 16 again where 8 do not suffice.
constexpr int MOST = 16;
constexpr int MAX_COLS = 1 << 29;   // column indexes are 32-bit
constexpr int WIDE = 512, WIDE_PER_SM = 3;      // threads of a block on a row too wide for registers, blocks on an SM
constexpr int CHAIN = 256;          // values that a thread adds up in fp32 there

// What a forward pass leaves for the backward one, a value a row each: the mean as mean + rest (rest may be NULL:
// zero), and r.  Its rounding to one fp32 value, 2^-25 of the mean, would stand in xh as that part of the mean over
// the spread.
template <typename F>
struct Stats {
  F* mean;
  F* rest;
  F* rstd;
};

struct Weights {
  const void* w;
  const void* b;
  int dtype;
  float minus_zero;
};

// V of them from i on, a multiple of V: 16 bytes a load where the weights are aligned so.
template <int V, typename W>
__device__ __forceinline__ void load_weights_of(float (&w)[V], const W* p) {
  constexpr int N = 16 / (int)sizeof(W);
  if constexpr (V % 4 == 0) {
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      constexpr int M = V < N ? V : N;
#pragma unroll
      for (int j = 0; j < V; j += M) {
        const Vec<W, M> v = load_vec_nc<W, M>(p + j);
#pragma unroll
        for (int k = 0; k < M; k++) w[j + k] = to_f32(v.e[k]);
      }
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < V; k++) w[k] = to_f32(p[k]);
}
template <int V, typename W>
__device__ __forceinline__ void load_weights(float (&w)[V], const void* p, int64_t i, float none) {
  if (!p) {
#pragma unroll
    for (int k = 0; k < V; k++) w[k] = none;
  } else {
    load_weights_of<V>(w, reinterpret_cast<const W*>(p) + i);
  }
}
// f(a value of the weights' type).
template <typename F>
__device__ __forceinline__ void of_weights(int dtype, F f) {
  if (dtype == F16_DTYPE_FP32) f(0.0f);
  else if (dtype == F16_DTYPE_BF16) f(__nv_bfloat16());
  else f(__half());
}
__device__ __forceinline__ void store_from_f32(void* p, int dtype, int64_t i, float v) {
  if (dtype == F16_DTYPE_FP32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == F16_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
  else reinterpret_cast<__half*>(p)[i] = from_f32<__half>(v);
}

// Sums over the threads of a row (xor shuffles: every thread gets the same bits).  LANES: 1 to 16 at run
// time (0), 32, or a whole block (ROW_BLOCK), whose warps meet in `red`; consecutive calls alternate its
// halves, so one barrier a call is enough.  N: how many of the M values.
constexpr int ROW_BLOCK = 64;
// `low` gets the rounding error of the last addition between the warps of a block (Knuth's two-sum), where N is 1.
template <int LANES, int N, int M>
__device__ __forceinline__ void row_sums(float (&v)[M], int lanes, float (*red)[M][32], int& half, float* low = nullptr) {
  if constexpr (LANES == 0) {
    for (int o = lanes >> 1; o; o >>= 1)
#pragma unroll
      for (int k = 0; k < N; k++) v[k] += __shfl_xor_sync(~0u, v[k], o);
  } else {
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
      for (int k = 0; k < N; k++) v[k] += __shfl_xor_sync(~0u, v[k], o);
  }
  if constexpr (LANES == ROW_BLOCK) {
    float (*r)[32] = red[half];
    half ^= 1;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < N; k++) r[k][threadIdx.x >> 5] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = lane < warps ? r[k][lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
      for (int k = 0; k < N; k++) {
        const float other = __shfl_xor_sync(~0u, v[k], o), sum = v[k] + other;
        if (low && o == 1) {
          const float part = sum - v[k];
          *low = (v[k] - (sum - part)) + (other - part);
        }
        v[k] = sum;
      }
  }
}

// A thread's part of a row: NV loads of V values, `apart` values from one load to the next; bit j of `there`:
// load j lies in the row.  The others read as zero.
template <typename T, int V, int E>
struct Part {
  static constexpr int NV = E / V;
  Vec<T, V> v[NV];
  __device__ __forceinline__ void load(const T* p, int apart, unsigned there, bool full) {
    if (full) {
#pragma unroll
      for (int j = 0; j < NV; j++) v[j] = load_vec_nc<T, V>(p + j * apart);
    } else {
#pragma unroll
      for (int j = 0; j < NV; j++) {
        if (there >> j & 1) {
          v[j] = load_vec_nc<T, V>(p + j * apart);
        } else {
#pragma unroll
          for (int k = 0; k < V; k++) v[j].e[k] = from_f32<T>(0.0f);
        }
      }
    }
  }
  // The pair i of the thread's E values, and the way back.
  __device__ __forceinline__ Two pair(int i) const {
    if constexpr (V == 1) return two(to_f32(v[2 * i].e[0]), to_f32(v[2 * i + 1].e[0]));
    else return pair_of<T, V>(v[2 * i / V], i % (V / 2));
  }
  __device__ __forceinline__ void set(int i, Two t) {
    if constexpr (V == 1) {
      const float2 f = split(t);
      v[2 * i].e[0] = from_f32<T>(f.x);
      v[2 * i + 1].e[0] = from_f32<T>(f.y);
    } else {
      set_pair<T, V>(v[2 * i / V], i % (V / 2), t);
    }
  }
  __device__ __forceinline__ void store(T* p, int apart, unsigned there, bool full) const {
    if (full) {
#pragma unroll
      for (int j = 0; j < NV; j++) store_vec<T, V>(p + j * apart, v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < NV; j++)
        if (there >> j & 1) store_vec<T, V>(p + j * apart, v[j]);
    }
  }
};

// The thread's parts of its next rows, N tensors' of each: on their way into shared memory two rows ahead
// (one row a block in flight leaves HBM idle half of the time; 16,384 x 4,096 bf16, forward + backward: 2 / 3 / 4
// slots 54 + 82, 47 + 80, 48 + 80 us, and 80 + 106 from registers before the mean had two parts), or, where a load is narrower than the 4 bytes
// that can be copied so, one row ahead in registers.  A thread reads what it copied itself, so no barrier.
constexpr int SLOTS = 3;
template <typename T, int V, int E, int N>
struct Ring {
  static constexpr bool STAGED = V * sizeof(T) >= 4;
  static constexpr int NV = E / V, BYTES = V * (int)sizeof(T);
  typedef Vec<T, V> Unit;
  Unit* slots;              // [SLOTS][N][NV][threads], this thread's
  int threads, filled, taken;
  Part<T, V, E> next[STAGED ? 1 : N];
  static constexpr size_t bytes(int threads) { return STAGED ? (size_t)SLOTS * N * E * sizeof(T) * threads : 0; }
  __device__ __forceinline__ Ring(unsigned char* smem, int threads, unsigned there) : threads(threads), filled(0), taken(0) {
    slots = reinterpret_cast<Unit*>(smem) + threadIdx.x;
    if constexpr (STAGED) {
      if (there != (1u << NV) - 1) {      // what lies past the row's end is never copied: zero
        Unit zero;
#pragma unroll
        for (int k = 0; k < V; k++) zero.e[k] = from_f32<T>(0.0f);
#pragma unroll
        for (int i = 0; i < SLOTS * N * NV; i++) slots[i * threads] = zero;
      }
    }
  }
  // Row `live` of every tensor into the next slot.
  __device__ __forceinline__ void put(const T* const (&from)[N], int apart, unsigned there, bool full) {
    if constexpr (STAGED) {
      const unsigned to = (unsigned)__cvta_generic_to_shared(slots + filled * N * NV * threads);
#pragma unroll
      for (int n = 0; n < N; n++)
#pragma unroll
        for (int j = 0; j < NV; j++)
          if (full || there >> j & 1) {
            const unsigned at = to + (n * NV + j) * threads * BYTES;
            if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from[n] + j * apart) : "memory");
            else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from[n] + j * apart), "n"(BYTES) : "memory");
          }
      asm volatile("cp.async.commit_group;" ::: "memory");
      filled = filled + 1 == SLOTS ? 0 : filled + 1;
    } else {
#pragma unroll
      for (int n = 0; n < N; n++) next[n].load(from[n], apart, there, full);
    }
  }
  __device__ __forceinline__ void take(Part<T, V, E> (&row)[N]) {
    if constexpr (STAGED) {
      asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 2) : "memory");
#pragma unroll
      for (int n = 0; n < N; n++)
#pragma unroll
        for (int j = 0; j < NV; j++) row[n].v[j] = slots[((taken * N + n) * NV + j) * threads];
      taken = taken + 1 == SLOTS ? 0 : taken + 1;
    } else {
#pragma unroll
      for (int n = 0; n < N; n++) row[n] = next[n];
    }
  }
};

// Where a thread works: its row's place in the block, its first column, what it has of a row.
template <int V, int E, int LANES>
struct Place {
  int lanes, lane, group, per, apart;
  unsigned there;
  bool full;                    // every thread of the row has all its values
  __device__ __forceinline__ Place(int cols, int run_lanes) {
    lanes = LANES == 32 ? 32 : run_lanes;
    lane = LANES == ROW_BLOCK ? threadIdx.x : threadIdx.x & (lanes - 1);
    group = LANES == ROW_BLOCK ? 0 : threadIdx.x / lanes;
    per = LANES == ROW_BLOCK ? 1 : BLOCK / lanes;
    apart = lanes * V;
    there = 0;
#pragma unroll
    for (int j = 0; j < E / V; j++) there |= (unsigned)((j * lanes + lane) * V < cols) << j;
    full = cols == E * lanes;
  }
  // The column of value e of the thread.
  __device__ __forceinline__ int column(int e) const { return (e / V * lanes + lane) * V + e % V; }
};

// The thread's weights, or `none`: the branch on their type is outside the loop, so that all loads are under way
// together (inside, a small call took 10 us of loads one after the other).
template <int E, typename W, typename P>
__device__ __forceinline__ void load_columns_of(Two (&w)[E / 2], const W* p, const P& at, int cols, float none) {
  float f[E];
#pragma unroll
  for (int e = 0; e < E; e++) f[e] = at.column(e) < cols ? to_f32(__ldg(p + at.column(e))) : none;
#pragma unroll
  for (int i = 0; i < E / 2; i++) w[i] = two(f[2 * i], f[2 * i + 1]);
}
template <int E, typename P>
__device__ __forceinline__ void load_columns(Two (&w)[E / 2], const void* p, int dtype, const P& at, int cols, float none) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < E / 2; i++) w[i] = two(none);
  } else if (dtype == F16_DTYPE_FP32) {
    load_columns_of<E>(w, reinterpret_cast<const float*>(p), at, cols, none);
  } else if (dtype == F16_DTYPE_BF16) {
    load_columns_of<E>(w, reinterpret_cast<const __nv_bfloat16*>(p), at, cols, none);
  } else {
    load_columns_of<E>(w, reinterpret_cast<const __half*>(p), at, cols, none);
  }
}

// (total + low) / n, itself where that is a fp32 value (Markstein's correction of a product with 1 / n by its fused
// residual): the mean of equal values is the value.
__device__ __forceinline__ float mean_of(float total, float n, float inv) {
  const float q = total * inv;
  return fmaf(fmaf(-q, n, total), inv, q);
}
__device__ __forceinline__ float mean_of(float total, float low, float n, float inv) {
  const float q = total * inv;
  return fmaf(fmaf(-q, n, total) + low, inv, q);
}
// 1 / sqrt(var + eps) of a row from the sum of squares of its d, whose mean is delta.  EXACT: delta is what is left of
// a quotient, far below the d unless they are all zero; else it may be of their size, and the difference of rounded
// terms negative.
template <bool EXACT>
__device__ __forceinline__ float rstd_of(float squares, float delta, float n, float inv, float eps) {
  if (EXACT) return rsqrtf(fmaf(-delta, delta, squares * inv) + eps);
  const float var = squares < __int_as_float(0x7f800000) ? fmaf(-delta, delta, mean_of(squares, n, inv)) : squares;
  return rsqrtf((var < 0.0f ? 0.0f : var) + eps);
}
__device__ __forceinline__ void store_stats(const Stats<float>& st, int64_t row, float mu, float delta, float r) {
  const float mean = mu + delta;
  st.mean[row] = mean;
  if (st.rest) st.rest[row] = delta - (mean - mu);
  st.rstd[row] = r;
}
template <typename T> constexpr bool EXACT_SUM = sizeof(T) == 2;      // see the file's head
// xh = (x - mean) r + shift.
__device__ __forceinline__ float shift_of(const Stats<const float>& st, int64_t row, float r) {
  return st.rest ? -(st.rest[row] * r) : 0.0f;
}

__device__ __forceinline__ float sum_of(const Two (&s)[2]) {
  const float2 f = split(s[0] + s[1]);
  return f.x + f.y;
}

// s + a b with the product rounded by itself; where a row takes a block nothing is left to cancel, and the fused
// operation saves some time (16,384 x 4,096 bf16 47 us for 48, backward 80 for 82).
template <int LANES>
__device__ __forceinline__ Two plus_product(Two s, Two a, Two b, Two zero) {
  if constexpr (LANES == ROW_BLOCK) return fma2(a, b, s);
  else return s + fma2(a, b, zero);
}

template <typename T, int V, int E, int LANES>
__global__ void __maxnreg__(80)
    k_ln_fwd(const T* __restrict__ x, int64_t ldx, int64_t rows, int cols, Weights wb, float eps, T* __restrict__ y,
             int64_t ldy, Stats<float> stats, int lanes) {
  __shared__ float red[2][2][32];
  int half = 0;
  const Place<V, E, LANES> at(cols, lanes);
  const int64_t step = (int64_t)gridDim.x * at.per;
  Two w[E / 2], b[E / 2];
  load_columns<E>(w, wb.w, wb.dtype, at, cols, 1.0f);
  load_columns<E>(b, wb.b, wb.dtype, at, cols, 0.0f);
  int64_t row = (int64_t)blockIdx.x * at.per + at.group;
  T* to = y + row * ldy + at.lane * V;
  const float n = (float)cols, inv = 1.0f / n;
  typedef Ring<T, V, E, 1> Rows;
  extern __shared__ __align__(16) unsigned char smem[];
  Rows ring(smem, LANES == ROW_BLOCK ? blockDim.x : BLOCK, at.there);
  const T* from[1] = {x + row * ldx + at.lane * V};
  int64_t ahead = row;
  const auto put = [&] {
    const bool live = ahead < rows;
    ring.put(from, at.apart, live ? at.there : 0u, at.full && live);
    from[0] += step * ldx;
    ahead += step;
  };
  put();
  if (Rows::STAGED) put();
  // every thread of a warp (or block) makes the same number of rounds: the sums are theirs together
  for (int64_t first = (int64_t)blockIdx.x * at.per; first < rows; first += step, row += step, to += step * ldy) {
    Part<T, V, E> here[1];
    ring.take(here);
    put();
    Two v[E / 2], s[2] = {two(0.0f), two(0.0f)};
#pragma unroll
    for (int i = 0; i < E / 2; i++) {
      v[i] = here[0].pair(i);
      s[i & 1] = s[i & 1] + v[i];
    }
    float total[2] = {sum_of(s), 0.0f};
    constexpr bool EXACT = EXACT_SUM<T>;
    float mu, delta = 0.0f;
    if constexpr (EXACT && LANES == ROW_BLOCK) {
      float low;
      row_sums<LANES, 1>(total, at.lanes, red, half, &low);
      mu = mean_of(total[0], low, n, inv);
      delta = (fmaf(-mu, n, total[0]) + low) * inv;
    } else {
      row_sums<LANES, 1>(total, at.lanes, red, half);
      mu = mean_of(total[0], n, inv);
      if (EXACT) delta = fmaf(-mu, n, total[0]) * inv;
    }
    const Two minus = two(-mu);
#pragma unroll
    for (int i = 0; i < E / 2; i++) v[i] = v[i] + minus;
    if (!at.full) {              // what lies past the row's end is zero, not the mean's negative
#pragma unroll
      for (int i = 0; i < E / 2; i++) {
        const float2 f = split(v[i]);
        v[i] = two(at.there >> (2 * i / V) & 1 ? f.x : 0.0f, at.there >> ((2 * i + 1) / V) & 1 ? f.y : 0.0f);
      }
    }
    const Two zero = two(wb.minus_zero);
    Two d[2] = {two(0.0f), two(0.0f)};
    s[0] = s[1] = two(0.0f);
#pragma unroll
    for (int i = 0; i < E / 2; i++) {
      if (!EXACT) d[i & 1] = d[i & 1] + v[i];
      s[i & 1] = plus_product<LANES>(s[i & 1], v[i], v[i], zero);
    }
    total[0] = sum_of(s);
    if (EXACT) {
      row_sums<LANES, 1>(total, at.lanes, red, half);
    } else {
      total[1] = sum_of(d);
      row_sums<LANES, 2>(total, at.lanes, red, half);
      delta = mean_of(total[1], n, inv);
    }
    const float r = rstd_of<EXACT>(total[0], delta, n, inv, eps);
    if (row < rows) {
      if (at.lane == 0 && stats.mean) store_stats(stats, row, mu, delta, r);
      Part<T, V, E> out;
      const Two scale = two(r), off = two(EXACT ? -(delta * r) : -delta);
#pragma unroll
      for (int i = 0; i < E / 2; i++) out.set(i, fma2(EXACT ? fma2(v[i], scale, off) : (v[i] + off) * scale, w[i], b[i]));
      out.store(to, at.apart, at.there, at.full);
    }
  }
}

// Backward of the rows of one block, and its columns' sums part[block][0][cols] (dw) and
// part[block][1][cols] (db).  dx or part may be null.
template <typename T, int V, int E, int LANES>
__global__ void __maxnreg__(128)
    k_ln_bwd(const T* __restrict__ dy, int64_t ldg, const T* __restrict__ x, int64_t ldx, int64_t rows, int cols,
             Weights wb, Stats<const float> stats, T* __restrict__ dx, int64_t ldd, float* __restrict__ part, int lanes) {
  __shared__ float red[2][2][32];
  extern __shared__ __align__(16) unsigned char smem[];
  int half = 0;
  const Place<V, E, LANES> at(cols, lanes);
  const int64_t step = (int64_t)gridDim.x * at.per;
  Two w[E / 2], aw[E / 2], ab[E / 2];
  load_columns<E>(w, wb.w, wb.dtype, at, cols, 1.0f);
#pragma unroll
  for (int i = 0; i < E / 2; i++) aw[i] = ab[i] = two(0.0f);
  int64_t row = (int64_t)blockIdx.x * at.per + at.group;
  T* to = dx ? dx + row * ldd + at.lane * V : nullptr;
  const float inv = 1.0f / (float)cols;
  typedef Ring<T, V, E, 2> Rows;
  Rows ring(smem, LANES == ROW_BLOCK ? blockDim.x : BLOCK, at.there);
  const T* from[2] = {x + row * ldx + at.lane * V, dy + row * ldg + at.lane * V};
  int64_t ahead = row;
  const auto put = [&] {
    const bool live = ahead < rows;
    ring.put(from, at.apart, live ? at.there : 0u, at.full && live);
    from[0] += step * ldx;
    from[1] += step * ldg;
    ahead += step;
  };
  put();
  if (Rows::STAGED) put();
  float nmu = row < rows ? stats.mean[row] : 0.0f, nr = row < rows ? stats.rstd[row] : 0.0f;
  float nrest = row < rows && stats.rest ? stats.rest[row] : 0.0f;
  for (int64_t first = (int64_t)blockIdx.x * at.per; first < rows; first += step, row += step, to += step * ldd) {
    Part<T, V, E> here[2];
    ring.take(here);
    put();
    const Part<T, V, E>&cx = here[0], &cg = here[1];
    const Two minus = two(-nmu), scale = two(nr), shift = two(-(nrest * nr)), zero = two(wb.minus_zero);
    const float r = nr;
    nmu = row + step < rows ? stats.mean[row + step] : 0.0f;
    nr = row + step < rows ? stats.rstd[row + step] : 0.0f;
    nrest = row + step < rows && stats.rest ? stats.rest[row + step] : 0.0f;
    Two s1 = two(0.0f), s2 = two(0.0f);
    if (row < rows) {
#pragma unroll
      for (int i = 0; i < E / 2; i++) {
        const Two d = cg.pair(i), xh = fma2(cx.pair(i) + minus, scale, shift), g = LANES == ROW_BLOCK ? d * w[i] : fma2(d, w[i], zero);
        s1 = s1 + g;
        s2 = plus_product<LANES>(s2, g, xh, zero);
        aw[i] = fma2(d, xh, aw[i]);
        ab[i] = ab[i] + d;
      }
    }
    if (!dx) continue;
    const float2 f1 = split(s1), f2 = split(s2);
    float total[2] = {f1.x + f1.y, f2.x + f2.y};
    row_sums<LANES, 2>(total, at.lanes, red, half);
    if (row < rows) {
      const Two m1 = two(-total[0] * inv), m2 = two(-total[1] * inv), rr = two(r);
      Part<T, V, E> out;
#pragma unroll
      for (int i = 0; i < E / 2; i++) {
        const Two xh = fma2(cx.pair(i) + minus, scale, shift), g = LANES == ROW_BLOCK ? cg.pair(i) * w[i] : fma2(cg.pair(i), w[i], zero);
        out.set(i, plus_product<LANES>(g + m1, xh, m2, zero) * rr);
      }
      out.store(to, at.apart, at.there, at.full);
    }
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * cols;
  float sw[E], sb[E];
#pragma unroll
  for (int i = 0; i < E / 2; i++) {
    split(aw[i], sw[2 * i], sw[2 * i + 1]);
    split(ab[i], sb[2 * i], sb[2 * i + 1]);
  }
  if constexpr (LANES == ROW_BLOCK) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int c = at.column(e);
      if (c < cols) {
        out[c] = sw[e];
        out[cols + c] = sb[e];
      }
    }
  } else {
    // rows of one warp first (shuffles), then the warps' sums side by side in the ring's memory
    float* col_sum = reinterpret_cast<float*>(smem);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++)
      for (int o = 16; o >= at.lanes; o >>= 1) {
        sw[e] += __shfl_xor_sync(~0u, sw[e], o);
        sb[e] += __shfl_xor_sync(~0u, sb[e], o);
      }
    if ((int)(threadIdx.x & 31) < at.lanes) {
      float* mine = col_sum + (threadIdx.x >> 5) * 2 * cols;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const int c = at.column(e);
        if (c < cols) {
          mine[c] = sw[e];
          mine[cols + c] = sb[e];
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * cols; c += BLOCK) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < BLOCK / 32; w++) v += col_sum[w * 2 * cols + c];
      out[c] = v;
    }
  }
}

// Sums over a block of WIDE threads.
template <int N>
__device__ __forceinline__ void wide_sums(float (&v)[2], float (*red)[2][32], int& half) {
  row_sums<ROW_BLOCK, N>(v, WIDE, red, half);
}
__device__ __forceinline__ double wide_sum64(double v, double* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  const int lane = threadIdx.x & 31;
  if (lane == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < WIDE / 32 ? red[lane] : 0.0;
#pragma unroll
  for (int o = WIDE / 64; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return __shfl_sync(~0u, v, 0);
}

// The block's next row into L2, a line of 128 bytes a thread, while the present one's sums are made: forward with
// narrow loads only (13,000 x 9,001 fp32 257 -> 217 us; with 16-byte loads, and backward with any, it lost).
template <typename T>
__device__ __forceinline__ void fetch_ahead(const T* row, int cols) {
  constexpr int LINE = 128 / (int)sizeof(T);
  for (int c = threadIdx.x * LINE; c < cols; c += WIDE * LINE) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + c));
}

// Rows too wide for a block's registers: a block a row, V values a load, read again for each of the passes
// (the second and third hit L1 and L2), several loads under way a thread: 4,096 x 16,384 bf16 93 us forward, 92 + 52
// + 10 backward with the sums over rows, where one read of everything would take 41 and 61 (rows of up to some
// 100 KB would fit shared memory; a kernel that holds them there was not built).
template <typename T, int V>
__global__ void __launch_bounds__(WIDE, WIDE_PER_SM)
    k_ln_fwd_wide(const T* __restrict__ x, int64_t ldx, int64_t rows, int cols, Weights wb, float eps,
                  T* __restrict__ y, int64_t ldy, Stats<float> stats) {
  __shared__ float red[2][2][32];
  __shared__ double red64[WIDE / 32];         // read before the row's next barrier, written after it
  constexpr int UNROLL = V * sizeof(T) <= 4 ? 8 : V == 2 ? 4 : 2;
  int half = 0;
  const float n = (float)cols, inv = 1.0f / n;
  [[maybe_unused]] const double inv64 = 1.0 / (double)cols;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s[2], q[2] = {0.0f, 0.0f};
    double sum64 = 0.0;
    for (int begin = 0; begin < cols; begin += WIDE * CHAIN) {
      const int end = cols - begin < WIDE * CHAIN ? cols : begin + WIDE * CHAIN;
      s[0] = 0.0f;
#pragma unroll UNROLL
      for (int c = begin + threadIdx.x * V; c < end; c += WIDE * V) {
        const Vec<T, V> v = load_vec<T, V>(xr + c);
#pragma unroll
        for (int k = 0; k < V; k++) s[0] += to_f32(v.e[k]);
      }
      sum64 += (double)s[0];
    }
    if (V <= 2 && row + gridDim.x < rows) fetch_ahead(xr + gridDim.x * ldx, cols);
    float mu, delta = 0.0f;
    if constexpr (EXACT_SUM<T>) {
      const double total = wide_sum64(sum64, red64), q = total * inv64;
      const double mean = fma(fma(-q, (double)cols, total), inv64, q);          // as mean_of
      mu = (float)mean;
      delta = (float)(mean - (double)mu);
    } else {
      s[0] = (float)sum64;
      wide_sums<1>(s, red, half);
      mu = mean_of(s[0], n, inv);
    }
#pragma unroll UNROLL
    for (int c = threadIdx.x * V; c < cols; c += WIDE * V) {
      const Vec<T, V> v = load_vec<T, V>(xr + c);
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float d = to_f32(v.e[k]) - mu;
        q[0] = fmaf(d, d, q[0]);
        if (!EXACT_SUM<T>) q[1] += d;
      }
    }
    if constexpr (EXACT_SUM<T>) {
      wide_sums<1>(q, red, half);
    } else {
      wide_sums<2>(q, red, half);
      delta = mean_of(q[1], n, inv);
    }
    const float r = rstd_of<EXACT_SUM<T>>(q[0], delta, n, inv, eps);
    const float shift = -(delta * r);
    if (threadIdx.x == 0 && stats.mean) store_stats(stats, row, mu, delta, r);
    of_weights(wb.dtype, [&](auto type) {
      typedef decltype(type) W;
#pragma unroll UNROLL
      for (int c = threadIdx.x * V; c < cols; c += WIDE * V) {
        Vec<T, V> v = load_vec<T, V>(xr + c);
        float w[V], b[V];
        load_weights<V, W>(w, wb.w, c, 1.0f);
        load_weights<V, W>(b, wb.b, c, 0.0f);
#pragma unroll
        for (int k = 0; k < V; k++) v.e[k] = from_f32<T>(fmaf(EXACT_SUM<T> ? fmaf(to_f32(v.e[k]) - mu, r, shift) : (to_f32(v.e[k]) - mu - delta) * r, w[k], b[k]));
        store_vec<T, V>(y + row * ldy + c, v);
      }
    });
  }
}

// Their dx; the sums over rows are k_ln_cols's.
template <typename T, int V>
__global__ void __launch_bounds__(WIDE, WIDE_PER_SM)
    k_ln_bwd_wide(const T* __restrict__ dy, int64_t ldg, const T* __restrict__ x, int64_t ldx, int64_t rows, int cols,
                  Weights wb, Stats<const float> stats, T* __restrict__ dx, int64_t ldd) {
  __shared__ float red[2][2][32];
  constexpr int UNROLL = V * sizeof(T) <= 4 ? 8 : V == 2 ? 4 : 2;
  int half = 0;
  const float inv = 1.0f / (float)cols;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float mu = stats.mean[row], r = stats.rstd[row], shift = shift_of(stats, row, r);
    float s[2] = {0.0f, 0.0f};
    of_weights(wb.dtype, [&](auto type) {
      typedef decltype(type) W;
#pragma unroll UNROLL
      for (int c = threadIdx.x * V; c < cols; c += WIDE * V) {
        const Vec<T, V> xv = load_vec<T, V>(x + row * ldx + c), gv = load_vec<T, V>(dy + row * ldg + c);
        float w[V];
        load_weights<V, W>(w, wb.w, c, 1.0f);
#pragma unroll
        for (int k = 0; k < V; k++) {
          const float xh = fmaf(to_f32(xv.e[k]) - mu, r, shift), g = to_f32(gv.e[k]) * w[k];
          s[0] += g;
          s[1] = fmaf(g, xh, s[1]);
        }
      }
    });
    wide_sums<2>(s, red, half);
    const float m1 = s[0] * inv, m2 = s[1] * inv;
    of_weights(wb.dtype, [&](auto type) {
      typedef decltype(type) W;
#pragma unroll UNROLL
      for (int c = threadIdx.x * V; c < cols; c += WIDE * V) {
        const Vec<T, V> xv = load_vec<T, V>(x + row * ldx + c), gv = load_vec<T, V>(dy + row * ldg + c);
        Vec<T, V> o;
        float w[V];
        load_weights<V, W>(w, wb.w, c, 1.0f);
#pragma unroll
        for (int k = 0; k < V; k++) {
          const float xh = fmaf(to_f32(xv.e[k]) - mu, r, shift), g = to_f32(gv.e[k]) * w[k];
          o.e[k] = from_f32<T>(r * (g - m1 - xh * m2));
        }
        store_vec<T, V>(dx + row * ldd + c, o);
      }
    });
  }
}

// Column sums part[slice][0][cols] (dw) and part[slice][1][cols] (db) of wide rows: a thread has V columns
// (blockIdx.x) of the rows of a slice (blockIdx.y).
constexpr int COLS = 256;
template <typename T, int V>
__global__ void __launch_bounds__(COLS)
    k_ln_cols(const T* __restrict__ dy, int64_t ldg, const T* __restrict__ x, int64_t ldx, int64_t rows, int cols,
              Stats<const float> stats, float* __restrict__ part) {
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y, first = blockIdx.y * per, end = first + per < rows ? first + per : rows;
  const int64_t c = ((int64_t)blockIdx.x * COLS + threadIdx.x) * V;
  if (c >= cols) return;
  float aw[V], ab[V];
#pragma unroll
  for (int k = 0; k < V; k++) aw[k] = ab[k] = 0.0f;
  // R rows' loads are written out ahead of their sums: left to itself the compiler keeps few of them under way once a
  // row has three statistics (13,000 x 9,001 fp32: 16 / 8 / 2 rows 528, 173, 248 us, a plain loop 230; 4,096 x 16,384
  // bf16, 16 bytes a load: 6 / 4 / 2 / 1 rows 74, 56, 52, 56).
  constexpr int R = V * sizeof(T) <= 4 ? 8 : 2;
  const auto add = [&](int64_t row, auto count) {
    constexpr int N = decltype(count)::value;
    Vec<T, V> xv[N], gv[N];
    float mu[N], r[N], shift[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      xv[i] = load_vec_nc<T, V>(x + (row + i) * ldx + c);
      gv[i] = load_vec_nc<T, V>(dy + (row + i) * ldg + c);
      mu[i] = stats.mean[row + i];
      r[i] = stats.rstd[row + i];
      shift[i] = stats.rest ? stats.rest[row + i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      shift[i] *= -r[i];
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float d = to_f32(gv[i].e[k]);
        aw[k] = fmaf(d, fmaf(to_f32(xv[i].e[k]) - mu[i], r[i], shift[i]), aw[k]);
        ab[k] += d;
      }
    }
  };
  int64_t row = first;
  for (; row + R <= end; row += R) add(row, std::integral_constant<int, R>());
  for (; row < end; row++) add(row, std::integral_constant<int, 1>());
  float* out = part + blockIdx.y * 2 * (int64_t)cols + c;
#pragma unroll
  for (int k = 0; k < V; k++) {
    out[k] = aw[k];
    out[cols + k] = ab[k];
  }
}

// dw and db from the blocks' partial sums: 32 columns a block, 32 threads a column, in a fixed order.
__global__ void __launch_bounds__(1024) k_ln_wgrad(const float* __restrict__ part, int64_t nblk, int cols, void* dw, void* db,
                                                   int dtype) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float v = 0.0f;
  if (c < 2 * cols)
    for (int64_t r = threadIdx.y; r < nblk; r += 32) v += part[r * 2 * cols + c];
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

// How a row is spread: v values a load, e values a thread, `lanes` threads a row -- a power of two up to 32, or
// whole warps, the fewest that hold it; 0: the wide kernels.
struct Plan {
  int v, e, lanes, threads;
};

// `most`: values of a row that its threads' registers may take.
inline Plan plan_for(int cols, int v, int most) {
  Plan p = {v, MOST, 1, BLOCK};
  if (v <= 2) {
    p.e = cols <= 16 ? 4 : cols <= 8 * MAX_LANES ? 8 : MOST;
  }
  while (p.lanes < 32 && p.lanes * p.e < cols) p.lanes <<= 1;
  if (p.lanes * p.e < cols) p.lanes = cols > most ? 0 : (cols + 32 * p.e - 1) / (32 * p.e) * 32;
  p.threads = p.lanes > 32 ? p.lanes : p.lanes ? BLOCK : WIDE;
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

// Persistent warps per SM, which the registers allow (80 and 128 a thread).  Forward with 16 / 24 / 32 of them:
// 16,384 x 4,096 bf16 52 / 47 / 60 us, 100,003 x 215 fp16 36 / 29 / 37.
constexpr int FWD_WARPS = 24, BWD_WARPS = 16;

// Dynamic shared memory above 48 KB has to be asked for (on every device; it costs the host under a microsecond).
template <typename K>
int room_for(K kernel, size_t bytes) {
  if (bytes <= 40 * 1024) return F16_OK;          // with what a kernel declares itself
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess ? F16_OK : F16_ERR_CUDA;
}

// Most values of a row in registers; beyond them the wide kernels.  Backward a row has 512 threads (of 128 registers
// each); of 16 values in 2-byte loads some spill, so such rows end at 8 a thread (20,000 x 5,001 bf16 511 us, wide
// 234 + 135; fp32 383, wide 266 + 149).  Forward it may have 768 (of 80 registers; 8,000 x 12,288 bf16 73 us, wide 137;
// 3,000 x 12,001 bf16 57, 71), but not where a load is one fp32 value (13,000 x 9,001 250 us, wide 217).
template <typename T, bool BACK>
constexpr int most_of(int v) {
  if (BACK) return (sizeof(T) == 2 && v == 1 ? 8 : MOST) * MAX_LANES;
  return MOST * (sizeof(T) == 4 && v == 1 ? MAX_LANES : FWD_LANES);
}

// f(V, E, LANES) for a plan, as integral constants.
template <int N> using Int = std::integral_constant<int, N>;
template <typename T, bool BACK, typename F>
void with_plan(const Plan& p, F f) {
  constexpr int VW = 16 / sizeof(T);
  const auto of_warp = [&](auto v, auto e) { p.lanes == 32 ? f(v, e, Int<32>()) : f(v, e, Int<0>()); };
  const auto of_any = [&](auto v, auto e) { p.lanes > 32 ? f(v, e, Int<ROW_BLOCK>()) : of_warp(v, e); };
  if (p.v == VW) {
    of_any(Int<VW>(), Int<MOST>());
  } else if (p.v == 2) {
    if (p.e == 4) of_warp(Int<2>(), Int<4>());
    else if (p.e == 8) of_any(Int<2>(), Int<8>());
    else f(Int<2>(), Int<MOST>(), Int<ROW_BLOCK>());
  } else {
    if (p.e == 4) of_warp(Int<1>(), Int<4>());
    else if (p.e == 8) of_any(Int<1>(), Int<8>());
    else if constexpr (most_of<T, BACK>(1) > 8 * MAX_LANES) f(Int<1>(), Int<MOST>(), Int<ROW_BLOCK>());
  }
}

// g(V) for rows too wide for registers (4,000 x 9,002 fp16 backward 67 + 34 us by two values a load).
template <typename T, typename G>
void with_loads(const Plan& p, G g) {
  if (p.v == 16 / (int)sizeof(T)) g(Int<16 / (int)sizeof(T)>());
  else if (p.v == 2) g(Int<2>());
  else g(Int<1>());
}

template <typename T>
int forward(const T* x, int64_t rows, int cols, int64_t ldx, Weights wb, float eps, T* y, int64_t ldy,
            const Stats<float>& stats, cudaStream_t st) {
  const void* ptrs[2] = {x, y};
  const int64_t lds[2] = {ldx, ldy};
  const int v = vec_for(cols, sizeof(T), ptrs, lds, 2);
  const Plan p = plan_for(cols, v, most_of<T, false>(v));
  if (!p.lanes) {
    const int64_t grid = rows < WIDE_PER_SM * sm_count() ? rows : WIDE_PER_SM * sm_count();
    with_loads<T>(p, [&](auto v) {
      k_ln_fwd_wide<T, v()><<<(unsigned)grid, WIDE, 0, st>>>(x, ldx, rows, cols, wb, eps, y, ldy, stats);
    });
    return launch_status();
  }
  const unsigned grid = (unsigned)grid_rows(rows, p, FWD_WARPS);
  int rc = F16_OK;
  with_plan<T, false>(p, [&](auto v, auto e, auto lanes) {
    const auto k = k_ln_fwd<T, v(), e(), lanes()>;
    const size_t smem = Ring<T, v(), e(), 1>::bytes(p.threads);
    rc = room_for(k, smem);
    if (rc == F16_OK) k<<<grid, p.threads, smem, st>>>(x, ldx, rows, cols, wb, eps, y, ldy, stats, p.lanes);
  });
  return rc != F16_OK ? rc : launch_status();
}

// Slices of rows of k_ln_cols: four blocks an SM over all tiles of its columns.
inline int64_t col_tiles(int cols, int v) { return (cols + (int64_t)COLS * v - 1) / (COLS * v); }
inline int64_t col_slices(int64_t tiles) { return (4 * sm_count() + tiles - 1) / tiles; }

// Most blocks that write column sums of rows this wide, whatever their alignment and number.
template <typename T>
int64_t sum_blocks(int cols) {
  const int widths[3] = {16 / (int)sizeof(T), 2, 1};
  int64_t most = 0;
  for (int v : widths) {
    if (cols % v) continue;
    const Plan p = plan_for(cols, v, most_of<T, true>(v));
    const int64_t n = p.lanes ? grid_rows(INT64_MAX / 2, p, BWD_WARPS) : col_slices(col_tiles(cols, v));
    if (n > most) most = n;
  }
  return most;
}

template <typename T>
int backward(const T* dy, int64_t ldg, const T* x, int64_t ldx, int64_t rows, int cols, Weights wb,
             const Stats<const float>& stats, T* dx, int64_t ldd, float* part, int64_t part_floats, void* dw, void* db,
             cudaStream_t st) {
  const void* ptrs[3] = {dy, x, dx};
  const int64_t lds[3] = {ldg, ldx, ldd};
  const int v = vec_for(cols, sizeof(T), ptrs, lds, 3);
  const Plan p = plan_for(cols, v, most_of<T, true>(v));
  const int64_t room = part ? part_floats / (2 * (int64_t)cols) : 0;
  int64_t grid = p.lanes ? grid_rows(rows, p, BWD_WARPS) : 0;
  int rc = F16_OK;
  if (!p.lanes) {
    with_loads<T>(p, [&](auto v) {
      const int64_t blocks = rows < WIDE_PER_SM * sm_count() ? rows : WIDE_PER_SM * sm_count();
      if (dx) k_ln_bwd_wide<T, v()><<<(unsigned)blocks, WIDE, 0, st>>>(dy, ldg, x, ldx, rows, cols, wb, stats, dx, ldd);
      if (part) {
        const int64_t tiles = col_tiles(cols, v());
        grid = col_slices(tiles);
        if (grid > rows) grid = rows;
        if (grid > room) grid = room;
        k_ln_cols<T, v()><<<dim3((unsigned)tiles, (unsigned)grid), COLS, 0, st>>>(dy, ldg, x, ldx, rows, cols, stats, part);
      }
    });
  } else {
    if (part && grid > room) grid = room;
    with_plan<T, true>(p, [&](auto v, auto e, auto lanes) {
      const auto k = k_ln_bwd<T, v(), e(), lanes()>;
      const size_t ring = Ring<T, v(), e(), 2>::bytes(p.threads), sums = p.lanes <= 32 ? BLOCK / 32 * 2 * (size_t)cols * sizeof(float) : 0;
      const size_t smem = ring > sums ? ring : sums;
      rc = room_for(k, smem);
      if (rc == F16_OK) k<<<(unsigned)grid, p.threads, smem, st>>>(dy, ldg, x, ldx, rows, cols, wb, stats, dx, ldd, part, p.lanes);
    });
    if (rc != F16_OK) return rc;
  }
  rc = launch_status();
  if (rc != F16_OK || !part) return rc;
  k_ln_wgrad<<<(unsigned)((2 * (int64_t)cols + 31) / 32), dim3(32, 32), 0, st>>>(part, grid, cols, dw, db, wb.dtype);
  return launch_status();
}

inline bool is_dtype(int t) { return t == F16_DTYPE_BF16 || t == F16_DTYPE_FP16 || t == F16_DTYPE_FP32; }
inline int size_of(int t) { return t == F16_DTYPE_FP32 ? 4 : 2; }

}  // namespace ln
}  // namespace f16

using namespace f16;

extern "C" int f16_layer_norm_fwd_rest(const void* x, int64_t rows, int cols, int64_t ldx, int dtype, const void* weight,
                                       const void* bias, int wdtype, double eps, void* y, int64_t ldy, float* mean,
                                       float* rest, float* rstd, f16_stream_t stream) {
  if (!x || !y || rows <= 0 || cols <= 0 || ldx < 0 || ldy < cols || !ln::is_dtype(dtype) || !ln::is_dtype(wdtype) ||
      !mean != !rstd || (rest && !mean) || !(eps >= 0.0))
    return F16_ERR_ARG;
  if (cols > ln::MAX_COLS) return F16_ERR_TOO_LARGE;
  if (!aligned(x, ln::size_of(dtype)) || !aligned(y, ln::size_of(dtype)) || !aligned(weight, ln::size_of(wdtype)) ||
      !aligned(bias, ln::size_of(wdtype)))
    return F16_ERR_ALIGN;
  const ln::Weights wb = {weight, bias, wdtype, -0.0f};
  const ln::Stats<float> stats = {mean, rest, rstd};
  const cudaStream_t st = cu_stream(stream);
  if (dtype == F16_DTYPE_FP32)
    return ln::forward((const float*)x, rows, cols, ldx, wb, (float)eps, (float*)y, ldy, stats, st);
  if (dtype == F16_DTYPE_BF16)
    return ln::forward((const __nv_bfloat16*)x, rows, cols, ldx, wb, (float)eps, (__nv_bfloat16*)y, ldy, stats, st);
  return ln::forward((const __half*)x, rows, cols, ldx, wb, (float)eps, (__half*)y, ldy, stats, st);
}

extern "C" int f16_layer_norm_fwd(const void* x, int64_t rows, int cols, int64_t ldx, int dtype, const void* weight,
                                  const void* bias, int wdtype, double eps, void* y, int64_t ldy, float* mean,
                                  float* rstd, f16_stream_t stream) {
  return f16_layer_norm_fwd_rest(x, rows, cols, ldx, dtype, weight, bias, wdtype, eps, y, ldy, mean, nullptr, rstd, stream);
}

extern "C" int64_t f16_layer_norm_scratch_floats(int64_t rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  const int64_t a = ln::sum_blocks<float>(cols), b = ln::sum_blocks<__half>(cols), most = a > b ? a : b;
  return 2 * (int64_t)cols * (rows < most ? rows : most);
}

extern "C" int f16_layer_norm_bwd_rest(const void* dy, int64_t ldg, const void* x, int64_t ldx, int64_t rows, int cols,
                                       int dtype, const void* weight, int wdtype, const float* mean, const float* rest,
                                       const float* rstd, void* dx, int64_t ldd, void* dweight, void* dbias,
                                       float* scratch, int64_t scratch_floats, f16_stream_t stream) {
  if (!dy || !x || !mean || !rstd || rows <= 0 || cols <= 0 || ldg < 0 || ldx < 0 || (dx && ldd < cols) ||
      !ln::is_dtype(dtype) || !ln::is_dtype(wdtype))
    return F16_ERR_ARG;
  if (cols > ln::MAX_COLS) return F16_ERR_TOO_LARGE;
  const bool sums = dweight || dbias;
  if (!dx && !sums) return F16_OK;
  if (sums && (!scratch || scratch_floats < 2 * (int64_t)cols)) return F16_ERR_ARG;
  const int size = ln::size_of(dtype);
  if (!aligned(dy, size) || !aligned(x, size) || !aligned(dx, size) || !aligned(weight, ln::size_of(wdtype)))
    return F16_ERR_ALIGN;
  const ln::Weights wb = {weight, nullptr, wdtype, -0.0f};
  const ln::Stats<const float> stats = {mean, rest, rstd};
  float* part = sums ? scratch : nullptr;
  const cudaStream_t st = cu_stream(stream);
  if (dtype == F16_DTYPE_FP32)
    return ln::backward((const float*)dy, ldg, (const float*)x, ldx, rows, cols, wb, stats, (float*)dx, ldd, part,
                        scratch_floats, dweight, dbias, st);
  if (dtype == F16_DTYPE_BF16)
    return ln::backward((const __nv_bfloat16*)dy, ldg, (const __nv_bfloat16*)x, ldx, rows, cols, wb, stats,
                        (__nv_bfloat16*)dx, ldd, part, scratch_floats, dweight, dbias, st);
  return ln::backward((const __half*)dy, ldg, (const __half*)x, ldx, rows, cols, wb, stats, (__half*)dx, ldd, part,
                      scratch_floats, dweight, dbias, st);
}

extern "C" int f16_layer_norm_bwd(const void* dy, int64_t ldg, const void* x, int64_t ldx, int64_t rows, int cols,
                                  int dtype, const void* weight, int wdtype, const float* mean, const float* rstd,
                                  void* dx, int64_t ldd, void* dweight, void* dbias, float* scratch,
                                  int64_t scratch_floats, f16_stream_t stream) {
  return f16_layer_norm_bwd_rest(dy, ldg, x, ldx, rows, cols, dtype, weight, wdtype, mean, nullptr, rstd, dx, ldd, dweight,
                                 dbias, scratch, scratch_floats, stream);
}
