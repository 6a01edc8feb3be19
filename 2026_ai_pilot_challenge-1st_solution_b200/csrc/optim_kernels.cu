// optim_kernels.cu -- one AdamW step over many tensors: the gradients' norm and the update.
//
//   n = sqrt(sum g^2) over all tensors,  c = min(1, max_norm / (n + 1e-6)),  g' = c g
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by HBM: a step reads p, g, m, v and writes p, m, v once, and the norm reads g once more.  The
// tensors come as a table in the kernel's parameters (no device table to build or keep), their
// moments lie in flat buffers that begin a new block of QBLOCK values with every tensor.  Persistent
// blocks walk over pieces of PIECE values.  The norm is summed in fp64 over the blocks' partial sums,
// each block in the same order; the step counts live on the device and the last block to finish
// raises them, so a captured step counts when it is replayed.
//
// 8-bit moments: m as e4m3 and v as e5m2 in units of a fp32 scale for each QBLOCK values (the largest
// finite one becomes the type's largest; e5m2 for v because its range is the square of m's).  v moves
// by 1/1000 of itself a step, a code by 1/8 at least: rounded to nearest, moments would stay where
// they are.  They are rounded stochastically instead -- up with the probability of the part left over
// -- so that their expectation is the moment; the random bits are a splitmix64 hash of (seed, step,
// position), 16 for each moment.  v > 0 stays above zero, since p moves by 1 / sqrt(v).  A value that
// is not finite becomes a NaN code and leaves its block's scale alone.
//
// 16-bit parameters may have fp32 master copies; a master counts while it rounds to its parameter,
// else the parameter was set from outside and is taken instead.
#include <cuda_fp8.h>
#include "typed.cuh"

namespace f16 {
namespace opt {

constexpr int THREADS = 256;
constexpr int QBLOCK = F16_ADAMW_BLOCK;       // values of one scale: a warp's, 8 each
constexpr int PIECE = THREADS / 32 * QBLOCK;  // values of a block at a time
constexpr int NORM_PIECE = 4 * PIECE;         // of a block of the norm: eight loads in flight a thread
static_assert(QBLOCK == 256, "a lane holds two groups of four values of a warp's scale block");

struct Tensor {
  void* p;
  const void* g;
  int64_t n;
  int64_t at;       // first element in the flat buffers
};

// Tensors of one launch.  `first[i]`: pieces before tensor i.  A parameter block holds 32,764 bytes.
template <int N>
struct Table {
  Tensor t[N];
  int64_t first[N + 1];
  int32_t index[N];       // of the tensor's step count
  int count;
};
constexpr int SMALL = 64, LARGE = 720;
static_assert(sizeof(Table<LARGE>) + 256 <= 32764, "kernel parameters");

struct Hyper {
  double lr, b1, b2;
  float eps, decay;                 // decay: 1 - lr wd
  float keep1, new1, keep2, new2;   // b1, 1 - b1, b2, 1 - b2, each rounded from fp64
  double max_norm;
};

struct Flat {
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  float* master;
  int64_t* steps;
  unsigned* ticket;                 // blocks that have finished, 0 between launches
  const double* partial;            // squares of the gradients, or NULL: no clip
  int partials;
  float* norm;
  uint64_t seed;
};

__device__ __forceinline__ uint64_t mix64(uint64_t z) {
  z += 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}

template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& tab, int64_t piece) {
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first[mid] <= piece) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Four values from element i of a tensor on (zero past its end); `vec`: aligned for one load.
template <typename T>
__device__ __forceinline__ Vec<T, 4> load4(const T* p, int64_t i, int64_t n, bool vec) {
  Vec<T, 4> v;
  if (vec && i + 4 <= n) return load_vec<T, 4>(p + i);
#pragma unroll
  for (int k = 0; k < 4; k++) v.e[k] = i + k < n ? p[i + k] : from_f32<T>(0.0f);
  return v;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t i, int64_t n, bool vec, const Vec<T, 4>& v) {
  if (vec && i + 4 <= n) {
    store_vec<T, 4>(p + i, v);
  } else {
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (i + k < n) p[i + k] = v.e[k];
  }
}

__device__ __forceinline__ double block_sum(double v, double* s) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; w++) v += s[w];
  __syncthreads();
  return v;
}

// Sums of squares of the gradients: one fp64 value a block.
template <typename T, int N>
__global__ void __launch_bounds__(THREADS)
    k_grad_squares(const __grid_constant__ Table<N> tab, double* __restrict__ partial) {
  __shared__ double s[THREADS / 32];
  double sum = 0.0;
  const int64_t pieces = tab.first[tab.count];
  for (int64_t piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    const int i = tensor_of(tab, piece);
    const T* g = reinterpret_cast<const T*>(tab.t[i].g);
    const int64_t n = tab.t[i].n, at = (piece - tab.first[i]) * NORM_PIECE;
    const bool vec = (reinterpret_cast<uintptr_t>(g) & (4 * sizeof(T) - 1)) == 0;
    Vec<T, 4> v[8];
    if (vec && at + NORM_PIECE <= n) {
#pragma unroll
      for (int h = 0; h < 8; h++) v[h] = load_vec_nc<T, 4>(g + at + (h * THREADS + threadIdx.x) * 4);
    } else {
#pragma unroll
      for (int h = 0; h < 8; h++) v[h] = load4(g, at + (h * THREADS + threadIdx.x) * 4, n, vec);
    }
    float q = 0.0f;
#pragma unroll
    for (int h = 0; h < 8; h++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float f = to_f32(v[h].e[k]);
        q = fmaf(f, f, q);
      }
    sum += (double)q;
  }
  sum = block_sum(sum, s);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// x / s rounded towards zero (x >= 0, inv = 1 / s): a Newton step gives the nearest quotient, the sign of its
// residual says whether that lies above the true one.  What the rounding to a code below looks at are whole
// units of the quotient's last place, so it decides as the exact quotient would; the nearest one would
// fall on the wrong side of a code's border once in some 10^6 -- and often where a block's values all
// shrink alike, which makes the quotients codes again and again.
__device__ __forceinline__ float quotient_rz(float x, float s, float inv) {
  const float q0 = x * inv, q = fmaf(fmaf(-q0, s, x), inv, q0);
  return __int_as_float(__float_as_int(q) - (fmaf(-q, s, x) < 0.0f));
}

// x >= 0, at most `most`, rounded to `MANT` mantissa bits (subnormals below 2^LOW included): up where
// the 16 random bits and the part left over carry.
template <int MANT, int LOW>
__device__ __forceinline__ float round_carry(float x, unsigned bits, float most) {
  constexpr int DROP = 23 - MANT;
  const float low = __int_as_float((127 + LOW) << 23);
  x = fminf(x, most);
  const bool sub = x < low;                       // in [low, 2 low) a mantissa step is a subnormal one
  const float y = sub ? __fadd_rz(x, low) : x;
  const float r = __uint_as_float((__float_as_uint(y) + (bits << (DROP - 16))) & ~((1u << DROP) - 1));
  return sub ? r - low : r;
}

__device__ __forceinline__ float warp_max(float v) {
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}

__device__ __forceinline__ float2 unpack8(__nv_fp8x2_storage_t c, __nv_fp8_interpretation_t kind) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(c, kind);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

__device__ __forceinline__ float root_of(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

#define INF __int_as_float(0x7f800000)
#define NOT_A_NUMBER __int_as_float(0x7fffffff)

template <typename T, int N, int BITS, bool MASTER>
__global__ void __launch_bounds__(THREADS)
    k_adamw(const __grid_constant__ Table<N> tab, const __grid_constant__ Hyper hy, const __grid_constant__ Flat fl) {
  __shared__ double s[THREADS / 32];
  const int64_t pieces = tab.first[tab.count];
  float clip = 1.0f;
  if (fl.partial) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < fl.partials; i += THREADS) sum += fl.partial[i];
    const double norm = sqrt(block_sum(sum, s));
    const double c = hy.max_norm / (norm + 1e-6);
    clip = c < 1.0 || c != c ? (float)c : 1.0f;
    if (blockIdx.x == 0 && threadIdx.x == 0 && fl.norm) *fl.norm = (float)norm;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t step = -1;
  float rate = 0.0f, root = 0.0f;
  uint64_t key = 0;
  for (int64_t piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    const int i = tensor_of(tab, piece);
    const int64_t n = tab.t[i].n, at = (piece - tab.first[i]) * PIECE + warp * QBLOCK;
    T* p = reinterpret_cast<T*>(tab.t[i].p);
    const T* g = reinterpret_cast<const T*>(tab.t[i].g);
    const bool vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g)) & (4 * sizeof(T) - 1)) == 0;
    const int64_t flat = tab.t[i].at + at;
    const int64_t t = fl.steps[tab.index[i]] + 1;
    if (t != step) {
      // 1 - b^t by squaring, in fp64: 1 - 0.999 has three digits less than 0.999
      step = t;
      double x1 = hy.b1, x2 = hy.b2, p1 = 1.0, p2 = 1.0;
      for (int64_t e = t; e; e >>= 1) {
        if (e & 1) {
          p1 *= x1;
          p2 *= x2;
        }
        x1 *= x1;
        x2 *= x2;
      }
      rate = (float)(hy.lr / (1.0 - p1));
      root = (float)(1.0 / sqrt(1.0 - p2));
      key = mix64(fl.seed ^ mix64((uint64_t)t));
    }
    if (at >= n) continue;                         // the warp's part lies past the tensor's end
    Vec<T, 4> pv[2], gv[2];
    float m[2][4], v[2][4], ms[2][4];
    float m_unit = 0.0f, v_unit = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int64_t e = at + h * 128 + lane * 4;
      pv[h] = load4(p, e, n, vec);
      gv[h] = load4(g, e, n, vec);
    }
    if (BITS == 8) {
      m_unit = fl.m_scale[flat / QBLOCK];
      v_unit = fl.v_scale[flat / QBLOCK];
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int64_t f = flat + h * 128 + lane * 4;
      if (BITS == 8) {
        const uint32_t mc = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(fl.m) + f);
        const uint32_t vc = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(fl.v) + f);
        const float2 m0 = unpack8(mc & 0xffff, __NV_E4M3), m1 = unpack8(mc >> 16, __NV_E4M3);
        const float2 v0 = unpack8(vc & 0xffff, __NV_E5M2), v1 = unpack8(vc >> 16, __NV_E5M2);
        m[h][0] = m0.x * m_unit; m[h][1] = m0.y * m_unit; m[h][2] = m1.x * m_unit; m[h][3] = m1.y * m_unit;
        v[h][0] = v0.x * v_unit; v[h][1] = v0.y * v_unit; v[h][2] = v1.x * v_unit; v[h][3] = v1.y * v_unit;
      } else {
        const float4 mf = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(fl.m) + f);
        const float4 vf = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(fl.v) + f);
        m[h][0] = mf.x; m[h][1] = mf.y; m[h][2] = mf.z; m[h][3] = mf.w;
        v[h][0] = vf.x; v[h][1] = vf.y; v[h][2] = vf.z; v[h][3] = vf.w;
      }
      if (MASTER) {
        const float4 w = *reinterpret_cast<const float4*>(fl.master + f);
        ms[h][0] = w.x; ms[h][1] = w.y; ms[h][2] = w.z; ms[h][3] = w.w;
      }
    }
    // past the tensor's end the gradient and the moments are zero, and stay it
    float m_most = 0.0f, v_most = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int64_t e = at + h * 128 + lane * 4;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float gr = to_f32(gv[h].e[k]) * clip;
        // each product rounded by itself, as torch's expressions do
        m[h][k] = __fadd_rn(__fmul_rn(hy.keep1, m[h][k]), __fmul_rn(hy.new1, gr));
        v[h][k] = __fadd_rn(__fmul_rn(hy.keep2, v[h][k]), __fmul_rn(hy.new2, __fmul_rn(gr, gr)));
        float w = to_f32(pv[h].e[k]);
        if (MASTER) {
          Vec<T, 1> rounded, now;
          rounded.e[0] = from_f32<T>(ms[h][k]);
          now.e[0] = pv[h].e[k];
          w = rounded.r == now.r ? ms[h][k] : w;
        }
        // the change is good to some 2^-21 of itself (approximate root and quotient): far below the
        // parameter's rounding
        w = fmaf(w, hy.decay, -__fdividef(rate * m[h][k], fmaf(root_of(v[h][k]), root, hy.eps)));
        if (MASTER) ms[h][k] = w;
        pv[h].e[k] = from_f32<T>(w);
        if (BITS == 8) {
          m_most = fmaxf(m_most, fabsf(m[h][k]));         // a NaN does not count
          v_most = fmaxf(v_most, v[h][k]);
        }
      }
      store4(p, e, n, vec, pv[h]);
    }
    float mi = 0.0f, vi = 0.0f;
    if (BITS == 8) {
      const float tiny = __int_as_float(1 << 23);       // the smallest normal: its reciprocal is finite
      m_most = warp_max(m_most);
      v_most = warp_max(v_most);
      if (!(m_most < INF) || !(v_most < INF)) {         // an infinity somewhere: the largest finite ones
        m_most = v_most = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int k = 0; k < 4; k++) {
            m_most = fmaxf(m_most, fabsf(m[h][k]) < INF ? fabsf(m[h][k]) : 0.0f);
            v_most = fmaxf(v_most, v[h][k] < INF ? v[h][k] : 0.0f);
          }
        m_most = warp_max(m_most);
        v_most = warp_max(v_most);
      }
      m_unit = fmaxf(m_most * (1.0f / 448.0f), tiny);
      v_unit = fmaxf(v_most * (1.0f / 57344.0f), tiny);
      if (lane == 0) {
        fl.m_scale[flat / QBLOCK] = m_unit;
        fl.v_scale[flat / QBLOCK] = v_unit;
      }
      mi = 1.0f / m_unit;
      vi = 1.0f / v_unit;
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int64_t e = at + h * 128 + lane * 4, f = flat + h * 128 + lane * 4;
      if (e >= n) continue;
      if (BITS == 8) {
        const uint64_t word0 = mix64(key + (uint64_t)(f >> 1)), word1 = mix64(key + (uint64_t)(f >> 1) + 1);
        float mq[4], vq[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const unsigned bits = (unsigned)((k < 2 ? word0 : word1) >> (32 * (k & 1)));
          const float a = fabsf(m[h][k]), b = v[h][k];
          const float x = round_carry<3, -6>(quotient_rz(a, m_unit, mi), bits & 0xffff, 448.0f);
          const float y = round_carry<2, -14>(quotient_rz(b, v_unit, vi), bits >> 16, 57344.0f);
          mq[k] = a < INF ? copysignf(x, m[h][k]) : NOT_A_NUMBER;
          // 2^-16, the smallest code, for what is above zero
          vq[k] = b < INF ? (b > 0.0f ? fmaxf(y, 1.52587890625e-05f) : 0.0f) : NOT_A_NUMBER;
        }
        const uint32_t mc = __nv_cvt_float2_to_fp8x2(make_float2(mq[0], mq[1]), __NV_SATFINITE, __NV_E4M3) |
                            (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(mq[2], mq[3]), __NV_SATFINITE, __NV_E4M3) << 16;
        const uint32_t vc = __nv_cvt_float2_to_fp8x2(make_float2(vq[0], vq[1]), __NV_SATFINITE, __NV_E5M2) |
                            (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(vq[2], vq[3]), __NV_SATFINITE, __NV_E5M2) << 16;
        *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(fl.m) + f) = mc;
        *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(fl.v) + f) = vc;
      } else {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(fl.m) + f) = make_float4(m[h][0], m[h][1], m[h][2], m[h][3]);
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(fl.v) + f) = make_float4(v[h][0], v[h][1], v[h][2], v[h][3]);
      }
      if (MASTER) {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (e + k >= n) ms[h][k] = 0.0f;
        *reinterpret_cast<float4*>(fl.master + f) = make_float4(ms[h][0], ms[h][1], ms[h][2], ms[h][3]);
      }
    }
  }
  // every block has read its counts before its ticket; the last one to take one raises them
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicInc(fl.ticket, gridDim.x - 1) == gridDim.x - 1;
  }
  __syncthreads();
  if (last)
    for (int i = threadIdx.x; i < tab.count; i += THREADS) fl.steps[tab.index[i]] += 1;
}

constexpr int BLOCKS_PER_SM = 4;

#undef INF
#undef NOT_A_NUMBER

template <int N>
void fill(Table<N>& tab, int piece, int count, void* const* p, const void* const* g, const int64_t* n, const int64_t* at,
          const int32_t* index) {
  int64_t pieces = 0;
  for (int i = 0; i < count; i++) {
    tab.t[i] = {p ? p[i] : nullptr, g[i], n[i], at ? at[i] : 0};
    tab.index[i] = index ? index[i] : 0;
    tab.first[i] = pieces;
    pieces += (n[i] + piece - 1) / piece;
  }
  tab.first[count] = pieces;
  tab.count = count;
}

inline unsigned blocks_for(int64_t pieces) {
  const int64_t most = (int64_t)sm_count() * BLOCKS_PER_SM;
  return (unsigned)(pieces < most ? pieces : most);
}

template <typename T, int N>
int squares(int count, const void* const* g, const int64_t* n, double* partial, int room, int* used, cudaStream_t st) {
  Table<N> tab;
  fill<N>(tab, NORM_PIECE, count, nullptr, g, n, nullptr, nullptr);
  unsigned grid = blocks_for(tab.first[count]);
  if ((int)grid > room) grid = room;
  k_grad_squares<T, N><<<grid, THREADS, 0, st>>>(tab, partial);
  *used = (int)grid;
  return launch_status();
}

template <typename T, int N>
int update(int count, void* const* p, const void* const* g, const int64_t* n, const int64_t* at, const int32_t* index,
           const Hyper& hy, const Flat& fl, int bits, cudaStream_t st) {
  Table<N> tab;
  fill<N>(tab, PIECE, count, p, g, n, at, index);
  const unsigned grid = blocks_for(tab.first[count]);
  const auto go = [&](auto k) { k<<<grid, THREADS, 0, st>>>(tab, hy, fl); };
  if constexpr (sizeof(T) == 4) {
    bits == 8 ? go(k_adamw<T, N, 8, false>) : go(k_adamw<T, N, 32, false>);
  } else if (fl.master) {
    bits == 8 ? go(k_adamw<T, N, 8, true>) : go(k_adamw<T, N, 32, true>);
  } else {
    bits == 8 ? go(k_adamw<T, N, 8, false>) : go(k_adamw<T, N, 32, false>);
  }
  return launch_status();
}

inline bool is_dtype(int t) { return t == F16_DTYPE_BF16 || t == F16_DTYPE_FP16 || t == F16_DTYPE_FP32; }

}  // namespace opt
}  // namespace f16

using namespace f16;

extern "C" int f16_grad_squares(int count, const void* const* grads_host, const int64_t* numel_host, int dtype,
                                double* partial, int room, int* used_host, f16_stream_t stream) {
  if (count <= 0 || !grads_host || !numel_host || !partial || !used_host || !opt::is_dtype(dtype)) return F16_ERR_ARG;
  const size_t size = dtype == F16_DTYPE_FP32 ? 4 : 2;
  for (int i = 0; i < count; i++) {
    if (!grads_host[i] || numel_host[i] <= 0) return F16_ERR_ARG;
    if (!aligned(grads_host[i], size)) return F16_ERR_ALIGN;
  }
  *used_host = 0;
  const cudaStream_t st = cu_stream(stream);
  for (int i = 0; i < count; i += opt::LARGE) {
    const int n = count - i < opt::LARGE ? count - i : opt::LARGE;
    if (*used_host >= room) return F16_ERR_TOO_LARGE;
    int used = 0, rc;
    const auto go = [&](auto tag) {
      typedef decltype(tag) T;
      return n <= opt::SMALL
                 ? opt::squares<T, opt::SMALL>(n, grads_host + i, numel_host + i, partial + *used_host, room - *used_host, &used, st)
                 : opt::squares<T, opt::LARGE>(n, grads_host + i, numel_host + i, partial + *used_host, room - *used_host, &used, st);
    };
    rc = dtype == F16_DTYPE_FP32 ? go(0.0f) : dtype == F16_DTYPE_BF16 ? go(__nv_bfloat16()) : go(__half());
    if (rc != F16_OK) return rc;
    *used_host += used;
  }
  return F16_OK;
}

extern "C" int f16_adamw_step(const f16_adamw_args* a, f16_stream_t stream) {
  if (!a || a->count <= 0 || !a->params_host || !a->grads_host || !a->numel_host || !a->first_host || !a->index_host ||
      !a->exp_avg || !a->exp_avg_sq || !a->steps || !a->ticket || !opt::is_dtype(a->dtype) ||
      (a->state_bits != 32 && a->state_bits != 8) || (a->state_bits == 8 && (!a->exp_avg_scale || !a->exp_avg_sq_scale)) ||
      (a->master && a->dtype == F16_DTYPE_FP32) || (a->partial && a->partials <= 0))
    return F16_ERR_ARG;
  const size_t size = a->dtype == F16_DTYPE_FP32 ? 4 : 2;
  if (!aligned(a->exp_avg, 16) || !aligned(a->exp_avg_sq, 16) || !aligned(a->master, 16)) return F16_ERR_ALIGN;
  for (int i = 0; i < a->count; i++) {
    if (!a->params_host[i] || !a->grads_host[i] || a->numel_host[i] <= 0 || a->first_host[i] < 0 ||
        a->first_host[i] % opt::QBLOCK || a->index_host[i] < 0)
      return F16_ERR_ARG;
    if (!aligned(a->params_host[i], size) || !aligned(a->grads_host[i], size)) return F16_ERR_ALIGN;
  }
  opt::Hyper hy;
  hy.lr = a->lr;
  hy.b1 = a->beta1;
  hy.b2 = a->beta2;
  hy.eps = (float)a->eps;
  hy.decay = (float)(1.0 - a->lr * a->weight_decay);
  hy.keep1 = (float)a->beta1;
  hy.new1 = (float)(1.0 - a->beta1);
  hy.keep2 = (float)a->beta2;
  hy.new2 = (float)(1.0 - a->beta2);
  hy.max_norm = a->max_norm;
  opt::Flat fl = {a->exp_avg, a->exp_avg_sq, a->exp_avg_scale, a->exp_avg_sq_scale, a->master, a->steps, a->ticket,
                  a->partial, a->partials, a->norm, a->seed};
  const cudaStream_t st = cu_stream(stream);
  for (int i = 0; i < a->count; i += opt::LARGE) {
    const int n = a->count - i < opt::LARGE ? a->count - i : opt::LARGE;
    const auto go = [&](auto tag) {
      typedef decltype(tag) T;
      return n <= opt::SMALL ? opt::update<T, opt::SMALL>(n, a->params_host + i, a->grads_host + i, a->numel_host + i,
                                                          a->first_host + i, a->index_host + i, hy, fl, a->state_bits, st)
                             : opt::update<T, opt::LARGE>(n, a->params_host + i, a->grads_host + i, a->numel_host + i,
                                                          a->first_host + i, a->index_host + i, hy, fl, a->state_bits, st);
    };
    const int rc = a->dtype == F16_DTYPE_FP32 ? go(0.0f) : a->dtype == F16_DTYPE_BF16 ? go(__nv_bfloat16()) : go(__half());
    if (rc != F16_OK) return rc;
  }
  return F16_OK;
}
