// optim_kernels.cu -- one AdamW step over many tensors: the gradients' norm and the update.
//
//   n = sqrt(sum g^2) over all tensors,  c = min(1, max_norm / (n + 1e-6)),  g' = c g
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by HBM: a step reads p, g, m, v and writes p, m, v once, and the norm reads g once more.  The
// tensors come as a table in the kernel's parameters (no device table to build or keep), their
// moments lie in flat buffers that begin a new block of QBLOCK values with every tensor.  Persistent
// blocks walk over pieces of PIECE values.  The norm's squares are added 32 at a time in fp32, then in fp64, each
// block in the same order; the step counts live on the device and the last block to finish
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
//
// Measured on a B200 whose copy makes 6.55 TB/s (norm + update, us, with a cold L2): 252 million fp32 parameters with
// 8-bit moments 167 + 814 (92%, 76% of that rate), 300 tensors with 22 million bf16 parameters, fp32 moments and masters
// 14 + 120, 1.3 million fp32 parameters 4 + 10; 252 million bf16 parameters with 8-bit moments 95 + 808, with masters 95 +
// 933 (48% and 74%: the same instructions over fewer bytes).  The 8-bit update is bound by the instructions of its roundings (integer
// pipe 60%, 2.7 of 4 issue slots), not by HBM; pairs of values in one instruction brought it from 956 to 847.
#include <cuda_fp8.h>
#include "typed.cuh"

namespace f16 {
namespace opt {

constexpr int THREADS = 256;
// Resident update blocks, each walking over its share: 64 registers a thread (80 and three blocks: +4% with 8-bit moments,
// +7% with the next block's values copied to shared memory ahead).
constexpr int BLOCKS_PER_SM = 4;
constexpr int NORM_BLOCKS_PER_SM = 4;
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
  float eps, decay, minus_zero;     // decay: 1 - lr wd
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

// x / s rounded towards zero (x >= 0, inv = 1 / s): a Newton step with a fused residual (Markstein's method) gives
// the nearest quotient, the sign of its residual says whether that lies above the true one.  What the rounding to a code below looks at are whole
// units of the quotient's last place, so it decides as the exact quotient would; the nearest one would
// fall on the wrong side of a code's border once in some 10^6 -- and often where a block's values all
// shrink alike, which makes the quotients codes again and again.
__device__ __forceinline__ Two quotient_rz(Two x, Two minus_s, Two inv) {
  const Two q0 = x * inv, q = fma2(fma2(q0, minus_s, x), inv, q0);
  const float2 f = split(q), res = split(fma2(q, minus_s, x));
  return two(__int_as_float(__float_as_int(f.x) + (__float_as_int(res.x) >> 31)),
             __int_as_float(__float_as_int(f.y) + (__float_as_int(res.y) >> 31)));
}

// x >= 0 rounded to `MANT` mantissa bits (subnormals below 2^LOW included): up where the 16 random bits
// and the part left over carry.  A carry above the type's largest is taken back by the conversion to it,
// which saturates.
template <int MANT, int LOW>
__device__ __forceinline__ float round_carry(float x, unsigned bits) {
  constexpr int DROP = 23 - MANT;
  const float low = __int_as_float((127 + LOW) << 23);
  const bool sub = x < low;
  if (sub) x = __fadd_rz(x, low);                 // in [low, 2 low) a mantissa step is a subnormal one
  float r = __uint_as_float((__float_as_uint(x) + (bits << (DROP - 16))) & ~((1u << DROP) - 1));
  if (sub) r -= low;
  return r;
}

constexpr unsigned INF_BITS = 0x7f800000u;        // of sizes as integers: finite < infinite < NaN

// The moments' sizes that make their block's scales: the largest finite ones, as integers.
__device__ __forceinline__ void block_sizes(const Two (&m)[2][2], const Two (&v)[2][2], unsigned& m_most,
                                            unsigned& v_most, bool& finite) {
  const auto most = [](const Two (&t)[2][2], unsigned below) {
    unsigned a = 0;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const float2 f = split(t[h][k]);
        const unsigned x = __float_as_uint(f.x) & 0x7fffffffu, y = __float_as_uint(f.y) & 0x7fffffffu;
        a = max(a, max(x < below ? x : 0u, y < below ? y : 0u));
      }
    return __reduce_max_sync(~0u, a);
  };
  m_most = most(m, 0xffffffffu);
  v_most = most(v, 0xffffffffu);
  finite = m_most < INF_BITS && v_most < INF_BITS;
  if (!finite) {
    m_most = most(m, INF_BITS);
    v_most = most(v, INF_BITS);
  }
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

// What a step's update of one tensor needs beside its values.
struct Numbers {
  float clip, rate, root;       // of the gradient; lr / (1 - b1^t); 1 / sqrt(1 - b2^t)
  uint64_t key;
};

// The parameter after the step.  The change is good to some 2^-21 of itself (approximate root and
// reciprocal): far below the parameter's rounding.
__device__ __forceinline__ float changed(float w, float m, float v, const Hyper& hy, const Numbers& nu) {
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(fmaf(root_of(v), nu.root, hy.eps)));
  return fmaf(-(nu.rate * m), inv, w * hy.decay);
}

template <typename T>
__device__ __forceinline__ bool same(T a, T b) {
  Vec<T, 1> x, y;
  x.e[0] = a;
  y.e[0] = b;
  return x.r == y.r;
}

// A warp's QBLOCK values from element `at` of a tensor on.  FULL: all of them exist, aligned for loads of
// four.  Else the gradient, the moments and the master are zero past the tensor's end, and stay it.
template <typename T, int BITS, bool MASTER, bool FULL>
__device__ __forceinline__ void update_block(T* p, const T* g, int64_t n, int64_t at, int64_t flat, bool vec,
                                             const Hyper& hy, const Flat& fl, const Numbers& nu) {
  const int lane4 = (threadIdx.x & 31) * 4;
  Vec<T, 4> pv[2], gv[2];
  Two m[2][2], v[2][2];
  float ms[2][4];
  float m_unit = 0.0f, v_unit = 0.0f;
  if (FULL) {
    p += at + lane4;
    g += at + lane4;
  }
#pragma unroll
  for (int h = 0; h < 2; h++) {
    gv[h] = FULL ? load_vec_nc<T, 4>(g + h * 128) : load4(g, at + h * 128 + lane4, n, vec);
    pv[h] = FULL ? load_vec<T, 4>(p + h * 128) : load4<T>(p, at + h * 128 + lane4, n, vec);
  }
  if (BITS == 8) {
    const uint32_t* mp = reinterpret_cast<const uint32_t*>(reinterpret_cast<uint8_t*>(fl.m) + flat + lane4);
    const uint32_t* vp = reinterpret_cast<const uint32_t*>(reinterpret_cast<uint8_t*>(fl.v) + flat + lane4);
    const uint32_t mc[2] = {mp[0], mp[32]}, vc[2] = {vp[0], vp[32]};
    m_unit = fl.m_scale[flat / QBLOCK];
    v_unit = fl.v_scale[flat / QBLOCK];
    const Two mu = two(m_unit), vu = two(v_unit);
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const float2 a = unpack8(mc[h] >> (16 * k) & 0xffff, __NV_E4M3), b = unpack8(vc[h] >> (16 * k) & 0xffff, __NV_E5M2);
        m[h][k] = two(a.x, a.y) * mu;
        v[h][k] = two(b.x, b.y) * vu;
      }
  } else {
    const float4* mp = reinterpret_cast<const float4*>(reinterpret_cast<float*>(fl.m) + flat + lane4);
    const float4* vp = reinterpret_cast<const float4*>(reinterpret_cast<float*>(fl.v) + flat + lane4);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const float4 a = mp[32 * h], b = vp[32 * h];
      m[h][0] = two(a.x, a.y);
      m[h][1] = two(a.z, a.w);
      v[h][0] = two(b.x, b.y);
      v[h][1] = two(b.z, b.w);
    }
  }
  float4* wp = reinterpret_cast<float4*>(fl.master + flat + lane4);
  if (MASTER) {
#pragma unroll
    for (int h = 0; h < 2; h++) *reinterpret_cast<float4*>(ms[h]) = wp[32 * h];
  }
  const Two zero = two(hy.minus_zero), clip = two(nu.clip), keep1 = two(hy.keep1), new1 = two(hy.new1), keep2 = two(hy.keep2), new2 = two(hy.new2);
#pragma unroll
  for (int h = 0; h < 2; h++) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const Two gr = pair_of<T, 4>(gv[h], k) * clip;
      // each product rounded by itself, as torch's expressions do (a product and a sum of pairs are made one
      // fused operation by the assembler; with a zero added that it does not know the product stays)
      m[h][k] = fma2(keep1, m[h][k], zero) + fma2(new1, gr, zero);
      v[h][k] = fma2(keep2, v[h][k], zero) + fma2(new2, fma2(gr, gr, zero), zero);
      const float2 mf = split(m[h][k]), vf = split(v[h][k]);
      float2 w = split(pair_of<T, 4>(pv[h], k));
      if (MASTER) {
        w.x = same(from_f32<T>(ms[h][2 * k]), pv[h].e[2 * k]) ? ms[h][2 * k] : w.x;
        w.y = same(from_f32<T>(ms[h][2 * k + 1]), pv[h].e[2 * k + 1]) ? ms[h][2 * k + 1] : w.y;
      }
      w.x = changed(w.x, mf.x, vf.x, hy, nu);
      w.y = changed(w.y, mf.y, vf.y, hy, nu);
      if (MASTER) {
        ms[h][2 * k] = FULL || at + h * 128 + lane4 + 2 * k < n ? w.x : 0.0f;
        ms[h][2 * k + 1] = FULL || at + h * 128 + lane4 + 2 * k + 1 < n ? w.y : 0.0f;
      }
      set_pair<T, 4>(pv[h], k, two(w.x, w.y));
    }
    if (FULL) store_vec<T, 4>(p + h * 128, pv[h]);
    else store4(p, at + h * 128 + lane4, n, vec, pv[h]);
    if (MASTER) wp[32 * h] = *reinterpret_cast<const float4*>(ms[h]);
  }
  if (!FULL && nu.clip != nu.clip) {              // what lies past the end is zero, not 0 times a NaN
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const int i = h * 128 + lane4 + 2 * k;
        const float2 a = split(m[h][k]), b = split(v[h][k]);
        m[h][k] = two(at + i < n ? a.x : 0.0f, at + i + 1 < n ? a.y : 0.0f);
        v[h][k] = two(at + i < n ? b.x : 0.0f, at + i + 1 < n ? b.y : 0.0f);
      }
  }
  if (BITS == 8) {
    unsigned m_most, v_most;
    bool finite;
    block_sizes(m, v, m_most, v_most, finite);
    const float tiny = __int_as_float(1 << 23);         // the smallest normal: its reciprocal is finite
    m_unit = fmaxf(__uint_as_float(m_most) * (1.0f / 448.0f), tiny);
    v_unit = fmaxf(__uint_as_float(v_most) * (1.0f / 57344.0f), tiny);
    if (lane4 == 0) {
      fl.m_scale[flat / QBLOCK] = m_unit;
      fl.v_scale[flat / QBLOCK] = v_unit;
    }
    const Two mu = two(-m_unit), vu = two(-v_unit), mi = two(1.0f / m_unit), vi = two(1.0f / v_unit);
    uint32_t* mp = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(fl.m) + flat + lane4);
    uint32_t* vp = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(fl.v) + flat + lane4);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint64_t first = nu.key + (uint64_t)((flat + h * 128 + lane4) >> 1);
      uint32_t mc = 0, vc = 0;
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const uint64_t word = mix64(first + k);
        const unsigned lo = (unsigned)word, hi = (unsigned)(word >> 32);
        const float2 mf = split(m[h][k]), vf = split(v[h][k]);
        const float2 mq = split(quotient_rz(two(fabsf(mf.x), fabsf(mf.y)), mu, mi)), vq = split(quotient_rz(v[h][k], vu, vi));
        float2 a = make_float2(copysignf(round_carry<3, -6>(mq.x, lo & 0xffff), mf.x),
                               copysignf(round_carry<3, -6>(mq.y, hi & 0xffff), mf.y));
        float2 b = make_float2(round_carry<2, -14>(vq.x, lo >> 16), round_carry<2, -14>(vq.y, hi >> 16));
        const float least = 1.52587890625e-05f;                         // 2^-16, the smallest code above zero
        if (vf.x > 0.0f) b.x = fmaxf(b.x, least);
        if (vf.y > 0.0f) b.y = fmaxf(b.y, least);
        if (!finite) {
          const float nan = __int_as_float(0x7fffffff);
          if ((__float_as_uint(mf.x) & 0x7fffffffu) >= INF_BITS) a.x = nan;
          if ((__float_as_uint(mf.y) & 0x7fffffffu) >= INF_BITS) a.y = nan;
          if ((__float_as_uint(vf.x) & 0x7fffffffu) >= INF_BITS) b.x = nan;
          if ((__float_as_uint(vf.y) & 0x7fffffffu) >= INF_BITS) b.y = nan;
        }
        mc |= (uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) << (16 * k);
        vc |= (uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E5M2) << (16 * k);
      }
      mp[32 * h] = mc;
      vp[32 * h] = vc;
    }
  } else {
    float4* mp = reinterpret_cast<float4*>(reinterpret_cast<float*>(fl.m) + flat + lane4);
    float4* vp = reinterpret_cast<float4*>(reinterpret_cast<float*>(fl.v) + flat + lane4);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const float2 a = split(m[h][0]), b = split(m[h][1]), c = split(v[h][0]), d = split(v[h][1]);
      mp[32 * h] = make_float4(a.x, a.y, b.x, b.y);
      vp[32 * h] = make_float4(c.x, c.y, d.x, d.y);
    }
  }
}

template <typename T, int N, int BITS, bool MASTER>
__global__ void __launch_bounds__(THREADS, BLOCKS_PER_SM)
    k_adamw(const __grid_constant__ Table<N> tab, const __grid_constant__ Hyper hy, const __grid_constant__ Flat fl) {
  __shared__ double s[THREADS / 32];
  const int64_t pieces = tab.first[tab.count];
  Numbers nu = {1.0f, 0.0f, 0.0f, 0};
  if (fl.partial) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < fl.partials; i += THREADS) sum += fl.partial[i];
    const double norm = sqrt(block_sum(sum, s));
    const double c = hy.max_norm / (norm + 1e-6);
    nu.clip = c < 1.0 || c != c ? (float)c : 1.0f;
    if (blockIdx.x == 0 && threadIdx.x == 0 && fl.norm) *fl.norm = (float)norm;
  }
  int64_t step = -1;
  for (int64_t piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    const int i = tensor_of(tab, piece);
    const int64_t n = tab.t[i].n, at = (piece - tab.first[i]) * PIECE + (threadIdx.x >> 5) * QBLOCK;
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
      nu.rate = (float)(hy.lr / (1.0 - p1));
      nu.root = (float)(1.0 / sqrt(1.0 - p2));
      nu.key = mix64(fl.seed ^ mix64((uint64_t)t));
    }
    if (at >= n) continue;                         // the warp's part lies past the tensor's end
    if (vec && at + QBLOCK <= n) update_block<T, BITS, MASTER, true>(p, g, n, at, flat, vec, hy, fl, nu);
    else update_block<T, BITS, MASTER, false>(p, g, n, at, flat, vec, hy, fl, nu);
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

inline unsigned blocks_for(int64_t pieces, int per_sm) {
  const int64_t most = (int64_t)sm_count() * per_sm;
  return (unsigned)(pieces < most ? pieces : most);
}

template <typename T, int N>
int squares(int count, const void* const* g, const int64_t* n, double* partial, int room, int* used, cudaStream_t st) {
  Table<N> tab;
  fill<N>(tab, NORM_PIECE, count, nullptr, g, n, nullptr, nullptr);
  unsigned grid = blocks_for(tab.first[count], NORM_BLOCKS_PER_SM);
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
  const unsigned grid = blocks_for(tab.first[count], BLOCKS_PER_SM);
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
  hy.minus_zero = -0.0f;
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
