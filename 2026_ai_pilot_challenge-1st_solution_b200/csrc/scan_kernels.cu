// scan_kernels.cu -- a gated linear recurrence over time, its gradient, and its single step.
//
//   h_t = a_t h_{t-1} + b_t        a_t given, b_t = x_t                       (raw)
//                                  a_t = f = sigmoid(gate_t), b_t = (1-f) x_t  (gated)
//
// for every channel (a sequence's feature) by itself; a reset at t drops h_{t-1} (h_t = b_t: an
// episode begins), steps from a sequence's length on leave the state as it is.  Backward, with G_t
// the gradient of h_t:  G_t = dh_t + a_{t+1} G_{t+1} (no second term where t+1 resets),
//   raw:    da_t = G_t h_{t-1},                      dx_t = G_t
//   gated:  dgate_t = G_t (h_{t-1} - x_t) f (1-f),   dx_t = G_t (1-f)
//
// All of it is bound by HBM: forward reads gate and x and writes h, backward reads gate, x and dh
// and writes two gradients.  h is not read back: the forward pass leaves the fp32 state before
// every CHUNK steps (4 / CHUNK bytes a value), from which the backward pass repeats the chunk in
// registers, so its h_{t-1} are the fp32 ones and not the rounded outputs.
//
// A thread owns the V channels of 4 bytes (two 16-bit values, or one where rows are not aligned for
// that), a warp 32 neighbours of them, and takes CHUNK steps at a time into registers.
//  * Many channels (k_scan<SPLIT = false>): a warp walks through time alone, the state in registers.
//  * Few (SPLIT = true): the warps of a block, and the blocks of a cluster, take consecutive chunks of
//    the same channels.  A chunk maps the state before it to A h + B; the (A, B) of a block's warps
//    meet in shared memory, those of the cluster's blocks in every block's shared memory (DSMEM), each
//    warp folds those before it into its own first state and repeats its chunk from registers.  Data
//    is read once, the order of all sums is fixed, and the blocks of a cluster are resident together,
//    so nothing spins on memory.
// A chunk that a reset cuts passes nothing of the state before it on.  That is kept as A = NaN, a
// selection (never a product with 0), so that an infinity or NaN left by the episode before does not
// leak: a coefficient that is NaN itself makes B NaN as well, so the two cannot be confused.
#include <cooperative_groups.h>
#include <type_traits>
#include "typed.cuh"

namespace cg = cooperative_groups;

namespace f16 {
namespace scan {

constexpr int CHUNK = F16_SCAN_CHUNK;     // steps in registers at a time, between saved states
constexpr int MAX_WARPS = 16;             // of a block on consecutive chunks
constexpr int MAX_CLUSTER = 8;            // blocks of a cluster on consecutive chunks
constexpr int WIDE_WARPS = 4;             // of a block whose warps have channels of their own
constexpr int WIDE_BLOCKS = 5, WIDE_GRAD_BLOCKS = 3;      // of those on an SM: 96 and 168 registers a thread
static_assert(CHUNK <= 32, "resets of a chunk are bits of one word");

typedef f16_scan_args Args;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A step's coefficients in one register.  Gated: the smaller one of f and 1 - f, e / (1 + e) with
// e = exp(-|gate|), with the gate's sign: negative, it is f.  The other is its difference from 1, which
// is at least 1/2 and so keeps every digit.  Raw: the coefficient itself.
template <bool GATED>
__device__ __forceinline__ float packed_gate(float g) {
  if (!GATED) return g;
  const float e = ex2(-1.4426950408889634f * fabsf(g));
  return copysignf(e * rcp(1.0f + e), g);
}
template <bool GATED>
__device__ __forceinline__ void coefficients(float s, float& a, float& k) {
  if (GATED) {
    const float small = fabsf(s), big = 1.0f - small;
    const bool neg = __float_as_int(s) < 0;
    a = neg ? small : big;
    k = neg ? big : small;
  } else {
    a = s;
    k = 1.0f;
  }
}

// h -> A h + B, where A is not NaN (cut) and h not zero (so that an overflown A cannot make NaN of it).
__device__ __forceinline__ float pass_through(float A, float B, float h) {
  return A != A || h == 0.0f ? B : fmaf(A, h, B);
}

struct Lane {
  int64_t b, d, c;      // sequence, feature, channel = b dim + d
  bool live;            // the channel exists
  bool together;        // all channels of the warp belong to one sequence
  int len;              // the sequence's steps
};

// Called by whole warps: c is the first of the lane's channels.
__device__ __forceinline__ Lane lane_of(const Args& p, int64_t c) {
  Lane l;
  l.c = c;
  l.live = c < p.batch * p.dim;
  l.b = l.live ? c / p.dim : 0;
  l.d = l.live ? c - l.b * p.dim : 0;
  const int64_t first = __shfl_sync(~0u, l.b, 0);
  if (!l.live) l.b = first;
  l.together = __all_sync(~0u, l.b == first);
  l.len = (int)p.steps;
  if (p.lengths) {
    const int64_t n = p.lengths[l.b];
    l.len = (int)(n < 0 ? 0 : n < p.steps ? n : p.steps);
  }
  return l;
}

__device__ __forceinline__ bool reset_at(const Args& p, int64_t b, int64_t t) {
  const int64_t i = b * p.reset_b + t * p.reset_t;
  return p.reset_bytes == 1 ? __ldg(reinterpret_cast<const uint8_t*>(p.reset) + i) != 0
                            : __ldg(reinterpret_cast<const float*>(p.reset) + i) != 0.0f;
}

// Bit i: step t0 + i (of the n from t0 on) resets the lane's sequence.  Called by whole warps: where a warp
// has one sequence its lanes read a step each.
__device__ __forceinline__ unsigned resets_of(const Args& p, const Lane& l, int t0, int n) {
  if (!p.reset) return 0;
  if (l.together) {
    const int lane = threadIdx.x & 31, m = l.len - t0 < CHUNK ? l.len - t0 : CHUNK;
    return __ballot_sync(~0u, t0 >= 0 && lane < m && reset_at(p, l.b, t0 + lane));
  }
  unsigned m = 0;
#pragma unroll 1
  for (int i = 0; i < n; i++) m |= (unsigned)reset_at(p, l.b, t0 + i) << i;
  return m;
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Vec<T, V>& v, float (&f)[V]) {
  if constexpr (sizeof(T) == 2 && V == 2) {
    float2 two;
    if constexpr (std::is_same<T, __half>::value) {
      two = __half22float2(*reinterpret_cast<const __half2*>(&v));
    } else {
      two = make_float2(__uint_as_float(v.r << 16), __uint_as_float(v.r & 0xffff0000u));
    }
    f[0] = two.x;
    f[1] = two.y;
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) f[k] = to_f32(v.e[k]);
  }
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> pack(const float (&f)[V]) {
  Vec<T, V> v;
  if constexpr (std::is_same<T, __nv_bfloat16>::value && V == 2) {
    const __nv_bfloat162 two = __floats2bfloat162_rn(f[0], f[1]);
    v.r = *reinterpret_cast<const unsigned*>(&two);
  } else if constexpr (std::is_same<T, __half>::value && V == 2) {
    const __half2 two = __floats2half2_rn(f[0], f[1]);
    v.r = *reinterpret_cast<const unsigned*>(&two);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) v.e[k] = from_f32<T>(f[k]);
  }
  return v;
}

// A tensor's element (t0, b, d), and how far it is to the next step's.
template <typename T>
struct Line {
  T* p;
  int64_t st;
  __device__ __forceinline__ Line(const void* base, int64_t st, int64_t sb, const Lane& l, int t0)
      : p(reinterpret_cast<T*>(const_cast<void*>(base)) + l.b * sb + l.d + (int64_t)t0 * st), st(st) {}
};
// One step on.  Opaque, so that a chunk's addresses are made one after the other and not all kept.
template <typename T>
__device__ __forceinline__ void advance(T*& q, int64_t by) {
  q += by;
  asm volatile("" : "+l"(q));
}

// The first n of CHUNK steps (ALL: every one); the others are left alone.
template <typename T, int V, bool ALL>
__device__ __forceinline__ void load_chunk(Vec<T, V> (&v)[CHUNK], Line<T> at, int n) {
#pragma unroll
  for (int i = 0; i < CHUNK; i++) {
    if (ALL || i < n) v[i] = load_vec_nc<T, V>(at.p);
    advance(at.p, at.st);
  }
}
template <typename T, int V>
__device__ __forceinline__ void load_chunk(Vec<T, V> (&v)[CHUNK], const Line<T>& at, int n, bool all) {
  if (all) load_chunk<T, V, true>(v, at, n);
  else load_chunk<T, V, false>(v, at, n);
}

template <int V>
__device__ __forceinline__ void load_state(float (&h)[V], const float* p, const Lane& l) {
#pragma unroll
  for (int k = 0; k < V; k++) h[k] = p && l.live ? p[l.c + k] : 0.0f;
}
template <int V>
__device__ __forceinline__ void store_state(float* p, const float (&h)[V], const Lane& l) {
  if (p && l.live) {
#pragma unroll
    for (int k = 0; k < V; k++) p[l.c + k] = h[k];
  }
}

// What the warps of a block and the blocks of a cluster tell one another, twice (a tile's is still
// read while the next one's is written).
template <int V>
struct Shared {
  float2 warp[2][MAX_WARPS][32][V];
  float2 block[2][MAX_CLUSTER][32][V];
};

// (A, B) of this warp's chunk in, the state before the chunk out; `carry`, the state before the tile,
// becomes the state after it.
template <int V>
__device__ __forceinline__ void join(Shared<V>& s, int half, int warps, int blocks, int rank, const float (&A)[V],
                                     const float (&B)[V], float (&carry)[V], float (&before)[V]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < V; k++) s.warp[half][warp][lane][k] = make_float2(A[k], B[k]);
  __syncthreads();
  if (blocks > 1) {
    // the block's own map, to block `warp` of the cluster: the first `blocks` warps each serve one
    // (a tile of a cluster has as many warps as blocks at least)
    if (warp < blocks) {
      Shared<V>* there = cg::this_cluster().map_shared_rank(&s, warp);
#pragma unroll
      for (int k = 0; k < V; k++) {
        float2 all = s.warp[half][0][lane][k];
        for (int w = 1; w < warps; w++) {
          const float2 m = s.warp[half][w][lane][k];
          all.y = pass_through(m.x, m.y, all.y);
          all.x = m.x * all.x;              // NaN (cut) stays NaN
        }
        there->block[half][rank][lane][k] = all;
      }
    }
    cg::this_cluster().sync();
  }
#pragma unroll
  for (int k = 0; k < V; k++) {
    float h = carry[k], mine = h;
    if (blocks > 1) {
      for (int r = 0; r < blocks; r++) {
        if (r == rank) mine = h;
        const float2 m = s.block[half][r][lane][k];
        h = pass_through(m.x, m.y, h);
      }
    }
    float at = mine;
    for (int w = 0; w < warps; w++) {
      if (w == warp) before[k] = at;
      if (w == warp && blocks > 1) break;
      const float2 m = s.warp[half][w][lane][k];
      at = pass_through(m.x, m.y, at);
    }
    carry[k] = blocks > 1 ? h : at;
  }
}

// The steps of a chunk from the state h on, written to `out`.  PLAIN: every lane has all CHUNK steps and no
// reset among them.  s: the packed coefficients (gated; raw ones are read from g).
template <typename T, int V, bool GATED, bool PLAIN>
__device__ __forceinline__ void walk(const Vec<T, V> (&g)[CHUNK], const float (&s)[GATED ? CHUNK : 1][V],
                                     const Vec<T, V> (&x)[CHUNK], unsigned cut, int n, int left, bool live, Line<T> out,
                                     float (&h)[V]) {
#pragma unroll
  for (int i = 0; i < CHUNK; i++) {
    float xf[V], gf[V], o[V];
    unpack<T, V>(x[i], xf);
    if (!GATED) unpack<T, V>(g[i], gf);
#pragma unroll
    for (int k = 0; k < V; k++) {
      float a, c;
      coefficients<GATED>(GATED ? s[i][k] : gf[k], a, c);
      const float b = GATED ? c * xf[k] : xf[k];
      if (PLAIN) {
        h[k] = fmaf(a, h[k], b);
        o[k] = h[k];
      } else {
        if (i < n) h[k] = cut >> i & 1 ? b : fmaf(a, h[k], b);
        o[k] = i < n ? h[k] : 0.0f;
      }
    }
    if (PLAIN || (live && i < left)) store_vec<T, V>(out.p, pack<T, V>(o));
    advance(out.p, out.st);
  }
}

template <typename T, int V, bool GATED>
__device__ __forceinline__ void pack_gates(const Vec<T, V> (&g)[CHUNK], float (&s)[GATED ? CHUNK : 1][V]) {
  if constexpr (GATED) {
#pragma unroll
    for (int i = 0; i < CHUNK; i++) {
      float gf[V];
      unpack<T, V>(g[i], gf);
#pragma unroll
      for (int k = 0; k < V; k++) s[i][k] = packed_gate<true>(gf[k]);
    }
  }
}

template <typename T, int V, bool GATED, bool SPLIT>
__global__ void __launch_bounds__(SPLIT ? 32 * MAX_WARPS : 32 * WIDE_WARPS, SPLIT ? 1 : WIDE_BLOCKS)
    k_scan(const __grid_constant__ Args p, int blocks) {
  const int warp = threadIdx.x >> 5, warps = SPLIT ? blockDim.x >> 5 : 1;
  const int rank = SPLIT ? (int)(blockIdx.x % blocks) : 0;
  const int64_t group = SPLIT ? blockIdx.x / blocks : (int64_t)blockIdx.x * WIDE_WARPS + warp;
  const Lane l = lane_of(p, (group * 32 + (threadIdx.x & 31)) * V);
  const int tile = CHUNK * (SPLIT ? warps * blocks : 1), T_ = (int)p.steps;
  float h[V];
  load_state<V>(h, p.h0, l);
  if (SPLIT && blocks > 1) cg::this_cluster().sync();      // every block has begun
  const int mine = SPLIT ? (rank * warps + warp) * CHUNK : 0;
  const auto steps_at = [&](int t0) { return l.live ? (l.len - t0 < CHUNK ? l.len - t0 : CHUNK) : 0; };
  Vec<T, V> g[CHUNK], x[CHUNK];
  const auto fetch = [&](int t0) {
    const int n = steps_at(t0);
    const bool all = __all_sync(~0u, n == CHUNK);
    load_chunk<T, V>(g, Line<T>(p.gate, p.gate_t, p.gate_b, l, t0), n, all);
    load_chunk<T, V>(x, Line<T>(p.x, p.x_t, p.x_b, l, t0), n, all);
    return resets_of(p, l, t0, n);
  };
  int half = 0;
  for (int base = 0; base < T_; base += tile, half ^= 1) {
    const int t0 = base + mine, left = T_ - t0, n = steps_at(t0);
    const unsigned cut = fetch(t0);
    const bool plain = __all_sync(~0u, n == CHUNK && cut == 0);
    float s[GATED ? CHUNK : 1][V];
    pack_gates<T, V, GATED>(g, s);
    float before[V];
    if (SPLIT) {
      __shared__ Shared<V> sh;
      float A[V], B[V];
#pragma unroll
      for (int k = 0; k < V; k++) {
        A[k] = 1.0f;
        B[k] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < CHUNK; i++) {
        float xf[V], gf[V];
        unpack<T, V>(x[i], xf);
        if (!GATED) unpack<T, V>(g[i], gf);
#pragma unroll
        for (int k = 0; k < V; k++) {
          float a, c;
          coefficients<GATED>(GATED ? s[i][k] : gf[k], a, c);
          const float b = GATED ? c * xf[k] : xf[k];
          if (i < n) {
            const bool r = cut >> i & 1;
            A[k] = r ? __int_as_float(0x7fffffff) : A[k] * a;
            B[k] = r ? b : fmaf(a, B[k], b);
          }
        }
      }
      join<V>(sh, half, warps, blocks, rank, A, B, h, before);
      // h is the state after the tile now; the chunk is repeated from `before`
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) before[k] = h[k];
    }
    if (p.saved && left > 0) store_state<V>(p.saved + (int64_t)(t0 / CHUNK) * p.batch * p.dim, before, l);
    const Line<T> out(p.h, p.h_t, p.h_b, l, t0);
    if (plain) walk<T, V, GATED, true>(g, s, x, 0, CHUNK, CHUNK, true, out, before);
    else walk<T, V, GATED, false>(g, s, x, cut, n, left, l.live, out, before);
    if (!SPLIT) {
#pragma unroll
      for (int k = 0; k < V; k++) h[k] = before[k];
    }
  }
  if (!SPLIT || (rank == 0 && warp == 0)) store_state<V>(p.hn, h, l);
}

// The steps of a chunk again from the saved state h, then their gradients from the last one back; carry: the
// gradient that reaches the chunk's last state, then the one that leaves its first.
// Gated: with d_t = f (h_{t-1} - x_t), dx_t = G k and dgate_t = dx_t d_t.
template <typename T, int V, bool GATED, bool PLAIN>
__device__ __forceinline__ void walk_back(const Vec<T, V> (&g)[CHUNK], const float (&s)[GATED ? CHUNK : 1][V],
                                          const Vec<T, V> (&x)[CHUNK], const Vec<T, V> (&dh)[CHUNK], unsigned cut, int n,
                                          int left, bool live, Line<T> dg, bool want_g, Line<T> dx, bool want_x,
                                          float (&h)[V], float (&carry)[V]) {
  float d[CHUNK][V];
#pragma unroll
  for (int i = 0; i < CHUNK; i++) {
    float xf[V], gf[V];
    unpack<T, V>(x[i], xf);
    if (!GATED) unpack<T, V>(g[i], gf);
#pragma unroll
    for (int k = 0; k < V; k++) {
      float a, c;
      coefficients<GATED>(GATED ? s[i][k] : gf[k], a, c);
      const float b = GATED ? c * xf[k] : xf[k];
      const bool r = !PLAIN && (cut >> i & 1);
      const float hp = r ? 0.0f : h[k];
      d[i][k] = GATED ? a * (hp - xf[k]) : hp;
      h[k] = r ? b : fmaf(a, hp, b);
    }
  }
  const int last = CHUNK - 1;
  dg.p += last * dg.st;
  dx.p += last * dx.st;
#pragma unroll
  for (int i = CHUNK - 1; i >= 0; i--) {
    float gf[V], df[V], og[V], ox[V];
    unpack<T, V>(dh[i], df);
    if (!GATED) unpack<T, V>(g[i], gf);
#pragma unroll
    for (int k = 0; k < V; k++) {
      float a, c;
      coefficients<GATED>(GATED ? s[i][k] : gf[k], a, c);
      const float G = df[k] + carry[k];
      ox[k] = GATED ? G * c : G;
      og[k] = ox[k] * d[i][k];
      if (PLAIN) {
        carry[k] = a * G;
      } else {
        if (i < n) carry[k] = cut >> i & 1 ? 0.0f : a * G;
        if (i >= n) og[k] = ox[k] = 0.0f;
      }
    }
    if (PLAIN || (live && i < left)) {
      if (want_g) store_vec<T, V>(dg.p, pack<T, V>(og));
      if (want_x) store_vec<T, V>(dx.p, pack<T, V>(ox));
    }
    advance(dg.p, -dg.st);
    advance(dx.p, -dx.st);
  }
}

// Backward: tiles and chunks from the last to the first, the carried value the gradient of the state
// before the steps already done.
template <typename T, int V, bool GATED, bool SPLIT>
__global__ void __launch_bounds__(SPLIT ? 32 * MAX_WARPS : 32 * WIDE_WARPS, SPLIT ? 1 : WIDE_GRAD_BLOCKS)
    k_scan_grad(const __grid_constant__ Args p, int blocks) {
  const int warp = threadIdx.x >> 5, warps = SPLIT ? blockDim.x >> 5 : 1;
  const int rank = SPLIT ? (int)(blockIdx.x % blocks) : 0;
  const int64_t group = SPLIT ? blockIdx.x / blocks : (int64_t)blockIdx.x * WIDE_WARPS + warp;
  const Lane l = lane_of(p, (group * 32 + (threadIdx.x & 31)) * V);
  const int T_ = (int)p.steps, chunks = (T_ + CHUNK - 1) / CHUNK, tile = SPLIT ? warps * blocks : 1;
  float carry[V];
  load_state<V>(carry, p.dhn, l);
  if (SPLIT && blocks > 1) cg::this_cluster().sync();
  int half = 0;
  for (int done = 0; done < chunks; done += tile, half ^= 1) {
    const int q = chunks - 1 - (done + (SPLIT ? rank * warps + warp : 0));      // below 0: nothing left
    const int t0 = q * CHUNK, left = q < 0 ? 0 : T_ - t0;
    const int n = l.live && q >= 0 ? (l.len - t0 < CHUNK ? l.len - t0 : CHUNK) : 0;
    const bool all = __all_sync(~0u, n == CHUNK);
    Vec<T, V> g[CHUNK], x[CHUNK], dh[CHUNK];
    load_chunk<T, V>(g, Line<T>(p.gate, p.gate_t, p.gate_b, l, t0), n, all);
    if (p.dh) {
      load_chunk<T, V>(dh, Line<T>(p.dh, p.dh_t, p.dh_b, l, t0), n, all);
    } else {
#pragma unroll
      for (int i = 0; i < CHUNK; i++)
#pragma unroll
        for (int k = 0; k < V; k++) dh[i].e[k] = from_f32<T>(0.0f);
    }
    load_chunk<T, V>(x, Line<T>(p.x, p.x_t, p.x_b, l, t0), n, all);
    const unsigned cut = resets_of(p, l, t0, n);
    const bool plain = __all_sync(~0u, n == CHUNK && cut == 0);
    float h[V], c_in[V];
    load_state<V>(h, n > 0 ? p.saved + (int64_t)q * p.batch * p.dim : nullptr, l);
    float s[GATED ? CHUNK : 1][V];
    pack_gates<T, V, GATED>(g, s);
    if (SPLIT) {
      __shared__ Shared<V> sh;
      float A[V], B[V];
#pragma unroll
      for (int k = 0; k < V; k++) {
        A[k] = 1.0f;
        B[k] = 0.0f;
      }
#pragma unroll
      for (int i = CHUNK - 1; i >= 0; i--) {
        float gf[V], df[V];
        unpack<T, V>(dh[i], df);
        if (!GATED) unpack<T, V>(g[i], gf);
#pragma unroll
        for (int k = 0; k < V; k++) {
          float a, c;
          coefficients<GATED>(GATED ? s[i][k] : gf[k], a, c);
          if (i < n) {
            const bool r = cut >> i & 1;
            A[k] = r ? __int_as_float(0x7fffffff) : A[k] * a;
            B[k] = r ? 0.0f : a * (df[k] + B[k]);
          }
        }
      }
      join<V>(sh, half, warps, blocks, rank, A, B, carry, c_in);
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) c_in[k] = carry[k];
    }
    const Line<T> dg(p.dgate, p.dgate_t, p.dgate_b, l, t0), dx(p.dx, p.dx_t, p.dx_b, l, t0);
    const bool want_g = p.dgate, want_x = p.dx;
    if (plain) walk_back<T, V, GATED, true>(g, s, x, dh, 0, CHUNK, CHUNK, true, dg, want_g, dx, want_x, h, c_in);
    else walk_back<T, V, GATED, false>(g, s, x, dh, cut, n, left, l.live, dg, want_g, dx, want_x, h, c_in);
    if (!SPLIT) {
#pragma unroll
      for (int k = 0; k < V; k++) carry[k] = c_in[k];
    }
  }
  if (!SPLIT || (rank == 0 && warp == 0)) store_state<V>(p.dh0, carry, l);
}

// One step over [batch][dim], the fp32 state updated in place: elementwise, V values a thread.
template <typename T, int V, bool GATED>
__global__ void __launch_bounds__(256)
    k_scan_step(const T* __restrict__ gate, int64_t gate_b, const T* __restrict__ x, int64_t x_b, int64_t batch, int64_t dim,
                const void* __restrict__ reset, int reset_bytes, int64_t reset_b, float* __restrict__ state,
                int64_t state_b, T* __restrict__ out, int64_t out_b) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, per = dim / V;
  if (i >= batch * per) return;
  const int64_t row = batch * per <= 0xffffffffll ? (unsigned)i / (unsigned)per : i / per, d = (i - row * per) * V;
  const Vec<T, V> g = load_vec_nc<T, V>(gate + row * gate_b + d), xv = load_vec_nc<T, V>(x + row * x_b + d);
  bool cut = false;
  if (reset)
    cut = reset_bytes == 1 ? reinterpret_cast<const uint8_t*>(reset)[row * reset_b] != 0
                           : reinterpret_cast<const float*>(reset)[row * reset_b] != 0.0f;
  float* s = state + row * state_b + d;
  float h[V];
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 4) *reinterpret_cast<float4*>(h + k) = *reinterpret_cast<const float4*>(s + k);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) h[k] = s[k];
  }
  Vec<T, V> o;
#pragma unroll
  for (int k = 0; k < V; k++) {
    float a, c;
    coefficients<GATED>(packed_gate<GATED>(to_f32(g.e[k])), a, c);
    const float b = GATED ? c * to_f32(xv.e[k]) : to_f32(xv.e[k]);
    h[k] = cut ? b : fmaf(a, h[k], b);
    o.e[k] = from_f32<T>(h[k]);
  }
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 4) *reinterpret_cast<float4*>(s + k) = *reinterpret_cast<const float4*>(h + k);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) s[k] = h[k];
  }
  store_vec<T, V>(out + row * out_b + d, o);
}

// Warps that keep an SM's loads going; fewer channel groups than this many on every SM and the work is
// split along time as well.
constexpr int WARPS_PER_SM = 16;

struct Shape {
  bool split;
  int warps, blocks;      // on consecutive chunks: of a block, of a cluster
  int64_t grid;
};

inline Shape shape_for(int64_t channels, int64_t steps, int v) {
  const int64_t groups = (channels + 32 * v - 1) / (32 * v), want = (int64_t)sm_count() * WARPS_PER_SM;
  const int64_t chunks = (steps + CHUNK - 1) / CHUNK;
  Shape s = {false, 1, 1, (groups + WIDE_WARPS - 1) / WIDE_WARPS};
  if (chunks == 1 || groups * 2 > want) return s;
  s.split = true;
  while (s.warps < MAX_WARPS && s.warps < chunks && groups * s.warps < want) s.warps *= 2;
  while (s.blocks < MAX_CLUSTER && s.warps * s.blocks < chunks && groups * s.warps * s.blocks < want) s.blocks *= 2;
  if (s.blocks > s.warps) s.blocks = s.warps;
  s.grid = groups * s.blocks;
  return s;
}

template <typename K>
int launch(K kernel, const Args& p, const Shape& s, cudaStream_t st) {
  if (s.grid > 0x7fffffff) return F16_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)s.grid);
  cfg.blockDim = dim3(32 * (s.split ? s.warps : WIDE_WARPS));
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  if (s.blocks > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)s.blocks, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  (void)cudaLaunchKernelEx(&cfg, kernel, p, s.blocks);
  return launch_status();
}

template <typename T, int V, bool GATED>
int run(const Args& p, bool grad, cudaStream_t st) {
  const Shape s = shape_for(p.batch * p.dim, p.steps, V);
  if (grad) return s.split ? launch(k_scan_grad<T, V, GATED, true>, p, s, st) : launch(k_scan_grad<T, V, GATED, false>, p, s, st);
  return s.split ? launch(k_scan<T, V, GATED, true>, p, s, st) : launch(k_scan<T, V, GATED, false>, p, s, st);
}

template <typename T, int V>
int run_kind(const Args& p, bool grad, cudaStream_t st) {
  return p.gated ? run<T, V, true>(p, grad, st) : run<T, V, false>(p, grad, st);
}

inline bool pairs(const void* p, int64_t t, int64_t b) { return !p || (aligned(p, 4) && t % 2 == 0 && b % 2 == 0); }

template <typename T>
int run_type(const Args& p, bool grad, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    const bool two = p.dim % 2 == 0 && pairs(p.gate, p.gate_t, p.gate_b) && pairs(p.x, p.x_t, p.x_b) &&
                     (grad ? pairs(p.dh, p.dh_t, p.dh_b) && pairs(p.dgate, p.dgate_t, p.dgate_b) && pairs(p.dx, p.dx_t, p.dx_b)
                           : pairs(p.h, p.h_t, p.h_b));
    if (two) return run_kind<T, 2>(p, grad, st);
  }
  return run_kind<T, 1>(p, grad, st);
}

inline int check(const Args* p, bool grad) {
  if (!p || !p->gate || !p->x || p->steps <= 0 || p->batch <= 0 || p->dim <= 0 ||
      (p->reset && p->reset_bytes != 1 && p->reset_bytes != 4))
    return F16_ERR_ARG;
  if (p->dtype != F16_DTYPE_BF16 && p->dtype != F16_DTYPE_FP16 && p->dtype != F16_DTYPE_FP32) return F16_ERR_ARG;
  if (grad ? !p->saved || (!p->dh && !p->dhn) : !p->h) return F16_ERR_ARG;
  if (p->steps > 0x7fffffff - 32 * CHUNK * MAX_WARPS * MAX_CLUSTER) return F16_ERR_TOO_LARGE;
  const int size = p->dtype == F16_DTYPE_FP32 ? 4 : 2;
  if (!aligned(p->gate, size) || !aligned(p->x, size) || !aligned(p->h, size) || !aligned(p->dh, size) ||
      !aligned(p->dgate, size) || !aligned(p->dx, size) || (p->reset_bytes == 4 && !aligned(p->reset, 4)))
    return F16_ERR_ALIGN;
  return F16_OK;
}

inline int go(const Args* p, bool grad, f16_stream_t stream) {
  const int rc = check(p, grad);
  if (rc != F16_OK) return rc;
  const cudaStream_t st = cu_stream(stream);
  if (p->dtype == F16_DTYPE_FP32) return run_type<float>(*p, grad, st);
  if (p->dtype == F16_DTYPE_BF16) return run_type<__nv_bfloat16>(*p, grad, st);
  return run_type<__half>(*p, grad, st);
}

template <typename T>
int step(const void* gate, int64_t gate_b, const void* x, int64_t x_b, int64_t batch, int64_t dim, int gated, const void* reset,
         int reset_bytes, int64_t reset_b, float* state, int64_t state_b, void* out, int64_t out_b, cudaStream_t st) {
  constexpr int W = 16 / sizeof(T);
  const bool wide = dim % W == 0 && aligned(gate, 16) && aligned(x, 16) && aligned(out, 16) && aligned(state, 16) &&
                    gate_b % W == 0 && x_b % W == 0 && out_b % W == 0 && state_b % 4 == 0;
  const int64_t n = batch * (dim / (wide ? W : 1)), grid = (n + 255) / 256;
  if (grid > 0x7fffffff) return F16_ERR_TOO_LARGE;
  const auto go = [&](auto k) {
    k<<<(unsigned)grid, 256, 0, st>>>((const T*)gate, gate_b, (const T*)x, x_b, batch, dim, reset, reset_bytes, reset_b,
                                      state, state_b, (T*)out, out_b);
  };
  if (wide) gated ? go(k_scan_step<T, W, true>) : go(k_scan_step<T, W, false>);
  else gated ? go(k_scan_step<T, 1, true>) : go(k_scan_step<T, 1, false>);
  return launch_status();
}

}  // namespace scan
}  // namespace f16

using namespace f16;

extern "C" int64_t f16_scan_saved_floats(int64_t steps, int64_t batch, int64_t dim) {
  if (steps <= 0 || batch <= 0 || dim <= 0) return 0;
  return (steps + scan::CHUNK - 1) / scan::CHUNK * batch * dim;
}

extern "C" int f16_scan_fwd(const f16_scan_args* args, f16_stream_t stream) { return scan::go(args, false, stream); }

extern "C" int f16_scan_bwd(const f16_scan_args* args, f16_stream_t stream) { return scan::go(args, true, stream); }

extern "C" int f16_scan_step(const void* gate, int64_t gate_b, const void* x, int64_t x_b, int64_t batch, int64_t dim,
                             int dtype, int gated, const void* reset, int reset_bytes, int64_t reset_b, float* state,
                             int64_t state_b, void* h, int64_t h_b, f16_stream_t stream) {
  if (!gate || !x || !state || !h || batch <= 0 || dim <= 0 || state_b < dim || h_b < dim ||
      (reset && reset_bytes != 1 && reset_bytes != 4))
    return F16_ERR_ARG;
  const int size = dtype == F16_DTYPE_FP32 ? 4 : 2;
  if (!aligned(gate, size) || !aligned(x, size) || !aligned(h, size) || !aligned(state, 4) ||
      (reset && reset_bytes == 4 && !aligned(reset, 4)))
    return F16_ERR_ALIGN;
  const cudaStream_t st = cu_stream(stream);
  switch (dtype) {
    case F16_DTYPE_FP32:
      return scan::step<float>(gate, gate_b, x, x_b, batch, dim, gated, reset, reset_bytes, reset_b, state, state_b, h, h_b, st);
    case F16_DTYPE_BF16:
      return scan::step<__nv_bfloat16>(gate, gate_b, x, x_b, batch, dim, gated, reset, reset_bytes, reset_b, state, state_b, h,
                                       h_b, st);
    case F16_DTYPE_FP16:
      return scan::step<__half>(gate, gate_b, x, x_b, batch, dim, gated, reset, reset_bytes, reset_b, state, state_b, h, h_b,
                                st);
  }
  return F16_ERR_ARG;
}
