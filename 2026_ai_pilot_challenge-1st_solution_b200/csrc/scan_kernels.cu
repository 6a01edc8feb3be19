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
//  * Many channels: a warp walks through time alone, the state in registers (k_scan, k_scan_grad).
//  * Few: time is cut into segments as well, enough of them to fill the GPU.  A segment maps the state
//    before it to A h + B; k_scan_fold makes (A, B) of every segment, k_scan_starts the states between them,
//    and then the same kernels walk through all segments at once.  That reads the coefficients and one
//    more input a second time (what L2 still holds of them from there: the walk begins at the end where the
//    fold stopped), but no block waits for another, and the order of all sums is fixed.
// A segment that a reset cuts passes nothing of the state before it on.  That is kept as A = NaN, a
// selection (never a product with 0), so that an infinity or NaN left by the episode before does not
// leak: a coefficient that is NaN itself makes B NaN as well, so the two cannot be confused.
//
// Measured on a B200 whose copy makes 6.55 TB/s, with a cold L2 (gated bf16, us, and the share of that rate of the
// bytes a pass has to move): time not cut, 64 steps x 16,384 x 128, forward 155 (83%), backward 279 (75%); cut,
// 65,536 steps x 1 x 1,024, fold + starts + walk 61 + 6 + 72 (44%) and 60 + 7 + 121 (55%); single step, fp32,
// 131,072 x 128, 52 (99%).  What the cut costs is the fold's second read; without it that case's 16 warps
// would walk through 65,536 steps alone.
#include "typed.cuh"

namespace f16 {
namespace scan {

constexpr int CHUNK = F16_SCAN_CHUNK;     // steps in registers at a time, between saved states
constexpr int WARPS = 4;                  // of a block, each with channels (and a segment) of its own
// Blocks on an SM: 96, 128 and 80 registers a thread.
constexpr int WALK_BLOCKS = 5, GRAD_BLOCKS = 4, FOLD_BLOCKS = 6;
constexpr int MAX_SEGMENT = F16_SCAN_SEGMENT;      // most steps of a segment
constexpr int64_t MAX_STEPS = 0x7fffffff - 2 * CHUNK;     // time indexes are 32-bit
// Time is cut where the channels give fewer than ENOUGH_PER_SM warps an SM, into so many segments that there
// are WARPS_PER_SM, but no more than MAX_CUTS (k_scan_starts takes so many at once) while they are not too long.
// Forward + backward, us, gated bf16, with 4 / 6 / 8 / 10 warps an SM: 1,024 steps cut 198 / 283 / 365 / 450, not cut
// 272 / 313 / 325 / 369; 4,096 steps cut 693 / 1,036 / 1,358 / 1,671, not cut 1,046 / 1,200 / 1,252 / 1,454.
// With segments for 16 / 32 / 48 / 64 / 96 / 128 warps an SM: 65,536 x 1 x 1,024 bf16 339 / 344 / 337 / 326 / 330 / 327,
// 512 x 64 x 512 bf16 109 / 103 / 100 / 101 / 101 / 107, 4,096 x 16 x 128 fp32 80 / 85 / 85 / 82 / 83 / 85.
constexpr int ENOUGH_PER_SM = 7, WARPS_PER_SM = 64, MAX_CUTS = 1024;
static_assert(CHUNK == 16, "the resets of a chunk are half a word");

typedef f16_scan_args Args;

// V channels of a lane as one value: a float, or a pair computed with by one instruction.
template <int V> struct Lanes { typedef float type; };
template <> struct Lanes<2> { typedef Two type; };

__device__ __forceinline__ float fma2(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float less(float a, float b) { return a - b; }
__device__ __forceinline__ Two less(Two a, Two b) { return fma2(b, two(-1.0f), a); }
__device__ __forceinline__ float part(float v, int) { return v; }
__device__ __forceinline__ float part(Two v, int k) {
  const float2 f = split(v);
  return k ? f.y : f.x;
}
__device__ __forceinline__ void join(float& v, float x, float) { v = x; }
__device__ __forceinline__ void join(Two& v, float x, float y) { v = two(x, y); }
template <typename P> __device__ __forceinline__ P all_of(float x);
template <> __device__ __forceinline__ float all_of<float>(float x) { return x; }
template <> __device__ __forceinline__ Two all_of<Two>(float x) { return two(x); }

// The types' values as fp32 and back.
template <typename T, int V>
__device__ __forceinline__ typename Lanes<V>::type widen(const Vec<T, V>& v) {
  if constexpr (V == 2) return pair_of<T, V>(v, 0);
  else return to_f32(v.e[0]);
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> narrow(typename Lanes<V>::type f) {
  Vec<T, V> v;
  if constexpr (V == 2) set_pair<T, V>(v, 0, f);
  else v.e[0] = from_f32<T>(f);
  return v;
}

// f = sigmoid(g) and k = 1 - f: with e = exp(g), k = 1 / (1 + e), and f = e k where g is at most zero.  Above,
// f is 1 - k, whose only error of its own is one rounding: e k of an open gate (g above 17, where f rounds to 1) often
// is 1 - 2^-24, an error that is the same at every step of a steady gate and adds up over a sequence (0.4% of the
// state over 65,536 steps).
// e is 2^t, t = g / ln 2 rounded once: an error of up to |t| / 2 units of t's last place, which a small f or k would
// show (63 half steps at a gate of 80).  So what t is off by, g - t ln 2 with ln 2 in two parts (Cody and Waite's
// reduction), multiplies e by 1 + itself.  f and k are good to 12 half steps (2^-24) of themselves, 2^t (2^-22) and
// the reciprocal (2^-23) being most of it; below 2^-126 they are zero.  It costs three product-sums for a pair: 64 x
// 16,384 x 128 bf16 155 + 279 us, 150 + 287 with t alone and the gates worked out twice in the backward pass.
// Gates are held at 88 to either side, where e is 0 or k is 0 (an infinite t has no remainder).
__device__ __forceinline__ float capped(float g) {
  float c;
  asm("min.NaN.xorsign.abs.f32 %0, %1, 0f42B00000;" : "=f"(c) : "f"(g));
  return c;
}
__device__ __forceinline__ float exp2_of(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f, LN2_LOW = -1.9046542e-9f;     // ln 2 = LN2 + LN2_LOW
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// k, and f as e k whatever the gate is.
__device__ __forceinline__ void sigmoid_closed(float g, float& f, float& k) {
  g = capped(g);
  const float t = g * LOG2E, rest = fmaf(t, -LN2_LOW, fmaf(t, -LN2, g)), e0 = exp2_of(t), e = fmaf(e0, rest, e0);
  k = reciprocal(1.0f + e);
  f = e * k;
}
__device__ __forceinline__ void sigmoid_closed(Two g, Two& f, Two& k) {
  const float2 at = split(g);
  g = two(capped(at.x), capped(at.y));
  const Two t = g * two(LOG2E), rest = fma2(t, two(-LN2_LOW), fma2(t, two(-LN2), g));
  const float2 ts = split(t);
  const Two e0 = two(exp2_of(ts.x), exp2_of(ts.y)), e = fma2(e0, rest, e0);
  const float2 d = split(e + two(1.0f));
  k = two(reciprocal(d.x), reciprocal(d.y));
  f = e * k;
}
__device__ __forceinline__ void sigmoid(float g, float& f, float& k) {
  sigmoid_closed(g, f, k);
  f = g > 0.0f ? 1.0f - k : f;
}
__device__ __forceinline__ void sigmoid(Two g, Two& f, Two& k) {
  sigmoid_closed(g, f, k);
  const float2 at = split(g), closed = split(f), open = split(fma2(k, two(-1.0f), two(1.0f)));
  f = two(at.x > 0.0f ? open.x : closed.x, at.y > 0.0f ? open.y : closed.y);
}

// A step's coefficient a and inflow b; k: 1 - a (gated only).
template <bool GATED, typename P>
__device__ __forceinline__ void step_of(P g, P x, P& a, P& b, P& k) {
  if (GATED) {
    sigmoid(g, a, k);
    b = k * x;
  } else {
    a = g;
    b = x;
    k = g;
  }
}

// How the work is cut: `groups` of 32 V channels, `segments` of `length` steps (a multiple of CHUNK).
struct Shape {
  int64_t groups;
  int segments, length;
  float2* maps;           // (A, B) of [segments][channels], or NULL: one segment
  float* starts;          // the state (gradient) that enters [segments][channels]
};

// h -> A h + B, where A is not NaN (cut) and h not zero (so that an overflown A cannot make NaN of it).
__device__ __forceinline__ float pass_through(float2 m, float h) {
  return m.x != m.x || h == 0.0f ? m.y : fmaf(m.x, h, m.y);
}
// First m, then n.
__device__ __forceinline__ float2 then(float2 m, float2 n) { return make_float2(n.x * m.x, pass_through(n, m.y)); }
__device__ __forceinline__ float cut_mark() { return __int_as_float(0x7fffffff); }

struct Lane {
  int64_t b, d, c;      // sequence, feature, channel = b dim + d
  bool live;            // the channel exists
  int64_t first;        // the warp's first sequence, and how many it has channels of
  int seqs;
  bool together;        // one
  int len;              // the sequence's steps
};

// Called by whole warps: c is the first of the lane's channels.
__device__ __forceinline__ Lane lane_of(const Args& p, int64_t c) {
  Lane l;
  l.c = c;
  l.live = c < p.batch * p.dim;
  l.b = !l.live ? 0 : p.batch * p.dim <= 0xffffffffll ? (unsigned)c / (unsigned)p.dim : c / p.dim;
  l.d = l.live ? c - l.b * p.dim : 0;
  l.first = __shfl_sync(~0u, l.b, 0);
  if (!l.live) l.b = l.first;
  l.seqs = (int)__reduce_max_sync(~0u, (unsigned)(l.b - l.first)) + 1;
  l.together = l.seqs == 1;
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

// Bit i of resets_of: step t0 + i of the CHUNK from t0 on resets the lane's sequence (past the sequence's length
// it says nothing).  Called by whole warps, whose lanes read a step of a sequence each, two sequences at a
// time; those of the first two ahead of the time they are wanted (reset_ahead).
__device__ __forceinline__ bool reset_ahead(const Args& p, const Lane& l, int t0, int pair = 0) {
  const int lane = threadIdx.x & 31, t = t0 + lane % CHUNK, seq = 2 * pair + lane / CHUNK;
  return p.reset && t0 >= 0 && t < p.steps && seq < l.seqs && reset_at(p, l.first + seq, t);
}
__device__ __forceinline__ unsigned resets_of(const Args& p, const Lane& l, int t0, bool ahead) {
  if (!p.reset) return 0;
  unsigned word = __ballot_sync(~0u, ahead);
  const int seq = (int)(l.b - l.first);
  for (int pair = 1; 2 * pair < l.seqs; pair++) {
    const unsigned next = __ballot_sync(~0u, reset_ahead(p, l, t0, pair));
    if (seq >> 1 == pair) word = next;
  }
  return seq & 1 ? word >> CHUNK : word & ((1u << CHUNK) - 1);
}
__device__ __forceinline__ unsigned resets_of(const Args& p, const Lane& l, int t0) {
  return resets_of(p, l, t0, reset_ahead(p, l, t0));
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
__device__ __forceinline__ typename Lanes<V>::type load_state(const float* p, const Lane& l) {
  typename Lanes<V>::type v;
  const bool there = p && l.live;
  join(v, there ? p[l.c] : 0.0f, there && V > 1 ? p[l.c + V - 1] : 0.0f);
  return v;
}
template <int V>
__device__ __forceinline__ void store_state(float* p, typename Lanes<V>::type v, const Lane& l) {
  if (p && l.live) {
#pragma unroll
    for (int k = 0; k < V; k++) p[l.c + k] = part(v, k);
  }
}
// Where `yes`, y instead of x.
__device__ __forceinline__ float pick(bool yes, float y, float x) { return yes ? y : x; }
__device__ __forceinline__ Two pick(bool yes, Two y, Two x) {
  const float2 a = split(y), b = split(x);
  return two(yes ? a.x : b.x, yes ? a.y : b.y);
}

// The steps of a chunk from the state h on, written to `out`.  PLAIN: every lane has all CHUNK steps and no
// reset among them.
template <typename T, int V, bool GATED, bool PLAIN, typename P>
__device__ __forceinline__ void walk(const Vec<T, V> (&g)[CHUNK], const Vec<T, V> (&x)[CHUNK], unsigned cut, int n,
                                     int left, bool live, Line<T> out, P& h) {
#pragma unroll
  for (int i = 0; i < CHUNK; i++) {
    if (!PLAIN && i >= left) break;
    P a, b, k;
    step_of<GATED>(widen(g[i]), widen(x[i]), a, b, k);
    P o;
    if (PLAIN) {
      o = h = fma2(a, h, b);
    } else {
      h = pick(i < n, pick(cut >> i & 1, b, fma2(a, h, b)), h);
      o = pick(i < n, h, all_of<P>(0.0f));
    }
    if (PLAIN || live) store_vec<T, V>(out.p, narrow<T, V>(o));
    advance(out.p, out.st);
  }
}

// The warp's segment and channels; false: there are none.  The last task first: see the file's head.
__device__ __forceinline__ bool task_of(const Args& p, const Shape& sh, int v, bool last_first, int& segment, Lane& l) {
  int64_t task = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  const int64_t tasks = sh.groups * sh.segments;
  if (task >= tasks) return false;
  if (last_first) task = tasks - 1 - task;
  segment = (int)(task / sh.groups);
  l = lane_of(p, ((task - segment * sh.groups) * 32 + (threadIdx.x & 31)) * v);
  return true;
}

// How many of the CHUNK steps from t0 on the lane's sequence has.
__device__ __forceinline__ int steps_of(const Lane& l, int t0) {
  return l.live ? (l.len - t0 < CHUNK ? l.len - t0 : CHUNK) : 0;
}

template <typename T, int V, bool GATED>
__global__ void __launch_bounds__(32 * WARPS, WALK_BLOCKS) k_scan(const __grid_constant__ Args p, const __grid_constant__ Shape sh) {
  int segment;
  Lane l;
  if (!task_of(p, sh, V, sh.maps, segment, l)) return;
  const int steps = (int)p.steps, begin = segment * sh.length;
  const int end = steps - begin < sh.length ? steps : begin + sh.length;
  const int64_t channels = p.batch * p.dim;
  typename Lanes<V>::type h = load_state<V>(segment ? sh.starts + segment * channels : p.h0, l);
  for (int t0 = begin; t0 < end; t0 += CHUNK) {
    const int n = steps_of(l, t0), left = steps - t0;
    const bool all = __all_sync(~0u, n == CHUNK);
    Vec<T, V> g[CHUNK], x[CHUNK];
    load_chunk<T, V>(g, Line<T>(p.gate, p.gate_t, p.gate_b, l, t0), n, all);
    load_chunk<T, V>(x, Line<T>(p.x, p.x_t, p.x_b, l, t0), n, all);
    const unsigned cut = resets_of(p, l, t0);
    const bool plain = all && __all_sync(~0u, cut == 0);
    if (p.saved) store_state<V>(p.saved + (int64_t)(t0 / CHUNK) * channels, h, l);
    const Line<T> out(p.h, p.h_t, p.h_b, l, t0);
    if (plain) walk<T, V, GATED, true>(g, x, 0, CHUNK, CHUNK, true, out, h);
    else walk<T, V, GATED, false>(g, x, cut, n, left, l.live, out, h);
  }
  if (end == steps) store_state<V>(p.hn, h, l);
}

// A chunk's steps folded into (A, B).
template <typename T, int V, bool GATED, bool BACK, bool PLAIN, typename P>
__device__ __forceinline__ void fold(const Vec<T, V> (&g)[CHUNK], const Vec<T, V> (&x)[CHUNK], unsigned cut, int n, P& A, P& B) {
#pragma unroll
  for (int j = 0; j < CHUNK; j++) {
    const int i = BACK ? CHUNK - 1 - j : j;
    P a, b, k;
    step_of<GATED>(widen(g[i]), widen(x[i]), a, b, k);
    const P nextA = A * a, nextB = BACK ? a * (widen(x[i]) + B) : fma2(a, B, b);
    if (PLAIN) {
      A = nextA;
      B = nextB;
    } else {
      const bool r = cut >> i & 1;
      A = pick(i < n, pick(r, all_of<P>(cut_mark()), nextA), A);
      B = pick(i < n, pick(r, BACK ? all_of<P>(0.0f) : b, nextB), B);
    }
  }
}

// (A, B) of the warp's segment: of the states, or (BACK) of their gradients in reverse time, where B gathers
// what the segment's own dh send to the state before it.
template <typename T, int V, bool GATED, bool BACK>
__global__ void __launch_bounds__(32 * WARPS, FOLD_BLOCKS)
    k_scan_fold(const __grid_constant__ Args p, const __grid_constant__ Shape sh) {
  int segment;
  Lane l;
  if (!task_of(p, sh, V, false, segment, l)) return;
  const int steps = (int)p.steps, begin = segment * sh.length;
  const int end = steps - begin < sh.length ? steps : begin + sh.length;
  const int chunks = (end - begin + CHUNK - 1) / CHUNK;
  typedef typename Lanes<V>::type P;
  P A = all_of<P>(1.0f), B = all_of<P>(0.0f);
  for (int c = 0; c < chunks; c++) {
    const int t0 = begin + (BACK ? chunks - 1 - c : c) * CHUNK, n = steps_of(l, t0);
    const bool all = __all_sync(~0u, n == CHUNK);
    Vec<T, V> g[CHUNK], x[CHUNK];
    load_chunk<T, V>(g, Line<T>(p.gate, p.gate_t, p.gate_b, l, t0), n, all);
    if (!BACK || p.dh) {
      load_chunk<T, V>(x, BACK ? Line<T>(p.dh, p.dh_t, p.dh_b, l, t0) : Line<T>(p.x, p.x_t, p.x_b, l, t0), n, all);
    } else {
#pragma unroll
      for (int i = 0; i < CHUNK; i++) x[i] = narrow<T, V>(all_of<P>(0.0f));
    }
    const unsigned cut = resets_of(p, l, t0);
    if (all && __all_sync(~0u, cut == 0)) fold<T, V, GATED, BACK, true>(g, x, 0, CHUNK, A, B);
    else fold<T, V, GATED, BACK, false>(g, x, cut, n, A, B);
  }
  if (l.live) {
    float2* out = sh.maps + segment * (p.batch * p.dim) + l.c;
#pragma unroll
    for (int k = 0; k < V; k++) out[k] = make_float2(part(A, k), part(B, k));
  }
}

// What enters each segment, from the first on (BACK: the last): the maps of the segments before it, folded in
// order.  A channel has `parts` threads, each with START_EACH consecutive segments at a time; `first`: what
// enters the first one, or NULL.
constexpr int START_THREADS = 256, START_EACH = 16, START_PARTS = 64;
template <bool BACK>
__global__ void __launch_bounds__(START_THREADS)
    k_scan_starts(const __grid_constant__ Shape sh, int64_t channels, const float* first, int parts) {
  __shared__ float2 of_part[START_THREADS];
  const int block = START_THREADS / parts, mine = threadIdx.x / block, k = threadIdx.x % block;
  const int64_t c = (int64_t)blockIdx.x * block + k;
  const bool live = c < channels;
  float h = first && live ? first[c] : 0.0f;
  for (int base = 0; base < sh.segments; base += parts * START_EACH) {
    const int begin = base + mine * START_EACH, count = sh.segments - begin < START_EACH ? sh.segments - begin : START_EACH;
    const auto at = [&](int i) { return (BACK ? sh.segments - 1 - i : i) * channels + c; };
    float2 m[START_EACH], all = make_float2(1.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < START_EACH; i++) m[i] = live && i < count ? sh.maps[at(begin + i)] : make_float2(1.0f, 0.0f);
    float enter = h;
    if (parts > 1) {
#pragma unroll
      for (int i = 0; i < START_EACH; i++)
        if (i < count) all = then(all, m[i]);
      of_part[threadIdx.x] = all;
      __syncthreads();
#pragma unroll 8
      for (int w = 0; w < parts; w++) {
        if (w == mine) enter = h;
        h = pass_through(of_part[w * block + k], h);
      }
    }
#pragma unroll
    for (int i = 0; i < START_EACH; i++)
      if (i < count) {
        if (live) sh.starts[at(begin + i)] = enter;
        enter = pass_through(m[i], enter);
      }
    if (parts == 1) h = enter;
    else __syncthreads();
  }
}

// A chunk of the backward pass's three inputs, as the lane's own values: in shared memory, where the copies of
// the next chunk land while this one is worked on (4-byte lanes), or in registers.  Backward of 64 x 16,384 x 128
// bf16: copies of 16 bytes 280 us, of each lane's own 4 bytes 338, chunks in registers 412; the gates worked out twice in
// place of kept 301.  Values of 2 bytes at odd widths or addresses are loaded into registers: 64 x 16,384 x 127, no
// resets, 199 + 330, of 128 channels 146 + 247.
constexpr int STAGES = 2;
template <typename T, int V, bool STAGED> struct Inputs;
template <typename T, int V> struct Inputs<T, V, true> {
  typedef unsigned Buffer[STAGES][3][CHUNK][32 * WARPS];
  unsigned* mine;
  bool with_dh;
  // Rows by 16 bytes: a lane copies the four lanes' channels that begin at (b, d), of a sequence of `len` steps
  // (0: there are none).  Where a unit lies in one sequence and is aligned in all inputs.
  bool rows;
  int b, d, len;
  __device__ __forceinline__ Inputs(Buffer& buf, const Args& p, const Lane& l) : mine(&buf[0][0][0][threadIdx.x]), with_dh(p.dh) {
    const auto whole = [&](const void* q, int64_t st, int64_t sb) {
      return (reinterpret_cast<uintptr_t>(q) & 15) == 0 && ((st | sb) & (4 * V - 1)) == 0;
    };
    rows = p.dim % (4 * V) == 0 && p.dim <= 0x7fffffff && p.batch <= 0x7fffffff && whole(p.gate, p.gate_t, p.gate_b) &&
           whole(p.x, p.x_t, p.x_b) && (!with_dh || whole(p.dh, p.dh_t, p.dh_b));
    const int first = (threadIdx.x & 7) * 4;
    b = __shfl_sync(~0u, (int)l.b, first);
    d = __shfl_sync(~0u, (int)l.d, first);
    len = __shfl_sync(~0u, l.live ? l.len : 0, first);
  }
  __device__ __forceinline__ unsigned* at(int stage, int which, int i) const {
    return mine + ((stage * 3 + which) * CHUNK + i) * 32 * WARPS;
  }
  __device__ __forceinline__ Vec<T, V> get(int stage, int which, int i) const {
    Vec<T, V> v;
    v.r = *at(stage, which, i);
    return v;
  }
  __device__ __forceinline__ Vec<T, V> gate(int stage, int i) const { return get(stage, 0, i); }
  __device__ __forceinline__ Vec<T, V> x(int stage, int i) const { return get(stage, 1, i); }
  __device__ __forceinline__ typename Lanes<V>::type dh(int stage, int i) const {
    return with_dh ? widen(get(stage, 2, i)) : all_of<typename Lanes<V>::type>(0.0f);
  }
  // A gate's f and 1 - f from the first pass over the chunk to the second, in place of its gate and x: of one
  // channel both, of two the smaller one, with the sign set where that is f.
  static constexpr bool KEEPS = true;
  __device__ __forceinline__ void keep(int stage, int i, float g, float f, float k) const {
    *at(stage, 0, i) = __float_as_uint(g > 0.0f ? 1.0f - k : f);
    *at(stage, 1, i) = __float_as_uint(k);
  }
  __device__ __forceinline__ void keep(int stage, int i, Two g, Two f, Two k) const {
    const float2 of = split(g), a = split(f), b = split(k);
    *at(stage, 0, i) = __float_as_uint(of.x > 0.0f ? b.x : -a.x);
    *at(stage, 1, i) = __float_as_uint(of.y > 0.0f ? b.y : -a.y);
  }
  __device__ __forceinline__ void kept(int stage, int i, float& f, float& k) const {
    f = __uint_as_float(*at(stage, 0, i));
    k = __uint_as_float(*at(stage, 1, i));
  }
  __device__ __forceinline__ void kept(int stage, int i, Two& f, Two& k) const {
    const float x = __uint_as_float(*at(stage, 0, i)), y = __uint_as_float(*at(stage, 1, i));
    const float bx = 1.0f - fabsf(x), by = 1.0f - fabsf(y);
    const bool ox = __float_as_int(x) >= 0, oy = __float_as_int(y) >= 0;
    f = two(ox ? bx : -x, oy ? by : -y);
    k = two(ox ? x : bx, oy ? y : by);
  }
  // Every lane its own 4 bytes.
  __device__ __forceinline__ void copy(int stage, int which, Line<T> from, int n) {
    unsigned to = (unsigned)__cvta_generic_to_shared(at(stage, which, 0));
#pragma unroll
    for (int i = 0; i < CHUNK; i++) {
      if (i < n) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + i * 128 * WARPS), "l"(from.p) : "memory");
      advance(from.p, from.st);
    }
  }
  // Eight lanes a row: 16 bytes each.
  __device__ __forceinline__ void copy_rows(int stage, int which, const void* base, int64_t st, int64_t sb, int t0, int n) {
    const int lane = threadIdx.x & 31, row = lane >> 3, col = lane & 7;
    const T* from = reinterpret_cast<const T*>(base) + b * sb + d + (int64_t)(t0 + row) * st;
    unsigned to = (unsigned)__cvta_generic_to_shared(at(stage, which, row) - lane + 4 * col);
#pragma unroll
    for (int i = 0; i < CHUNK / 4; i++) {
      if (row + 4 * i < n) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * 4 * 128 * WARPS), "l"(from) : "memory");
      advance(from, 4 * st);
    }
  }
  __device__ __forceinline__ void fetch(const Args& p, const Lane& l, int stage, int t0, bool there) {
    if (rows) {
      __syncwarp();             // every lane has read what this stage held
      const int m = there ? len - t0 : 0;
      copy_rows(stage, 0, p.gate, p.gate_t, p.gate_b, t0, m);
      copy_rows(stage, 1, p.x, p.x_t, p.x_b, t0, m);
      if (with_dh) copy_rows(stage, 2, p.dh, p.dh_t, p.dh_b, t0, m);
    } else {
      const int n = there ? steps_of(l, t0) : 0;
      const Line<T> g(p.gate, p.gate_t, p.gate_b, l, t0), x(p.x, p.x_t, p.x_b, l, t0), d(p.dh, p.dh_t, p.dh_b, l, t0);
      copy(stage, 0, g, n);
      copy(stage, 1, x, n);
      if (with_dh) copy(stage, 2, d, n);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // The chunk fetched before the last one has landed, what the other lanes copied of it as well.
  __device__ __forceinline__ void wait() {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    if (rows) __syncwarp();
  }
};
template <typename T, int V> struct Inputs<T, V, false> {
  typedef int Buffer;
  static constexpr bool KEEPS = false;
  Vec<T, V> in[3][CHUNK];
  bool with_dh;
  __device__ __forceinline__ Inputs(Buffer&, const Args& p, const Lane&) : with_dh(p.dh) {}
  __device__ __forceinline__ Vec<T, V> gate(int, int i) const { return in[0][i]; }
  __device__ __forceinline__ Vec<T, V> x(int, int i) const { return in[1][i]; }
  __device__ __forceinline__ typename Lanes<V>::type dh(int, int i) const {
    return with_dh ? widen(in[2][i]) : all_of<typename Lanes<V>::type>(0.0f);
  }
  __device__ __forceinline__ void load(const Args& p, const Lane& l, int t0, int n) {
    const bool all = __all_sync(~0u, n == CHUNK);
    load_chunk<T, V>(in[0], Line<T>(p.gate, p.gate_t, p.gate_b, l, t0), n, all);
    load_chunk<T, V>(in[1], Line<T>(p.x, p.x_t, p.x_b, l, t0), n, all);
    if (with_dh) load_chunk<T, V>(in[2], Line<T>(p.dh, p.dh_t, p.dh_b, l, t0), n, all);
  }
};

// The steps of a chunk again from the saved state h, then their gradients from the last one back; carry: the
// gradient that reaches the chunk's last state, then the one that leaves its first.
// Gated: with d_t = f (h_{t-1} - x_t), dx_t = G k and dgate_t = dx_t d_t.
template <typename T, int V, bool GATED, bool PLAIN, typename I, typename P>
__device__ __forceinline__ void walk_back(const I& in, int stage, unsigned cut, int n, int left, bool live,
                                          Line<T> dg, bool want_g, Line<T> dx, bool want_x, P h, P& carry) {
  const P zero = all_of<P>(0.0f);
  P d[CHUNK];
#pragma unroll
  for (int i = 0; i < CHUNK; i++) {
    if (!PLAIN && i >= left) break;
    P a, b, k;
    const P xf = widen(in.x(stage, i)), g = widen(in.gate(stage, i));
    if constexpr (GATED && I::KEEPS) {
      sigmoid_closed(g, a, k);         // only for the chunk's own states: over 16 steps f's bias is 2^-20 at most
      b = k * xf;
      in.keep(stage, i, g, a, k);
    } else {
      step_of<GATED>(g, xf, a, b, k);
    }
    const bool r = !PLAIN && (cut >> i & 1);
    const P hp = PLAIN ? h : pick(r, zero, h);
    d[i] = GATED ? a * less(hp, xf) : hp;
    h = PLAIN ? fma2(a, hp, b) : pick(r, b, fma2(a, hp, b));
  }
  // where they are not kept in shared memory the gates are read and worked out again: registers do not hold them
  asm volatile("" ::: "memory");
  // what reaches a step's state from the step after it is pass * carry
  P pass = all_of<P>(1.0f);
  const int last = !PLAIN && left < CHUNK ? left - 1 : CHUNK - 1;
  dg.p += last * dg.st;
  dx.p += last * dx.st;
#pragma unroll
  for (int i = CHUNK - 1; i >= 0; i--) {
    if (!PLAIN && i >= left) continue;
    P a, b, k;
    if constexpr (GATED && I::KEEPS) in.kept(stage, i, a, k);
    else step_of<GATED>(widen(in.gate(stage, i)), zero, a, b, k);
    const P G = fma2(pass, carry, in.dh(stage, i));
    P ox = GATED ? G * k : G, og = ox * d[i];
    if (PLAIN) {
      pass = a;
      carry = G;
    } else {
      const bool r = cut >> i & 1;
      pass = pick(i < n, pick(r, zero, a), pass);
      carry = pick(i < n, pick(r, zero, G), carry);
      ox = pick(i < n, ox, zero);
      og = pick(i < n, og, zero);
    }
    if (PLAIN || live) {
      if (want_g) store_vec<T, V>(dg.p, narrow<T, V>(og));
      if (want_x) store_vec<T, V>(dx.p, narrow<T, V>(ox));
    }
    advance(dg.p, -dg.st);
    advance(dx.p, -dx.st);
  }
  carry = pass * carry;
}

// Backward: chunks from the segment's last to its first, the carried value the gradient of the state
// before the steps already done.
template <typename T, int V, bool GATED>
__global__ void __launch_bounds__(32 * WARPS, GRAD_BLOCKS)
    k_scan_grad(const __grid_constant__ Args p, const __grid_constant__ Shape sh) {
  constexpr bool STAGED = V * sizeof(T) == 4;
  typedef Inputs<T, V, STAGED> In;
  typedef typename Lanes<V>::type P;
  __shared__ __align__(16) typename In::Buffer buffer;
  int segment;
  Lane l;
  if (!task_of(p, sh, V, sh.maps, segment, l)) return;
  const int steps = (int)p.steps, begin = segment * sh.length;
  const int end = steps - begin < sh.length ? steps : begin + sh.length;
  const int64_t channels = p.batch * p.dim;
  P carry = load_state<V>(end < steps ? sh.starts + segment * channels : p.dhn, l);
  In in(buffer, p, l);
  int stage = 0;
  const int first = begin + (end - begin - 1) / CHUNK * CHUNK;
  const auto saved_at = [&](int t0) {
    return load_state<V>(t0 >= begin && steps_of(l, t0) > 0 ? p.saved + (int64_t)(t0 / CHUNK) * channels : nullptr, l);
  };
  if constexpr (STAGED) in.fetch(p, l, 0, first, true);
  P h = saved_at(first), h_next = h;
  bool ahead = reset_ahead(p, l, first);
  for (int t0 = first; t0 >= begin; t0 -= CHUNK, h = h_next) {
    const int n = steps_of(l, t0), left = steps - t0, next = t0 - CHUNK;
    const unsigned cut = resets_of(p, l, t0, ahead);
    if constexpr (STAGED) in.fetch(p, l, stage ^ 1, next, next >= begin);
    h_next = saved_at(next);
    if (next >= begin) ahead = reset_ahead(p, l, next);
    if constexpr (STAGED) in.wait();
    else in.load(p, l, t0, n);
    const bool plain = __all_sync(~0u, n == CHUNK && cut == 0);
    const Line<T> dg(p.dgate, p.dgate_t, p.dgate_b, l, t0), dx(p.dx, p.dx_t, p.dx_b, l, t0);
    const bool want_g = p.dgate, want_x = p.dx;
    if (plain) walk_back<T, V, GATED, true>(in, stage, 0, CHUNK, CHUNK, true, dg, want_g, dx, want_x, h, carry);
    else walk_back<T, V, GATED, false>(in, stage, cut, n, left, l.live, dg, want_g, dx, want_x, h, carry);
    stage ^= 1;
  }
  if (begin == 0) store_state<V>(p.dh0, carry, l);
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
    float a, b, c;
    step_of<GATED>(to_f32(g.e[k]), to_f32(xv.e[k]), a, b, c);
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

// Segments: a multiple of CHUNK steps, few enough that the fold's and the walk's warps fill the GPU.
inline Shape shape_for(int64_t channels, int64_t steps, int v) {
  Shape s = {(channels + 32 * v - 1) / (32 * v), 1, (int)((steps + CHUNK - 1) / CHUNK * CHUNK), nullptr, nullptr};
  const int64_t want = (int64_t)sm_count() * WARPS_PER_SM, chunks = (steps + CHUNK - 1) / CHUNK;
  if (s.groups >= (int64_t)sm_count() * ENOUGH_PER_SM || chunks < 2) return s;
  const int64_t cuts = (want + s.groups - 1) / s.groups;                 // at least two
  int64_t each = (chunks + cuts - 1) / cuts;                             // chunks of a segment
  if (each < (chunks + MAX_CUTS - 1) / MAX_CUTS) each = (chunks + MAX_CUTS - 1) / MAX_CUTS;
  if (each > MAX_SEGMENT / CHUNK) each = MAX_SEGMENT / CHUNK;
  s.length = (int)each * CHUNK;
  s.segments = (int)((chunks + each - 1) / each);
  return s;
}

inline int64_t scratch_for(const Shape& s, int64_t channels) { return s.segments > 1 ? 3 * s.segments * channels : 0; }

template <typename T, int V, bool GATED>
int run(const Args& p, bool grad, cudaStream_t st) {
  const int64_t channels = p.batch * p.dim;
  Shape s = shape_for(channels, p.steps, V);
  if (s.segments > 1 && p.scratch && p.scratch_floats >= scratch_for(s, channels)) {
    s.maps = reinterpret_cast<float2*>(p.scratch);
    s.starts = p.scratch + 2 * s.segments * channels;
  } else {
    s.segments = 1;
    s.length = (int)((p.steps + CHUNK - 1) / CHUNK * CHUNK);
  }
  const int64_t grid = (s.groups * s.segments + WARPS - 1) / WARPS;
  if (grid > 0x7fffffff) return F16_ERR_TOO_LARGE;
  const unsigned blocks = (unsigned)grid, threads = 32 * WARPS;
  int parts = 1;
  while (parts < START_PARTS && parts * START_EACH < s.segments) parts *= 2;
  const int64_t starts = (channels + START_THREADS / parts - 1) / (START_THREADS / parts);
  if (s.maps && starts > 0x7fffffff) return F16_ERR_TOO_LARGE;
  if (s.maps) {
    if (grad) {
      k_scan_fold<T, V, GATED, true><<<blocks, threads, 0, st>>>(p, s);
      k_scan_starts<true><<<(unsigned)starts, START_THREADS, 0, st>>>(s, channels, p.dhn, parts);
    } else {
      k_scan_fold<T, V, GATED, false><<<blocks, threads, 0, st>>>(p, s);
      k_scan_starts<false><<<(unsigned)starts, START_THREADS, 0, st>>>(s, channels, p.h0, parts);
    }
  }
  if (grad) k_scan_grad<T, V, GATED><<<blocks, threads, 0, st>>>(p, s);
  else k_scan<T, V, GATED><<<blocks, threads, 0, st>>>(p, s);
  return launch_status();
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
  if (p->steps > MAX_STEPS || p->batch > INT64_MAX / 16 / p->dim) return F16_ERR_TOO_LARGE;
  const int size = p->dtype == F16_DTYPE_FP32 ? 4 : 2;
  if (!aligned(p->gate, size) || !aligned(p->x, size) || !aligned(p->h, size) || !aligned(p->dh, size) ||
      !aligned(p->dgate, size) || !aligned(p->dx, size) || (p->reset && p->reset_bytes == 4 && !aligned(p->reset, 4)) ||
      !aligned(p->scratch, 8))
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

extern "C" int64_t f16_scan_scratch_floats(int64_t steps, int64_t batch, int64_t dim) {
  if (steps <= 0 || batch <= 0 || dim <= 0 || batch > INT64_MAX / 16 / dim || steps > scan::MAX_STEPS) return 0;
  const int64_t one = scan::scratch_for(scan::shape_for(batch * dim, steps, 1), batch * dim),
                two = scan::scratch_for(scan::shape_for(batch * dim, steps, 2), batch * dim);
  return one > two ? one : two;
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
