// Log probability of one given token per row of logits, the row's entropy and its most likely
// alternatives, and the gradient of the first two with respect to the logits.  With z = x / temperature
// and m the row's maximum, of the logits as they are:
//   e_j = e^((x_j - m) / temperature)      S = sum e_j      T = sum (x_j - m) e_j      lse = m / temperature + log S
//   logprob = (x_t - m) / temperature - log S      entropy = log S - T / (S temperature)      p_j = e^(z_j - lse)
// Everything but lse is formed from differences of logits: m / temperature need not even be finite (logits of the
// type's lowest value at a temperature below 1), and a constant added to a row changes nothing.  The gradient, too: from lse
// alone, log p_j would have lse's rounding, 8 % of a gradient at logits near 1000 and a temperature of 0.7.
//   dx_j = ( g_l (1[j = t] - p_j) - g_h p_j (log p_j + entropy) ) / temperature
//
// Forward: ONE pass over the logits.  Every thread keeps a running (m, S, T) of its own, m the largest
// logit so far: log S and -T / S are then both positive, and nothing cancels in the entropy of a row that is nearly
// certain (letting m lag by up to 6, to rescale less often, left 7e-7 in it, whatever the entropy was).  A batch's
// exponentials are added to each other before they are added to S, of which they are a small part then.
// The partial results of threads, warps and CTAs are joined by the same rule.  A row belongs
// to a CLUSTER of CTAs (1 for many rows, up to 16 for a few): the join over a long row goes through
// distributed shared memory, so there is one launch, no workspace, no atomic and a fixed order -- the
// result is bit-reproducible.
//
// The top k <= 32: keys of 64 bits (order-preserving value bits, then the complement of the index, so that
// equal logits go to the lowest index) are collected in shared memory from elements that reach a bound T
// below which the k-th best cannot lie, and ranked by counting: with n keys a thread reads n words to find its
// key's place.  T first comes from the maxima of the threads' first vectors: of F full warps each has
// ceil(k / F) lanes whose maximum is at least its ceil(k / F)-th largest, so the smallest of those is reached by k
// elements at least; then it is the k-th best of what has been ranked, after 1, 4, 16, ... batches, so that about 3 k
// elements pass in between.  Where too many pass (rows of ties, ascending rows), the CTA reads its columns once more
// and every warp keeps a list of 32 that is sorted over its lanes.  Keeping such lists from the start took 69 us for 64
// rows of 151936 fp32 logits with k = 20, nearly all of it in some hundred insertions per warp.
//
// Backward: reads the logits, writes the gradient; one exponential per element.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "forge_host.h"

namespace cg = cooperative_groups;

namespace forge {
namespace loss {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_CLUSTER = 16;
constexpr int MAX_TOP = 32;
constexpr float LOG2E = 1.44269504088896340736f;

struct Params {
  const uint8_t* logits;
  const long long* targets;
  float* logprobs;
  float* entropy;
  float* lse;
  float* top_logprobs;
  long long* top_ids;
  float* row_max;
  float* log_sum;
  float* stats;                          // partial mode: (rows, 5) = m, S, T, target's logit, target found
  unsigned long long* keys;              // partial mode: (rows, top_k)
  long long vocab, ld, ignore_index, vocab_start, vocab_total;
  int top_k;
  float inv_t;                           // 1 / temperature
};

struct Acc {
  float m, s, t;                         // m and t in units of the logits
};

// a NaN stays a NaN (fmaxf would drop it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (m, S, T) of two disjoint sets of columns -> of their union.  A set without a finite logit has m = -inf
// and S = T = 0 (or NaN, if it holds a NaN): it must not enter the differences below.  c: log2 e / temperature.
__device__ __forceinline__ Acc join(const Acc& a, const Acc& b, float c) {
  if (a.m == -INFINITY) return Acc{b.m, a.s + b.s, a.t + b.t};
  if (b.m == -INFINITY) return Acc{a.m, a.s + b.s, a.t + b.t};
  const float m = fmaxf(a.m, b.m);
  const float da = a.m - m, db = b.m - m;
  const float fa = exp2_approx(da * c), fb = exp2_approx(db * c);
  // one of da, db is zero; the other may be so low that its factor is 0, and 0 * -inf would be NaN
  const float ta = fa > 0.0f ? fa * (a.t + da * a.s) : 0.0f * a.s;
  const float tb = fb > 0.0f ? fb * (b.t + db * b.s) : 0.0f * b.s;
  return Acc{m, fa * a.s + fb * b.s, ta + tb};
}

// over the lanes of a warp: the maximum first, then plain sums
__device__ __forceinline__ Acc warp_join(const Acc& a, float c) {
  float m = a.m, s = a.s, t = a.t;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (a.m != -INFINITY) {
    const float d = a.m - m, f = exp2_approx(d * c);
    t = f > 0.0f ? f * (t + d * s) : 0.0f * s;
    s *= f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  return Acc{m, s, t};
}

// ----- sorted lists of 32 keys, one per lane, descending ------------------------------------------
typedef unsigned long long u64;

__device__ __forceinline__ u64 make_key(float x, uint32_t index) {
  uint32_t u = __float_as_uint(x + 0.0f);             // -0 becomes +0: they are equal
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (static_cast<u64>(u) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ float key_value(u64 k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ uint32_t key_index(u64 k) { return 0xffffffffu - static_cast<uint32_t>(k); }

__device__ __forceinline__ u64 warp_merge(u64 a, u64 b, int lane);

// the lanes' keys in descending order: a bitonic network
__device__ __forceinline__ u64 warp_sort(u64 c, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const u64 d = __shfl_xor_sync(0xffffffffu, c, o);
      const bool larger = ((lane & o) == 0) == ((lane & size) == 0);
      c = (larger == (c > d)) ? c : d;
    }
  }
  return c;
}

// every lane offers one key (0: none); the list keeps the best 32, `floor` is its k-th entry
__device__ __forceinline__ void warp_offer(u64& list, u64& floor, u64 key, int k, int lane) {
  uint32_t mask = __ballot_sync(0xffffffffu, key > floor);
  if (__popc(mask) > 4) {
    list = warp_merge(list, warp_sort(key, lane), lane);
    floor = __shfl_sync(0xffffffffu, list, k - 1);
    return;
  }
  while ((mask = __ballot_sync(0xffffffffu, key > floor)) != 0) {
    const int src = __ffs(mask) - 1;
    const u64 x = __shfl_sync(0xffffffffu, key, src);
    const int pos = __popc(__ballot_sync(0xffffffffu, list > x));
    const u64 up = __shfl_up_sync(0xffffffffu, list, 1);
    if (lane == pos) list = x;
    else if (lane > pos) list = up;
    floor = __shfl_sync(0xffffffffu, list, k - 1);
    if (lane == src) key = 0;
  }
}

// the best 32 of two descending lists, descending: the larger of a[i], b[31 - i] is a bitonic
// sequence, five exchange steps sort it
__device__ __forceinline__ u64 warp_merge(u64 a, u64 b, int lane) {
  const u64 r = __shfl_sync(0xffffffffu, b, 31 - lane);
  u64 c = a > r ? a : r;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 d = __shfl_xor_sync(0xffffffffu, c, o);
    c = (((lane & o) == 0) == (c > d)) ? c : d;
  }
  return c;
}

// ----- one thread's running sums ------------------------------------------------------------------
struct Run {
  float m;                               // the largest logit so far
  float nm;                              // -m, or 0 while there is no finite logit
  float2 s, t;                           // two interleaved partial sums
};

__device__ __forceinline__ void rebase(Run& r, float vmax, float c) {
  if (r.m != -INFINITY) {
    const float d = r.m - vmax;
    const float f = exp2_approx(d * c);
    const float df = f > 0.0f ? d : 0.0f;
    r.t.x = f * (r.t.x + df * r.s.x);
    r.t.y = f * (r.t.y + df * r.s.y);
    r.s.x *= f;
    r.s.y *= f;
  }
  r.m = vmax;
  r.nm = -vmax;
}

// adds N logits whose masked (-inf) ones have been replaced by a finite number so low that its exponential is 0 and the
// product in T stays 0
template <int N>
__device__ __forceinline__ void accumulate(float nm, float2& s, float2& t, const float (&x)[N], float c) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 z = fadd2(make_float2(x[i], x[i + 1]), make_float2(nm, nm));
    const float2 y = fmul2(z, make_float2(c, c));
    const float2 e = make_float2(exp2_approx(y.x), exp2_approx(y.y));
    s = fadd2(s, e);
    t = ffma2(e, z, t);
  }
}
// the same for logits as they are, into the running sums
template <int N>
__device__ __forceinline__ void accumulate_raw(Run& r, const float (&x)[N], float c) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float z = x[i] + r.nm;
    const float e = exp2_approx(z * c);
    r.s.x += e;
    r.t.x = __fmaf_rn(e, max_nan(z, -3.0e38f), r.t.x);
  }
}

template <int DT>
struct Vec;
template <>
struct Vec<DT_BF16> {
  static constexpr int N = 8, ES = 2;
  static __device__ __forceinline__ __nv_bfloat162 as2(uint32_t u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); }
  static __device__ __forceinline__ void unpack(const uint4& q, float (&x)[8]) {
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  // -inf -> the lowest finite number, two at a time (a NaN stays one)
  static __device__ __forceinline__ uint4 unmask(const uint4& q) {
    uint4 o;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(o.x) : "r"(q.x), "r"(0xff7fff7fu));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(o.y) : "r"(q.y), "r"(0xff7fff7fu));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(o.z) : "r"(q.z), "r"(0xff7fff7fu));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(o.w) : "r"(q.w), "r"(0xff7fff7fu));
    return o;
  }
  static __device__ __forceinline__ float max_of(const uint4& q) {
    const __nv_bfloat162 m = __hmax2(__hmax2(as2(q.x), as2(q.y)), __hmax2(as2(q.z), as2(q.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float one(const uint8_t* p) {
    return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p)) << 16);
  }
  // the vector's first element, which it loses
  static __device__ __forceinline__ float pop(uint4& q) {
    const float x = __uint_as_float(q.x << 16);
    q.x = __funnelshift_r(q.x, q.y, 16);
    q.y = __funnelshift_r(q.y, q.z, 16);
    q.z = __funnelshift_r(q.z, q.w, 16);
    q.w >>= 16;
    return x;
  }
};
template <>
struct Vec<DT_F32> {
  static constexpr int N = 4, ES = 4;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&x)[4]) {
    x[0] = __uint_as_float(q.x); x[1] = __uint_as_float(q.y);
    x[2] = __uint_as_float(q.z); x[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 unmask(const uint4& q) {
    return make_uint4(__float_as_uint(max_nan(__uint_as_float(q.x), -3.0e38f)), __float_as_uint(max_nan(__uint_as_float(q.y), -3.0e38f)),
                      __float_as_uint(max_nan(__uint_as_float(q.z), -3.0e38f)), __float_as_uint(max_nan(__uint_as_float(q.w), -3.0e38f)));
  }
  static __device__ __forceinline__ float max_of(const uint4& q) {
    return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
  }
  static __device__ __forceinline__ float one(const uint8_t* p) { return *reinterpret_cast<const float*>(p); }
  static __device__ __forceinline__ float pop(uint4& q) {
    const float x = __uint_as_float(q.x);
    q = make_uint4(q.y, q.z, q.w, 0);
    return x;
  }
};

__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
  uint4 q;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
               : "l"(p));
  return q;
}

constexpr int CAP = 512;                 // candidate keys
static_assert(WARPS * 32 <= CAP, "the warps' lists are ranked in the same array");

struct Shared {
  Acc warp_acc[WARPS];
  Acc cta_acc[MAX_CLUSTER];              // written by the cluster's CTAs into the first one's copy
};
struct alignas(16) TopShared {
  u64 cand[CAP];                         // keys
  uint32_t col[CAP];                     // columns of candidates that have no key yet
  u64 best[32];                          // ranked, descending
  u64 cta_keys[MAX_CLUSTER * 32];        // as cta_acc
  float warp_bound[WARPS];
  int count;
};

// The best 32 of cand[0 .. n) in order of rank, into best[] (0 where there are fewer); all threads call it.
__device__ __forceinline__ void rank_keys(const u64* cand, int n, u64* best) {
  if (threadIdx.x < 32) best[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const u64 mine = cand[i];
    if (mine == 0) continue;
    int above = 0;
    int j = 0;
    for (; j + 8 <= n; j += 8) {
#pragma unroll
      for (int u = 0; u < 8; u += 2) {
        const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(cand + j + u);
        above += (q.x > mine) + (q.y > mine);
      }
    }
    for (; j < n; ++j) above += cand[j] > mine;
    if (above < 32) best[above] = mine;
  }
  __syncthreads();
}

// what the joined row comes to; xt: the target's logit, `list`: the keys, over the lanes
__device__ __forceinline__ void write_row(const Params& p, long long row, const Acc& a, float xt, bool found, bool top,
                                          u64 list, int lane) {
  const float log_s = logf(a.s);
  if (lane == 0) {
    const long long t = p.targets ? p.targets[row] : p.ignore_index;
    const bool ignored = p.targets == nullptr || t == p.ignore_index;
    if (p.logprobs) p.logprobs[row] = ignored ? 0.0f : (found ? (xt - a.m) * p.inv_t - log_s : NAN);
    if (p.entropy) p.entropy[row] = log_s - a.t / a.s * p.inv_t;
    if (p.lse) p.lse[row] = a.m * p.inv_t + log_s;
    if (p.row_max) p.row_max[row] = a.m;
    if (p.log_sum) p.log_sum[row] = log_s;
  }
  if (top && lane < p.top_k) {
    // fewer than k comparable logits (NaN): any valid column
    p.top_ids[row * p.top_k + lane] = list != 0 ? static_cast<long long>(key_index(list)) : lane;
    p.top_logprobs[row * p.top_k + lane] = ((list != 0 ? key_value(list) : NAN) - a.m) * p.inv_t - log_s;
  }
}

// a CTA's columns: vectors [v_begin, v_end) from vbase on, the first of them column `head`, and `ones` single ones, those in
// front of `head` and those from `tail` on
struct Columns {
  const uint8_t* vbase;
  const uint8_t* base;
  int v_begin, v_end, head, tail, ones;
  uint32_t first;
};

// the best 32 keys of this warp's share of the CTA's columns, sorted over its lanes
template <int DT>
__device__ __noinline__ u64 rescan(const Columns& c, int top_k) {
  using V = Vec<DT>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 list = 0, floor_key = 0;
  for (int v0 = c.v_begin + warp * 32; v0 < c.v_end; v0 += THREADS) {
    const int v = v0 + lane;
    uint4 q = make_uint4(0, 0, 0, 0);
    if (v < c.v_end) q = load_stream(c.vbase + static_cast<long long>(v) * 16);
#pragma unroll 1
    for (int i = 0; i < V::N; ++i) {
      const float x = V::pop(q);
      warp_offer(list, floor_key, v < c.v_end ? make_key(x, c.first + c.head + v * V::N + i) : 0, top_k, lane);
    }
  }
  if (warp == 0) {
    const int col = lane < c.head ? lane : c.tail + (lane - c.head);
    const bool live = lane < c.ones;
    warp_offer(list, floor_key, live ? make_key(V::one(c.base + static_cast<long long>(live ? col : 0) * V::ES), c.first + col) : 0, top_k, lane);
  }
  return list;
}

// CTAs per SM: four of 64 registers (511 rows of 151936 fp32 logits take 69 us with three, 49 with four: one wave instead
// of two).  With the top k three: fewer registers cost more than the fourth CTA brings (300 rows of
// 128256 bf16 logits, k = 5: 31.2 against 33.8 us; 511 of 151936 fp32, k = 20, the other way: 79 against 71).
template <int DT, bool TOP>
__global__ void __launch_bounds__(THREADS, TOP ? 3 : 4) logprobs_kernel(const Params p, const int cs) {
  using V = Vec<DT>;
  constexpr int N = V::N, ES = V::ES;
  __shared__ Shared sh;
  __shared__ typename std::conditional<TOP, TopShared, char>::type top_raw;
  TopShared& top = reinterpret_cast<TopShared&>(top_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = blockIdx.x / cs;
  const int rank = blockIdx.x % cs;
  const uint8_t* base = p.logits + row * p.ld * ES;
  if (cs > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // columns: `head` up to the first 16-byte boundary, nv whole vectors shared out over the cluster, a tail
  const int mis = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / ES;
  const int vocab = static_cast<int>(p.vocab);
  const int head = mis < vocab ? mis : vocab;
  const int nv = (vocab - head) / N;
  const int tail0 = head + nv * N;
  const uint8_t* vbase = base + static_cast<long long>(head) * ES;
  // whole warps of vectors per CTA
  const int per = ((nv + cs - 1) / cs + 31) / 32 * 32;
  const int v_begin = min(rank * per, nv), v_end = min(v_begin + per, nv);

  const float c = p.inv_t * LOG2E;
  Run r;
  r.m = -INFINITY;
  r.nm = 0.0f;
  r.s = r.t = make_float2(0.0f, 0.0f);

  // the given token's logit, asked for now and used at the end
  const long long t = p.targets ? p.targets[row] : p.ignore_index;
  const long long tl = t - p.vocab_start;
  const bool found = rank == 0 && t != p.ignore_index && t >= 0 && t < p.vocab_total && tl >= 0 && tl < p.vocab;
  const float xt = found ? V::one(base + tl * ES) : 0.0f;

  constexpr int U = 4;
  float bound = -INFINITY;               // nothing below it can be among the best k
  // At most N - 1 single columns at either end: warp 0 of the first CTA, one per lane.
  const int n_one = rank == 0 ? head + vocab - tail0 : 0;
  if (TOP && threadIdx.x == 0) top.count = n_one;
  if (warp == 0 && lane < n_one) {
    const int col = lane < head ? lane : tail0 + (lane - head);
    const float x[1] = {V::one(base + static_cast<long long>(col) * ES)};
    if (x[0] > r.m) rebase(r, x[0], c);
    accumulate_raw<1>(r, x, c);
    if constexpr (TOP) top.col[lane] = col;
  }
  if constexpr (TOP) __syncthreads();
  int keyed = 0;                         // candidates below this have their keys in top.cand
  bool kept = true;                      // every candidate is in the list

  // vectors past the end are all masked
  auto load = [&](int v0, uint4 (&q)[U]) {
    const uint32_t lo = DT == DT_BF16 ? 0xff80ff80u : 0xff800000u;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * THREADS + threadIdx.x;
      q[u] = make_uint4(lo, lo, lo, lo);
      if (v < v_end) q[u] = load_stream(vbase + static_cast<long long>(v) * 16);
    }
  };
  uint4 q[U], ahead[U];
  load(v_begin, ahead);
  // (once at least: the last batch ranks the candidates)
  for (int v0 = v_begin, batch = 1, next_rank = 1; v0 < v_end || batch == 1; v0 += U * THREADS, ++batch) {
    const bool last = v0 + U * THREADS >= v_end;
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = ahead[u];
    if (!last) load(v0 + U * THREADS, ahead);
    float mx = V::max_of(q[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) mx = fmaxf(mx, V::max_of(q[u]));
    if (mx > r.m) rebase(r, mx, c);
    float2 s = make_float2(0.0f, 0.0f), t = s;
    // (a maximum as low as what stands for a masked logit: take them as they are)
    if (r.m > -1.0e38f) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[N];
        V::unpack(V::unmask(q[u]), x);
        accumulate<N>(r.nm, s, t, x, c);
      }
    }
    const float tt = t.x + t.y;
    if (r.m > -1.0e38f && tt == tt) {
      r.s = fadd2(r.s, s);
      r.t = fadd2(r.t, t);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[N];
        V::unpack(q[u], x);
        accumulate_raw<N>(r, x, c);
      }
    }
    if constexpr (TOP) {
      if (batch == 1) {
        // the first bound, from the threads' maxima of this batch
        const int full = min(WARPS, (v_end - v_begin) / 32);         // warps whose first vectors are all live
        if (full > 0 && warp < full) {
          const int need = (p.top_k + full - 1) / full;
          uint32_t key = static_cast<uint32_t>(make_key(mx, 0) >> 32);
          uint32_t best = 0;
          for (int i = 0; i < need; ++i) {
            best = __reduce_max_sync(0xffffffffu, key);
            const int first = __ffs(__ballot_sync(0xffffffffu, key == best)) - 1;
            if (lane == first) key = 0;
          }
          if (lane == 0) top.warp_bound[warp] = best == 0 ? -INFINITY : key_value(static_cast<u64>(best) << 32);
        }
        __syncthreads();
        if (full > 0) {
          bound = top.warp_bound[0];
          for (int w = 1; w < full; ++w) bound = fminf(bound, top.warp_bound[w]);
        }
      }
      if (kept && mx >= bound) {
        // one place in the list per thread for all of its candidates
        uint32_t mask = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float x[N];
          V::unpack(q[u], x);
#pragma unroll
          for (int i = 0; i < N; ++i) mask |= x[i] >= bound ? 1u << (u * N + i) : 0u;
          if (v0 + u * THREADS + static_cast<int>(threadIdx.x) >= v_end) mask &= (1u << (u * N)) - 1u;
        }
        int at = atomicAdd(&top.count, __popc(mask));
#pragma unroll 1
        for (; mask != 0; mask &= mask - 1, ++at) {
          const int e = __ffs(mask) - 1;
          if (at < CAP) top.col[at] = head + (v0 + (e / N) * THREADS + static_cast<int>(threadIdx.x)) * N + e % N;
        }
      }
      if (batch == next_rank || last) {
        next_rank *= 4;
        __syncthreads();
        int n = top.count;
        __syncthreads();
        kept = n <= CAP;
        if (kept || last) {
          if (kept) {
            for (int i = keyed + static_cast<int>(threadIdx.x); i < n; i += THREADS) {
              const uint32_t col = top.col[i];
              top.cand[i] = make_key(V::one(base + static_cast<long long>(col) * ES), static_cast<uint32_t>(p.vocab_start) + col);
            }
          } else {
            // once more, each warp for itself
            const Columns cols{vbase, base, v_begin, v_end, head, tail0, n_one, static_cast<uint32_t>(p.vocab_start)};
            top.cand[warp * 32 + lane] = rescan<DT>(cols, p.top_k);
            n = WARPS * 32;
          }
          rank_keys(top.cand, n, top.best);
          if (!last) {
            if (threadIdx.x < 32) top.cand[threadIdx.x] = top.best[threadIdx.x];
            if (threadIdx.x == 0) top.count = 32;
            keyed = 32;
            const u64 kth = top.best[p.top_k - 1];
            if (kth != 0) bound = key_value(kth);
            __syncthreads();
          }
        }
      }
    }
  }

  Acc a{r.m, r.s.x + r.s.y, r.t.x + r.t.y};
  a = warp_join(a, c);
  if (lane == 0) sh.warp_acc[warp] = a;
  __syncthreads();
  if (warp == 0) a = warp_join(lane < WARPS ? sh.warp_acc[lane] : Acc{-INFINITY, 0.0f, 0.0f}, c);
  if (cs > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");       // the first CTA has started
    cg::cluster_group cluster = cg::this_cluster();
    if (warp == 0) {
      Shared* first = cluster.map_shared_rank(&sh, 0);
      if (lane == 0) first->cta_acc[rank] = a;
      if constexpr (TOP) {
        if (lane < p.top_k) cluster.map_shared_rank(&top, 0)->cta_keys[rank * p.top_k + lane] = top.best[lane];
      }
    }
    __syncwarp();
    cluster.sync();
    if (rank != 0) return;
    if (warp == 0) a = warp_join(lane < cs ? sh.cta_acc[lane] : Acc{-INFINITY, 0.0f, 0.0f}, c);
    if constexpr (TOP) rank_keys(top.cta_keys, cs * p.top_k, top.best);
  }
  if (warp != 0) return;

  const u64 key = TOP ? top.best[lane] : 0;
  if (p.stats != nullptr) {
    if (lane == 0) {
      float* s = p.stats + row * 5;
      s[0] = a.m; s[1] = a.s; s[2] = a.t; s[3] = xt; s[4] = found ? 1.0f : 0.0f;
    }
    if (TOP && lane < p.top_k) p.keys[row * p.top_k + lane] = key;
  } else {
    write_row(p, row, a, xt, found, TOP, key, lane);
  }
}

// Partial results of `parts` slices of the vocabulary (stats (parts, rows, 5), keys (parts, rows, k)) ->
// the rows' results.  One warp per row.
__global__ void __launch_bounds__(256) logprobs_join_kernel(const Params p, const float* stats, const u64* keys, int parts,
                                                            long long rows) {
  const int lane = threadIdx.x & 31;
  const long long row = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if (row >= rows) return;
  Acc a{-INFINITY, 0.0f, 0.0f};
  const float c = p.inv_t * LOG2E;
  float xt = 0.0f;
  bool found = false;
  u64 list = 0;
  for (int q = 0; q < parts; ++q) {
    const float* s = stats + (q * rows + row) * 5;
    a = join(a, Acc{s[0], s[1], s[2]}, c);
    if (s[4] != 0.0f) { xt = s[3]; found = true; }
    if (p.top_k > 0) list = warp_merge(list, lane < p.top_k ? keys[(q * rows + row) * p.top_k + lane] : 0, lane);
  }
  write_row(p, row, a, xt, found, p.top_k > 0, list, lane);
}

struct BackParams {
  const uint8_t* logits;
  uint8_t* grad;
  const long long* targets;
  const float* row_max;                  // or NULL, and log_sum is lse
  const float* log_sum;
  const float* entropy;
  const float* g_logprob;
  const float* g_entropy;
  long long vocab, ld, ld_grad, ignore_index, vocab_start, vocab_total;
  float inv_t;
};

template <int DT>
__device__ __forceinline__ uint4 pack(const float* x);
template <>
__device__ __forceinline__ uint4 pack<DT_BF16>(const float* x) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
  return make_uint4(u[0], u[1], u[2], u[3]);
}
template <>
__device__ __forceinline__ uint4 pack<DT_F32>(const float* x) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
template <int DT>
__device__ __forceinline__ void store_one(uint8_t* p, float x) {
  if constexpr (DT == DT_BF16) *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(float_to_bf16_bits(x));
  else *reinterpret_cast<float*>(p) = x;
}

// small CTAs with all of their loads in flight at once: 4095 x 151936 bf16 with an entropy gradient takes 367 us with 128
// threads of eight vectors each, 402 with four, 415 / 414 with 256 threads of four / eight, 472 with 512 of two
constexpr int BACK_THREADS = 128;
constexpr int BACK_VECS = 8;

// grid: (column chunks, rows folded over y and z)
template <int DT, bool ENT>
__global__ void __launch_bounds__(BACK_THREADS) logprobs_backward_kernel(const BackParams p, long long rows, int vec_per_cta) {
  using V = Vec<DT>;
  constexpr int N = V::N, ES = V::ES;
  // the last rows first: they are what the forward pass has left in the L2
  const long long row = rows - 1 - (blockIdx.y + static_cast<long long>(blockIdx.z) * gridDim.y);
  if (row < 0) return;
  const uint8_t* in = p.logits + row * p.ld * ES;
  uint8_t* out = p.grad + row * p.ld_grad * ES;
  const long long t = p.targets ? p.targets[row] : p.ignore_index;
  const bool ignored = t == p.ignore_index;
  const float gl = (ignored || p.g_logprob == nullptr) ? 0.0f
                   : (t < 0 || t >= p.vocab_total)     ? NAN
                                                       : p.g_logprob[row] * p.inv_t;
  const float c = p.inv_t * LOG2E;
  const float m = p.row_max ? p.row_max[row] : 0.0f;
  const float nl = -p.log_sum[row] * LOG2E;              // log2 p = (x - m) c + nl
  const float gh = ENT ? p.g_entropy[row] * p.inv_t : 0.0f;
  // dx = p (-gl - gh (log p + H)) + gl [j = t] = p (a + b log2 p) + ...
  const float a = ENT ? -gl - gh * p.entropy[row] : -gl;
  const float b = ENT ? -gh / LOG2E : 0.0f;
  const long long tl = t - p.vocab_start;                // column of the target, if it is one of these
  const bool here = !ignored && tl >= 0 && tl < p.vocab;
  auto one = [&](float x) {
    const float y = __fmaf_rn(x - m, c, nl);
    const float pr = exp2_approx(y);
    // (below -127 the probability is 0: p log p is then 0, too, however large b is)
    if constexpr (ENT) return __fmaf_rn(pr * b, max_nan(y, -127.0f), pr * a);
    else return pr * a;
  };
  const int mis = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(in) & 15)) & 15) / ES;
  const bool wide = (reinterpret_cast<uintptr_t>(in) & 15) == (reinterpret_cast<uintptr_t>(out) & 15);
  const long long head = mis < p.vocab ? mis : p.vocab;
  const long long nv = (p.vocab - head) / N;
  const long long v_begin = static_cast<long long>(blockIdx.x) * vec_per_cta;
  const long long v_end = v_begin + vec_per_cta < nv ? v_begin + vec_per_cta : nv;
  constexpr int U = BACK_VECS;
  if (gl == 0.0f && gh == 0.0f) {
    // neither result has a gradient (an ignored row, a padded one): zeros, whatever the row holds
    auto zero = [&](long long col) { store_one<DT>(out + col * ES, 0.0f); };
    for (long long v = v_begin + threadIdx.x; v < v_end; v += BACK_THREADS) {
      if (wide) {
        *reinterpret_cast<uint4*>(out + (head + v * N) * ES) = make_uint4(0, 0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) zero(head + v * N + i);
      }
    }
    const long long tail0 = head + nv * N;
    const int i = threadIdx.x;
    if (blockIdx.x == 0 && i < head + (p.vocab - tail0)) zero(i < head ? i : tail0 + (i - head));
    return;
  }
  for (long long v = v_begin + threadIdx.x; v < v_end; v += U * BACK_THREADS) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * BACK_THREADS < v_end) q[u] = load_stream(in + (head + (v + u * BACK_THREADS) * N) * ES);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long vv = v + u * BACK_THREADS;
      if (vv >= v_end) break;
      float x[N];
      V::unpack(q[u], x);
      const long long col = head + vv * N;
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = one(x[i]);
      if (here && tl >= col && tl < col + N) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (tl == col + i) x[i] += gl;
      }
      if (wide) {
        *reinterpret_cast<uint4*>(out + col * ES) = pack<DT>(x);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) store_one<DT>(out + (col + i) * ES, x[i]);
      }
    }
  }
  if (blockIdx.x == 0) {
    const long long tail0 = head + nv * N;
    const int n_one = static_cast<int>(head + (p.vocab - tail0));
    const int i = threadIdx.x;
    if (i < n_one) {
      const long long col = i < head ? i : tail0 + (i - head);
      float x = one(V::one(in + col * ES));
      if (here && tl == col) x += gl;
      store_one<DT>(out + col * ES, x);
    }
  }
}

static int check(const ForgeLogprobsArgs& a, const char* what) {
  if (a.rows < 0 || a.vocab < 0) return fail(FORGE_ERR_INVALID_ARG, "%s: negative dimension", what);
  if (a.dtype != FORGE_DT_BF16 && a.dtype != FORGE_DT_F32) return fail(FORGE_ERR_INVALID_ARG, "%s: unknown dtype %d", what, a.dtype);
  if (a.top_k < 0 || a.top_k > MAX_TOP) return fail(FORGE_ERR_INVALID_ARG, "%s: top_k must be 0 .. %d (got %d)", what, MAX_TOP, a.top_k);
  // log2 e / temperature is a number in fp32, and the exponential of the lowest logit over the temperature 0: a masked (-inf)
  // logit is taken for one of those
  if (!(a.temperature >= 1e-36 && a.temperature <= 1e36))
    return fail(FORGE_ERR_INVALID_ARG, "%s: temperature must be a positive number, 1e-36 .. 1e36 (got %g)", what, a.temperature);
  if (a.vocab_start < 0 || a.vocab_total < a.vocab_start + a.vocab || a.vocab_total > 0x7fffffffll)
    return fail(FORGE_ERR_SHAPE, "%s: columns [%lld, %lld) of a vocabulary of %lld", what, (long long)a.vocab_start,
                (long long)(a.vocab_start + a.vocab), (long long)a.vocab_total);
  if (a.top_k > a.vocab_total) return fail(FORGE_ERR_SHAPE, "%s: top_k (%d) exceeds the vocabulary (%lld)", what, a.top_k, (long long)a.vocab_total);
  if (a.rows > 0 && (a.vocab < 1 || a.ld < a.vocab)) return fail(FORGE_ERR_SHAPE, "%s: vocab=%lld ld=%lld", what, (long long)a.vocab, (long long)a.ld);
  if (a.rows * MAX_CLUSTER > 0x7fffffffll) return fail(FORGE_ERR_SHAPE, "%s: %lld rows", what, (long long)a.rows);
  auto off = [](const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  if (off(a.targets, 8) || off(a.logprobs, 4) || off(a.entropy, 4) || off(a.lse, 4) || off(a.top_logprobs, 4) || off(a.top_ids, 8) ||
      off(a.stats, 4) || off(a.keys, 8) || off(a.row_max, 4) || off(a.log_sum, 4))
    return fail(FORGE_ERR_ALIGNMENT, "%s: targets or outputs are not element-aligned", what);
  return FORGE_OK;
}

static Params make_params(const ForgeLogprobsArgs& a) {
  Params p;
  p.logits = static_cast<const uint8_t*>(a.logits);
  p.targets = reinterpret_cast<const long long*>(a.targets);
  p.logprobs = a.logprobs; p.entropy = a.entropy; p.lse = a.lse;
  p.row_max = a.row_max; p.log_sum = a.log_sum;
  p.top_logprobs = a.top_logprobs; p.top_ids = reinterpret_cast<long long*>(a.top_ids);
  p.stats = a.stats; p.keys = reinterpret_cast<u64*>(a.keys);
  p.vocab = a.vocab; p.ld = a.ld; p.ignore_index = a.ignore_index;
  p.vocab_start = a.vocab_start; p.vocab_total = a.vocab_total;
  p.top_k = a.top_k;
  p.inv_t = static_cast<float>(1.0 / a.temperature);
  return p;
}

template <int DT, bool TOP>
static int launch_forward(const Params& p, long long rows, int cs, int device, cudaStream_t stream) {
  auto* fn = logprobs_kernel<DT, TOP>;
  static std::atomic<uint64_t> allowed{0};             // devices on which clusters of sixteen have been allowed
  const uint64_t bit = 1ull << (device & 63);
  if (cs > 8 && !(allowed.load(std::memory_order_relaxed) & bit)) {
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "logprobs: cluster attribute: %s", cudaGetErrorString(e));
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * cs));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, fn, p, cs);
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "logprobs launch: %s", cudaGetErrorString(e));
  return FORGE_OK;
}

}  // namespace loss
}  // namespace forge

using namespace forge;

extern "C" int forge_logprobs_forward(const ForgeLogprobsArgs* args, void* cuda_stream) {
  if (args == nullptr) return fail(FORGE_ERR_INVALID_ARG, "forge_logprobs_forward: args is NULL");
  const ForgeLogprobsArgs& a = *args;
  int rc = loss::check(a, "forge_logprobs_forward");
  if (rc != FORGE_OK) return rc;
  if (a.rows == 0) return FORGE_OK;
  if (a.logits == nullptr) return fail(FORGE_ERR_INVALID_ARG, "forge_logprobs_forward: logits is NULL");
  const int es = a.dtype == FORGE_DT_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(a.logits) % es != 0) return fail(FORGE_ERR_ALIGNMENT, "forge_logprobs_forward: logits are not element-aligned");
  if (a.stats == nullptr && a.vocab != a.vocab_total)
    return fail(FORGE_ERR_INVALID_ARG, "forge_logprobs_forward: a slice of the vocabulary needs `stats`");
  if (a.top_k > 0 && (a.stats != nullptr ? a.keys == nullptr : (a.top_logprobs == nullptr || a.top_ids == nullptr)))
    return fail(FORGE_ERR_INVALID_ARG, "forge_logprobs_forward: top_k without its outputs");
  const DeviceInfo* di = current_device_info();
  if (di == nullptr) return FORGE_ERR_CUDA;
  if (di->cc_major != 10) return fail(FORGE_ERR_DEVICE, "device %d is sm_%d%d, not sm_100", di->device, di->cc_major, di->cc_minor);
  // A row is cut over a cluster while all CTAs are resident at once (nine tenths of the places that the kernel's launch
  // bounds leave, two CTAs per SM for clusters of eight and sixteen, which fill the GPU less well) and each still has four
  // vectors per thread to load: 64 rows of 128256 bf16 logits take 14.2 / 9.6 / 7.6 / 10.3 us over 1 / 2 / 4 / 8 CTAs a
  // row, 100 rows of 151936 fp32 logits 18.3 / 14.3 over 2 / 4, 4096 fp32 logits 4.7 / 5.9 over 1 / 2.  The first CTA
  // ranks the others' k keys each: with k = 20, 8 CTAs a row beat 16 (14.6 against 18.5 us for 16 rows).
  const long long vecs = a.vocab * es / 16;
  auto resident = [&](int n) { return a.rows * n * 10 <= (n > 4 ? 20ll : a.top_k > 0 ? 27ll : 36ll) * di->sm_count; };
  int cs = 1;
  while (cs < loss::MAX_CLUSTER && resident(cs * 2) && vecs > 4ll * cs * loss::THREADS && cs * 2 * a.top_k <= 192) cs *= 2;
  const loss::Params p = loss::make_params(a);
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  if (a.dtype == FORGE_DT_BF16)
    return a.top_k > 0 ? loss::launch_forward<DT_BF16, true>(p, a.rows, cs, di->device, s) : loss::launch_forward<DT_BF16, false>(p, a.rows, cs, di->device, s);
  return a.top_k > 0 ? loss::launch_forward<DT_F32, true>(p, a.rows, cs, di->device, s) : loss::launch_forward<DT_F32, false>(p, a.rows, cs, di->device, s);
}

extern "C" int forge_logprobs_join(const ForgeLogprobsArgs* args, const float* stats, const uint64_t* keys, int32_t parts,
                                   void* cuda_stream) {
  if (args == nullptr) return fail(FORGE_ERR_INVALID_ARG, "forge_logprobs_join: args is NULL");
  ForgeLogprobsArgs a = *args;
  a.vocab_start = 0;                       // the joined rows cover the whole vocabulary
  a.vocab = a.vocab_total;
  a.ld = a.vocab_total;
  int rc = loss::check(a, "forge_logprobs_join");
  if (rc != FORGE_OK) return rc;
  if (parts < 1) return fail(FORGE_ERR_INVALID_ARG, "forge_logprobs_join: parts = %d", parts);
  if (a.rows == 0) return FORGE_OK;
  if (stats == nullptr || (a.top_k > 0 && (keys == nullptr || a.top_logprobs == nullptr || a.top_ids == nullptr)))
    return fail(FORGE_ERR_INVALID_ARG, "forge_logprobs_join: null pointer");
  if (reinterpret_cast<uintptr_t>(stats) % 4 || reinterpret_cast<uintptr_t>(keys) % 8)
    return fail(FORGE_ERR_ALIGNMENT, "forge_logprobs_join: stats or keys are not element-aligned");
  const loss::Params p = loss::make_params(a);
  loss::logprobs_join_kernel<<<static_cast<unsigned>((a.rows + 7) / 8), 256, 0, static_cast<cudaStream_t>(cuda_stream)>>>(
      p, stats, reinterpret_cast<const loss::u64*>(keys), parts, a.rows);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "logprobs join launch: %s", cudaGetErrorString(e));
  return FORGE_OK;
}

extern "C" int forge_logprobs_backward(const ForgeLogprobsArgs* args, const float* g_logprob, const float* g_entropy, void* grad,
                                       int64_t ld_grad, void* cuda_stream) {
  if (args == nullptr) return fail(FORGE_ERR_INVALID_ARG, "forge_logprobs_backward: args is NULL");
  const ForgeLogprobsArgs& a = *args;
  int rc = loss::check(a, "forge_logprobs_backward");
  if (rc != FORGE_OK) return rc;
  if (a.rows == 0) return FORGE_OK;
  const bool apart = a.row_max != nullptr && a.log_sum != nullptr;
  if (a.logits == nullptr || (!apart && a.lse == nullptr) || grad == nullptr || (g_entropy != nullptr && a.entropy == nullptr))
    return fail(FORGE_ERR_INVALID_ARG, "forge_logprobs_backward: null pointer");
  if (ld_grad < a.vocab) return fail(FORGE_ERR_SHAPE, "forge_logprobs_backward: ld_grad=%lld", (long long)ld_grad);
  const int es = a.dtype == FORGE_DT_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(a.logits) % es != 0 || reinterpret_cast<uintptr_t>(grad) % es != 0 ||
      reinterpret_cast<uintptr_t>(g_logprob) % 4 != 0 || reinterpret_cast<uintptr_t>(g_entropy) % 4 != 0)
    return fail(FORGE_ERR_ALIGNMENT, "forge_logprobs_backward: tensors are not element-aligned");
  loss::BackParams p;
  p.logits = static_cast<const uint8_t*>(a.logits);
  p.grad = static_cast<uint8_t*>(grad);
  p.targets = reinterpret_cast<const long long*>(a.targets);
  p.row_max = apart ? a.row_max : nullptr; p.log_sum = apart ? a.log_sum : a.lse;
  p.entropy = a.entropy; p.g_logprob = g_logprob; p.g_entropy = g_entropy;
  p.vocab = a.vocab; p.ld = a.ld; p.ld_grad = ld_grad; p.ignore_index = a.ignore_index;
  p.vocab_start = a.vocab_start; p.vocab_total = a.vocab_total;
  p.inv_t = static_cast<float>(1.0 / a.temperature);
  const int vec_per_cta = loss::BACK_THREADS * loss::BACK_VECS;
  const long long vecs = a.vocab * es / 16;
  const long long chunks = std::max<long long>(1, (vecs + vec_per_cta - 1) / vec_per_cta);
  const unsigned gy = static_cast<unsigned>(std::min<int64_t>(a.rows, 32768));
  const unsigned gz = static_cast<unsigned>((a.rows + gy - 1) / gy);
  if (gz > 65535u) return fail(FORGE_ERR_SHAPE, "forge_logprobs_backward: %lld rows", (long long)a.rows);
  const dim3 grid(static_cast<unsigned>(chunks), gy, gz);
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  if (a.dtype == FORGE_DT_BF16) {
    if (g_entropy) loss::logprobs_backward_kernel<DT_BF16, true><<<grid, loss::BACK_THREADS, 0, s>>>(p, a.rows, vec_per_cta);
    else loss::logprobs_backward_kernel<DT_BF16, false><<<grid, loss::BACK_THREADS, 0, s>>>(p, a.rows, vec_per_cta);
  } else {
    if (g_entropy) loss::logprobs_backward_kernel<DT_F32, true><<<grid, loss::BACK_THREADS, 0, s>>>(p, a.rows, vec_per_cta);
    else loss::logprobs_backward_kernel<DT_F32, false><<<grid, loss::BACK_THREADS, 0, s>>>(p, a.rows, vec_per_cta);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "logprobs backward launch: %s", cudaGetErrorString(e));
  return FORGE_OK;
}
