// One AdamW step over a list of tensors of any sizes, and the common norm of a list of gradients.
//
// The tensors' pointers and sizes travel in the kernel's parameter block (up to MAX_TENSORS per launch),
// so a step is one launch, needs no descriptor in device memory and can be captured as it is.  The
// elements of all tensors are cut into chunks; a CTA finds its tensor by bisection of the chunks' prefix
// sums.  A thread owns 8 consecutive elements, so eight lanes own a quantisation block of 64 and agree on
// its absmax with three shuffles; the blocks run over a tensor's elements in memory order, which for a
// (V, H) weight with H % 64 == 0 is the layout of the fused path.  Same per-element arithmetic as the fused
// path (forge_update.cuh), but for the scales of the 8-bit moments (block_scale there: at most one ulp apart).  As there,
// an 8-bit second moment counts as at least 1e-8.
//
// Bound by memory: 3 element sizes of the parameter (read, write, gradient) and 2 of each moment.  A thread has the next
// pass's elements on their way while it updates this one's: 525 M bf16 parameters with e4m3 moments take 830 us (6.5 TB/s; 931
// where seconds of it have brought the SMs to the power cap), 984 without; fp32 throughout, with the norm before it, 132 M take
// 640 us: about 90 for the norm, which only reads, and 541 for the update (6.8 TB/s).
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include "forge_host.h"

namespace forge {
namespace multi {

constexpr int THREADS = 256;
constexpr int EPT = 8;                          // elements per thread and pass
constexpr int PASS = THREADS * EPT;             // 2048 elements
constexpr int MAX_TENSORS = 448;
constexpr int FEW_TENSORS = 112;                // a parameter block of 7 KB instead of 27: less to copy per launch

struct Item {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  long long n;
};

template <int CAP>
struct Params {
  Item item[CAP];
  int first_chunk[CAP + 1];                     // first chunk of each tensor; [count] = number of chunks
  int count;
  int passes;                                   // a chunk is this many passes of PASS elements
  const float* coef;                            // gradients are multiplied by *coef, if given
  const Hyper* hyper_device;
  Hyper hyper;
};

// largest i with first[i] <= c
__device__ __forceinline__ int find_tensor(const int* first, int count, int c) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int DT>
__device__ __forceinline__ void store8(void* base, long long i, const float (&x)[8]) {
  if constexpr (DT == DT_F32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
    q[0] = make_float4(x[0], x[1], x[2], x[3]);
    q[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[k]) : "f"(x[2 * k + 1]), "f"(x[2 * k]));
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + i) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}
template <int DT>
__device__ __forceinline__ void store1(void* base, long long i, float x) {
  if constexpr (DT == DT_F32) static_cast<float*>(base)[i] = x;
  else static_cast<uint16_t*>(base)[i] = static_cast<uint16_t>(float_to_bf16_bits(x));
}

__device__ __forceinline__ float absmax8(const float (&x)[8]) {
  const float a = fmax3(fabsf(x[0]), fabsf(x[1]), fabsf(x[2])), b = fmax3(fabsf(x[3]), fabsf(x[4]), fabsf(x[5]));
  return fmax3(fmaxf(a, b), fabsf(x[6]), fabsf(x[7]));
}

__device__ __forceinline__ bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// what a thread reads of eight consecutive elements
template <int DT>
struct Raw8 {
  uint4 q[DT == DT_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* base, long long i) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + i * (DT == DT_F32 ? 4 : 2));
#pragma unroll
    for (int k = 0; k < (DT == DT_F32 ? 2 : 1); ++k) q[k] = p[k];
  }
  __device__ __forceinline__ void load_some(const void* base, long long i, int live) {
    uint32_t u[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k < live) {
        if constexpr (DT == DT_F32) u[k] = static_cast<const uint32_t*>(base)[i + k];
        else u[k >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t*>(base)[i + k]) << (16 * (k & 1));
      }
    }
#pragma unroll
    for (int k = 0; k < (DT == DT_F32 ? 2 : 1); ++k) q[k] = make_uint4(u[4 * k], u[4 * k + 1], u[4 * k + 2], u[4 * k + 3]);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    if constexpr (DT == DT_F32) {
      x[0] = __uint_as_float(q[0].x); x[1] = __uint_as_float(q[0].y); x[2] = __uint_as_float(q[0].z); x[3] = __uint_as_float(q[0].w);
      x[4] = __uint_as_float(q[1].x); x[5] = __uint_as_float(q[1].y); x[6] = __uint_as_float(q[1].z); x[7] = __uint_as_float(q[1].w);
    } else {
      const uint32_t u[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[2 * k] = __uint_as_float(u[k] << 16);
        x[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
      }
    }
  }
};
struct RawCodes {
  uint2 q;
  __device__ __forceinline__ void load(const void* base, long long i) { q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(base) + i); }
  __device__ __forceinline__ void load_some(const void* base, long long i, int live) {
    uint32_t u[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < live) u[k >> 2] |= static_cast<uint32_t>(static_cast<const uint8_t*>(base)[i + k]) << (8 * (k & 3));
    q = make_uint2(u[0], u[1]);
  }
};

template <int W_DT, int G_DT, int ST>
struct Elements {
  static constexpr bool QUANT = ST == ST_INT8 || ST == ST_FP8_BLOCK;
  static constexpr int S_DT = ST == ST_F32 ? DT_F32 : DT_BF16;
  typedef typename std::conditional<QUANT, RawCodes, Raw8<S_DT>>::type State;
  Raw8<W_DT> p;
  Raw8<G_DT> g;
  State m, v;
  float sm, sv;
  // `live` of the eight elements from i exist; whole and aligned: wide loads
  __device__ __forceinline__ void load(const Item& it, long long i, int live, bool wide) {
    if (wide && live == EPT) {
      g.load(it.g, i);
      p.load(it.p, i);
      m.load(it.m, i);
      v.load(it.v, i);
    } else {
      g.load_some(it.g, i, live);
      p.load_some(it.p, i, live);
      m.load_some(it.m, i, live);
      v.load_some(it.v, i, live);
    }
    sm = sv = 1.0f;
    if (QUANT && live > 0) {
      sm = it.m_scale[i >> 6];
      sv = it.v_scale[i >> 6];
    }
  }
};

__device__ __forceinline__ int live_of(long long n, long long i) {
  const long long left = n - i;
  return left >= EPT ? EPT : (left > 0 ? static_cast<int>(left) : 0);
}

template <int W_DT, int G_DT, int ST, int CAP>
__global__ void __launch_bounds__(THREADS) multi_adamw_kernel(const __grid_constant__ Params<CAP> p) {
  constexpr bool QUANT = ST == ST_INT8 || ST == ST_FP8_BLOCK;
  constexpr int S_DT = ST == ST_F32 ? DT_F32 : DT_BF16;
  const int chunk = blockIdx.x;
  const int ti = find_tensor(p.first_chunk, p.count, chunk);
  const Item it = p.item[ti];
  const Hyper hy = p.hyper_device != nullptr ? *p.hyper_device : p.hyper;
  const float coef = p.coef != nullptr ? *p.coef : 1.0f;
  const long long begin = static_cast<long long>(chunk - p.first_chunk[ti]) * p.passes * PASS;
  const bool wide = aligned(it.p, 16) && aligned(it.g, 16) && aligned(it.m, QUANT ? 8 : 16) && aligned(it.v, QUANT ? 8 : 16);
  long long i0 = begin + threadIdx.x * EPT;
  int live = live_of(it.n, i0);
  Elements<W_DT, G_DT, ST> now, next;
  now.load(it, i0, live, wide);
#pragma unroll 1
  for (int pass = 0; pass < p.passes; ++pass) {
    // whole warps leave together (the block absmax is agreed on by shuffles)
    if (i0 - (threadIdx.x & 31) * EPT >= it.n) break;
    // the next pass's elements are on their way while this one's are updated
    const int live_next = pass + 1 < p.passes ? live_of(it.n, i0 + PASS) : 0;
    if (live_next > 0) next.load(it, i0 + PASS, live_next, wide);
    float w[EPT], g[EPT], m[EPT], v[EPT];
    now.g.get(g);
    now.p.get(w);
    if constexpr (QUANT) {
      uint32_t mq[2] = {now.m.q.x, now.m.q.y}, vq[2] = {now.v.q.x, now.v.q.y};
      if constexpr (ST == ST_INT8) {
#pragma unroll
        for (int j = 0; j < 2; ++j) { mq[j] ^= 0x80808080u; vq[j] ^= 0x80808080u; }
      }
#pragma unroll
      for (int k = 0; k < EPT; k += 2) {
        float2 m2, v2;
        if constexpr (ST == ST_INT8) {
          m2 = int8x2_to_float(mq[k >> 2], k & 3);
          v2 = int8x2_to_float(vq[k >> 2], k & 3);
        } else {
          e4m3x2_to_float(mq[k >> 2] >> (8 * (k & 3)), m2.x, m2.y);
          e4m3x2_to_float(vq[k >> 2] >> (8 * (k & 3)), v2.x, v2.y);
        }
        m2 = fmul2(m2, make_float2(now.sm, now.sm));
        v2 = fmul2(v2, make_float2(now.sv, now.sv));
        m[k] = m2.x; m[k + 1] = m2.y;
        v[k] = fmaxf(v2.x, 1e-8f); v[k + 1] = fmaxf(v2.y, 1e-8f);
      }
    } else {
      now.m.get(m);
      now.v.get(v);
    }
    if (p.coef != nullptr) {
#pragma unroll
      for (int k = 0; k < EPT; ++k) g[k] = f_mul(g[k], coef);
    }
#pragma unroll
    for (int k = 0; k < EPT; k += 2) {
      float2 m2 = make_float2(m[k], m[k + 1]), v2 = make_float2(v[k], v[k + 1]);
      const float2 w2 = adamw_update2(make_float2(w[k], w[k + 1]), make_float2(g[k], g[k + 1]), m2, v2, hy);
      w[k] = w2.x; w[k + 1] = w2.y;
      m[k] = m2.x; m[k + 1] = m2.y;
      v[k] = v2.x; v[k + 1] = v2.y;
    }
    uint32_t mo[2], vo[2];
    if constexpr (QUANT) {
      float am, av;
      if (live == EPT) {
        am = absmax8(m);
        av = absmax8(v);
      } else {
        // elements past the end of the tensor take no part in the last block's absmax
        am = av = 0.0f;
#pragma unroll
        for (int k = 0; k < EPT; ++k) {
          am = fmaxf(am, k < live ? fabsf(m[k]) : 0.0f);
          av = fmaxf(av, k < live ? fabsf(v[k]) : 0.0f);
        }
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
        av = fmaxf(av, __shfl_xor_sync(0xffffffffu, av, o));
      }
      const float sm_new = block_scale<ST == ST_INT8 ? 127 : 448>(am);
      const float sv_new = block_scale<ST == ST_INT8 ? 127 : 448>(av);
      const float rsm = f_rcp(sm_new), rsv = f_rcp(sv_new);
      const float2 nsm2 = make_float2(-sm_new, -sm_new), nsv2 = make_float2(-sv_new, -sv_new);
      const float2 rsm2 = make_float2(rsm, rsm), rsv2 = make_float2(rsv, rsv);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = 4 * j;
        const float2 qm01 = div2_by_rcp(make_float2(m[k], m[k + 1]), nsm2, rsm2);
        const float2 qm23 = div2_by_rcp(make_float2(m[k + 2], m[k + 3]), nsm2, rsm2);
        const float2 qv01 = div2_by_rcp(make_float2(v[k], v[k + 1]), nsv2, rsv2);
        const float2 qv23 = div2_by_rcp(make_float2(v[k + 2], v[k + 3]), nsv2, rsv2);
        if constexpr (ST == ST_INT8) {
          mo[j] = int8x4_pack(int8x2_round(qm01), int8x2_round(qm23));
          vo[j] = int8x4_pack(int8x2_round(qv01), int8x2_round(qv23));
        } else {
          mo[j] = e4m3x2_code_bits(qm01.x, qm01.y) | (e4m3x2_code_bits(qm23.x, qm23.y) << 16);
          vo[j] = e4m3x2_code_bits(qv01.x, qv01.y) | (e4m3x2_code_bits(qv23.x, qv23.y) << 16);
        }
      }
      if (live > 0 && (i0 & 63) == 0) {
        it.m_scale[i0 >> 6] = sm_new;
        it.v_scale[i0 >> 6] = sv_new;
      }
    }
    if (wide && live == EPT) {
      store8<W_DT>(it.p, i0, w);
      if constexpr (QUANT) {
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(it.m) + i0) = make_uint2(mo[0], mo[1]);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(it.v) + i0) = make_uint2(vo[0], vo[1]);
      } else {
        store8<S_DT>(it.m, i0, m);
        store8<S_DT>(it.v, i0, v);
      }
    } else {
#pragma unroll
      for (int k = 0; k < EPT; ++k) {
        if (k >= live) continue;
        store1<W_DT>(it.p, i0 + k, w[k]);
        if constexpr (QUANT) {
          static_cast<uint8_t*>(it.m)[i0 + k] = static_cast<uint8_t>(mo[k >> 2] >> (8 * (k & 3)));
          static_cast<uint8_t*>(it.v)[i0 + k] = static_cast<uint8_t>(vo[k >> 2] >> (8 * (k & 3)));
        } else {
          store1<S_DT>(it.m, i0 + k, m[k]);
          store1<S_DT>(it.v, i0 + k, v[k]);
        }
      }
    }
    now = next;
    i0 += PASS;
    live = live_next;
  }
}

// ----- common norm --------------------------------------------------------------------------------
struct NormItem {
  const void* g;
  long long n;
};
template <int CAP>
struct NormParams {
  NormItem item[CAP];
  int first_chunk[CAP + 1];
  int count;
  int passes;
  double* partial;                              // one sum per CTA of the launch
};

__device__ __forceinline__ double block_sum_d(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) t += red[i];
  return t;
}

// The sum of eight squares: in fp32, or, where that has left its range (a square above 3.4e38 or all of them so small that
// what is lost below 2^-149 would be missed), in fp64.  Zeros, of which an embedding's gradient mostly consists, are told apart
// before they are converted.
__device__ __forceinline__ double sum_of_squares(const float (&x)[EPT]) {
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < EPT; ++k) s = __fmaf_rn(x[k], x[k], s);
  if ((s >= 0x1p-100f && s < INFINITY) || s != s) return static_cast<double>(s);
  uint32_t any = 0;
#pragma unroll
  for (int k = 0; k < EPT; ++k) any |= __float_as_uint(x[k]) << 1;
  double d = 0.0;
  if (any != 0) {
#pragma unroll
    for (int k = 0; k < EPT; ++k) d = __fma_rn(static_cast<double>(x[k]), static_cast<double>(x[k]), d);
  }
  return d;
}

// squares are summed eight at a time in fp32 and from there on in fp64, in an order that does not
// depend on the run
template <int DT, int CAP>
__global__ void __launch_bounds__(THREADS) multi_norm_kernel(const __grid_constant__ NormParams<CAP> p) {
  __shared__ double red[THREADS / 32];
  const int chunk = blockIdx.x;
  const int ti = find_tensor(p.first_chunk, p.count, chunk);
  const NormItem it = p.item[ti];
  const long long begin = static_cast<long long>(chunk - p.first_chunk[ti]) * p.passes * PASS;
  const bool wide = aligned(it.g, 16);
  double sum = 0.0;
  constexpr int AT_ONCE = 4;                    // passes whose elements are on their way together
  for (int pass = 0; pass < p.passes; pass += AT_ONCE) {
    const long long i0 = begin + static_cast<long long>(pass) * PASS + threadIdx.x * EPT;
    Raw8<DT> raw[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const long long i = i0 + u * PASS;
      const int live = pass + u < p.passes ? live_of(it.n, i) : 0;
      if (wide && live == EPT) raw[u].load(it.g, i);
      else raw[u].load_some(it.g, i, live);
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      float x[EPT];
      raw[u].get(x);
      sum += sum_of_squares(x);
    }
  }
  const double t = block_sum_d(sum, red);
  if (threadIdx.x == 0) p.partial[blockIdx.x] = t;
}

// norm = sqrt of the partial sums; coef = min(1, max_norm / (norm + 1e-6))
__global__ void __launch_bounds__(1024) multi_norm_final_kernel(const double* partial, int n, float max_norm, float* norm, float* coef) {
  __shared__ double red[32];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += partial[i];
  s = block_sum_d(s, red);
  if (threadIdx.x == 0) {
    const float r = static_cast<float>(sqrt(s));
    *norm = r;
    if (coef != nullptr) {
      // (a norm beyond fp32 still has a factor, if a subnormal one: with r = inf it would be 0 and every gradient lost)
      const float q = isinf(r) && !isinf(s) ? static_cast<float>(max_norm / sqrt(s)) : max_norm / (r + 1e-6f);
      *coef = q > 1.0f ? 1.0f : q;              // a NaN stays one
    }
  }
}

// A chunk is as many passes as leave about eight CTAs for each of an SM's eight slots: enough to even out
// the ends of a launch, few enough that looking the tensor up costs nothing.
static int pick_passes(long long total, int sm_count) {
  const long long want = total / (static_cast<long long>(PASS) * sm_count * 64);
  return static_cast<int>(std::max<long long>(1, std::min<long long>(want, 8)));
}
static long long chunks_of(long long n, int passes) { return (n + static_cast<long long>(PASS) * passes - 1) / (static_cast<long long>(PASS) * passes); }

static constexpr long long MAX_CHUNKS = 0x7fffffffll;

template <int W_DT, int G_DT, int ST, int CAP>
static int launch_adamw(const ForgeMultiItem* const* items, int count, int passes, const ForgeMultiArgs& a, cudaStream_t stream) {
  Params<CAP> p;
  long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    const ForgeMultiItem& s = *items[i];
    p.item[i] = Item{s.param, s.grad, s.m, s.v, s.m_scale, s.v_scale, static_cast<long long>(s.numel)};
    p.first_chunk[i] = static_cast<int>(chunks);
    chunks += chunks_of(s.numel, passes);
  }
  if (chunks > MAX_CHUNKS) return fail(FORGE_ERR_SHAPE, "forge_multi_adamw: too many elements for one launch");
  p.first_chunk[count] = static_cast<int>(chunks);
  p.count = count;
  p.passes = passes;
  p.coef = a.grad_coef;
  p.hyper_device = static_cast<const Hyper*>(a.hyper_device);
  p.hyper = make_hyper(a.hyper);
  multi_adamw_kernel<W_DT, G_DT, ST, CAP><<<static_cast<unsigned>(chunks), THREADS, 0, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "multi-tensor AdamW launch: %s", cudaGetErrorString(e));
  return FORGE_OK;
}

template <int W_DT, int G_DT, int CAP>
static int by_state(const ForgeMultiItem* const* items, int count, int passes, const ForgeMultiArgs& a, cudaStream_t s) {
  switch (a.state_mode) {
    case FORGE_ST_F32: return launch_adamw<W_DT, G_DT, ST_F32, CAP>(items, count, passes, a, s);
    case FORGE_ST_BF16: return launch_adamw<W_DT, G_DT, ST_BF16, CAP>(items, count, passes, a, s);
    case FORGE_ST_INT8: return launch_adamw<W_DT, G_DT, ST_INT8, CAP>(items, count, passes, a, s);
    case FORGE_ST_FP8_BLOCK: return launch_adamw<W_DT, G_DT, ST_FP8_BLOCK, CAP>(items, count, passes, a, s);
  }
  return fail(FORGE_ERR_UNSUPPORTED, "forge_multi_adamw: state mode %d is not built", a.state_mode);
}

template <int CAP>
static int by_types(int w, int g, const ForgeMultiItem* const* items, int count, int passes, const ForgeMultiArgs& a, cudaStream_t s) {
  if (w == FORGE_DT_BF16) return g == FORGE_DT_BF16 ? by_state<DT_BF16, DT_BF16, CAP>(items, count, passes, a, s) : by_state<DT_BF16, DT_F32, CAP>(items, count, passes, a, s);
  return g == FORGE_DT_BF16 ? by_state<DT_F32, DT_BF16, CAP>(items, count, passes, a, s) : by_state<DT_F32, DT_F32, CAP>(items, count, passes, a, s);
}

template <int DT>
static int launch_norm(const ForgeNormItem* const* items, int count, int passes, double* partial, long long* used, cudaStream_t stream) {
  NormParams<MAX_TENSORS> p;
  long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    p.item[i] = NormItem{items[i]->grad, static_cast<long long>(items[i]->numel)};
    p.first_chunk[i] = static_cast<int>(chunks);
    chunks += chunks_of(items[i]->numel, passes);
  }
  p.first_chunk[count] = static_cast<int>(chunks);
  p.count = count;
  p.passes = passes;
  p.partial = partial;
  multi_norm_kernel<DT, MAX_TENSORS><<<static_cast<unsigned>(chunks), THREADS, 0, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "multi-tensor norm launch: %s", cudaGetErrorString(e));
  *used = chunks;
  return FORGE_OK;
}

static bool dtype_ok(int d) { return d == FORGE_DT_BF16 || d == FORGE_DT_F32; }

}  // namespace multi
}  // namespace forge

using namespace forge;

extern "C" int forge_multi_adamw(const ForgeMultiArgs* args, void* cuda_stream) {
  if (args == nullptr) return fail(FORGE_ERR_INVALID_ARG, "forge_multi_adamw: args is NULL");
  const ForgeMultiArgs& a = *args;
  if (a.count < 0 || (a.count > 0 && a.items == nullptr)) return fail(FORGE_ERR_INVALID_ARG, "forge_multi_adamw: bad item list");
  if (a.state_mode != FORGE_ST_F32 && a.state_mode != FORGE_ST_BF16 && a.state_mode != FORGE_ST_INT8 && a.state_mode != FORGE_ST_FP8_BLOCK)
    return fail(FORGE_ERR_UNSUPPORTED, "forge_multi_adamw: state mode %d is not built", a.state_mode);
  if (a.hyper_device == nullptr && a.hyper.step < 1) return fail(FORGE_ERR_INVALID_ARG, "step must be >= 1 (got %d)", a.hyper.step);
  if (reinterpret_cast<uintptr_t>(a.grad_coef) % 4 || reinterpret_cast<uintptr_t>(a.hyper_device) % 8)
    return fail(FORGE_ERR_ALIGNMENT, "forge_multi_adamw: grad_coef or hyper_device is not aligned");
  const bool quant = a.state_mode == FORGE_ST_INT8 || a.state_mode == FORGE_ST_FP8_BLOCK;
  const int ses = a.state_mode == FORGE_ST_F32 ? 4 : (a.state_mode == FORGE_ST_BF16 ? 2 : 1);
  long long total = 0;
  for (int i = 0; i < a.count; ++i) {
    const ForgeMultiItem& s = a.items[i];
    if (s.numel < 0) return fail(FORGE_ERR_INVALID_ARG, "forge_multi_adamw: tensor %d has %lld elements", i, (long long)s.numel);
    if (!multi::dtype_ok(s.param_dtype) || !multi::dtype_ok(s.grad_dtype))
      return fail(FORGE_ERR_INVALID_ARG, "forge_multi_adamw: tensor %d has an unknown dtype", i);
    if (s.numel == 0) continue;
    if (s.param == nullptr || s.grad == nullptr || s.m == nullptr || s.v == nullptr || (quant && (s.m_scale == nullptr || s.v_scale == nullptr)))
      return fail(FORGE_ERR_INVALID_ARG, "forge_multi_adamw: tensor %d has a null pointer", i);
    if (reinterpret_cast<uintptr_t>(s.param) % (s.param_dtype == FORGE_DT_BF16 ? 2 : 4) || reinterpret_cast<uintptr_t>(s.grad) % (s.grad_dtype == FORGE_DT_BF16 ? 2 : 4) ||
        reinterpret_cast<uintptr_t>(s.m) % ses || reinterpret_cast<uintptr_t>(s.v) % ses ||
        (quant && (reinterpret_cast<uintptr_t>(s.m_scale) % 4 || reinterpret_cast<uintptr_t>(s.v_scale) % 4)))
      return fail(FORGE_ERR_ALIGNMENT, "forge_multi_adamw: tensor %d is not element-aligned", i);
    total += s.numel;
  }
  if (total == 0) return FORGE_OK;
  const DeviceInfo* di = current_device_info();
  if (di == nullptr) return FORGE_ERR_CUDA;
  const int passes = multi::pick_passes(total, di->sm_count);
  if (total / multi::PASS + a.count > multi::MAX_CHUNKS) return fail(FORGE_ERR_SHAPE, "forge_multi_adamw: %lld elements", total);
  // one launch per combination of types and MAX_TENSORS tensors
  std::vector<const ForgeMultiItem*> list;
  try {
    list.reserve(a.count);
  } catch (...) {
    return fail(FORGE_ERR_INVALID_ARG, "forge_multi_adamw: out of host memory");
  }
  for (int combo = 0; combo < 4; ++combo) {
    const int w = combo & 1, g = combo >> 1;
    list.clear();
    for (int i = 0; i < a.count; ++i)
      if (a.items[i].numel > 0 && a.items[i].param_dtype == w && a.items[i].grad_dtype == g) list.push_back(&a.items[i]);
    for (size_t i = 0; i < list.size(); i += multi::MAX_TENSORS) {
      const int n = static_cast<int>(std::min<size_t>(multi::MAX_TENSORS, list.size() - i));
      cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
      const int rc = n <= multi::FEW_TENSORS ? multi::by_types<multi::FEW_TENSORS>(w, g, list.data() + i, n, passes, a, s)
                                             : multi::by_types<multi::MAX_TENSORS>(w, g, list.data() + i, n, passes, a, s);
      if (rc != FORGE_OK) return rc;
    }
  }
  return FORGE_OK;
}

static long long norm_total(const ForgeNormItem* items, int32_t count) {
  long long total = 0;
  for (int i = 0; i < count; ++i) total += items[i].numel > 0 ? items[i].numel : 0;
  return total;
}

// a chunk of the norm is 1 .. 64 passes long, so that there are never many partial sums
static int norm_passes(long long total) {
  return static_cast<int>(std::max<long long>(1, std::min<long long>(64, total / (static_cast<long long>(multi::PASS) * 148 * 8))));
}

extern "C" size_t forge_multi_norm_scratch_bytes(const ForgeNormItem* items, int32_t count) {
  if (items == nullptr || count <= 0) return 0;
  const int passes = norm_passes(norm_total(items, count));
  long long chunks = 0;
  for (int i = 0; i < count; ++i) chunks += items[i].numel > 0 ? multi::chunks_of(items[i].numel, passes) : 0;
  return static_cast<size_t>(chunks) * sizeof(double);
}

extern "C" int forge_multi_norm(const ForgeNormItem* items, int32_t count, double max_norm, float* norm, float* coef, void* scratch,
                                size_t scratch_bytes, void* cuda_stream) {
  if (count < 0 || (count > 0 && items == nullptr) || norm == nullptr) return fail(FORGE_ERR_INVALID_ARG, "forge_multi_norm: null pointer");
  if (coef != nullptr && !(max_norm > 0.0)) return fail(FORGE_ERR_INVALID_ARG, "forge_multi_norm: max_norm must be positive (got %g)", max_norm);
  for (int i = 0; i < count; ++i) {
    if (items[i].numel < 0 || !multi::dtype_ok(items[i].dtype) || (items[i].numel > 0 && items[i].grad == nullptr))
      return fail(FORGE_ERR_INVALID_ARG, "forge_multi_norm: bad tensor %d", i);
    if (reinterpret_cast<uintptr_t>(items[i].grad) % (items[i].dtype == FORGE_DT_BF16 ? 2 : 4))
      return fail(FORGE_ERR_ALIGNMENT, "forge_multi_norm: tensor %d is not element-aligned", i);
  }
  const size_t need = forge_multi_norm_scratch_bytes(items, count);
  if (need > scratch_bytes || (need > 0 && scratch == nullptr))
    return fail(FORGE_ERR_SCRATCH, "forge_multi_norm needs %zu bytes of scratch (got %zu)", need, scratch_bytes);
  if (reinterpret_cast<uintptr_t>(norm) % 4 || reinterpret_cast<uintptr_t>(coef) % 4)
    return fail(FORGE_ERR_ALIGNMENT, "forge_multi_norm: norm or coef is not aligned");
  if (reinterpret_cast<uintptr_t>(scratch) % sizeof(double)) return fail(FORGE_ERR_ALIGNMENT, "forge_multi_norm: scratch is not 8-byte aligned");
  if (need / sizeof(double) > static_cast<size_t>(multi::MAX_CHUNKS)) return fail(FORGE_ERR_SHAPE, "forge_multi_norm: too many elements");
  const int passes = norm_passes(norm_total(items, count));
  double* partial = static_cast<double*>(scratch);
  long long used = 0;
  std::vector<const ForgeNormItem*> list;
  try {
    list.reserve(count);
  } catch (...) {
    return fail(FORGE_ERR_INVALID_ARG, "forge_multi_norm: out of host memory");
  }
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  for (int dt = 0; dt < 2; ++dt) {
    list.clear();
    for (int i = 0; i < count; ++i)
      if (items[i].numel > 0 && items[i].dtype == dt) list.push_back(&items[i]);
    for (size_t i = 0; i < list.size(); i += multi::MAX_TENSORS) {
      const int n = static_cast<int>(std::min<size_t>(multi::MAX_TENSORS, list.size() - i));
      long long chunks = 0;
      const int rc = dt == FORGE_DT_BF16 ? multi::launch_norm<DT_BF16>(list.data() + i, n, passes, partial + used, &chunks, s)
                                         : multi::launch_norm<DT_F32>(list.data() + i, n, passes, partial + used, &chunks, s);
      if (rc != FORGE_OK) return rc;
      used += chunks;
    }
  }
  multi::multi_norm_final_kernel<<<1, 1024, 0, s>>>(partial, static_cast<int>(used), static_cast<float>(max_norm), norm, coef);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "multi-tensor norm launch: %s", cudaGetErrorString(e));
  return FORGE_OK;
}
