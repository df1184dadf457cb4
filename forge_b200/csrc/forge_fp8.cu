// Products in 8-bit floating point with one fp32 scale for each block of 128, and the quantiser that
// feeds them.
//
//   scale = absmax * fp32(1 / 448) + 1e-12, code = e4m3(x / scale)   over 1 x 128 blocks of a row (activations,
//   gradients) or 128 x 128 blocks (weights; their transpose has the transposed scales)
//   Y[m, n] = sum over kb of sx[m, kb] sw[n / 128, kb] * sum over the block's k of xq[m, k] wq[n, k]
//
// The inner sums are tensor-core products of 128 terms; the outer sum is held in fp32 registers.
#include <algorithm>
#include <atomic>

#include "forge_host.h"
#include "forge_ptx.cuh"

namespace forge {
namespace fp8 {

// ---------------------------------------------------------------------------------------------
// quantiser
// ---------------------------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ void load8(const uint8_t* p, int live, bool vec, float (&x)[8]) {
  if constexpr (DT == DT_BF16) {
    if (vec) {
      const uint4 q = *reinterpret_cast<const uint4*>(p);
      const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[2 * k] = __uint_as_float(u[k] << 16);
        x[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = k < live ? bf16_bits_to_float(reinterpret_cast<const uint16_t*>(p)[k]) : 0.0f;
    }
  } else {
    if (vec) {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = k < live ? reinterpret_cast<const float*>(p)[k] : 0.0f;
    }
  }
}

__device__ __forceinline__ float absmax8(const float (&x)[8]) {
  float m = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(x[k]));
  return m;
}

__device__ __forceinline__ uint2 codes8(const float (&x)[8], float scale, float rscale) {
  const float2 ns = make_float2(-scale, -scale), rs = make_float2(rscale, rscale);
  uint32_t o[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float2 a = div2_by_rcp(make_float2(x[4 * j], x[4 * j + 1]), ns, rs);
    const float2 b = div2_by_rcp(make_float2(x[4 * j + 2], x[4 * j + 3]), ns, rs);
    o[j] = e4m3x2_code_bits(a.x, a.y) | (e4m3x2_code_bits(b.x, b.y) << 16);
  }
  return make_uint2(o[0], o[1]);
}

struct QuantParams {
  const uint8_t* x;
  uint8_t* q;
  uint8_t* qt;                // transposed codes (C, R), or NULL (128 x 128 blocks only)
  float* scale;               // (R / block_rows, C / 128)
  float* scale_t;             // (C / 128, R / 128), with qt
  long long rows, cols, ld_x, ld_q, ld_qt;
};

// programmatic dependent launch: the kernel that follows may start / wait for the one before and see what it wrote
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// 1 x 128 blocks: sixteen lanes of eight columns each; a warp takes two neighbouring blocks of a row
template <int DT>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantParams p) {
  constexpr int ES = DT == DT_BF16 ? 2 : 4;
  allow_next();
  const int lane = threadIdx.x & 31;
  const long long cb = (p.cols + 127) / 128, pairs = (cb + 1) / 2;
  const long long unit = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const long long row = unit / pairs;
  if (row >= p.rows) return;
  const long long col = (unit % pairs) * 256 + lane * 8;
  const long long left = p.cols - col;
  const int live = left >= 8 ? 8 : (left > 0 ? static_cast<int>(left) : 0);
  const uint8_t* src = p.x + (row * p.ld_x + col) * ES;
  float x[8];
  load8<DT>(src, live, live == 8 && (reinterpret_cast<uintptr_t>(src) & 15) == 0, x);
  float m = absmax8(x);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float scale = block_scale<448>(m);
  const uint2 c = codes8(x, scale, f_rcp(scale));
  uint8_t* dst = p.q + row * p.ld_q + col;
  if (live == 8 && (reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
    *reinterpret_cast<uint2*>(dst) = c;
  } else {
    for (int k = 0; k < live; ++k) dst[k] = static_cast<uint8_t>((k < 4 ? c.x : c.y) >> (8 * (k & 3)));
  }
  if ((lane & 15) == 0 && live > 0) p.scale[row * cb + col / 128] = scale;
}

// eight consecutive elements as they lie in memory
template <int DT>
struct Raw8;
template <>
struct Raw8<DT_BF16> {
  uint4 q;
  __device__ __forceinline__ void load(const uint8_t* p, int live, bool vec) {
    if (vec) {
      q = *reinterpret_cast<const uint4*>(p);
    } else {
      uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < live) u[k >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[k]) << (16 * (k & 1));
      q = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
  // two at a time; a NaN is passed over, as by fmaxf
  __device__ __forceinline__ float absmax() const {
    auto as2 = [](uint32_t u) { u &= 0x7fff7fffu; return *reinterpret_cast<const __nv_bfloat162*>(&u); };
    const __nv_bfloat162 m = __hmax2(__hmax2(as2(q.x), as2(q.y)), __hmax2(as2(q.z), as2(q.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = __uint_as_float(u[k] << 16);
      x[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
    }
  }
};
template <>
struct Raw8<DT_F32> {
  float x[8];
  __device__ __forceinline__ void load(const uint8_t* p, int live, bool vec) { load8<DT_F32>(p, live, vec, x); }
  __device__ __forceinline__ float absmax() const { return absmax8(x); }
  __device__ __forceinline__ void get(float (&y)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = x[k];
  }
};

// 128 x 128 blocks: one CTA per block, a thread holds 8 x 8 elements, all of its loads in flight at once.  The transposed
// codes go through shared memory: four 4 x 4 byte transpositions in registers, then rows of 128 bytes whose 8-byte pieces
// are exchanged by row / 8, so that the sixteen threads that write one row each hit different banks.  14336 x 4096 bf16, both
// ways round: 39 us (6.0 TB/s) with five CTAs per SM, 54 with three, 71 with the elements held in fp32.
template <int DT>
__global__ void __launch_bounds__(256, DT == DT_BF16 ? 5 : 2) quantize_blocks_kernel(const QuantParams p) {
  constexpr int ES = DT == DT_BF16 ? 2 : 4;
  __shared__ __align__(16) uint8_t tile[128 * 128];
  __shared__ float red[8];
  const long long cb = (p.cols + 127) / 128, rb = (p.rows + 127) / 128;
  const long long bi = blockIdx.x / cb, bj = blockIdx.x % cb;
  const int tc = (threadIdx.x & 15) * 8, tr = (threadIdx.x >> 4) * 8;
  const long long col = bj * 128 + tc, row0 = bi * 128 + tr;
  const long long left = p.cols - col;
  const int live = left >= 8 ? 8 : (left > 0 ? static_cast<int>(left) : 0);
  Raw8<DT> x[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const uint8_t* src = p.x + ((row0 + r) * p.ld_x + col) * ES;
    const int n = row0 + r < p.rows ? live : 0;
    x[r].load(src, n, n == 8 && (reinterpret_cast<uintptr_t>(src) & 15) == 0);
  }
  float m = 0.0f;
#pragma unroll
  for (int r = 0; r < 8; ++r) m = fmaxf(m, x[r].absmax());
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, red[i]);
  const float scale = block_scale<448>(m), rscale = f_rcp(scale);
  uint2 c[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    float y[8];
    x[r].get(y);
    c[r] = codes8(y, scale, rscale);
    if (row0 + r >= p.rows) continue;
    uint8_t* dst = p.q + (row0 + r) * p.ld_q + col;
    if (live == 8 && (reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
      *reinterpret_cast<uint2*>(dst) = c[r];
    } else {
      for (int k = 0; k < live; ++k) dst[k] = static_cast<uint8_t>((k < 4 ? c[r].x : c[r].y) >> (8 * (k & 3)));
    }
  }
  if (threadIdx.x == 0) {
    p.scale[bi * cb + bj] = scale;
    if (p.qt != nullptr) p.scale_t[bj * rb + bi] = scale;
  }
  if (p.qt == nullptr) return;
  // column k of the 8 x 8 piece = row tc + k of the transposed tile, bytes tr .. tr + 7
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t t[2][4];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const uint32_t a0 = h ? c[4 * g].y : c[4 * g].x, a1 = h ? c[4 * g + 1].y : c[4 * g + 1].x;
      const uint32_t a2 = h ? c[4 * g + 2].y : c[4 * g + 2].x, a3 = h ? c[4 * g + 3].y : c[4 * g + 3].x;
      const uint32_t p01l = __byte_perm(a0, a1, 0x5140), p01h = __byte_perm(a0, a1, 0x7362);
      const uint32_t p23l = __byte_perm(a2, a3, 0x5140), p23h = __byte_perm(a2, a3, 0x7362);
      t[g][0] = __byte_perm(p01l, p23l, 0x5410);
      t[g][1] = __byte_perm(p01l, p23l, 0x7632);
      t[g][2] = __byte_perm(p01h, p23h, 0x5410);
      t[g][3] = __byte_perm(p01h, p23h, 0x7632);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)      // rows tc .. tc + 7 share tc / 8
      *reinterpret_cast<uint2*>(&tile[(tc + 4 * h + k) * 128 + (((tr ^ tc) & 0x78))]) = make_uint2(t[0][k], t[1][k]);
  }
  __syncthreads();
  const long long trow0 = bj * 128, tcol0 = bi * 128;
  const bool whole = tcol0 + 128 <= p.rows && (p.ld_qt & 15) == 0 && (reinterpret_cast<uintptr_t>(p.qt) & 15) == 0;
#pragma unroll
  for (int i = threadIdx.x; i < 128 * 8; i += 256) {
    const int r = i >> 3, pc = (i & 7) * 16, swap = r & 0x78;
    if (trow0 + r >= p.cols) continue;
    uint8_t* dst = p.qt + (trow0 + r) * p.ld_qt + tcol0 + pc;
    uint4 v = *reinterpret_cast<const uint4*>(&tile[r * 128 + ((pc ^ swap) & 0x70)]);
    if (swap & 8) v = make_uint4(v.z, v.w, v.x, v.y);
    if (whole) {
      *reinterpret_cast<uint4*>(dst) = v;
    } else {
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (tcol0 + pc + k < p.rows) dst[k] = static_cast<uint8_t>(u[k >> 2] >> (8 * (k & 3)));
    }
  }
}

// ---------------------------------------------------------------------------------------------
// product, one CTA per tile of 128 weight rows x NT tokens
// ---------------------------------------------------------------------------------------------
// The weight's rows are the rows of the accumulator (M = 128) and the tokens its columns, so that a few
// tokens cost a narrow product and the tile count does not fall with their number.  K is cut over the CTAs of
// a cluster where the tiles alone would leave SMs idle; the parts meet in distributed shared memory and are
// added in rank order.
struct Params {
  const float* sx;
  const float* sw;
  __nv_bfloat16* y;
  long long sx_row, sx_col, sw_row, sw_col, ld_y;   // strides of the scales in elements
  int M, N, KB;                                     // tokens, weight rows, K blocks
  int tiles_m;
  int split;
  int wide;                                         // rows of y are 16-byte aligned
  int early;                                        // launched while the kernel that writes X's codes may still run
  int* status;
};

enum : int { ERR_OP_EMPTY = 221, ERR_OP_FULL = 222, ERR_ACC_EMPTY = 223, ERR_ACC_FULL = 224, ERR_SC_EMPTY = 225, ERR_SC_FULL = 226 };
constexpr int SC_SLOTS = 8;                         // K blocks whose scales are in shared memory
constexpr int BK = 128;                             // bytes = elements
constexpr int A_BYTES = 128 * BK;
constexpr int ACC_BUFS = 4;
constexpr int THREADS = 384;                        // producer, MMA, two idle warps; eight epilogue warps

template <int NT>
struct Cfg {
  static constexpr int B_BYTES = NT * BK;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  // up to 64 tokens two CTAs share an SM (112 KB each); 128 take an SM's tensor memory alone
  static constexpr int STAGES = NT == 128 ? 6 : (NT == 64 ? 3 : (NT == 32 ? 4 : 5));
  // what the cluster's CTAs send for this CTA's tokens: at most NT + split - 1 rows of 128 sums.  With 128 tokens there is
  // no room for it beside the stages: it takes their place, once all CTAs of the cluster are done with theirs.
  static constexpr bool SHARED_RECV = NT == 128;
  static constexpr int RECV = (NT + 8) * 128 * 4;
  static constexpr int SMEM = 1024 + STAGES * STAGE + (SHARED_RECV ? 0 : RECV);      // + alignment slack; control words are static
  static constexpr int TMEM_COLS = ACC_BUFS * NT;
  static constexpr int MIN_CTAS = NT == 128 ? 1 : 2;
};

// 32 lanes x 8 consecutive columns
__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}

// the first barrier phase of a cluster: everybody has started
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster(uint32_t cluster_addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// instruction descriptor of kind::f8f6f4, e4m3 x e4m3 -> f32, both operands K-major
__host__ __device__ constexpr uint32_t make_idesc_e4m3(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t u;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
  return u;
}

constexpr int MAX_STAGES = 6;
struct Ctrl {
  uint64_t full[MAX_STAGES];
  uint64_t empty[MAX_STAGES];
  uint64_t acc_full[ACC_BUFS];
  uint64_t acc_empty[ACC_BUFS];
  uint64_t sc_full[SC_SLOTS];
  uint64_t sc_empty[SC_SLOTS];
  uint32_t tmem_base;
  int abort_word;
};

// The scales' products sx sw of one K block after the other, formed by two warps (64 threads) and handed to the
// epilogue through slots of W floats: loaded where they are used, they cost the epilogue a memory latency per K block.
// Four blocks are asked for at a time.  value(i, kb): what thread-slot i holds for block kb.
template <int W, typename F>
__device__ __forceinline__ bool feed_scales(float (*sc)[W], uint64_t* full, uint64_t* empty, int& it, int kb0, int kb1, volatile int* abort_word,
                                            F&& value) {
  const int t = threadIdx.x - 64;
  constexpr int PER = (W + 63) / 64;
  for (int kb = kb0; kb < kb1; kb += 4) {
    float v[4][PER];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < PER; ++i) v[u][i] = kb + u < kb1 && t + 64 * i < W ? value(t + 64 * i, kb + u) : 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (kb + u >= kb1) break;
      const int slot = it % SC_SLOTS;
      bool ok = mbar_wait(&empty[slot], ((it / SC_SLOTS) & 1) ^ 1, abort_word, ERR_SC_EMPTY);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return false;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (t + 64 * i < W) sc[slot][t + 64 * i] = v[u][i];
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(&full[slot]);
      ++it;
    }
  }
  return true;
}

template <int NT>
__global__ void __launch_bounds__(THREADS, Cfg<NT>::MIN_CTAS)
fp8_product_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Params p) {
  using C = Cfg<NT>;
  static_assert(C::STAGES <= MAX_STAGES, "one barrier pair per stage");
  __shared__ Ctrl ctrl;
  __shared__ __align__(16) float sc[SC_SLOTS][NT];
  extern __shared__ uint8_t smem_raw[];
  uint8_t* data = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_word = &ctrl.abort_word;
  const int rank = blockIdx.x % p.split;
  const int tile = blockIdx.x / p.split;
  // consecutive tiles share the weight's rows
  const int m0 = (tile % p.tiles_m) * NT, n0 = (tile / p.tiles_m) * 128;
  const int per = (p.KB + p.split - 1) / p.split;
  const int kb0 = min(p.KB, rank * per), kb1 = min(p.KB, kb0 + per);
  // where the sums of this CTA's tokens are: its own, if K is not cut, lie at the start of the stages (see below)
  float* recv = reinterpret_cast<float*>(p.split == 1 ? data : data + (C::SHARED_RECV ? NT * 512 : C::STAGES * C::STAGE));
  static_assert(!C::SHARED_RECV || NT * 512 + C::RECV <= C::STAGES * C::STAGE, "the sums fit where the stages were");
  // the tile's tokens, and how many of them each CTA of the cluster writes
  const int tokens = min(NT, p.M - m0), share = (tokens + p.split - 1) / p.split;
  // (waited for before anything is sent to another CTA: it has started)
  if (p.split > 1 && !C::SHARED_RECV) cluster_arrive_relaxed();
  const uint64_t pol_w = p.tiles_m > 1 ? policy_evict_normal() : policy_evict_first();

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) { mbar_init(&ctrl.full[i], 1); mbar_init(&ctrl.empty[i], 1); }
    for (int i = 0; i < ACC_BUFS; ++i) { mbar_init(&ctrl.acc_full[i], 1); mbar_init(&ctrl.acc_empty[i], 8); }
    for (int i = 0; i < SC_SLOTS; ++i) { mbar_init(&ctrl.sc_full[i], 2); mbar_init(&ctrl.sc_empty[i], 8); }
    ctrl.abort_word = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
    // the weight's first stages are on their way before the rest of the CTA is set up, and (early) before the tokens'
    // codes are known to be there
    for (int i = 0; i < C::STAGES && kb0 + i < kb1; ++i) {
      mbar_expect_tx(&ctrl.full[i], C::STAGE);
      tma_load_2d(data + i * C::STAGE, &tm_w, &ctrl.full[i], (kb0 + i) * BK, n0, pol_w);
    }
  }
  if (warp == 1) {
    tmem_alloc(&ctrl.tmem_base, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = ctrl.tmem_base;

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t pol_x = policy_evict_last();
      if (p.early) wait_for_previous();
      for (int i = 0; i < C::STAGES && kb0 + i < kb1; ++i)
        tma_load_2d(data + i * C::STAGE + A_BYTES, &tm_x, &ctrl.full[i], (kb0 + i) * BK, m0, pol_x);
      for (int kb = kb0 + C::STAGES, it = C::STAGES; kb < kb1; ++kb, ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(&ctrl.empty[s], ((it / C::STAGES) & 1) ^ 1, abort_word, ERR_OP_EMPTY)) break;
        uint8_t* a = data + s * C::STAGE;
        mbar_expect_tx(&ctrl.full[s], C::STAGE);
        tma_load_2d(a, &tm_w, &ctrl.full[s], kb * BK, n0, pol_w);
        tma_load_2d(a + A_BYTES, &tm_x, &ctrl.full[s], kb * BK, m0, pol_x);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_e4m3(128, NT);
      for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {
        const int s = it % C::STAGES, b = it % ACC_BUFS;
        if (!mbar_wait(&ctrl.acc_empty[b], ((it / ACC_BUFS) & 1) ^ 1, abort_word, ERR_ACC_EMPTY)) break;
        if (!mbar_wait(&ctrl.full[s], (it / C::STAGES) & 1, abort_word, ERR_OP_FULL)) break;
        tc_fence_after();
        const uint32_t a_addr = smem_u32(data + s * C::STAGE), b_addr = a_addr + A_BYTES;
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)
          umma_f8(tmem_base + b * NT, make_smem_desc_sw128(a_addr + k * 32, 16, 1024), make_smem_desc_sw128(b_addr + k * 32, 16, 1024),
                  idesc, k > 0 ? 1u : 0u);
        umma_commit(&ctrl.empty[s]);
        umma_commit(&ctrl.acc_full[b]);
      }
    }
  } else if (warp < 4) {
    if (p.early) wait_for_previous();
    const float* swp = p.sw + static_cast<long long>(n0 / 128) * p.sw_row;
    int it = 0;
    feed_scales<NT>(sc, ctrl.sc_full, ctrl.sc_empty, it, kb0, kb1, abort_word, [&](int i, int kb) {
      return m0 + i < p.M ? p.sx[static_cast<long long>(m0 + i) * p.sx_row + kb * p.sx_col] * swp[kb * p.sw_col] : 0.0f;
    });
  } else {
    // two warpgroups, each with half of the tokens
    constexpr int NC = NT / 2;
    const int quarter = warp & 3, c0 = ((warp - 4) >> 2) * NC;
    float acc[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[j] = 0.0f;
    for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {
      const int b = it % ACC_BUFS, slot = it % SC_SLOTS;
      bool ok = mbar_wait(&ctrl.sc_full[slot], (it / SC_SLOTS) & 1, abort_word, ERR_SC_FULL);
      ok = mbar_wait(&ctrl.acc_full[b], (it / ACC_BUFS) & 1, abort_word, ERR_ACC_FULL) && ok;
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      constexpr int STEP = NC < 32 ? NC : 32;
#pragma unroll
      for (int c = 0; c < NC; c += STEP) {
        uint32_t r[STEP];
        const uint32_t ta = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + b * NT + c0 + c;
        if constexpr (STEP == 8) tmem_ld_32x8(ta, r);
        else if constexpr (STEP == 16) tmem_ld_32x16(ta, r);
        else tmem_ld_32x32(ta, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < STEP; j += 4) {
          const float4 s4 = *reinterpret_cast<const float4*>(&sc[slot][c0 + c + j]);
          const float2 lo = ffma2(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), make_float2(s4.x, s4.y),
                                  make_float2(acc[c + j], acc[c + j + 1]));
          const float2 hi = ffma2(make_float2(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])), make_float2(s4.z, s4.w),
                                  make_float2(acc[c + j + 2], acc[c + j + 3]));
          acc[c + j] = lo.x; acc[c + j + 1] = lo.y; acc[c + j + 2] = hi.x; acc[c + j + 3] = hi.y;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&ctrl.acc_empty[b]);
        mbar_arrive(&ctrl.sc_empty[slot]);
      }
    }
    // Every product has completed (the last accumulator was signalled after all of them), so this CTA's operand stages are
    // free: its sums go there as [token][weight row].
    float* part = reinterpret_cast<float*>(data);
    const int r = quarter * 32 + lane;
#pragma unroll
    for (int j = 0; j < NC; ++j) part[(c0 + j) * 128 + r] = acc[j];
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  const bool failed = *abort_word != 0;
  if (failed) {
    // copies of this CTA may still be in flight: let them land before its shared memory goes
    const long long t0 = clock64();
    while (clock64() - t0 < 400000) __nanosleep(1000);
    if (threadIdx.x == 0 && p.status != nullptr) atomicCAS(p.status, 0, *abort_word);
  }
  __syncwarp();
  if (p.split > 1) {
    if (C::SHARED_RECV) cluster_arrive_relaxed();       // (now it means: this CTA no longer needs its stages)
    cluster_wait();
    // each token's sums go to the CTA that adds them up and writes them, row [this rank][token] there
    const float* part = reinterpret_cast<const float*>(data);
    for (int j = warp; j < tokens; j += THREADS / 32) {
      const float4 v = *reinterpret_cast<const float4*>(part + j * 128 + lane * 4);
      st_cluster(map_to_cta(smem_u32(recv + (rank * share + j % share) * 128 + lane * 4), j / share), v);
    }
    __syncwarp();
    cluster_sync_all();                                  // all sums have arrived; nothing is sent after this
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
  // this CTA's tokens: eight weight rows per lane, sixteen lanes per token, the parts added in the order of the ranks
  const int j1 = min(tokens - rank * share, share);
  const int r8 = (threadIdx.x & 15) * 8;
  for (int j = threadIdx.x >> 4; j < j1 && !failed; j += THREADS / 16) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.0f;
    for (int q = 0; q < p.split; ++q) {
      const float4 a = *reinterpret_cast<const float4*>(recv + (q * share + j) * 128 + r8);
      const float4 c = *reinterpret_cast<const float4*>(recv + (q * share + j) * 128 + r8 + 4);
      v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
      v[4] += c.x; v[5] += c.y; v[6] += c.z; v[7] += c.w;
    }
    __nv_bfloat16* dst = p.y + static_cast<long long>(m0 + rank * share + j) * p.ld_y + n0 + r8;
    if (p.wide && n0 + r8 + 8 <= p.N) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (n0 + r8 + k < p.N) dst[k] = __float2bfloat16_rn(v[k]);
    }
  }
}

// sets a kernel's shared-memory limit once per device
template <typename F>
static int allow_smem(F* fn, int bytes, std::atomic<uint64_t>& done, int device) {
  const uint64_t bit = 1ull << (device & 63);
  if (done.load(std::memory_order_relaxed) & bit) return FORGE_OK;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "fp8 product: shared memory attribute: %s", cudaGetErrorString(e));
  done.fetch_or(bit, std::memory_order_relaxed);
  return FORGE_OK;
}

// a launch of clusters; `early`: it may begin before the kernel in front of it in the stream has ended
struct Launch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  Launch(int ctas, int threads, int smem, int cluster, bool early, cudaStream_t stream) {
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = early ? 2 : 1;
  }
};

template <int NT>
static int launch_product(const CUtensorMap& tw, const CUtensorMap& tx, const Params& p, int ctas, int device, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  auto* fn = fp8_product_kernel<NT>;
  const int rc = allow_smem(fn, Cfg<NT>::SMEM, done, device);
  if (rc != FORGE_OK) return rc;
  Launch l(ctas, THREADS, Cfg<NT>::SMEM, p.split, p.early, stream);
  cudaError_t e = cudaLaunchKernelEx(&l.cfg, fn, tw, tx, p);
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "fp8 product launch: %s", cudaGetErrorString(e));
  return FORGE_OK;
}

// ---------------------------------------------------------------------------------------------
// product, a pair of CTAs per tile of 256 tokens x 256 (or 128) weight rows
// ---------------------------------------------------------------------------------------------
// For many tokens.  The pair's MMA (cta_group::2) reads each CTA's 128 tokens and half of the tile's weight rows from that
// CTA's shared memory, so a CTA stages 32 KB per K block for 128 x 256 x 128 products, half of what single CTAs of
// 128 x 128 stage per product.  Tokens are the accumulator's
// rows: a thread's scale is then one number per K block, sx[its token, kb] sw[its 128 weight rows, kb].  Every K block
// goes to an accumulator of its own (two of 256 columns, four of 128); eight warps add it, scaled, to 128 fp32 registers each thread
// while the tensor cores work on the next one.
//
// 4096 x 14336 x 4096: 228 us, 2.1 PFLOP/s.  The MMAs alone, on operands that stay in place, take 156 us; with the copies of
// the operands 194 (four or five stages alike: the copies and the MMAs' operand reads share the shared memory's
// bandwidth); the rest is the hand-over of an accumulator per K block.  Four column groups of 64 instead of two of 128
// (less work per warp, but 112 registers are too few): 245 to 270 us; 32 columns per fetch instead of 16: 233 us.
namespace pair {
constexpr int STAGES = 5;
constexpr int GROUPS = 2;                             // epilogue warpgroups, each with half of the columns
constexpr int THREADS = 128 + GROUPS * 128;           // producer, MMA, two idle warps; the epilogue
constexpr int TMEM_COLS = 512;

// W: weight rows of a tile
template <int W>
struct Cfg {
  static constexpr int B_BYTES = W / 2 * BK;          // each CTA's half of them
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int COLS = W / GROUPS;
  static constexpr int ACCS = TMEM_COLS / W;          // accumulators
  static constexpr int SMEM = 1024 + STAGES * STAGE + 128 * W * 2;
};
constexpr int MAX_ACCS = 4;

struct Ctrl {
  uint64_t full[STAGES];
  uint64_t empty[STAGES];
  uint64_t acc_full[MAX_ACCS];
  uint64_t acc_empty[MAX_ACCS];
  uint32_t tmem_base;
  int abort_word;
};

__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

constexpr int STEP = 16;                              // columns fetched from tensor memory at a time
// acc += s * STEP columns of the accumulator
template <int N>
__device__ __forceinline__ void add_scaled(float2 (&acc)[N], int at, const uint32_t (&r)[STEP], float s) {
  const float2 s2 = make_float2(s, s);
#pragma unroll
  for (int j = 0; j < STEP / 2; ++j)
    acc[at + j] = ffma2(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), s2, acc[at + j]);
}

template <int W>
__global__ void __launch_bounds__(THREADS, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                const __grid_constant__ CUtensorMap tm_out, const Params p) {
  constexpr int STAGE = Cfg<W>::STAGE, COLS = Cfg<W>::COLS, ACCS = Cfg<W>::ACCS;
  static_assert(ACCS <= MAX_ACCS, "one barrier pair per accumulator");
  __shared__ Ctrl ctrl;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* data = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* out_buf = data + STAGES * STAGE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_word = &ctrl.abort_word;
  const uint32_t cta_rank = cluster_ctarank();
  const int first_tile = static_cast<int>(cluster_id_x()), tile_step = static_cast<int>(gridDim.x) / 2;
  const int num_tiles = p.tiles_m * ((p.N + W - 1) / W);

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) { mbar_init(&ctrl.full[i], 1); mbar_init(&ctrl.empty[i], 1); }
    for (int i = 0; i < ACCS; ++i) { mbar_init(&ctrl.acc_full[i], 1); mbar_init(&ctrl.acc_empty[i], 8 * GROUPS); }
    ctrl.abort_word = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&ctrl.tmem_base, TMEM_COLS);
    tmem_relinquish_pair();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
    if (p.wide) prefetch_tmap(&tm_out);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();          // the peer's barriers exist before anyone signals them
  tc_fence_after();
  const uint32_t tmem_base = ctrl.tmem_base;

  if (warp < 4) {
    setmaxnreg_dec<40>();
    if (warp == 0 && lane == 0) {
      const uint64_t pol = policy_evict_normal();
      if (p.early) wait_for_previous();
      int it = 0;
      for (int tile = first_tile; tile < num_tiles; tile += tile_step) {
        const int m0 = (tile % p.tiles_m) * 256 + static_cast<int>(cta_rank) * 128;
        const int n0 = (tile / p.tiles_m) * W + static_cast<int>(cta_rank) * (W / 2);
        for (int kb = 0; kb < p.KB; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&ctrl.empty[s], ((it / STAGES) & 1) ^ 1, abort_word, ERR_OP_EMPTY)) goto done;
          uint8_t* a = data + s * STAGE;
          // both CTAs' copies count on the leader's barrier, which expects the bytes of both
          const uint32_t full_leader = map_to_cta(smem_u32(&ctrl.full[s]), 0);
          if (cta_rank == 0) mbar_expect_tx(&ctrl.full[s], 2 * STAGE);
          tma_load_2d_pair(a, &tm_x, full_leader, kb * BK, m0, pol);
          tma_load_2d_pair(a + A_BYTES, &tm_w, full_leader, kb * BK, n0, pol);
        }
      }
    } else if (warp == 1 && lane == 0 && cta_rank == 0) {
      constexpr uint32_t idesc = make_idesc_e4m3(256, W);
      int it = 0;
      for (int tile = first_tile; tile < num_tiles; tile += tile_step) {
        for (int kb = 0; kb < p.KB; ++kb, ++it) {
          const int s = it % STAGES, b = it % ACCS;
          if (!mbar_wait(&ctrl.acc_empty[b], ((it / ACCS) & 1) ^ 1, abort_word, ERR_ACC_EMPTY)) goto done;
          if (!mbar_wait(&ctrl.full[s], (it / STAGES) & 1, abort_word, ERR_OP_FULL)) goto done;
          tc_fence_after();
          const uint32_t a_addr = smem_u32(data + s * STAGE), b_addr = a_addr + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            umma_f8_pair(tmem_base + b * W, make_smem_desc_sw128(a_addr + k * 32, 16, 1024),
                         make_smem_desc_sw128(b_addr + k * 32, 16, 1024), idesc, k > 0 ? 1u : 0u);
          umma_commit_pair(&ctrl.empty[s], 3);
          umma_commit_pair(&ctrl.acc_full[b], 3);
        }
      }
    }
  } else {
    setmaxnreg_inc<232>();     // 256 x 232 + 128 x 40 = 384 x 168, the registers of the launch
    const int quarter = warp & 3, group = (warp - 4) >> 2;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + group * COLS;
    uint8_t* stage = out_buf + (group * 4 + quarter) * (32 * COLS * 2);          // boxes of 32 rows x 64 columns
    const uint32_t empty_leader = map_to_cta(smem_u32(&ctrl.acc_empty[0]), 0);
    const uint64_t pol = policy_evict_normal();
    if (p.early) wait_for_previous();
    int it = 0;
    for (int tile = first_tile; tile < num_tiles; tile += tile_step) {
      const int row = (tile % p.tiles_m) * 256 + static_cast<int>(cta_rank) * 128 + quarter * 32 + lane;
      const int col = (tile / p.tiles_m) * W + group * COLS;
      const bool live = row < p.M && col < p.N;
      const float* sx = p.sx + static_cast<long long>(live ? row : 0) * p.sx_row;
      const float* sw = p.sw + static_cast<long long>(live ? col / 128 : 0) * p.sw_row;
      // Two blocks ahead, and multiplied only when the product is wanted.  (Four at a time in a loop unrolled by four, or
      // fed by the two idle warps through shared memory: 250 and 255 us instead of 228 for 4096 x 14336 x 4096.)
      float2 s0 = make_float2(0.0f, 0.0f), s1 = s0;
      if (live) {
        s0 = make_float2(*sx, *sw);
        if (p.KB > 1) s1 = make_float2(sx[p.sx_col], sw[p.sw_col]);
        sx += 2 * p.sx_col;
        sw += 2 * p.sw_col;
      }
      float2 acc[COLS / 2];
#pragma unroll
      for (int j = 0; j < COLS / 2; ++j) acc[j] = make_float2(0.0f, 0.0f);
#pragma unroll 1
      for (int kb = 0; kb < p.KB; ++kb, ++it) {
        const int b = it % ACCS;
        const float s = s0.x * s0.y;
        s0 = s1;
        if (live && kb + 2 < p.KB) {
          s1 = make_float2(*sx, *sw);
          sx += p.sx_col;
          sw += p.sw_col;
        }
        bool ok = mbar_wait(&ctrl.acc_full[b], (it / ACCS) & 1, abort_word, ERR_ACC_FULL);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) goto done;
        tc_fence_after();
        const uint32_t ta = lane_addr + b * W;
        // two fetches in flight: each is asked for again as soon as its columns have been added
        uint32_t r0[STEP], r1[STEP];
        tmem_ld_32x16(ta, r0);
        tmem_ld_32x16(ta + STEP, r1);
#pragma unroll
        for (int c = 0; c < COLS; c += 2 * STEP) {
          tmem_ld_wait();
          if (c + 2 * STEP >= COLS) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(empty_leader + b * 8);
          }
          add_scaled(acc, c / 2, r0, s);
          if (c + 2 * STEP < COLS) tmem_ld_32x16(ta + c + 2 * STEP, r0);
          add_scaled(acc, c / 2 + STEP / 2, r1, s);
          if (c + 2 * STEP < COLS) tmem_ld_32x16(ta + c + 3 * STEP, r1);
        }
      }
      if (p.wide) {
        if (lane == 0) tma_store_wait_read<0>();                       // the last tile's store has left the staging tile
        __syncwarp();
#pragma unroll
        for (int j = 0; j < COLS / 8; ++j) {
          // columns 8j .. 8j + 7: box j / 8, 16-byte piece j % 8 of the row's 128 bytes
          uint8_t* dst = stage + (j >> 3) * 4096 + lane * 128;
          *reinterpret_cast<uint4*>(dst + (((j & 7) ^ (lane & 7)) << 4)) =
              make_uint4(pack_bf16(acc[4 * j].x, acc[4 * j].y), pack_bf16(acc[4 * j + 1].x, acc[4 * j + 1].y),
                         pack_bf16(acc[4 * j + 2].x, acc[4 * j + 2].y), pack_bf16(acc[4 * j + 3].x, acc[4 * j + 3].y));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (row < p.M) {                                             // lane 0: the warp's first row
#pragma unroll
            for (int c = 0; c < COLS; c += 64)
              if (col + c < p.N) tma_store_2d(&tm_out, stage + c * 64, col + c, row, pol);
          }
          tma_store_commit();
        }
        __syncwarp();
      } else if (live) {
        __nv_bfloat16* dst = p.y + static_cast<long long>(row) * p.ld_y + col;
#pragma unroll
        for (int j = 0; j < COLS; ++j)
          if (col + j < p.N) dst[j] = __float2bfloat16_rn(j & 1 ? acc[j / 2].y : acc[j / 2].x);
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
  }

done:
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_word != 0) {
    const long long t0 = clock64();
    while (clock64() - t0 < 400000) __nanosleep(1000);
    if (threadIdx.x == 0 && p.status != nullptr) atomicCAS(p.status, 0, *abort_word);
    __syncthreads();
  }
  cluster_sync_all();          // the peer's shared memory and barriers stay valid until both are done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

template <int W>
static int launch(const CUtensorMap& tx, const CUtensorMap& tw, const CUtensorMap& ty, const Params& p, int pairs, int device,
                  cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const int rc = allow_smem(fp8_pair_kernel<W>, Cfg<W>::SMEM, done, device);
  if (rc != FORGE_OK) return rc;
  Launch l(2 * pairs, THREADS, Cfg<W>::SMEM, 2, p.early, stream);
  cudaError_t e = cudaLaunchKernelEx(&l.cfg, fp8_pair_kernel<W>, tx, tw, ty, p);
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "fp8 product launch: %s", cudaGetErrorString(e));
  return FORGE_OK;
}
}  // namespace pair

}  // namespace fp8
}  // namespace forge

using namespace forge;

extern "C" int forge_fp8_quantize(const ForgeFp8QuantizeArgs* args, void* cuda_stream) {
  if (args == nullptr) return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_quantize: args is NULL");
  const ForgeFp8QuantizeArgs& a = *args;
  if (a.rows < 0 || a.cols < 0) return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_quantize: negative dimension");
  if (a.dtype != FORGE_DT_BF16 && a.dtype != FORGE_DT_F32) return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_quantize: unknown dtype %d", a.dtype);
  if (a.block_rows != 1 && a.block_rows != 128) return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_quantize: block_rows must be 1 or 128 (got %d)", a.block_rows);
  if (a.rows == 0 || a.cols == 0) return FORGE_OK;
  if (a.x == nullptr || a.codes == nullptr || a.scales == nullptr) return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_quantize: null pointer");
  if (a.codes_t != nullptr && (a.block_rows != 128 || a.scales_t == nullptr || a.ld_codes_t < a.rows))
    return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_quantize: transposed codes need 128 x 128 blocks, scales_t and a pitch of at least `rows`");
  if (a.ld_x < a.cols || a.ld_codes < a.cols) return fail(FORGE_ERR_SHAPE, "forge_fp8_quantize: ld_x=%lld ld_codes=%lld cols=%lld", (long long)a.ld_x, (long long)a.ld_codes, (long long)a.cols);
  if (reinterpret_cast<uintptr_t>(a.x) % (a.dtype == FORGE_DT_BF16 ? 2 : 4)) return fail(FORGE_ERR_ALIGNMENT, "forge_fp8_quantize: x is not element-aligned");
  if (reinterpret_cast<uintptr_t>(a.scales) % 4 || (a.codes_t != nullptr && reinterpret_cast<uintptr_t>(a.scales_t) % 4))
    return fail(FORGE_ERR_ALIGNMENT, "forge_fp8_quantize: scales are not aligned");
  fp8::QuantParams p;
  p.x = static_cast<const uint8_t*>(a.x);
  p.q = static_cast<uint8_t*>(a.codes);
  p.qt = static_cast<uint8_t*>(a.codes_t);
  p.scale = a.scales; p.scale_t = a.scales_t;
  p.rows = a.rows; p.cols = a.cols; p.ld_x = a.ld_x; p.ld_q = a.ld_codes; p.ld_qt = a.ld_codes_t;
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  const int64_t cb = (a.cols + 127) / 128;
  const int64_t ctas = a.block_rows == 1 ? (a.rows * ((cb + 1) / 2) + 7) / 8 : cb * ((a.rows + 127) / 128);
  if (ctas > 0x7fffffffll) return fail(FORGE_ERR_SHAPE, "forge_fp8_quantize: %lld x %lld is too large", (long long)a.rows, (long long)a.cols);
  const unsigned g = static_cast<unsigned>(ctas);
  if (a.block_rows == 1) {
    if (a.dtype == FORGE_DT_BF16) fp8::quantize_rows_kernel<DT_BF16><<<g, 256, 0, s>>>(p);
    else fp8::quantize_rows_kernel<DT_F32><<<g, 256, 0, s>>>(p);
  } else {
    if (a.dtype == FORGE_DT_BF16) fp8::quantize_blocks_kernel<DT_BF16><<<g, 256, 0, s>>>(p);
    else fp8::quantize_blocks_kernel<DT_F32><<<g, 256, 0, s>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "fp8 quantise launch: %s", cudaGetErrorString(e));
  return FORGE_OK;
}

static int check_product(const ForgeFp8ProductArgs& a, const char* what) {
  if (a.M < 0 || a.N < 0 || a.K < 0) return fail(FORGE_ERR_INVALID_ARG, "%s: negative dimension", what);
  if (a.M == 0 || a.N == 0) return FORGE_OK;
  if (a.K < 1) return fail(FORGE_ERR_SHAPE, "%s: K must be at least 1", what);
  if (a.M > 0x7fffff00ll || a.N > 0x7fffff00ll || a.K > 0x7fffff00ll) return fail(FORGE_ERR_SHAPE, "%s: dimension too large", what);
  if (a.x_codes == nullptr || a.x_scales == nullptr || a.w_codes == nullptr || a.w_scales == nullptr || a.y == nullptr)
    return fail(FORGE_ERR_INVALID_ARG, "%s: null pointer", what);
  if (!aligned16(a.x_codes) || !aligned16(a.w_codes) || a.ld_x % 16 || a.ld_w % 16)
    return fail(FORGE_ERR_ALIGNMENT, "%s: codes must start on 16-byte boundaries and have row pitches that are multiples of 16", what);
  if (a.ld_x < a.K || a.ld_w < a.K || a.ld_y < a.N) return fail(FORGE_ERR_SHAPE, "%s: row pitch smaller than the row", what);
  if (reinterpret_cast<uintptr_t>(a.y) % 2 || reinterpret_cast<uintptr_t>(a.x_scales) % 4 || reinterpret_cast<uintptr_t>(a.w_scales) % 4 ||
      reinterpret_cast<uintptr_t>(a.status) % 4)
    return fail(FORGE_ERR_ALIGNMENT, "%s: y, scales or status are not element-aligned", what);
  return FORGE_OK;
}

static int run_product(const ForgeFp8ProductArgs& a, bool early, cudaStream_t stream) {
  const DeviceInfo* di = current_device_info();
  if (di == nullptr) return FORGE_ERR_CUDA;
  if (di->cc_major != 10) return fail(FORGE_ERR_DEVICE, "device %d is sm_%d%d, not sm_100", di->device, di->cc_major, di->cc_minor);
  fp8::Params p;
  p.sx = a.x_scales; p.sw = a.w_scales;
  p.y = static_cast<__nv_bfloat16*>(a.y);
  p.sx_row = a.x_scale_row; p.sx_col = a.x_scale_col; p.sw_row = a.w_scale_row; p.sw_col = a.w_scale_col;
  p.ld_y = a.ld_y;
  p.M = static_cast<int>(a.M); p.N = static_cast<int>(a.N);
  p.KB = static_cast<int>((a.K + fp8::BK - 1) / fp8::BK);
  p.wide = aligned16(a.y) && a.ld_y % 8 == 0;
  p.early = early;
  p.status = a.status;

  const int nt = a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= 64 ? 64 : 128;
  p.tiles_m = static_cast<int>((a.M + nt - 1) / nt);
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * ((a.N + 127) / 128);
  // K is cut until the CTAs fill the GPU once (two per SM up to 64 tokens), each with two K blocks at least
  const int64_t slots = static_cast<int64_t>(di->sm_count) * (nt == 128 ? 1 : 2);
  p.split = 1;
  // (clusters of eight leave a few SMs of every GPC unused: count on three quarters)
  while (p.split < 8 && tiles * p.split * 2 <= (p.split == 4 ? slots * 3 / 4 : slots) && p.KB >= p.split * 4) p.split *= 2;
  if (tiles * p.split > 0x7fffffffll) return fail(FORGE_ERR_SHAPE, "forge_fp8_product: too many tiles");

  // Pairs of CTAs where they need fewer rounds of K blocks over the GPU than the tiles of 128 x 128, a round taking about
  // as long in both (0.55 us).  With K = 4096, pairs / tiles: 256 x 14336 23.5 / 42 us, 512 x 14336 39 / 78,
  // 4096 x 14336 228 / 478, 512 x 1024 20 / 13.5 (K cut in four), 128 x 4096 21 / 14.  Tiles of half the weight rows where
  // one round holds them, a round taking three quarters as long: 512 x 4096 19.5 us, 22.7 without, with K = 14336 53 and 61.
  // (As the last, partial round of many tiles they are not worth it: a kernel that does both is 2 % slower per whole tile.)
  const int64_t tiles_m = (a.M + 255) / 256, pair_slots = di->sm_count / 2;
  const int64_t pair_tiles = tiles_m * ((a.N + 255) / 256), half_tiles = tiles_m * ((a.N + 127) / 128);
  const bool halves = half_tiles <= pair_slots;
  const int64_t pair_time = halves ? p.KB * 3 / 4 : (pair_tiles + pair_slots - 1) / pair_slots * p.KB;
  const int64_t tile_time = (tiles * p.split + slots - 1) / slots * ((p.KB + p.split - 1) / p.split);
  const bool pairs = nt == 128 && pair_time < tile_time;
  CUtensorMap tw, tx, ty;
  int rc = encode_tmap_2d(&tw, a.w_codes, 1, false, a.N, a.K, a.ld_w, fp8::BK, pairs && halves ? 64 : 128, 128);
  if (rc != FORGE_OK) return rc;
  rc = encode_tmap_2d(&tx, a.x_codes, 1, false, a.M, a.K, a.ld_x, fp8::BK, nt, 128);
  if (rc != FORGE_OK) return rc;
  if (pairs) {
    ty = tx;                                   // not used without aligned rows
    if (p.wide) {
      rc = encode_tmap_2d(&ty, a.y, 2, true, a.M, a.N, a.ld_y, 64, 32, 128);
      if (rc != FORGE_OK) return rc;
    }
    p.tiles_m = static_cast<int>(tiles_m);
    p.split = 1;
    if (halves) return fp8::pair::launch<128>(tx, tw, ty, p, static_cast<int>(half_tiles), di->device, stream);
    return fp8::pair::launch<256>(tx, tw, ty, p, static_cast<int>(std::min<int64_t>(pair_tiles, pair_slots)), di->device, stream);
  }
  const int ctas = static_cast<int>(tiles * p.split);
  switch (nt) {
    case 16: return fp8::launch_product<16>(tw, tx, p, ctas, di->device, stream);
    case 32: return fp8::launch_product<32>(tw, tx, p, ctas, di->device, stream);
    case 64: return fp8::launch_product<64>(tw, tx, p, ctas, di->device, stream);
    default: return fp8::launch_product<128>(tw, tx, p, ctas, di->device, stream);
  }
}

extern "C" int forge_fp8_product(const ForgeFp8ProductArgs* args, void* cuda_stream) {
  if (args == nullptr) return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_product: args is NULL");
  const int rc = check_product(*args, "forge_fp8_product");
  if (rc != FORGE_OK || args->M == 0 || args->N == 0) return rc;
  return run_product(*args, false, static_cast<cudaStream_t>(cuda_stream));
}

extern "C" int forge_fp8_linear(const ForgeFp8QuantizeArgs* x, const ForgeFp8ProductArgs* product, void* cuda_stream) {
  if (x == nullptr || product == nullptr) return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_linear: null pointer");
  const ForgeFp8ProductArgs& a = *product;
  if (x->block_rows != 1 || x->codes_t != nullptr || x->rows != a.M || x->cols != a.K || x->codes != a.x_codes || x->ld_codes != a.ld_x ||
      x->scales != a.x_scales || a.x_scale_row != (a.K + 127) / 128 || a.x_scale_col != 1)
    return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_linear: the quantiser's output is not the product's X");
  int rc = check_product(a, "forge_fp8_linear");
  if (rc != FORGE_OK || a.M == 0 || a.N == 0) return rc;
  rc = forge_fp8_quantize(x, cuda_stream);
  if (rc != FORGE_OK) return rc;
  // The product may start under the quantiser: what it reads before that has ended (the weight) was written before
  // the quantiser was launched, and the quantiser was launched after all work in front of it.
  return run_product(a, true, static_cast<cudaStream_t>(cuda_stream));
}
