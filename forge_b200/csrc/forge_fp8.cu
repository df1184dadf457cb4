// Products in 8-bit floating point with one fp32 scale for each block of 128, and the quantiser that
// feeds them.
//
//   scale = absmax * fp32(1 / 448) + 1e-12, code = e4m3(x / scale)   over 1 x 128 blocks of a row (activations,
//   gradients) or 128 x 128 blocks (weights; their transpose has the transposed scales)
//   Y[m, n] = sum over kb of sx[m, kb] sw[n / 128, kb] * sum over the block's k of xq[m, k] wq[n, k]
//
// The inner sums are tensor-core products of 128 terms; the outer sum is held in fp32 registers.
#include <cooperative_groups.h>

#include <algorithm>

#include "forge_host.h"
#include "forge_ptx.cuh"

namespace cg = cooperative_groups;

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

// 1 x 128 blocks: sixteen lanes of eight columns each; a warp takes two neighbouring blocks of a row
template <int DT>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantParams p) {
  constexpr int ES = DT == DT_BF16 ? 2 : 4;
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

// 128 x 128 blocks: one CTA per block, a thread holds 8 x 8 elements.  The transposed codes go through
// shared memory: four 4 x 4 byte transpositions in registers, then rows of 128 bytes.
template <int DT>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const QuantParams p) {
  constexpr int ES = DT == DT_BF16 ? 2 : 4;
  constexpr int PITCH = 128 + 16;
  __shared__ __align__(16) uint8_t tile[128 * PITCH];
  __shared__ float red[8];
  const long long cb = (p.cols + 127) / 128, rb = (p.rows + 127) / 128;
  const long long bi = blockIdx.x / cb, bj = blockIdx.x % cb;
  const int tc = (threadIdx.x & 15) * 8, tr = (threadIdx.x >> 4) * 8;
  const long long col = bj * 128 + tc, row0 = bi * 128 + tr;
  const long long left = p.cols - col;
  const int live = left >= 8 ? 8 : (left > 0 ? static_cast<int>(left) : 0);
  float x[8][8];
  float m = 0.0f;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const uint8_t* src = p.x + ((row0 + r) * p.ld_x + col) * ES;
    const int n = row0 + r < p.rows ? live : 0;
    load8<DT>(src, n, n == 8 && (reinterpret_cast<uintptr_t>(src) & 15) == 0, x[r]);
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) m = fmaxf(m, absmax8(x[r]));
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
    c[r] = codes8(x[r], scale, rscale);
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
    for (int k = 0; k < 4; ++k) *reinterpret_cast<uint2*>(&tile[(tc + 4 * h + k) * PITCH + tr]) = make_uint2(t[0][k], t[1][k]);
  }
  __syncthreads();
  const long long trow0 = bj * 128, tcol0 = bi * 128;
  const bool whole = tcol0 + 128 <= p.rows && (p.ld_qt & 15) == 0 && (reinterpret_cast<uintptr_t>(p.qt) & 15) == 0;
  for (int i = threadIdx.x; i < 128 * 8; i += 256) {
    const int r = i >> 3, pc = (i & 7) * 16;
    if (trow0 + r >= p.cols) continue;
    uint8_t* dst = p.qt + (trow0 + r) * p.ld_qt + tcol0 + pc;
    const uint4 v = *reinterpret_cast<const uint4*>(&tile[r * PITCH + pc]);
    if (whole) {
      *reinterpret_cast<uint4*>(dst) = v;
    } else {
      for (int k = 0; k < 16 && tcol0 + pc + k < p.rows; ++k) dst[k] = tile[r * PITCH + pc + k];
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
  int* status;
};

enum : int { ERR_OP_EMPTY = 221, ERR_OP_FULL = 222, ERR_ACC_EMPTY = 223, ERR_ACC_FULL = 224 };
constexpr int BK = 128;                             // bytes = elements
constexpr int A_BYTES = 128 * BK;
constexpr int ACC_BUFS = 4;
constexpr int THREADS = 256;

template <int NT>
struct Cfg {
  static constexpr int B_BYTES = NT * BK;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  // up to 64 tokens two CTAs share an SM (112 KB each); 128 take an SM's tensor memory alone
  static constexpr int STAGES = NT == 128 ? 6 : (NT == 64 ? 4 : 5);
  static constexpr int SMEM = 1024 + STAGES * STAGE;      // + alignment slack; control words are static
  static constexpr int TMEM_COLS = ACC_BUFS * NT;
  static constexpr int MIN_CTAS = NT == 128 ? 1 : 2;
};

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

struct Ctrl {
  uint64_t full[8];
  uint64_t empty[8];
  uint64_t acc_full[ACC_BUFS];
  uint64_t acc_empty[ACC_BUFS];
  uint32_t tmem_base;
  int abort_word;
};

template <int NT>
__global__ void __launch_bounds__(THREADS, Cfg<NT>::MIN_CTAS)
fp8_product_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Params p) {
  using C = Cfg<NT>;
  __shared__ Ctrl ctrl;
  __shared__ __align__(16) float sc[2][NT];
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

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) { mbar_init(&ctrl.full[i], 1); mbar_init(&ctrl.empty[i], 1); }
    for (int i = 0; i < ACC_BUFS; ++i) { mbar_init(&ctrl.acc_full[i], 1); mbar_init(&ctrl.acc_empty[i], 4); }
    ctrl.abort_word = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&ctrl.tmem_base, C::TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = ctrl.tmem_base;

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t pol_w = p.tiles_m > 1 ? policy_evict_normal() : policy_evict_first();
      const uint64_t pol_x = policy_evict_last();
      for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {
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
  } else if (warp >= 4) {
    const int quarter = warp & 3, e = threadIdx.x - 128;
    float acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = 0.0f;
    // this thread fetches the scale of token m0 + e for the coming blocks
    const bool has = e < NT && m0 + e < p.M;
    const float* sxp = p.sx + static_cast<long long>(m0 + (has ? e : 0)) * p.sx_row;
    const float* swp = p.sw + static_cast<long long>(n0 / 128) * p.sw_row;
    auto fetch = [&](int kb) { return has && kb < kb1 ? sxp[kb * p.sx_col] * swp[kb * p.sw_col] : 0.0f; };
    float s_next = fetch(kb0), s_next2 = fetch(kb0 + 1);
    bool ok = true;
    for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {
      const int b = it % ACC_BUFS;
      if (e < NT) sc[it & 1][e] = s_next;
      s_next = s_next2;
      s_next2 = fetch(kb + 2);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      ok = mbar_wait(&ctrl.acc_full[b], (it / ACC_BUFS) & 1, abort_word, ERR_ACC_FULL) && ok;
      tc_fence_after();
      __syncwarp();
      constexpr int STEP = NT < 32 ? 16 : 32;
#pragma unroll
      for (int c = 0; c < NT; c += STEP) {
        uint32_t r[STEP];
        const uint32_t ta = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + b * NT + c;
        if constexpr (STEP == 16) tmem_ld_32x16(ta, r);
        else tmem_ld_32x32(ta, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < STEP; j += 4) {
          const float4 s4 = *reinterpret_cast<const float4*>(&sc[it & 1][c + j]);
          const float2 lo = ffma2(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), make_float2(s4.x, s4.y),
                                  make_float2(acc[c + j], acc[c + j + 1]));
          const float2 hi = ffma2(make_float2(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])), make_float2(s4.z, s4.w),
                                  make_float2(acc[c + j + 2], acc[c + j + 3]));
          acc[c + j] = lo.x; acc[c + j + 1] = lo.y; acc[c + j + 2] = hi.x; acc[c + j + 3] = hi.y;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctrl.acc_empty[b]);
    }
    // Every product has completed (the last accumulator was signalled after all of them), so the operand
    // stages are free: the part goes there as [token][weight row].
    float* part = reinterpret_cast<float*>(data);
    const int r = quarter * 32 + lane;
#pragma unroll
    for (int j = 0; j < NT; ++j) part[j * 128 + r] = acc[j];
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
  cg::cluster_group cluster = cg::this_cluster();
  if (p.split > 1) cluster.sync();
  {
    // this CTA's share of the tile's tokens: eight weight rows per lane, sixteen lanes per token
    const int tokens = min(NT, p.M - m0);
    const int share = (tokens + p.split - 1) / p.split;
    const int j1 = min(tokens, (rank + 1) * share);
    const int r8 = (threadIdx.x & 15) * 8;
    for (int j = rank * share + (threadIdx.x >> 4); j < j1; j += THREADS / 16) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.0f;
      for (int q = 0; q < p.split; ++q) {
        const float* part = reinterpret_cast<const float*>(p.split > 1 ? cluster.map_shared_rank(data, q) : data);
        const float4 a = *reinterpret_cast<const float4*>(part + j * 128 + r8);
        const float4 c = *reinterpret_cast<const float4*>(part + j * 128 + r8 + 4);
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += c.x; v[5] += c.y; v[6] += c.z; v[7] += c.w;
      }
      __nv_bfloat16* dst = p.y + static_cast<long long>(m0 + j) * p.ld_y + n0 + r8;
      if (failed) continue;
      if (p.wide && n0 + r8 + 8 <= p.N) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (n0 + r8 + k < p.N) dst[k] = __float2bfloat16_rn(v[k]);
      }
    }
  }
  if (p.split > 1) cluster.sync();          // a part stays until every CTA of the cluster has read it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

template <int NT>
static int launch_product(const CUtensorMap& tw, const CUtensorMap& tx, const Params& p, int ctas, cudaStream_t stream) {
  auto* fn = fp8_product_kernel<NT>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<NT>::SMEM);
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "fp8 product: shared memory attribute: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = Cfg<NT>::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, fn, tw, tx, p);
  if (e != cudaSuccess) return fail(FORGE_ERR_CUDA, "fp8 product launch: %s", cudaGetErrorString(e));
  return FORGE_OK;
}

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

extern "C" int forge_fp8_product(const ForgeFp8ProductArgs* args, void* cuda_stream) {
  if (args == nullptr) return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_product: args is NULL");
  const ForgeFp8ProductArgs& a = *args;
  if (a.M < 0 || a.N < 0 || a.K < 0) return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_product: negative dimension");
  if (a.M == 0 || a.N == 0) return FORGE_OK;
  if (a.K < 1) return fail(FORGE_ERR_SHAPE, "forge_fp8_product: K must be at least 1");
  if (a.M > 0x7fffff00ll || a.N > 0x7fffff00ll || a.K > 0x7fffff00ll) return fail(FORGE_ERR_SHAPE, "forge_fp8_product: dimension too large");
  if (a.x_codes == nullptr || a.x_scales == nullptr || a.w_codes == nullptr || a.w_scales == nullptr || a.y == nullptr)
    return fail(FORGE_ERR_INVALID_ARG, "forge_fp8_product: null pointer");
  if (!aligned16(a.x_codes) || !aligned16(a.w_codes) || a.ld_x % 16 || a.ld_w % 16)
    return fail(FORGE_ERR_ALIGNMENT, "forge_fp8_product: codes must start on 16-byte boundaries and have row pitches that are multiples of 16");
  if (a.ld_x < a.K || a.ld_w < a.K || a.ld_y < a.N) return fail(FORGE_ERR_SHAPE, "forge_fp8_product: row pitch smaller than the row");
  if (reinterpret_cast<uintptr_t>(a.y) % 2) return fail(FORGE_ERR_ALIGNMENT, "forge_fp8_product: y is not element-aligned");
  const DeviceInfo* di = current_device_info();
  if (di == nullptr) return FORGE_ERR_CUDA;
  if (di->cc_major != 10) return fail(FORGE_ERR_DEVICE, "device %d is sm_%d%d, not sm_100", di->device, di->cc_major, di->cc_minor);

  const int nt = a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= 64 ? 64 : 128;
  CUtensorMap tw, tx;
  int rc = encode_tmap_2d(&tw, a.w_codes, 1, false, a.N, a.K, a.ld_w, fp8::BK, 128, 128);
  if (rc != FORGE_OK) return rc;
  rc = encode_tmap_2d(&tx, a.x_codes, 1, false, a.M, a.K, a.ld_x, fp8::BK, nt, 128);
  if (rc != FORGE_OK) return rc;
  fp8::Params p;
  p.sx = a.x_scales; p.sw = a.w_scales;
  p.y = static_cast<__nv_bfloat16*>(a.y);
  p.sx_row = a.x_scale_row; p.sx_col = a.x_scale_col; p.sw_row = a.w_scale_row; p.sw_col = a.w_scale_col;
  p.ld_y = a.ld_y;
  p.M = static_cast<int>(a.M); p.N = static_cast<int>(a.N);
  p.KB = static_cast<int>((a.K + fp8::BK - 1) / fp8::BK);
  p.tiles_m = static_cast<int>((a.M + nt - 1) / nt);
  p.wide = aligned16(a.y) && a.ld_y % 8 == 0;
  p.status = a.status;
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * ((a.N + 127) / 128);
  // K is cut until the CTAs fill the GPU once (two per SM up to 64 tokens), each with two K blocks at least
  const int64_t slots = static_cast<int64_t>(di->sm_count) * (nt == 128 ? 1 : 2);
  p.split = 1;
  while (p.split < 8 && tiles * p.split * 2 <= slots && p.KB >= p.split * 4) p.split *= 2;
  if (tiles * p.split > 0x7fffffffll) return fail(FORGE_ERR_SHAPE, "forge_fp8_product: too many tiles");
  const int ctas = static_cast<int>(tiles * p.split);
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  switch (nt) {
    case 16: return fp8::launch_product<16>(tw, tx, p, ctas, s);
    case 32: return fp8::launch_product<32>(tw, tx, p, ctas, s);
    case 64: return fp8::launch_product<64>(tw, tx, p, ctas, s);
    default: return fp8::launch_product<128>(tw, tx, p, ctas, s);
  }
}
