// Linear layers in 8-bit integers: out[m][n] = (sum_k q[m][k] w[n][k]) * s[m] * w_scale[n] + bias[n], with the rows of the
// activations quantised to q = x / s by their largest magnitude.
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>

#include "stages.h"
#include "umma.cuh"

namespace xf {

// ---------------------------------------------------------------------------------------------
// Rows to 8 bits: s = max |x| / 127 (in 32 bits), q = x / s rounded to the nearest whole number, ties to even, exactly.
//
// t = x * (1 / s) is within 2e-5 of the quotient.  Where it lies that near to a border between two numbers the residual
// x - q s decides: it has no more bits than a float32 holds, so the fused multiply-add is exact.
// A row whose scale would be subnormal becomes zeros with scale 0; a row that holds something not finite zeros with scale NaN.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int quantise(float x, float s, float r) {
  const float t = x * r;
  float q = rintf(t);
  if (fabsf(t - q) > 0.4999f) {
    const float e = fmaf(-q, s, x), h = 0.5f * s;
    if (fabsf(e) > h || (fabsf(e) == h && (int(q) & 1))) q += copysignf(1.f, e);
  }
  return int(q);
}

template <typename T, int V>
struct RowPiece;  // V elements that are loaded at once
template <>
struct RowPiece<bf16, 8> {
  uint4 u;
  __device__ __forceinline__ void load(const bf16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ float at(int i) const {
    const uint32_t w = i < 2 ? u.x : i < 4 ? u.y : i < 6 ? u.z : u.w;
    return i & 1 ? bf16_hi(w) : bf16_lo(w);
  }
};
template <>
struct RowPiece<float, 4> {
  float4 u;
  __device__ __forceinline__ void load(const float* p) { u = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ float at(int i) const { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }
};
template <typename T>
struct RowPiece<T, 1> {
  T u;
  __device__ __forceinline__ void load(const T* p) { u = *p; }
  __device__ __forceinline__ float at(int) const { return float(u); }
};

struct QuantArgs {
  const void* x;
  long long ldx, M, ldq;
  int8_t* q;
  float* scale;
  int K, pitch, log_tpr;  // pitch: bytes of a row that are written (zeros from K on); threads for each row
};

constexpr int QUANT_ELEMS = 32;  // of a row, in a thread's registers

// `HELD`: the row stays in registers between the two passes over it
template <typename T, int V, bool HELD>
__global__ void __launch_bounds__(1024) quantise_rows_kernel(const QuantArgs a) {
  constexpr int NV = QUANT_ELEMS / V;
  __shared__ uint32_t part[32];
  const int tpr = 1 << a.log_tpr, t = threadIdx.x & (tpr - 1), rows = blockDim.x >> a.log_tpr;
  const long long m = (long long)blockIdx.x * rows + (threadIdx.x >> a.log_tpr);
  pdl_wait();
  pdl_launch();
  const bool in = m < a.M;
  const T* x = static_cast<const T*>(a.x) + (in ? m : 0) * a.ldx;
  const int nv = in ? a.K / V : 0;  // (V > 1: K is a multiple of V)
  RowPiece<T, V> p[NV];
  uint32_t most = 0;  // of the magnitudes' bits: orders floats, with what is not finite on top
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * tpr < nv) p[i].load(x + (long long)(t + i * tpr) * V);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * tpr < nv) {
#pragma unroll
        for (int v = 0; v < V; ++v) most = max(most, __float_as_uint(p[i].at(v)) & 0x7fffffffu);
      }
  } else {
    for (int i = t; i < nv; i += tpr) {
      p[0].load(x + (long long)i * V);
#pragma unroll
      for (int v = 0; v < V; ++v) most = max(most, __float_as_uint(p[0].at(v)) & 0x7fffffffu);
    }
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (tpr > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
    __syncthreads();
    const int w0 = (threadIdx.x >> a.log_tpr) << (a.log_tpr - 5);
    most = 0;
    for (int w = 0; w < tpr / 32; ++w) most = max(most, part[w0 + w]);
  }
  if (!in) return;
  float s = __uint_as_float(most) / 127.f, r;
  const bool fine = most < 0x7f800000u, some = fine && s >= FLT_MIN;
  if (!some) s = fine ? 0.f : __uint_as_float(0x7fffffffu);
  r = some ? 1.f / s : 0.f;
  if (t == 0) a.scale[m] = s;
  int8_t* q = a.q + m * a.ldq;
  auto put = [&](const RowPiece<T, V>& pc, int i) {
    if constexpr (V == 1) {
      q[i] = int8_t(some ? quantise(pc.at(0), s, r) : 0);
    } else {
      uint32_t w[V / 4];
#pragma unroll
      for (int g = 0; g < V / 4; ++g) {
        w[g] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[g] |= uint32_t((some ? quantise(pc.at(4 * g + e), s, r) : 0) & 255) << (8 * e);
      }
      if constexpr (V == 8) *reinterpret_cast<uint2*>(q + (long long)i * 8) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(q + (long long)i * 4) = w[0];
    }
  };
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * tpr < nv) put(p[i], t + i * tpr);
  } else {
    for (int i = t; i < nv; i += tpr) {
      p[0].load(x + (long long)i * V);
      put(p[0], i);
    }
  }
  for (int i = a.K + t; i < a.pitch; i += tpr) q[i] = 0;
}

template <typename T, int V>
static void launch_quantise_wide(QuantArgs a, cudaStream_t st) {
  a.log_tpr = 5;
  while ((1 << a.log_tpr) * QUANT_ELEMS < a.K && a.log_tpr < 10) ++a.log_tpr;
  const bool held = (1 << a.log_tpr) * QUANT_ELEMS >= a.K;
  const int threads = std::max(128, 1 << a.log_tpr), rows = threads >> a.log_tpr;
  const unsigned grid = (unsigned)((a.M + rows - 1) / rows);
  if (held) launch_pdl(quantise_rows_kernel<T, V, true>, dim3(grid), threads, 0, st, a);
  else launch_pdl(quantise_rows_kernel<T, V, false>, dim3(grid), threads, 0, st, a);
}

static int launch_quantise(Ctx* c, const void* x, int f32, long long ldx, long long M, int K, int8_t* q, long long ldq, int pitch, float* scale,
                           cudaStream_t st) {
  QuantArgs a{x, ldx, M, ldq, q, scale, K, pitch, 0};
  const int wide = f32 ? 4 : 8;
  const bool vec = K % wide == 0 && ldx % wide == 0 && (uintptr_t)x % 16 == 0 && ldq % wide == 0 && (uintptr_t)q % wide == 0;
  ProfScope ps(c, XFOLD_K_LAYERNORM, st);
  if (f32) vec ? launch_quantise_wide<float, 4>(a, st) : launch_quantise_wide<float, 1>(a, st);
  else vec ? launch_quantise_wide<bf16, 8>(a, st) : launch_quantise_wide<bf16, 1>(a, st);
  return check_launch(c, "quantise_rows_kernel");
}

// ---------------------------------------------------------------------------------------------
// The product: persistent and warp-specialised like gemm_tn_kernel, on tcgen05.mma kind::i8 with 32-bit sums in tensor memory.
//   warp 0      : TMA producer, 128-byte-swizzled K-major tiles of 128 bytes along K
//   warp 1      : tcgen05.mma issuer; owns the tensor memory (2 accumulators)
//   warps 2..9  : epilogue: scales, bias, rounding; each warp's 32 x 32 parts leave through its own staging tiles
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void umma_i8_if(uint32_t go, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(go)
      : "memory");
}
// signed 8 bits x signed 8 bits -> signed 32 bits, both operands K-major
__host__ __device__ constexpr uint32_t make_idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

constexpr int I8_BM = 128, I8_BK = 128, I8_THREADS = 320;
constexpr uint32_t I8_OUT_WARP = 4096;  // staging of an epilogue warp: two [32][32] tiles of 16 bits or one of 32

template <int BN>
struct I8Cfg {
  static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr uint32_t A_BYTES = I8_BM * I8_BK, B_BYTES = BN * I8_BK, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr uint32_t OFF_OUT = STAGES * STAGE_BYTES, OFF_BAR = OFF_OUT + 8 * I8_OUT_WARP;
  static constexpr uint32_t SMEM_BYTES = OFF_BAR + 256 + 1024;
};

struct I8Args {
  int M, N, K, tiles_m, tiles_n;
  const float *x_scale, *w_scale, *bias;
  void* out;
  long long ldo;
  int by_tma;  // the result's rows can leave by TMA (16-byte alignment)
  int early_b; // the weights are older than the kernel before
  int* status;
};

template <int BN, typename OutT>
__global__ void __launch_bounds__(I8_THREADS, 1)
i8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmO,
               const I8Args p) {
  using Cfg = I8Cfg<BN>;
  constexpr int STAGES = Cfg::STAGES;
  constexpr bool F32 = sizeof(OutT) == 4;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __reduce_max_sync(0xffffffffu, threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const AbortCtx ab{cta_abort, p.status};
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&tfull[s], 1);
      mbar_init(&tempty[s], 8);
    }
    *cta_abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __reduce_max_sync(0xffffffffu, *tmem_slot);
  const int KB = (p.K + I8_BK - 1) / I8_BK;
  const long long total = (long long)p.tiles_m * p.tiles_n;

  if (warp == 0) {
    const uint32_t go = elect_one();
    uint32_t stage = 0, phase = 0;
    bool okay = true;
    // the first tile's weights are on their way before the wait for the kernel before
    int pre = 0;
    if (p.early_b && blockIdx.x < total)
      for (; pre < STAGES && pre < KB; ++pre) {
        mbar_arrive_expect_tx_if(go, &full[pre], Cfg::STAGE_BYTES);
        tma_load_3d_if(go, smem + pre * Cfg::STAGE_BYTES + Cfg::A_BYTES, &tmB, &full[pre], pre * I8_BK, int(blockIdx.x % p.tiles_n) * BN, 0);
      }
    pdl_wait();
    pdl_launch();
    for (long long t = blockIdx.x; t < total && okay; t += gridDim.x) {
      const int tn = int(t % p.tiles_n), tm = int(t / p.tiles_n);
      for (int kb = 0; kb < KB; ++kb) {
        uint8_t* sA = smem + stage * Cfg::STAGE_BYTES;
        if (pre > 0) {
          --pre;
        } else {
          if (!mbar_wait_warp(&empty[stage], phase ^ 1u, ab, XF_ERR_WAIT_EMPTY)) { okay = false; break; }
          mbar_arrive_expect_tx_if(go, &full[stage], Cfg::STAGE_BYTES);
          tma_load_3d_if(go, sA + Cfg::A_BYTES, &tmB, &full[stage], kb * I8_BK, tn * BN, 0);
        }
        tma_load_3d_if(go, sA, &tmA, &full[stage], kb * I8_BK, tm * I8_BM, 0);
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    pdl_wait();
    pdl_launch();
    const uint32_t go = elect_one();
    constexpr uint32_t idesc = make_idesc_i8(I8_BM, BN);
    uint32_t stage = 0, phase = 0, it = 0;
    bool okay = true;
    for (long long t = blockIdx.x; t < total && okay; t += gridDim.x, ++it) {
      const uint32_t buf = it & 1u, aphase = (it >> 1) & 1u;
      if (!mbar_wait_warp(&tempty[buf], aphase ^ 1u, ab, XF_ERR_WAIT_TMEM_EMPTY)) break;
      tc_fence_after();
      const uint32_t d = tmem_base + buf * BN;
      for (int kb = 0; kb < KB; ++kb) {
        if (!mbar_wait_warp(&full[stage], phase, ab, XF_ERR_WAIT_FULL)) { okay = false; break; }
        tc_fence_after();
        const uint32_t sA = smem_u32(smem + stage * Cfg::STAGE_BYTES);
        const uint64_t ad = make_sdesc(sA, 16u, 1024), bd = make_sdesc(sA + Cfg::A_BYTES, 16u, 1024);
#pragma unroll
        for (int k = 0; k < I8_BK / 32; ++k)  // 32 bytes along K inside the swizzled row
          umma_i8_if(go, d, ad + 2 * k, bd + 2 * k, idesc, (kb | k) ? 1u : 0u);
        umma_commit_if(go, &empty[stage]);
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
      if (okay) umma_commit_if(go, &tfull[buf]);
    }
  } else {
    pdl_wait();
    pdl_launch();
    const uint32_t go = elect_one();
    const int q = warp & 3, ch = (warp - 2) >> 2;
    uint8_t* stage_out = smem + Cfg::OFF_OUT + (warp - 2) * I8_OUT_WARP;
    uint32_t it = 0, ochunk = 0;
    for (long long t = blockIdx.x; t < total; t += gridDim.x, ++it) {
      const int tn = int(t % p.tiles_n), tm = int(t / p.tiles_n);
      const uint32_t buf = it & 1u, aphase = (it >> 1) & 1u;
      const int row0 = tm * I8_BM + q * 32;
      const float rs = row0 + lane < p.M ? p.x_scale[row0 + lane] : 0.f;
      float cb = 0.f, cs = 0.f;  // this lane's element of the column vectors
      auto fetch_cols = [&](int c) {
        const int col = tn * BN + c * 64 + ch * 32 + lane;
        cs = col < p.N ? p.w_scale[col] : 0.f;
        cb = p.bias && col < p.N ? p.bias[col] : 0.f;
      };
      fetch_cols(0);
      if (!mbar_wait(&tfull[buf], aphase, ab, XF_ERR_WAIT_TMEM_FULL)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + buf * BN + (uint32_t(q * 32) << 16);
      const int nch = min(BN / 64, (p.N - tn * BN + 63) / 64);
#pragma unroll 1
      for (int c = 0; c < nch; ++c, ++ochunk) {
        const int colw = tn * BN + c * 64 + ch * 32;
        uint8_t* so = F32 ? stage_out : stage_out + (ochunk & 1u) * (I8_OUT_WARP / 2);
        uint32_t r[32];
        tmem_ld32(taddr + c * 64 + ch * 32, r);
        tmem_ld_wait();
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = float(int(r[e]));
        // the store that last used this staging tile must have read it out
        if constexpr (F32) tma_store_wait_read<0>();
        else tma_store_wait_read<1>();
        __syncwarp();
        // every row needs all 32 elements of the column vectors: they pass through the free staging tile
        float* sv = reinterpret_cast<float*>(so);
        sv[lane] = cb;
        sv[32 + lane] = cs;
        __syncwarp();
        if (c + 1 < nch) fetch_cols(c + 1);
#pragma unroll  // (the scales' product first: a sum times a large scale of its row alone could overflow)
        for (int e = 0; e < 8; ++e) {
          const float4 fb = reinterpret_cast<const float4*>(sv)[e], fs = reinterpret_cast<const float4*>(sv)[8 + e];
          v[4 * e] = fmaf(v[4 * e], rs * fs.x, fb.x);
          v[4 * e + 1] = fmaf(v[4 * e + 1], rs * fs.y, fb.y);
          v[4 * e + 2] = fmaf(v[4 * e + 2], rs * fs.z, fb.z);
          v[4 * e + 3] = fmaf(v[4 * e + 3], rs * fs.w, fb.w);
        }
        __syncwarp();
        if constexpr (F32) {
#pragma unroll
          for (int g = 0; g < 8; ++g)  // 128-byte rows, 128-byte swizzle
            *reinterpret_cast<float4*>(so + lane * 128 + ((uint32_t(g) ^ uint32_t(lane & 7)) << 4)) =
                make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
        } else {
#pragma unroll
          for (int g = 0; g < 4; ++g)  // 64-byte rows, 64-byte swizzle
            *reinterpret_cast<uint4*>(so + lane * 64 + ((uint32_t(g) ^ uint32_t((lane >> 1) & 3)) << 4)) =
                make_uint4(pack_bf16x2(v[8 * g], v[8 * g + 1]), pack_bf16x2(v[8 * g + 2], v[8 * g + 3]),
                           pack_bf16x2(v[8 * g + 4], v[8 * g + 5]), pack_bf16x2(v[8 * g + 6], v[8 * g + 7]));
        }
        if (p.by_tma) {
          fence_proxy_async_smem();
          __syncwarp();
          tma_store_3d_if(colw < p.N && row0 < p.M ? go : 0u, &tmO, so, colw, row0, 0);
        } else {
          // rows that start at any element: a row's 32 elements by the 32 lanes
          __syncwarp();
          if (colw + lane < p.N) {
            OutT* o = static_cast<OutT*>(p.out) + (long long)row0 * p.ldo + colw + lane;
            const int rows = min(32, p.M - row0);
            for (int rr = 0; rr < rows; ++rr, o += p.ldo) {
              if constexpr (F32)
                *o = *reinterpret_cast<const float*>(so + rr * 128 + ((uint32_t(lane >> 2) ^ uint32_t(rr & 7)) << 4) + (lane & 3) * 4);
              else
                *o = *reinterpret_cast<const bf16*>(so + rr * 64 + ((uint32_t(lane >> 3) ^ uint32_t((rr >> 1) & 3)) << 4) + (lane & 7) * 2);
            }
          }
          __syncwarp();
        }
        tma_store_commit();  // empty groups count too: the wait is by number
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[buf]);
    }
    tma_store_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  if (*cta_abort && threadIdx.x == 0) {
    // give TMA copies that were already in flight time to land before the CTA's memory is released
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000) {}
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}

template <int BN, typename OutT>
static int launch_i8_one(Ctx* c, const CUtensorMap& tmA, const int8_t* w, long long ldw, I8Args a, cudaStream_t st) {
  using Cfg = I8Cfg<BN>;
  auto kern = i8_gemm_kernel<BN, OutT>;
  static bool attr_done[8] = {false};
  if (!attr_done[c->device & 7]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
    if (e != cudaSuccess) return fail(c, XFOLD_ERR_LAUNCH, "int8 product: %s", cudaGetErrorString(e));
    attr_done[c->device & 7] = true;
  }
  CUtensorMap tmB, tmO = tmA;
  if (!make_tmap_3d(&tmB, TMAP_U8, w, a.K, a.N, 1, ldw, (uint64_t)ldw * a.N, I8_BK, BN, 1, 128))
    return fail(c, XFOLD_ERR_ARG, "int8 product: cannot encode the weights' tensor map");
  a.tiles_n = (a.N + BN - 1) / BN;
  constexpr int elem = sizeof(OutT);
  a.by_tma = (uintptr_t)a.out % 16 == 0 && a.ldo * elem % 16 == 0;
  if (a.by_tma && !make_tmap_3d(&tmO, elem == 4 ? TMAP_F32 : TMAP_BF16, a.out, a.N, a.M, 1, a.ldo, (uint64_t)a.ldo * a.M, 32, 32, 1, 32 * elem))
    return fail(c, XFOLD_ERR_ARG, "int8 product: cannot encode the result's tensor map");
  const long long total = (long long)a.tiles_m * a.tiles_n;
  ProfScope ps(c, XFOLD_K_LINEAR, st);
  launch_pdl(kern, dim3((unsigned)std::min<long long>(total, c->sm_count)), I8_THREADS, Cfg::SMEM_BYTES, st, tmA, tmB, tmO, a);
  return check_launch(c, "i8_gemm_kernel");
}

template <typename OutT>
static int launch_i8(Ctx* c, const int8_t* x, long long ldx, const float* x_scale, long long M, int K, const int8_t* w, long long ldw, int N,
                     const float* w_scale, const float* bias, OutT* out, long long ldo, int early_b, cudaStream_t st) {
  I8Args a{};
  a.M = (int)M; a.N = N; a.K = K;
  a.tiles_m = (int)((M + I8_BM - 1) / I8_BM);
  a.x_scale = x_scale; a.w_scale = w_scale; a.bias = bias;
  a.out = out; a.ldo = ldo;
  a.early_b = early_b;
  a.status = c->d_status;
  CUtensorMap tmA;
  if (!make_tmap_3d(&tmA, TMAP_U8, x, K, M, 1, ldx, (uint64_t)ldx * M, I8_BK, I8_BM, 1, 128))
    return fail(c, XFOLD_ERR_ARG, "int8 product: cannot encode the activations' tensor map");
  switch (gemm_tile_n(c, M, N, (K + 1) / 2, 1, 256, 64)) {
    case 256: return launch_i8_one<256, OutT>(c, tmA, w, ldw, a, st);
    case 128: return launch_i8_one<128, OutT>(c, tmA, w, ldw, a, st);
    default: return launch_i8_one<64, OutT>(c, tmA, w, ldw, a, st);
  }
}

static int i8_check(Ctx* c, long long M, int K, int N) {
  if (M < 0 || K < 1 || N < 0) return fail(c, XFOLD_ERR_ARG, "int8 linear: sizes");
  // 127 * 127 * K stays within the 32-bit sums
  if (K > 131072) return fail(c, XFOLD_ERR_ARG, "int8 linear: K up to 131072");
  if (M >= (1ll << 31) - 128 || N >= (1 << 30)) return fail(c, XFOLD_ERR_ARG, "int8 linear: too many rows");
  return XFOLD_OK;
}

static int i8_operand(Ctx* c, const void* p, long long ld, int K, const char* what) {
  if (!p || (uintptr_t)p % 16 || ld % 16 || ld < K)
    return fail(c, XFOLD_ERR_ARG, "int8 linear: %s start at 16-byte boundaries, rows a multiple of 16 bytes apart", what);
  return XFOLD_OK;
}

static int i8_product(Ctx* c, const int8_t* x, long long ldx, const float* x_scale, long long M, int K, const int8_t* w, long long ldw, int N,
                      const float* w_scale, const float* bias, void* out, int out_f32, long long ldo, int early_b, cudaStream_t st) {
  if (out_f32 != 0 && out_f32 != 1) return fail(c, XFOLD_ERR_ARG, "int8 linear: type of the result");
  if (!x_scale || !w_scale || !out || ldo < N || (uintptr_t)out % (out_f32 ? 4 : 2)) return fail(c, XFOLD_ERR_ARG, "int8 linear: scales and result");
  if (int rc = i8_operand(c, x, ldx, K, "activations")) return rc;
  if (int rc = i8_operand(c, w, ldw, K, "weights")) return rc;
  return out_f32 ? launch_i8(c, x, ldx, x_scale, M, K, w, ldw, N, w_scale, bias, (float*)out, ldo, early_b, st)
                 : launch_i8(c, x, ldx, x_scale, M, K, w, ldw, N, w_scale, bias, (bf16*)out, ldo, early_b, st);
}

static long long pad16(long long k) { return (k + 15) & ~15ll; }

}  // namespace xf

using namespace xf;

extern "C" {

int xfold_quantize_rows_fwd(xfold_ctx* cx, const void* x, int is_f32, long long ldx, long long M, int K, void* q, long long ldq, float* scale,
                            void* stream) {
  if (!cx) return XFOLD_ERR_ARG;
  Ctx* c = reinterpret_cast<Ctx*>(cx);
  CallLock call(c);
  if (int rc = i8_check(c, M, K, 0)) return rc;
  if (!M) return XFOLD_OK;
  if (is_f32 != 0 && is_f32 != 1) return fail(c, XFOLD_ERR_ARG, "quantise rows: type");
  if (!x || !q || !scale || ldx < K || (uintptr_t)x % (is_f32 ? 4 : 2)) return fail(c, XFOLD_ERR_ARG, "quantise rows: null or misaligned argument");
  if (ldq < K) return fail(c, XFOLD_ERR_ARG, "quantise rows: rows of the result are too near to each other");
  DeviceGuard dev(c);
  return launch_quantise(c, x, is_f32, ldx, M, K, (int8_t*)q, ldq, (int)std::min(ldq, pad16(K)), scale, (cudaStream_t)stream);
}

int xfold_linear_int8_quantized_fwd(xfold_ctx* cx, const void* x, long long ldx, const float* x_scale, long long M, int K, const void* w,
                                    long long ldw, int N, const float* w_scale, const float* bias, void* out, int out_is_f32, long long ldo,
                                    void* stream) {
  if (!cx) return XFOLD_ERR_ARG;
  Ctx* c = reinterpret_cast<Ctx*>(cx);
  CallLock call(c);
  if (int rc = i8_check(c, M, K, N)) return rc;
  if (!M || !N) return XFOLD_OK;
  DeviceGuard dev(c);
  return i8_product(c, (const int8_t*)x, ldx, x_scale, M, K, (const int8_t*)w, ldw, N, w_scale, bias, out, out_is_f32, ldo, c->static_weights,
                    (cudaStream_t)stream);
}

size_t xfold_linear_int8_workspace_bytes(long long M, int K) {
  return M > 0 && K > 0 ? align_up((size_t)M * pad16(K), 1024) + align_up((size_t)M * 4, 1024) + 1024 : 0;
}

int xfold_linear_int8_fwd(xfold_ctx* cx, const void* x, int is_f32, long long ldx, long long M, int K, const void* w, long long ldw, int N,
                          const float* w_scale, const float* bias, void* out, int out_is_f32, long long ldo, void* ws, size_t ws_bytes,
                          void* stream) {
  if (!cx) return XFOLD_ERR_ARG;
  Ctx* c = reinterpret_cast<Ctx*>(cx);
  CallLock call(c);
  if (int rc = i8_check(c, M, K, N)) return rc;
  if (!M || !N) return XFOLD_OK;
  if (is_f32 != 0 && is_f32 != 1) return fail(c, XFOLD_ERR_ARG, "int8 linear: type");
  if (!x || ldx < K || (uintptr_t)x % (is_f32 ? 4 : 2)) return fail(c, XFOLD_ERR_ARG, "int8 linear: null or misaligned activations");
  Carver cv(ws, ws_bytes);
  int8_t* q = (int8_t*)cv.take((size_t)M * pad16(K));
  float* scale = (float*)cv.take((size_t)M * 4);
  if (!ws || (uintptr_t)ws % 16 || !cv.ok()) return fail(c, XFOLD_ERR_ARG, "int8 linear: workspace too small (%zu < %zu) or misaligned", ws_bytes, cv.off);
  // what the product would refuse is refused before the first launch
  if (int rc = i8_operand(c, w, ldw, K, "weights")) return rc;
  if (!w_scale || !out || ldo < N || (uintptr_t)out % (out_is_f32 ? 4 : 2)) return fail(c, XFOLD_ERR_ARG, "int8 linear: scales and result");
  DeviceGuard dev(c);
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = launch_quantise(c, x, is_f32, ldx, M, K, q, pad16(K), (int)pad16(K), scale, st)) return rc;
  // the quantisation starts behind what wrote the weights, and the product is launched behind its start
  return i8_product(c, q, pad16(K), scale, M, K, (const int8_t*)w, ldw, N, w_scale, bias, out, out_is_f32, ldo, 1, st);
}

}  // extern "C"
