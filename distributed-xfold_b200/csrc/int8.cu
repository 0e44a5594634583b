// Linear layers in 8-bit integers: out[m][n] = (sum_k q[m][k] w[n][k]) * s[m] * w_scale[n] + bias[n], with the rows of the
// activations quantised to q = x / s by their largest magnitude.
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cfloat>

#include "stages.h"
#include "umma.cuh"

namespace xf {

// ---------------------------------------------------------------------------------------------
// Rows to 8 bits: s = max |x| / 127 (in 32 bits), q = x / s rounded to the nearest whole number, ties to even, exactly.
//
// One element: t = x * (1 / s) is within 2e-5 of the quotient.  Where it lies that near to a border between two numbers the
// residual x - q s decides: it has no more bits than a float32 holds, so the fused multiply-add is exact.
// A row whose scale would be subnormal becomes zeros with scale 0; a row that holds something not finite zeros with scale NaN.
// Bound by its instructions: nine for an element, and 300 for a warp (8192 x 4096 in 16 bits: 25 us, of which 15 are the bytes').
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

// A row's scale by the bits of its largest magnitude, its reciprocal in two parts, and how near to a half a remainder is taken
// for one.
struct RowScale {
  float s, r, r_low, near;
  bool some;
  __device__ __forceinline__ explicit RowScale(uint32_t most) {
    s = __uint_as_float(most) / 127.f;
    const bool fine = most < 0x7f800000u;
    some = fine && s >= FLT_MIN;
    if (!some) s = fine ? 0.f : __uint_as_float(0x7fffffffu);
    r = some ? 1.f / s : 0.f;
    const bool low = some && s < 1e20f;  // (r_low of larger scales would be subnormal)
    r_low = low ? fmaf(-r, s, 1.f) * r : 0.f;
    near = low ? 1.2e-7f : 1e-4f;
  }
};

struct QuantArgs {
  const void* x;
  long long ldx, M, ldq;
  int8_t* q;
  float* scale;
  int K, pitch, log_tpr;  // pitch: bytes of a row that are written (zeros from K on); threads for each row
  int wide_q;             // rows of q start at 8-byte boundaries
};

// (a call of its own: rare, and eight times as long as the common way)
__device__ __noinline__ uint2 quantise_one_by_one(float4 x, float4 y, float s, float r) {
  const uint32_t lo = __byte_perm(__byte_perm(quantise(x.x, s, r), quantise(x.y, s, r), 0x0040),
                                  __byte_perm(quantise(x.z, s, r), quantise(x.w, s, r), 0x0040), 0x5410);
  return make_uint2(lo, __byte_perm(__byte_perm(quantise(y.x, s, r), quantise(y.y, s, r), 0x0040),
                                    __byte_perm(quantise(y.z, s, r), quantise(y.w, s, r), 0x0040), 0x5410));
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}

// Eight neighbouring elements of a row as they lie in memory.  ALIGNED: rows start at 16-byte boundaries, and K is a multiple of 8.
template <typename T, bool ALIGNED>
struct Eight {
  static constexpr int W = sizeof(T) * 2, PER = 4 / sizeof(T);  // words; elements of a word
  uint32_t w[W];

  // elements 8 i .. 8 i + 7 of a row; elements from `n` on are zero
  __device__ __forceinline__ void load(const QuantArgs& a, const T* row, long long i, int n) {
    const T* at = row + i * 8;
    if constexpr (ALIGNED) {
#pragma unroll
      for (int g = 0; g < W / 4; ++g) *reinterpret_cast<uint4*>(w + 4 * g) = reinterpret_cast<const uint4*>(at)[g];
      return;
    }
    // the 16-byte pieces around them, and a shift.  Of the first and the last row a piece could reach beyond the array.
    const uintptr_t addr = reinterpret_cast<uintptr_t>(at), from = addr & ~uintptr_t(15);
    const uintptr_t first = reinterpret_cast<uintptr_t>(a.x), last = first + ((a.M - 1) * a.ldx + a.K) * sizeof(T);
    if (from >= first && from + 4 * W + 16 <= last) {
      uint32_t u[W + 4];
#pragma unroll
      for (int g = 0; g < W / 4 + 1; ++g) *reinterpret_cast<uint4*>(u + 4 * g) = reinterpret_cast<const uint4*>(from)[g];
      const bool two = addr & 8, one = addr & 4;
#pragma unroll
      for (int e = 0; e < W + 2; ++e) u[e] = two ? u[e + 2] : u[e];
#pragma unroll
      for (int e = 0; e < W + 1; ++e) u[e] = one ? u[e + 1] : u[e];
#pragma unroll
      for (int e = 0; e < W; ++e) w[e] = sizeof(T) == 2 ? __funnelshift_r(u[e], u[e + 1], (addr & 2) * 8) : u[e];
      if (n < 8) {
#pragma unroll
        for (int e = 0; e < W; ++e) w[e] = e * PER + PER <= n ? w[e] : e * PER < n ? w[e] & 0xffffu : 0u;
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < W; ++e) {
      w[e] = 0;
      if constexpr (sizeof(T) == 2) {
        if (2 * e < n) w[e] = reinterpret_cast<const uint16_t*>(at)[2 * e];
        if (2 * e + 1 < n) w[e] |= uint32_t(reinterpret_cast<const uint16_t*>(at)[2 * e + 1]) << 16;
      } else if (e < n) {
        w[e] = reinterpret_cast<const uint32_t*>(at)[e];
      }
    }
  }
  // the largest magnitude's bits so far (in 16 bits: of the elements at even and odd places)
  __device__ __forceinline__ void most(uint32_t& m) const {
#pragma unroll
    for (int e = 0; e < W; ++e) m = sizeof(T) == 2 ? max_u16x2(m, w[e] & 0x7fff7fffu) : max(m, w[e] & 0x7fffffffu);
  }
  __device__ __forceinline__ float2 pair(int j) const {
    if constexpr (sizeof(T) == 2) return make_float2(bf16_lo(w[j]), bf16_hi(w[j]));
    else return make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
  }
  // All eight quantised.  Added to 1.5 * 2^23 a product is rounded to a whole number, whose low bits are the sum's: t from x r,
  // corrected by what the quotient differs from it, d = x (r + r_low) - t, which rounds two times at 2^-25.  Where d is that near
  // to a half the eight are taken one by one.  (Without r_low, within 1e-4 of a half, half the warps with 16-bit numbers would:
  // their quotients by the largest of them are near to halves often.)
  __device__ __forceinline__ uint2 quantised(float s, float r, float r_low, float near) const {
    constexpr float BIG = 12582912.f;
    const float2 big = make_float2(BIG, BIG), minus = make_float2(-1.f, -1.f), r2 = make_float2(r, r), l2 = make_float2(r_low, r_low),
                 quarter = make_float2(-0.25f, -0.25f);
    uint32_t q[8];
    float least = 1.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = pair(j), t = ffma2(x, r2, big), d = ffma2(x, l2, ffma2(x, r2, ffma2(t, minus, big))), y = fadd2(t, d);
      const float2 e = ffma2(d, d, quarter);  // near to a half: d's distance to it
      least = fminf(least, fminf(fabsf(e.x), fabsf(e.y)));
      q[2 * j] = __float_as_uint(y.x);
      q[2 * j + 1] = __float_as_uint(y.y);
    }
    if (least < near) {
      const float2 u = pair(0), v = pair(1), x = pair(2), y = pair(3);
      return quantise_one_by_one(make_float4(u.x, u.y, v.x, v.y), make_float4(x.x, x.y, y.x, y.y), s, r);
    }
    return make_uint2(__byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410));
  }
};

template <typename T>
constexpr int QUANT_PIECES = 8 / sizeof(T);  // of eight elements of a row, in 16 of a thread's registers (32: long batches a tenth faster, others slower)

// `HELD`: the row stays in registers between the two passes over it
template <typename T, bool ALIGNED, bool HELD>
__global__ void __launch_bounds__(1024) quantise_rows_kernel(const QuantArgs a) {
  __shared__ uint32_t part[32];
  const int tpr = 1 << a.log_tpr, t = threadIdx.x & (tpr - 1), rows = blockDim.x >> a.log_tpr;
  const long long m = (long long)blockIdx.x * rows + (threadIdx.x >> a.log_tpr);
  pdl_wait();
  pdl_launch();
  const bool in = m < a.M;
  const T* x = static_cast<const T*>(a.x) + (in ? m : 0) * a.ldx;
  const int pieces = in ? (a.K + 7) / 8 : 0;
  Eight<T, ALIGNED> p[HELD ? QUANT_PIECES<T> : 1];
  uint32_t most = 0;  // of the magnitudes' bits: orders floats, with what is not finite on top
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < QUANT_PIECES<T>; ++i)
      if (t + i * tpr < pieces) p[i].load(a, x, t + i * tpr, a.K - (t + i * tpr) * 8);
#pragma unroll
    for (int i = 0; i < QUANT_PIECES<T>; ++i)
      if (t + i * tpr < pieces) p[i].most(most);
  } else {
    for (int i = t; i < pieces; i += tpr) {
      p[0].load(a, x, i, a.K - i * 8);
      p[0].most(most);
    }
  }
  if (sizeof(T) == 2) most = max(most & 0xffffu, most >> 16) << 16;
  most = __reduce_max_sync(0xffffffffu, most);
  if (tpr > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
    __syncthreads();
    const int w0 = (threadIdx.x >> a.log_tpr) << (a.log_tpr - 5);
    most = 0;
#pragma unroll 4
    for (int w = 0; w < tpr / 32; ++w) most = max(most, part[w0 + w]);
  }
  if (!in) return;
  const RowScale r(most);
  if (t == 0) a.scale[m] = r.s;
  int8_t* q = a.q + m * a.ldq;
  auto put = [&](uint2 w, int i) {
    if (a.wide_q) {
      *reinterpret_cast<uint2*>(q + (long long)i * 8) = w;
    } else {
      for (int e = 0; e < 8 && i * 8 + e < a.pitch; ++e) q[i * 8 + e] = int8_t((e < 4 ? w.x : w.y) >> (e & 3) * 8);
    }
  };
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < QUANT_PIECES<T>; ++i)
      if (t + i * tpr < pieces) put(r.some ? p[i].quantised(r.s, r.r, r.r_low, r.near) : make_uint2(0, 0), t + i * tpr);
  } else {
    for (int i = t; i < pieces; i += tpr) {
      p[0].load(a, x, i, a.K - i * 8);
      put(r.some ? p[0].quantised(r.s, r.r, r.r_low, r.near) : make_uint2(0, 0), i);
    }
  }
  for (int i = pieces + t; i * 8 < a.pitch; i += tpr) put(make_uint2(0, 0), i);
}

template <typename T>
static void launch_quantise_of(QuantArgs a, bool aligned, cudaStream_t st) {
  a.log_tpr = 5;
  while ((1 << a.log_tpr) * QUANT_PIECES<T> * 8 < a.K && a.log_tpr < 10) ++a.log_tpr;
  const bool held = (1 << a.log_tpr) * QUANT_PIECES<T> * 8 >= a.K;
  const int threads = std::max(128, 1 << a.log_tpr), rows = threads >> a.log_tpr;
  const unsigned grid = (unsigned)((a.M + rows - 1) / rows);
  auto kern = aligned ? (held ? quantise_rows_kernel<T, true, true> : quantise_rows_kernel<T, true, false>)
                      : (held ? quantise_rows_kernel<T, false, true> : quantise_rows_kernel<T, false, false>);
  launch_pdl(kern, dim3(grid), threads, 0, st, a);
}

// pitch: a multiple of 8 where rows of q start at 8-byte boundaries
static int launch_quantise(Ctx* c, const void* x, int f32, long long ldx, long long M, int K, int8_t* q, long long ldq, int pitch, float* scale,
                           cudaStream_t st) {
  QuantArgs a{x, ldx, M, ldq, q, scale, K, pitch, 0, 0};
  const bool aligned = K % 8 == 0 && (uintptr_t)x % 16 == 0 && (M == 1 || ldx * (f32 ? 4 : 2) % 16 == 0);
  a.wide_q = (uintptr_t)q % 8 == 0 && (M == 1 || ldq % 8 == 0) && pitch % 8 == 0;
  ProfScope ps(c, XFOLD_K_LAYERNORM, st);
  if (f32) launch_quantise_of<float>(a, aligned, st);
  else launch_quantise_of<bf16>(a, aligned, st);
  return check_launch(c, "quantise_rows_kernel");
}

// ---------------------------------------------------------------------------------------------
// The product: persistent and warp-specialised like gemm_tn_kernel, on tcgen05.mma kind::i8 with 32-bit sums in tensor memory.
//   warp 0      : TMA producer, 128-byte-swizzled K-major tiles of 128 bytes along K
//   warp 1      : tcgen05.mma issuer; owns the tensor memory (2 accumulators)
//   warps 2..9  : epilogue: scales, bias, rounding; each warp's 32 x 32 parts leave through its own staging tiles
// 8192 x 4096 x 4096: 96 us at 1965 MHz, 2.9 PTOP/s (the library's 91), and 111 (105) where the power limit holds the clock at 1.4
// GHz; bound by the tensor cores and the operands' trip from L2.  Rows that start in the middle of a sector cost a third of it
// (5000^3: 103 us at rows 5056 bytes apart, 143 at 5008).  Clusters that share K of one tile, as gemm_split_kernel's, were slower at most sizes.
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

// sum * rs * ws + bias.  The scales' product first: a sum times a large scale alone could overflow.  Where that product is subnormal
// and would lose bits, or beyond all numbers and not to be had by a sum of 0, the larger scale first: in the one case it is less than
// 2^23, in the other no result but 0 is a number.
__device__ __forceinline__ float i8_scaled(float sum, float rs, float ws, float bias) {
  const float p = rs * ws;
  if (fabsf(p) >= FLT_MIN && fabsf(p) <= FLT_MAX) return fmaf(sum, p, bias);
  const bool row = fabsf(rs) > fabsf(ws);
  return fmaf(sum * (row ? rs : ws), row ? ws : rs, bias);
}

constexpr int I8_MOST_K = 131072;  // sums from -127 * 128 K to 128 * 128 K
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
        // whether a scale of the columns (zero aside) and a row's make a product that i8_scaled has to look at
        const uint32_t size = __float_as_uint(fabsf(cs));
        const float least = __uint_as_float(__reduce_min_sync(0xffffffffu, size ? size : 0x7f800000u)),
                    most = __uint_as_float(__reduce_max_sync(0xffffffffu, size));
        const bool odd = __any_sync(0xffffffffu, rs != 0.f && !(fabsf(rs) * least >= FLT_MIN && fabsf(rs) * most <= FLT_MAX));
        tmem_ld_wait();
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = float(int(r[e]));
        if (p.K == I8_MOST_K) {  // products of -128 alone: their sum, 2^31, is the one that wraps around, to what no other sum is
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = r[e] == 0x80000000u ? 2147483648.f : v[e];
        }
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
        const float4 *fb = reinterpret_cast<const float4*>(sv), *fs = fb + 8;
        if (!odd) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 b = fb[e], f = fs[e];
            v[4 * e] = fmaf(v[4 * e], rs * f.x, b.x);
            v[4 * e + 1] = fmaf(v[4 * e + 1], rs * f.y, b.y);
            v[4 * e + 2] = fmaf(v[4 * e + 2], rs * f.z, b.z);
            v[4 * e + 3] = fmaf(v[4 * e + 3], rs * f.w, b.w);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 b = fb[e], f = fs[e];
            v[4 * e] = i8_scaled(v[4 * e], rs, f.x, b.x);
            v[4 * e + 1] = i8_scaled(v[4 * e + 1], rs, f.y, b.y);
            v[4 * e + 2] = i8_scaled(v[4 * e + 2], rs, f.z, b.z);
            v[4 * e + 3] = i8_scaled(v[4 * e + 3], rs, f.w, b.w);
          }
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
  static std::atomic<bool> attr_done[8];
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

// ---------------------------------------------------------------------------------------------
// Few rows (a decoding step): bound by the weights, which are read once, 16 bytes to a lane, two channels to a warp, straight
// into the dot products of four bytes.  With one or two rows every CTA quantises them for itself while its weights are on their
// way, and the whole layer is one launch.  (4096 x 4096, weights from memory: one row 6.7 us, by quantise_rows_kernel and the
// tensor cores' tiles, of which there are but 64, 13.4; four rows, quantised before, 6.6 against 12.1; of eight rows the dot products
// take as long as the tiles.)
// ---------------------------------------------------------------------------------------------
constexpr int ROWS_MOST = 4, ROWS_SMEM = 48 * 1024 - 1024;  // rows; bytes of quantised rows in shared memory
constexpr int ROWS_C = 2, ROWS_U = 4;                       // channels of a warp; pieces of each that a lane has on their way

struct RowsArgs {
  QuantArgs x;            // (quantised rows: x, ldx, M, K, and the scales)
  const int8_t* w;
  long long ldw;
  int N;
  const float *w_scale, *bias;
  void* out;
  long long ldo;
  int out_f32;
};

// 16 bytes of a row of K; what lies behind it is zero, and not read
__device__ __forceinline__ uint4 sixteen(const int8_t* row, int piece, int K) {
  const int8_t* at = row + (long long)piece * 16;
  if (piece * 16 + 16 <= K) return *reinterpret_cast<const uint4*>(at);
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (piece * 16 + e < K) v[e / 4] |= uint32_t(uint8_t(at[e])) << (e % 4 * 8);
  return make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename T, int MB>
__global__ void __launch_bounds__(256) i8_rows_kernel(const RowsArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ float scale[MB];
  __shared__ uint32_t part[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = a.x.K, pieces = (K + 15) / 16, M = (int)a.x.M;
  const int n0 = (blockIdx.x * 8 + warp) * ROWS_C;
  pdl_wait();
  pdl_launch();
  uint4 w[ROWS_C][ROWS_U];
  auto load = [&](int u, int piece) {
#pragma unroll
    for (int c = 0; c < ROWS_C; ++c) {
      w[c][u] = make_uint4(0, 0, 0, 0);
      if (n0 + c < a.N && piece < pieces) w[c][u] = sixteen(a.w + (n0 + c) * a.ldw, piece, K);
    }
  };
#pragma unroll
  for (int u = 0; u < ROWS_U; ++u) load(u, u * 32 + lane);

  // the rows in 8 bits, 256 / MB threads to each
  constexpr int TPR = 256 / MB;
  const int m = threadIdx.x / TPR, t = threadIdx.x % TPR;
  int8_t* q = reinterpret_cast<int8_t*>(smem_raw) + (size_t)m * pieces * 16;
  if constexpr (sizeof(T) == 1) {
    const int8_t* row = static_cast<const int8_t*>(a.x.x) + m * a.x.ldx;
    for (int i = t; i < pieces; i += TPR)
      reinterpret_cast<uint4*>(q)[i] = m < M ? sixteen(row, i, K) : make_uint4(0, 0, 0, 0);
    if (t == 0) scale[m] = m < M ? a.x.scale[m] : 0.f;
  } else {
    const T* row = static_cast<const T*>(a.x.x) + m * a.x.ldx;
    const int eights = m < M ? (K + 7) / 8 : 0;
    Eight<T, false> p;
    uint32_t most = 0;
    for (int i = t; i < eights; i += TPR) {
      p.load(a.x, row, i, K - i * 8);
      p.most(most);
    }
    if (sizeof(T) == 2) most = max(most & 0xffffu, most >> 16) << 16;
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) part[warp] = most;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TPR / 32; ++k) most = max(most, part[m * (TPR / 32) + k]);
    const RowScale r(most);
    if (t == 0) scale[m] = r.s;
    for (int i = t; i < pieces * 2; i += TPR) {
      uint2 v = make_uint2(0, 0);
      if (i < eights && r.some) {
        p.load(a.x, row, i, K - i * 8);
        v = p.quantised(r.s, r.r, r.r_low, r.near);
      }
      reinterpret_cast<uint2*>(q)[i] = v;
    }
  }
  __syncthreads();

  int sum[ROWS_C][MB] = {};
  for (int base = 0; base < pieces; base += 32 * ROWS_U) {
#pragma unroll
    for (int u = 0; u < ROWS_U; ++u) {
      const int piece = base + u * 32 + lane;
      if (piece < pieces) {
#pragma unroll
        for (int r = 0; r < MB; ++r) {
          const int4 x = reinterpret_cast<const int4*>(smem_raw)[r * pieces + piece];
#pragma unroll
          for (int c = 0; c < ROWS_C; ++c) {
            int d = __dp4a(x.x, int(w[c][u].x), sum[c][r]);
            d = __dp4a(x.y, int(w[c][u].y), d);
            d = __dp4a(x.z, int(w[c][u].z), d);
            sum[c][r] = __dp4a(x.w, int(w[c][u].w), d);
          }
        }
      }
      load(u, piece + 32 * ROWS_U);
    }
  }
  int mine = 0;  // lane c * MB + r: row r of channel c
#pragma unroll
  for (int c = 0; c < ROWS_C; ++c)
#pragma unroll
    for (int r = 0; r < MB; ++r) {
      const int all = __reduce_add_sync(0xffffffffu, sum[c][r]);
      if (lane == c * MB + r) mine = all;
    }
  const int n = n0 + lane / MB, r = lane % MB;
  if (lane < ROWS_C * MB && n < a.N && r < M) {
    const float y = i8_scaled(float(mine), scale[r], a.w_scale[n], a.bias ? a.bias[n] : 0.f);
    if (a.out_f32) static_cast<float*>(a.out)[r * a.ldo + n] = y;
    else static_cast<bf16*>(a.out)[r * a.ldo + n] = __float2bfloat16(y);
  }
}

static int rows_bound(long long M) { return M <= 1 ? 1 : M <= 2 ? 2 : 4; }
static bool i8_few_rows(long long M, int K) { return M <= ROWS_MOST && rows_bound(M) * ((K + 15ll) / 16 * 16) <= ROWS_SMEM; }
// beyond this a CTA takes longer to quantise the rows than a launch costs (2 x 4096: 7.6 us, by two launches 7.8; 4 x 4096: 12.5
// and 9)
static bool i8_one_launch(long long M, int K) { return i8_few_rows(M, K) && (long long)rows_bound(M) * K <= 8192; }

template <typename T>
static int launch_i8_rows(Ctx* c, const RowsArgs& a, cudaStream_t st) {
  const int mb = rows_bound(a.x.M);
  auto kern = mb == 1 ? i8_rows_kernel<T, 1> : mb == 2 ? i8_rows_kernel<T, 2> : i8_rows_kernel<T, 4>;
  ProfScope ps(c, XFOLD_K_LINEAR, st);
  launch_pdl(kern, dim3((a.N + 8 * ROWS_C - 1) / (8 * ROWS_C)), 256, (size_t)mb * ((a.x.K + 15) / 16 * 16), st, a);
  return check_launch(c, "i8_rows_kernel");
}

static int i8_check(Ctx* c, long long M, int K, int N) {
  if (M < 0 || K < 1 || N < 0) return fail(c, XFOLD_ERR_ARG, "int8 linear: sizes");
  if (K > I8_MOST_K) return fail(c, XFOLD_ERR_ARG, "int8 linear: K up to 131072");
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
  if (i8_few_rows(M, K))
    return launch_i8_rows<int8_t>(c, {{x, ldx, M, 0, nullptr, const_cast<float*>(x_scale), K, 0, 0, 0}, w, ldw, N, w_scale, bias, out, ldo, out_f32}, st);
  return out_f32 ? launch_i8(c, x, ldx, x_scale, M, K, w, ldw, N, w_scale, bias, (float*)out, ldo, early_b, st)
                 : launch_i8(c, x, ldx, x_scale, M, K, w, ldw, N, w_scale, bias, (bf16*)out, ldo, early_b, st);
}

static long long pad16(long long k) { return (k + 15) & ~15ll; }
// distance of quantised rows: whole sectors of the L2 (5000^3: 142 us at rows 5008 bytes apart, 127 at 5056)
static long long pad64(long long k) { return (k + 63) & ~63ll; }

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
  return launch_quantise(c, x, is_f32, ldx, M, K, (int8_t*)q, ldq, (int)std::min(ldq, pad64(K)), scale, (cudaStream_t)stream);
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
  return i8_product(c, (const int8_t*)x, ldx, x_scale, M, K, (const int8_t*)w, ldw, N, w_scale, bias, out, out_is_f32, ldo, 0,
                    (cudaStream_t)stream);  // (the kernel before may have made the weights)
}

size_t xfold_linear_int8_workspace_bytes(long long M, int K) {
  return M > 0 && K > 0 && !i8_one_launch(M, K) ? align_up((size_t)M * pad64(K), 1024) + align_up((size_t)M * 4, 1024) + 1024 : 0;
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
  // what the product would refuse is refused before the first launch
  if (out_is_f32 != 0 && out_is_f32 != 1) return fail(c, XFOLD_ERR_ARG, "int8 linear: type of the result");
  if (int rc = i8_operand(c, w, ldw, K, "weights")) return rc;
  if (!w_scale || !out || ldo < N || (uintptr_t)out % (out_is_f32 ? 4 : 2)) return fail(c, XFOLD_ERR_ARG, "int8 linear: scales and result");
  DeviceGuard dev(c);
  cudaStream_t st = (cudaStream_t)stream;
  if (i8_one_launch(M, K)) {
    const RowsArgs a{{x, ldx, M, 0, nullptr, nullptr, K, 0, 0, 0}, (const int8_t*)w, ldw, N, w_scale, bias, out, ldo, out_is_f32};
    return is_f32 ? launch_i8_rows<float>(c, a, st) : launch_i8_rows<bf16>(c, a, st);
  }
  Carver cv(ws, ws_bytes);
  int8_t* q = (int8_t*)cv.take((size_t)M * pad64(K));
  float* scale = (float*)cv.take((size_t)M * 4);
  if (!ws || (uintptr_t)ws % 16 || !cv.ok()) return fail(c, XFOLD_ERR_ARG, "int8 linear: workspace too small (%zu < %zu) or misaligned", ws_bytes, cv.off);
  if (int rc = launch_quantise(c, x, is_f32, ldx, M, K, q, pad64(K), (int)pad16(K), scale, st)) return rc;
  // the quantisation starts behind what wrote the weights, and the product is launched behind its start
  return i8_product(c, q, pad64(K), scale, M, K, (const int8_t*)w, ldw, N, w_scale, bias, out, out_is_f32, ldo, 1, st);
}

}  // extern "C"
