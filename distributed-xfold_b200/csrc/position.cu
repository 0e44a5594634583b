// Positions in attention: a learned bias of the logits by buckets of relative position, with the gradient of its table, and
// the norms of queries and keys for each head together with the rotation by position, with their gradients.  All of them are
// bound by what they read and write; the compiler's fast approximations stay off here (see build.py).
#include <cuda_fp16.h>

#include <algorithm>

#include "stages.h"
#include "umma.cuh"

namespace xf {

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---------------------------------------------------------------------------------------------
// Relative position bias: out[h][i][j] = table[b(i, j)][h],
//   b(i, j) = lut[clamp(k_pos[j] - q_pos[i], -reach, reach) + reach], or the table's last row where the groups differ.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int offset_in_lut(int kp, int qp, int reach) {
  int d;
  asm("sub.sat.s32 %0, %1, %2;" : "=r"(d) : "r"(kp), "r"(qp));
  return min(max(d, -reach), reach) + reach;
}

struct RelShared {  // what both directions read of the positions
  const int* lut;
  const int *q_pos, *k_pos, *q_grp, *k_grp;
  int reach, nb, H, Sq, Sk;
};

// a lut entry that names no row of the table: row nb + 1
__device__ __forceinline__ void stage_lut(const RelShared& s, uint16_t* lut, int step = 1) {
  for (int i = threadIdx.x; i < 2 * s.reach + 1; i += blockDim.x) {
    const int b = s.lut[i];
    lut[i] = uint16_t((b >= 0 && b < s.nb ? b : s.nb + 1) * step);
  }
}
// the positions that a query's buckets end at: a key's place in the lut is min(max(its position, low), high) - (query's - reach)
__device__ __forceinline__ int low_end(int qp, int reach) { return max(qp, -0x7fffffff - 1 + reach) - reach; }
__device__ __forceinline__ int high_end(int qp, int reach) { return min(qp, 0x7fffffff - reach) + reach; }

struct RelFwdArgs {
  RelShared s;
  const float* table;
  void* out;
  long long pitch;  // elements from one query's keys to the next's
  int cols;         // columns written: Sk, or the pitch where the rest is zero
  int hg, log_cx;   // heads per CTA; chunks of columns side by side in a CTA (a power of two)
};

__device__ __forceinline__ void rel_value(float v, float& o) { o = v; }
__device__ __forceinline__ void rel_value(float v, bf16& o) { o = __float2bfloat16(v); }
// the attention kernel's operand, as the other producers of pair biases write it
__device__ __forceinline__ void rel_value(float v, __half& o) {
  o = __float2half_rn(fminf(fmaxf(v * 1.4426950408889634f, -60000.f), 60000.f));
}

template <typename E, int V>
struct alignas(sizeof(E) * V) RelPiece {
  E e[V];
};

// A thread keeps V columns and goes down the rows: their positions stay in registers, and a row's buckets serve all heads of
// the CTA.  Where the V columns share a bucket (beyond the reach, or in another group) a head's value is fetched once.
template <typename E, int V>
__global__ void __launch_bounds__(256) rel_bias_kernel(const RelFwdArgs a) {
  extern __shared__ uint8_t smem_raw[];
  const RelShared& s = a.s;
  const int rows_tab = s.nb + 2, h0 = blockIdx.z * a.hg, hn = min(a.hg, s.H - h0);
  E* tab = reinterpret_cast<E*>(smem_raw);  // [hg][nb + 2]: row nb is zero, row nb + 1 not a number
  uint16_t* lut = reinterpret_cast<uint16_t*>(smem_raw + (((size_t)a.hg * rows_tab * sizeof(E) + 15) & ~size_t(15)));
  pdl_wait();
  pdl_launch();
  stage_lut(s, lut);
  for (int i = threadIdx.x; i < hn * rows_tab; i += 256) {
    const int h = i / rows_tab, b = i % rows_tab;
    rel_value(b < s.nb ? a.table[(long long)b * s.H + h0 + h] : b == s.nb ? 0.f : __int_as_float(0x7fffffff), tab[i]);
  }
  __syncthreads();
  const int cx = 1 << a.log_cx, ry = 256 >> a.log_cx;
  const long long col = ((long long)blockIdx.x * cx + (threadIdx.x & (cx - 1))) * V;
  if (col >= a.cols) return;
  int kp[V], kg[V], pmin = 0x7fffffff, pmax = -0x7fffffff - 1;
  bool whole = true;  // one group, no padding
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const bool in = col + v < s.Sk;
    kp[v] = in ? s.k_pos[col + v] : 0;
    kg[v] = in && s.k_grp ? s.k_grp[col + v] : 0;
    whole = whole && in && kg[v] == kg[0];
    pmin = min(pmin, kp[v]);
    pmax = max(pmax, kp[v]);
  }
  for (int i = blockIdx.y * ry + (threadIdx.x >> a.log_cx); i < s.Sq; i += gridDim.y * ry) {
    const int qp = s.q_pos[i], qg = s.q_grp ? s.q_grp[i] : 0;
    E* dst = static_cast<E*>(a.out) + ((long long)h0 * s.Sq + i) * a.pitch + col;
    const long long plane = (long long)s.Sq * a.pitch;
    const int lo = offset_in_lut(pmin, qp, s.reach), hi = offset_in_lut(pmax, qp, s.reach);
    const bool other = whole && kg[0] != qg;
    if (other || (whole && lo == hi)) {
      const E* t = tab + (other ? s.nb - 1 : int(lut[lo]));
#pragma unroll 4
      for (int h = 0; h < hn; ++h, t += rows_tab, dst += plane) {
        RelPiece<E, V> p;
#pragma unroll
        for (int v = 0; v < V; ++v) p.e[v] = *t;
        *reinterpret_cast<RelPiece<E, V>*>(dst) = p;
      }
    } else {
      int b[V];
#pragma unroll
      for (int v = 0; v < V; ++v)
        b[v] = col + v >= s.Sk ? s.nb : kg[v] != qg ? s.nb - 1 : int(lut[offset_in_lut(kp[v], qp, s.reach)]);
      const E* t = tab;
#pragma unroll 4
      for (int h = 0; h < hn; ++h, t += rows_tab, dst += plane) {
        RelPiece<E, V> p;
#pragma unroll
        for (int v = 0; v < V; ++v) p.e[v] = t[b[v]];
        *reinterpret_cast<RelPiece<E, V>*>(dst) = p;
      }
    }
  }
}

template <typename E, int V>
static void launch_rel_fwd(Ctx* c, RelFwdArgs a, cudaStream_t st) {
  const int chunks = (a.cols + V - 1) / V;
  a.log_cx = 0;
  while ((1 << a.log_cx) < chunks && a.log_cx < 8) ++a.log_cx;
  const int cx = 1 << a.log_cx, ry = 256 / cx, gx = (chunks + cx - 1) / cx, gy_most = (a.s.Sq + ry - 1) / ry;
  // heads of a CTA: as many as 32 KB of table hold, fewer where the SMs would otherwise have nothing to do
  a.hg = std::max(1, std::min(a.s.H, int(32768 / ((a.s.nb + 2) * sizeof(E)))));
  while (a.hg > 1 && (long long)gx * gy_most * ((a.s.H + a.hg - 1) / a.hg) < c->sm_count) a.hg = (a.hg + 1) / 2;
  const int gz = (a.s.H + a.hg - 1) / a.hg;
  const int gy = (int)std::max(1ll, std::min({(long long)gy_most, 8ll * c->sm_count / std::max(1ll, (long long)gx * gz), 65535ll}));
  const size_t smem = (((size_t)a.hg * (a.s.nb + 2) * sizeof(E) + 15) & ~size_t(15)) + (2 * a.s.reach + 1) * 2;
  ProfScope ps(c, XFOLD_K_MASK_BIAS, st);
  launch_pdl(rel_bias_kernel<E, V>, dim3(gx, gy, gz), 256, smem, st, a);
}

// ---------------------------------------------------------------------------------------------
// Gradient of the table: dtable[b][h] = sum over (i, j) with b(i, j) = b of grad[h][i][j].
//
// A warp keeps 32 V columns of one head, V neighbours to a lane, and goes down its rows.  Of each 32 columns (a group of
// lanes) a row's entries lie before the reach, behind it or in another group of tokens, all of them: then a lane adds its V to
// one of three sums in registers, at two dozen instructions for 512 bytes.  Or they do not: a band along the diagonal.  Its
// rows are put into shared memory and taken a column to a lane, into sums [nb + 2][32 lanes] of the warp's (a lane's bank is its
// own: no conflicts, no atomics, and the order of the sum is always the same).
// The rows of a CTA lie `slices` apart, so that every warp has its share of the band.  CTAs leave their sums in the workspace; a
// second kernel adds them.
// ---------------------------------------------------------------------------------------------
struct RelBwdArgs {
  RelShared s;
  const void* grad;
  long long sh, sq;       // strides of heads and queries, in elements
  float* partial;         // [H][slices][nb]
  int slices;             // CTAs for each head: rows slice, slice + slices, ...
  int cblocks, row_sets;  // blocks of 32 V columns; sets of rows that warps take such a block in
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }

constexpr int REL_ROWS = 8, REL_HALF = 4;  // rows of a warp that are on their way together; that lie in shared memory
template <int V>
__host__ __device__ constexpr size_t rel_bwd_warp_bytes() { return REL_HALF * 512 + 32 * V * 8; }  // rows; columns' positions, groups

// sum of a piece
__device__ __forceinline__ float piece_sum(const RelPiece<float, 4>& p) { return (p.e[0] + p.e[1]) + (p.e[2] + p.e[3]); }
__device__ __forceinline__ float piece_sum(const RelPiece<bf16, 8>& p) {
  const uint4 u = *reinterpret_cast<const uint4*>(&p);
  float2 t = make_float2(bf16_lo(u.x), bf16_hi(u.x));
  sum2(u.y, t);
  sum2(u.z, t);
  sum2(u.w, t);
  return t.x + t.y;
}

template <typename E, int V, bool VEC, bool GROUPS>
__global__ void __launch_bounds__(256, VEC ? 3 : 2) rel_bias_grad_kernel(const RelBwdArgs a) {
  static_assert(sizeof(E) * V == 16, "a row's 32 V columns take 512 bytes");
  constexpr int W = 32 * V, SHARE = 32 / V;  // columns of a warp; lanes whose neighbours make 32 columns
  extern __shared__ __align__(16) uint8_t smem_raw[];
  const RelShared& s = a.s;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hrows = s.nb + 2;
  uint8_t* own = smem_raw + warp * rel_bwd_warp_bytes<V>();
  E* srow = reinterpret_cast<E*>(own);  // [REL_HALF][W]
  int* skp = reinterpret_cast<int*>(own + REL_HALF * 512);
  int* skg = skp + W;
  float* sums = reinterpret_cast<float*>(smem_raw + warps * rel_bwd_warp_bytes<V>());
  uint16_t* lut = reinterpret_cast<uint16_t*>(sums + (size_t)warps * hrows * 32);
  float* acc = sums + (size_t)warp * hrows * 32 + lane;
  pdl_wait();
  pdl_launch();
  const int h = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  const int rows = (s.Sq - slice + a.slices - 1) / a.slices;  // of this CTA
  const E* g0 = static_cast<const E*>(a.grad) + (long long)h * a.sh;
  float before = 0.f, behind = 0.f, others = 0.f;
  bool staged = false;  // (the table of buckets and the sums are made while the first unit's rows are on their way)
  auto stage = [&]() {
    stage_lut(s, lut, 32);  // (at most 1025 * 32)
    for (int b = 0; b < hrows; ++b) acc[b * 32] = 0.f;
    named_bar_sync(1, blockDim.x);
    staged = true;
  };
  for (int unit = warp; unit < a.cblocks * a.row_sets; unit += warps) {
    const int c0 = unit % a.cblocks * W, set = unit / a.cblocks, c1 = c0 + lane * V;
    RelPiece<E, V> x[REL_ROWS];
    int qp = 0, qg = 0;  // lane u: of row u of the batch
    const E* next = g0 + ((long long)set * a.slices + slice) * a.sq + (VEC && c1 < s.Sk ? c1 : 0);
    const long long step = (long long)a.row_sets * a.slices * a.sq;
    auto load = [&](int n0) {  // rows n0, n0 + row_sets, ..; rows and columns beyond the last are read as the last, and not added
      const int last = (rows - 1 - n0) / a.row_sets;
#pragma unroll
      for (int u = 0; u < REL_ROWS; ++u) {
        const E* row = next + min(u, last) * step;
        if constexpr (VEC) {
          x[u] = *reinterpret_cast<const RelPiece<E, V>*>(row);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) x[u].e[v] = row[min(c0 + v * 32 + lane, s.Sk - 1)];
        }
      }
      next += REL_ROWS * step;
      const int i = min(n0 + (lane & (REL_ROWS - 1)) * a.row_sets, rows - 1) * a.slices + slice;
      qp = s.q_pos[i];
      if (GROUPS) qg = s.q_grp[i];
    };
    if (set < rows) load(set);
    __syncwarp();
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int j = min(c0 + v * 32 + lane, s.Sk - 1);
      skp[v * 32 + lane] = s.k_pos[j];
      if (GROUPS) skg[v * 32 + lane] = s.k_grp[j];
    }
    if (!staged) stage();
    __syncwarp();
    // the lane's 32 columns: before the reach of rows at `after` or later, behind that of rows at `until` or earlier
    int lo = skp[lane * V], hi = lo, grp = GROUPS ? skg[lane * V] : 0, gmax = grp;  // (columns beyond the last repeat it)
#pragma unroll
    for (int v = 1; v < V; ++v) {
      lo = min(lo, skp[lane * V + v]); hi = max(hi, skp[lane * V + v]);
      if (GROUPS) { grp = min(grp, skg[lane * V + v]); gmax = max(gmax, skg[lane * V + v]); }
    }
#pragma unroll
    for (int o = 1; o < SHARE; o <<= 1) {
      lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o)); hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      if (GROUPS) { grp = min(grp, __shfl_xor_sync(0xffffffffu, grp, o)); gmax = max(gmax, __shfl_xor_sync(0xffffffffu, gmax, o)); }
    }
    const bool fits = hi <= 0x7fffffff - s.reach && lo >= s.reach - 0x7fffffff;  // (else as a band)
    const int after = fits ? hi + s.reach : 0, until = fits ? lo - s.reach : 0;
    const bool mine = c1 < s.Sk, same = grp == gmax && fits;
    for (int n0 = set; n0 < rows; n0 += REL_ROWS * a.row_sets) {
      const int bp = qp, bg = qg;
#pragma unroll
      for (int half = 0; half < REL_ROWS; half += REL_HALF) {
        uint32_t band = 0;  // lane u: the lanes of row u whose columns lie in the band
#pragma unroll
        for (int u = half; u < half + REL_HALF; ++u) {
          if (n0 + u * a.row_sets < rows) {
            const int p = __shfl_sync(0xffffffffu, bp, u), g = GROUPS ? __shfl_sync(0xffffffffu, bg, u) : 0;
            const bool other = GROUPS && same && grp != g, in = same && (!GROUPS || grp == g), bef = in && after <= p, beh = in && until >= p;
            const bool out = other || bef || beh;
            const uint32_t b = __ballot_sync(0xffffffffu, mine && !out);
            E* row = srow + (u - half) * W;
            if constexpr (!VEC) {  // a lane's columns lie apart: everything passes through shared memory
#pragma unroll
              for (int v = 0; v < V; ++v) row[v * 32 + lane] = x[u].e[v];
              __syncwarp();
              x[u] = *reinterpret_cast<const RelPiece<E, V>*>(row + lane * V);
#pragma unroll
              for (int v = 0; v < V; ++v)
                if (c1 + v >= s.Sk) x[u].e[v] = E(0.f);
            } else if (b) {
              *reinterpret_cast<RelPiece<E, V>*>(row + lane * V) = x[u];
            }
            const float t = mine ? piece_sum(x[u]) : 0.f;
            if (beh) behind += t;  // (with a reach of nothing a key at the query's own position is on both sides)
            else if (bef) before += t;
            if (GROUPS && other) others += t;
            if (lane == u) band = b;
          }
        }
        __syncwarp();
        if (half + REL_HALF == REL_ROWS && n0 + REL_ROWS * a.row_sets < rows) load(n0 + REL_ROWS * a.row_sets);
        uint32_t todo = __ballot_sync(0xffffffffu, band != 0);
        while (todo) {
          const int u = __ffs(todo) - 1;
          todo &= todo - 1;
          const int p = __shfl_sync(0xffffffffu, bp, u), g = GROUPS ? __shfl_sync(0xffffffffu, bg, u) : 0;
          const int low = low_end(p, s.reach), high = high_end(p, s.reach);
          const E* row = srow + (u - half) * W + lane;
          uint32_t b = __shfl_sync(0xffffffffu, band, u);
          do {
            const int at = (__ffs(b) - 1) / SHARE * 32;  // the first 32 columns left
            b &= ~(((1u << SHARE) - 1) << (at / 32 * SHARE));
            int k = lut[min(max(skp[at + lane], low), high) - p + s.reach];
            if (GROUPS && skg[at + lane] != g) k = (s.nb - 1) * 32;
            if (c0 + at + lane < s.Sk) acc[k] += to_float(row[at]);
          } while (b);
        }
        __syncwarp();
      }
    }
  }
  if (!staged) stage();
  acc[lut[0]] += before;
  acc[lut[2 * s.reach]] += behind;
  acc[(s.nb - 1) * 32] += others;
  __syncthreads();
  // four threads for a bucket, eight lanes' sums of every warp to each
  for (int b = threadIdx.x >> 2; b < (s.nb + 7) / 8 * 8; b += blockDim.x >> 2) {
    float t = 0.f;
    if (b < s.nb)
      for (int w = 0; w < warps; ++w) {
        const float4* q = reinterpret_cast<const float4*>(sums + ((size_t)w * hrows + b) * 32) + (threadIdx.x & 3) * 2;
        t += ((q[0].x + q[0].y) + (q[0].z + q[0].w)) + ((q[1].x + q[1].y) + (q[1].z + q[1].w));
      }
    t += __shfl_xor_sync(0xffffffffu, t, 1);
    t += __shfl_xor_sync(0xffffffffu, t, 2);
    if (b < s.nb && (threadIdx.x & 3) == 0) a.partial[((long long)h * a.slices + slice) * s.nb + b] = t;
  }
}

// dtable[b][h] = sum of the CTAs' parts, a warp for each
__global__ void __launch_bounds__(256) rel_bias_grad_sum_kernel(const float* partial, float* dtable, int nb, int H, int ctas) {
  const int o = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch();
  if (o >= nb * H) return;
  const int b = o / H, h = o % H;
  float t = 0.f;
  for (int i = lane; i < ctas; i += 32) t += partial[((long long)h * ctas + i) * nb + b];
  t = warp_total(t);
  if (lane == 0) dtable[o] = t;
}

struct RelBwdPlan {
  int warps, slices, cblocks, row_sets;
  size_t smem;
};
// CTAs for each head: three or two to an SM, by their registers and their sums' room
static int rel_bwd_slices(int nb, int H, int Sq, bool vec, int sms) {
  const int per_sm = vec && (size_t)(nb + 2) * 128 * 8 <= 36 * 1024 ? 3 : 2;
  return std::max(1, std::min(per_sm * sms / H, (Sq + 7) / 8));
}
static RelBwdPlan rel_bwd_plan(int nb, int H, int Sq, int Sk, int reach, int V, bool vec, int sms) {
  RelBwdPlan p;
  const size_t per_warp = (size_t)(nb + 2) * 128 + (V == 8 ? rel_bwd_warp_bytes<8>() : rel_bwd_warp_bytes<4>()), rest = (2 * reach + 1) * 2;
  p.warps = 8;
  while (p.warps > 1 && p.warps * per_warp + rest > 113 * 1024) p.warps /= 2;
  p.smem = p.warps * per_warp + rest;
  p.slices = rel_bwd_slices(nb, H, Sq, vec, sms);
  p.cblocks = (Sk + 32 * V - 1) / (32 * V);
  // sets of rows: the warps' rounds over the units are to come out even, but a unit costs about as much as four rows to begin
  const int rows = (Sq + p.slices - 1) / p.slices;
  double best = 1e30;
  for (int n = 1; n <= 8; n *= 2) {
    const double cost = double((p.cblocks * n + p.warps - 1) / p.warps) * ((rows + n - 1) / n + 4);
    if (cost < best) {
      best = cost;
      p.row_sets = n;
    }
  }
  return p;
}

template <typename E, int V, bool VEC>
static int launch_rel_bwd(Ctx* c, RelBwdArgs a, const RelBwdPlan& p, cudaStream_t st) {
  auto kern = a.s.k_grp ? rel_bias_grad_kernel<E, V, VEC, true> : rel_bias_grad_kernel<E, V, VEC, false>;
  static bool attr_done[8] = {false};
  if (!attr_done[c->device & 7]) {
    cudaError_t e = cudaFuncSetAttribute(rel_bias_grad_kernel<E, V, VEC, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(rel_bias_grad_kernel<E, V, VEC, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return fail(c, XFOLD_ERR_LAUNCH, "relative bias gradient: %s", cudaGetErrorString(e));
    attr_done[c->device & 7] = true;
  }
  ProfScope ps(c, XFOLD_K_MASK_BIAS, st);
  launch_pdl(kern, dim3(a.s.H * a.slices), p.warps * 32, p.smem, st, a);
  return check_launch(c, "rel_bias_grad_kernel");
}

static int rel_check(Ctx* c, int nb, int H, int reach, int Sq, int Sk, const void* lut, const void* qp, const void* kp,
                     const void* qg, const void* kg) {
  if (Sq < 0 || Sk < 0 || H < 1 || nb < 1) return fail(c, XFOLD_ERR_ARG, "relative bias: sizes");
  if (nb > 1024 || reach < 0 || reach > 4096) return fail(c, XFOLD_ERR_ARG, "relative bias: up to 1024 buckets and a reach up to 4096");
  if (H > 65535) return fail(c, XFOLD_ERR_ARG, "relative bias: too many heads");
  if (!lut || (Sq && !qp) || (Sk && !kp)) return fail(c, XFOLD_ERR_ARG, "relative bias: null argument");
  if ((qg != nullptr) != (kg != nullptr) && Sq && Sk) return fail(c, XFOLD_ERR_ARG, "relative bias: groups of queries and keys come together");
  return XFOLD_OK;
}

// ---------------------------------------------------------------------------------------------
// Norms of queries and keys for each head, and the rotation by position.
//   y = x * rsqrt(mean(x^2) + eps) * w * scale; of its first `rot` elements the pairs (a, b) become
//   (a cos t - b sin t, b cos t + a sin t), t = position * freq of the pair.
// Pairs are (i, i + rot / 2), or neighbours (2 i, 2 i + 1).
//
// G lanes share a head; a lane holds two pieces of V elements that rotate into each other: of the halves, or 2 V neighbours
// (beyond `rot`: 2 V neighbours that do not rotate).  Its place in the head is the same for all heads, so weights, cosines and
// sines stay in registers while a warp goes through its token's heads.  Angles are made once for a token and warp, in turns and
// in 64 bits until the whole turns are gone: 32 bits would lose far positions.
// ---------------------------------------------------------------------------------------------
struct QkTensor {
  const void *x, *d;  // d: gradient of the result (backward)
  void* y;
  long long xb, xt, xh, db, dt, dh, yb, yt, yh;  // strides of batch, token and head, in elements
  const float* w;
  float scale;
  int H, passes;
};
struct QkArgs {
  QkTensor t[2];
  const double* freqs;
  const int* pos;
  long long pos_b;
  int B, S, D, rot, log_g, parts, per_part;
  float eps;
  float* partial;  // backward: [CTAs][2][D]
};

template <int BYTES>
struct PieceOf;
template <> struct PieceOf<16> { typedef uint4 type; };
template <> struct PieceOf<8> { typedef uint2 type; };
template <> struct PieceOf<4> { typedef uint32_t type; };
template <> struct PieceOf<2> { typedef uint16_t type; };

template <typename T, int V>
struct Piece {
  typename PieceOf<sizeof(T) * V>::type raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const decltype(raw)*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<decltype(raw)*>(p) = raw; }
  __device__ __forceinline__ void clear() { raw = decltype(raw){}; }
  __device__ __forceinline__ void get(float (&f)[V]) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = to_float(e[v]);
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if constexpr (sizeof(T) == 4) e[v] = f[v];
      else e[v] = __float2bfloat16(f[v]);
    }
  }
};

// slots (pairs of pieces) of a lane: heads are at most 256 wide, so 32 lanes with pieces of 4 hold one
template <int V>
__host__ __device__ constexpr int qk_slots() { return V >= 4 ? 1 : 4 / V; }

// where the pieces of slot sl lie; < 0: behind the head's end
template <int V, bool NEIGH>
__device__ __forceinline__ void qk_place(const QkArgs& a, int sl, int& pa, int& pb, int& angle) {
  const int turning = a.rot / (2 * V);
  if (sl < turning) {
    pa = NEIGH ? 2 * V * sl : V * sl;
    pb = NEIGH ? pa + V : pa + a.rot / 2;
    angle = V * sl;
  } else {
    pa = 2 * V * sl;  // = rot + 2 V (sl - turning)
    pb = pa + V;
    angle = -1;
    if (pa >= a.D) pa = -1;
  }
}

// the pairs of (x, y) turned by their angles (SIGN -1: back)
template <int V, bool NEIGH, int SIGN>
__device__ __forceinline__ void qk_turn(float (&x)[V], float (&y)[V], const float2 (&cs)[V]) {
  if constexpr (NEIGH && V > 1) {
#pragma unroll
    for (int v = 0; v < V; v += 2) {  // the pair of angle v / 2 lies in x, that of angle V / 2 + v / 2 in y
      const float2 c = cs[v / 2], d = cs[V / 2 + v / 2];
      const float sx = SIGN * c.y, sy = SIGN * d.y;
      const float x0 = x[v], x1 = x[v + 1], y0 = y[v], y1 = y[v + 1];
      x[v] = x0 * c.x - x1 * sx;
      x[v + 1] = x1 * c.x + x0 * sx;
      y[v] = y0 * d.x - y1 * sy;
      y[v + 1] = y1 * d.x + y0 * sy;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float p = x[v], q = y[v], sn = SIGN * cs[v].y;
      x[v] = p * cs[v].x - q * sn;
      y[v] = q * cs[v].x + p * sn;
    }
  }
}

// cosines and sines of a token's angles, by a warp, into shared memory, and from there those of the lane's slots
template <int V, bool NEIGH>
__device__ __forceinline__ void qk_angles(const QkArgs& a, int b, int t, float2* sm, const int (&angle)[qk_slots<V>()],
                                          float2 (&cs)[qk_slots<V>()][V]) {
  const int lane = threadIdx.x & 31;
  const double p = a.pos ? a.pos[b * a.pos_b + t] : t;
  __syncwarp();
  for (int i = lane; i < a.rot / 2; i += 32) {
    const double turns = p * (a.freqs[i] * 0.15915494309189533577);  // 1 / (2 pi)
    float c, s;
    sincospif(2.f * float(turns - rint(turns)), &s, &c);
    sm[i] = make_float2(c, s);
  }
  __syncwarp();
#pragma unroll
  for (int n = 0; n < qk_slots<V>(); ++n)
#pragma unroll
    for (int v = 0; v < V; ++v) cs[n][v] = angle[n] >= 0 ? sm[angle[n] + v] : make_float2(1.f, 0.f);
}

__device__ __forceinline__ float group_total(float v, int log_g) {
  for (int o = 1; o < (1 << log_g); o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int QK_WARPS = 4;

template <typename T, int V, bool NEIGH>
__global__ void __launch_bounds__(QK_WARPS * 32) qk_norm_rotate_kernel(const QkArgs a) {
  constexpr int NS = qk_slots<V>();
  constexpr int U = NS == 1 ? 4 : 1;  // heads whose loads are on their way together
  __shared__ float2 sm[QK_WARPS][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * QK_WARPS + warp;
  pdl_wait();
  pdl_launch();
  if (item >= (long long)a.B * a.S * a.parts) return;
  const int part = int(item % a.parts);
  const long long token = item / a.parts;
  const int b = int(token / a.S), t = int(token % a.S);
  int pa[NS], pb[NS], angle[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) qk_place<V, NEIGH>(a, (lane & ((1 << a.log_g) - 1)) + n * 32, pa[n], pb[n], angle[n]);
  float2 cs[NS][V];
  qk_angles<V, NEIGH>(a, b, t, sm[warp], angle, cs);
  const int per_pass = 32 >> a.log_g, sub = lane >> a.log_g;
  const float inv_d = 1.f / a.D;
  int p0 = part * a.per_part, p1 = p0 + a.per_part;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const QkTensor& q = a.t[which];
    const int first = max(p0, 0), last = min(p1, q.passes);
    p0 -= q.passes;
    p1 -= q.passes;
    if (first >= last) continue;
    float wa[NS][V], wb[NS][V];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        wa[n][v] = (q.w && pa[n] >= 0 ? q.w[pa[n] + v] : 1.f) * q.scale;
        wb[n][v] = (q.w && pa[n] >= 0 ? q.w[pb[n] + v] : 1.f) * q.scale;
      }
    const T* src = static_cast<const T*>(q.x) + b * q.xb + t * q.xt;
    T* dst = static_cast<T*>(q.y) + b * q.yb + t * q.yt;
    for (int p = first; p < last; p += U) {
      Piece<T, V> xa[U][NS], xb[U][NS];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = (p + u) * per_pass + sub;
        const bool in = p + u < last && h < q.H;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          if (in && pa[n] >= 0) {
            xa[u][n].load(src + h * q.xh + pa[n]);
            xb[u][n].load(src + h * q.xh + pb[n]);
          } else {
            xa[u][n].clear();
            xb[u][n].clear();
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = (p + u) * per_pass + sub;
        const bool in = p + u < last && h < q.H;
        float fa[NS][V], fb[NS][V], ss = 0.f;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          xa[u][n].get(fa[n]);
          xb[u][n].get(fb[n]);
#pragma unroll
          for (int v = 0; v < V; ++v) ss += fa[n][v] * fa[n][v] + fb[n][v] * fb[n][v];
        }
        const float r = rsqrtf(group_total(ss, a.log_g) * inv_d + a.eps);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            fa[n][v] = fa[n][v] * r * wa[n][v];
            fb[n][v] = fb[n][v] * r * wb[n][v];
          }
          if (angle[n] >= 0) qk_turn<V, NEIGH, 1>(fa[n], fb[n], cs[n]);
          if (in && pa[n] >= 0) {
            xa[u][n].set(fa[n]);
            xb[u][n].set(fb[n]);
            xa[u][n].store(dst + h * q.yh + pa[n]);
            xb[u][n].store(dst + h * q.yh + pb[n]);
          }
        }
      }
    }
  }
}

// Backward, with g = the gradient turned back, times the scale, and r = rsqrt(mean(x^2) + eps):
//   dw_i = sum over tokens and heads of g_i x_i r;  dx = r (g w - x r^2 mean(g w x)).
// A lane's place in the head is always the same, so the weights' gradients are sums in its registers until the end.
template <typename T, int V, bool NEIGH>
__global__ void __launch_bounds__(QK_WARPS * 32) qk_norm_rotate_grad_kernel(const QkArgs a) {
  constexpr int NS = qk_slots<V>();
  constexpr int U = NS == 1 ? 2 : 1;
  __shared__ float2 sm[QK_WARPS][128];
  __shared__ float red[2][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch();
  int pa[NS], pb[NS], angle[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) qk_place<V, NEIGH>(a, (lane & ((1 << a.log_g) - 1)) + n * 32, pa[n], pb[n], angle[n]);
  const int per_pass = 32 >> a.log_g, sub = lane >> a.log_g;
  const float inv_d = 1.f / a.D;
  float da[2][NS][V], db[2][NS][V];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int v = 0; v < V; ++v) da[w][n][v] = db[w][n][v] = 0.f;
  const long long items = (long long)a.B * a.S * a.parts;
  for (long long item = (long long)blockIdx.x * QK_WARPS + warp; item < items; item += (long long)gridDim.x * QK_WARPS) {
    const int part = int(item % a.parts);
    const long long token = item / a.parts;
    const int b = int(token / a.S), t = int(token % a.S);
    float2 cs[NS][V];
    qk_angles<V, NEIGH>(a, b, t, sm[warp], angle, cs);
    int p0 = part * a.per_part, p1 = p0 + a.per_part;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const QkTensor& q = a.t[which];
      const int first = max(p0, 0), last = min(p1, q.passes);
      p0 -= q.passes;
      p1 -= q.passes;
      if (first >= last) continue;
      float wa[NS][V], wb[NS][V];
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          wa[n][v] = q.w && pa[n] >= 0 ? q.w[pa[n] + v] : 1.f;
          wb[n][v] = q.w && pa[n] >= 0 ? q.w[pb[n] + v] : 1.f;
        }
      const T* src = static_cast<const T*>(q.x) + b * q.xb + t * q.xt;
      const T* grd = static_cast<const T*>(q.d) + b * q.db + t * q.dt;
      T* dst = static_cast<T*>(q.y) + b * q.yb + t * q.yt;
      for (int p = first; p < last; p += U) {
        Piece<T, V> xa[U][NS], xb[U][NS], ga[U][NS], gb[U][NS];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = (p + u) * per_pass + sub;
          const bool in = p + u < last && h < q.H;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            if (in && pa[n] >= 0) {
              xa[u][n].load(src + h * q.xh + pa[n]);
              xb[u][n].load(src + h * q.xh + pb[n]);
              ga[u][n].load(grd + h * q.dh + pa[n]);
              gb[u][n].load(grd + h * q.dh + pb[n]);
            } else {
              xa[u][n].clear();
              xb[u][n].clear();
              ga[u][n].clear();
              gb[u][n].clear();
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = (p + u) * per_pass + sub;
          const bool in = p + u < last && h < q.H;
          float fa[NS][V], fb[NS][V], ea[NS][V], eb[NS][V], ss = 0.f, sg = 0.f;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            xa[u][n].get(fa[n]);
            xb[u][n].get(fb[n]);
            ga[u][n].get(ea[n]);
            gb[u][n].get(eb[n]);
            if (angle[n] >= 0) qk_turn<V, NEIGH, -1>(ea[n], eb[n], cs[n]);
#pragma unroll
            for (int v = 0; v < V; ++v) {
              ea[n][v] *= q.scale;
              eb[n][v] *= q.scale;
              ss += fa[n][v] * fa[n][v] + fb[n][v] * fb[n][v];
              sg += fa[n][v] * (ea[n][v] * wa[n][v]) + fb[n][v] * (eb[n][v] * wb[n][v]);
            }
          }
          const float r = rsqrtf(group_total(ss, a.log_g) * inv_d + a.eps);
          const float m = group_total(sg, a.log_g) * inv_d * r * r;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
              da[which][n][v] += ea[n][v] * fa[n][v] * r;
              db[which][n][v] += eb[n][v] * fb[n][v] * r;
              fa[n][v] = r * (ea[n][v] * wa[n][v] - fa[n][v] * m);
              fb[n][v] = r * (eb[n][v] * wb[n][v] - fb[n][v] * m);
            }
            if (in && pa[n] >= 0) {
              xa[u][n].set(fa[n]);
              xb[u][n].set(fb[n]);
              xa[u][n].store(dst + h * q.yh + pa[n]);
              xb[u][n].store(dst + h * q.yh + pb[n]);
            }
          }
        }
      }
    }
  }
  // lanes with the same place in other heads, then the warps one after the other
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int v = 0; v < V; ++v)
        for (int o = 1 << a.log_g; o < 32; o <<= 1) {
          da[w][n][v] += __shfl_xor_sync(0xffffffffu, da[w][n][v], o);
          db[w][n][v] += __shfl_xor_sync(0xffffffffu, db[w][n][v], o);
        }
  }
  for (int turn = 0; turn < QK_WARPS; ++turn) {
    if (warp == turn && sub == 0) {
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int n = 0; n < NS; ++n)
          if (pa[n] >= 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
              red[w][pa[n] + v] = (turn ? red[w][pa[n] + v] : 0.f) + da[w][n][v];
              red[w][pb[n] + v] = (turn ? red[w][pb[n] + v] : 0.f) + db[w][n][v];
            }
          }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * a.D; i += QK_WARPS * 32) a.partial[(long long)blockIdx.x * 2 * a.D + i] = red[i / a.D][i % a.D];
}

__global__ void __launch_bounds__(256) qk_weight_grad_kernel(const float* partial, float* dqw, float* dkw, int D, int ctas) {
  const int o = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch();
  if (o >= 2 * D) return;
  float* dst = o < D ? dqw : dkw;
  if (!dst) return;
  float t = 0.f;
  for (int i = lane; i < ctas; i += 32) t += partial[(long long)i * 2 * D + o];
  t = warp_total(t);
  if (lane == 0) dst[o % D] = t;
}

static int qk_ctas(const Ctx* c) { return 4 * c->sm_count; }

// the widest pieces that sizes, strides and addresses allow
static int qk_piece(const QkArgs& a, int elem, bool grad) {
  int V = 16 / elem;
  auto fits = [&](int v) {
    if (a.rot % (2 * v) || (a.D - a.rot) % (2 * v)) return false;
    for (const QkTensor& q : a.t) {
      if (!q.H) continue;
      long long all = q.xb | q.xt | q.xh | q.yb | q.yt | q.yh | (grad ? q.db | q.dt | q.dh : 0);
      uintptr_t ptr = (uintptr_t)q.x | (uintptr_t)q.y | (grad ? (uintptr_t)q.d : 0);
      if (all % v || ptr % (v * elem)) return false;
    }
    return true;
  };
  while (V > 1 && !fits(V)) V /= 2;
  return V;
}

template <typename T, int V, bool GRAD>
static void launch_qk_one(Ctx* c, QkArgs& a, int neighbours, int grid, cudaStream_t st) {
  if constexpr (GRAD) {
    if (neighbours) launch_pdl(qk_norm_rotate_grad_kernel<T, V, true>, dim3(grid), QK_WARPS * 32, 0, st, a);
    else launch_pdl(qk_norm_rotate_grad_kernel<T, V, false>, dim3(grid), QK_WARPS * 32, 0, st, a);
  } else {
    if (neighbours) launch_pdl(qk_norm_rotate_kernel<T, V, true>, dim3(grid), QK_WARPS * 32, 0, st, a);
    else launch_pdl(qk_norm_rotate_kernel<T, V, false>, dim3(grid), QK_WARPS * 32, 0, st, a);
  }
}

template <bool GRAD>
static void launch_qk_wide(Ctx* c, QkArgs& a, int f32, int V, int neighbours, int grid, cudaStream_t st) {
  if (f32) {
    if (V == 4) launch_qk_one<float, 4, GRAD>(c, a, neighbours, grid, st);
    else if (V == 2) launch_qk_one<float, 2, GRAD>(c, a, neighbours, grid, st);
    else launch_qk_one<float, 1, GRAD>(c, a, neighbours, grid, st);
  } else {
    if (V == 8) launch_qk_one<bf16, 8, GRAD>(c, a, neighbours, grid, st);
    else if (V == 4) launch_qk_one<bf16, 4, GRAD>(c, a, neighbours, grid, st);
    else if (V == 2) launch_qk_one<bf16, 2, GRAD>(c, a, neighbours, grid, st);
    else launch_qk_one<bf16, 1, GRAD>(c, a, neighbours, grid, st);
  }
}

template <bool GRAD>
static int launch_qk(Ctx* c, QkArgs a, int f32, int neighbours, cudaStream_t st, float* dqw = nullptr, float* dkw = nullptr) {
  const int V = qk_piece(a, f32 ? 4 : 2, GRAD), slots = (a.D / 2 + V - 1) / V;
  a.log_g = 0;
  while ((1 << a.log_g) < slots && a.log_g < 5) ++a.log_g;
  int passes = 0;
  for (QkTensor& q : a.t) {
    q.passes = (q.H + (32 >> a.log_g) - 1) / (32 >> a.log_g);
    passes += q.passes;
  }
  // a warp for each token, or several where that leaves warps without work
  const long long tokens = (long long)a.B * a.S, want = 16ll * c->sm_count;
  a.parts = (int)std::max(1ll, std::min<long long>(passes, want / std::max(1ll, tokens)));
  a.per_part = (passes + a.parts - 1) / a.parts;
  a.parts = (passes + a.per_part - 1) / a.per_part;
  const long long ctas = (tokens * a.parts + QK_WARPS - 1) / QK_WARPS;
  if (ctas > 0x7fffffffll) return fail(c, XFOLD_ERR_ARG, "qk norm: too many tokens");
  const int grid = GRAD ? (int)std::min<long long>(ctas, qk_ctas(c)) : (int)ctas;
  {
    ProfScope ps(c, XFOLD_K_LAYERNORM, st);
    launch_qk_wide<GRAD>(c, a, f32, V, neighbours, grid, st);
  }
  if (int rc = check_launch(c, "qk_norm_rotate")) return rc;
  if (!dqw && !dkw) return XFOLD_OK;
  ProfScope ps(c, XFOLD_K_LAYERNORM, st);
  launch_pdl(qk_weight_grad_kernel, dim3((2 * a.D + 7) / 8), 256, 0, st, (const float*)a.partial, dqw, dkw, a.D, grid);
  return check_launch(c, "qk_weight_grad_kernel");
}

// the call's description as the kernels take it
static int qk_fill(Ctx* c, const xfold_qk_norm* n, QkArgs& a, bool grad, const char* what) {
  if (!n) return fail(c, XFOLD_ERR_ARG, "%s: null argument", what);
  if (n->B < 0 || n->S < 0 || n->Hq < 0 || n->Hk < 0 || n->D < 2 || n->D > 256 || n->D % 2)
    return fail(c, XFOLD_ERR_ARG, "%s: sizes (heads of an even width up to 256)", what);
  if (n->rot < 0 || n->rot > n->D || n->rot % 2 || (n->rot && !n->freqs)) return fail(c, XFOLD_ERR_ARG, "%s: an even part of a head is rotated, with its frequencies", what);
  if (n->is_f32 != 0 && n->is_f32 != 1) return fail(c, XFOLD_ERR_ARG, "%s: type", what);
  if (!(n->eps >= 0.f)) return fail(c, XFOLD_ERR_ARG, "%s: eps", what);
  a = QkArgs{};
  a.B = n->B; a.S = n->S; a.D = n->D; a.rot = n->rot;
  a.freqs = n->freqs; a.pos = n->positions; a.pos_b = n->pos_batch_stride;
  a.eps = n->eps;
  const xfold_heads *x[2] = {&n->q, &n->k}, *y[2] = {&n->q_result, &n->k_result}, *d[2] = {&n->q_grad, &n->k_grad};
  for (int i = 0; i < 2; ++i) {
    QkTensor& t = a.t[i];
    t.H = i ? n->Hk : n->Hq;
    t.w = i ? n->k_weight : n->q_weight;
    t.scale = i ? 1.f : n->q_scale;
    if (!t.H || !a.B || !a.S) continue;
    if (!x[i]->at || !y[i]->at || (grad && !d[i]->at)) return fail(c, XFOLD_ERR_ARG, "%s: null argument", what);
    t.x = x[i]->at; t.xb = x[i]->batch; t.xt = x[i]->token; t.xh = x[i]->head;
    t.y = const_cast<void*>(y[i]->at); t.yb = y[i]->batch; t.yt = y[i]->token; t.yh = y[i]->head;
    if (grad) { t.d = d[i]->at; t.db = d[i]->batch; t.dt = d[i]->token; t.dh = d[i]->head; }
    if (((uintptr_t)t.x | (uintptr_t)t.y | (uintptr_t)t.d) % (n->is_f32 ? 4 : 2)) return fail(c, XFOLD_ERR_ARG, "%s: alignment", what);
  }
  return XFOLD_OK;
}

}  // namespace xf

using namespace xf;

extern "C" {

int xfold_relative_bias_fwd(xfold_ctx* cx, const float* table, int num_buckets, int H, const int* buckets, int reach, const int* q_pos,
                            const int* k_pos, const int* q_group, const int* k_group, int Sq, int Sk, int form, void* out,
                            void* stream) {
  if (!cx) return XFOLD_ERR_ARG;
  Ctx* c = reinterpret_cast<Ctx*>(cx);
  CallLock call(c);
  if (int rc = rel_check(c, num_buckets, H, reach, Sq, Sk, buckets, q_pos, k_pos, q_group, k_group)) return rc;
  if (form < 0 || form > 2) return fail(c, XFOLD_ERR_ARG, "relative bias: form");
  if (!Sq || !Sk) return XFOLD_OK;
  if (!table || !out) return fail(c, XFOLD_ERR_ARG, "relative bias: null argument");
  DeviceGuard dev(c);
  cudaStream_t st = (cudaStream_t)stream;
  RelFwdArgs a{};
  a.s = RelShared{buckets, q_pos, k_pos, q_group, k_group, reach, num_buckets, H, Sq, Sk};
  a.table = table;
  a.out = out;
  a.pitch = form == XFOLD_BIAS_PREPARED ? pad8(Sk) : Sk;
  a.cols = (int)a.pitch;
  const int elem = form == XFOLD_BIAS_F32 ? 4 : 2, wide = 16 / elem;
  if ((uintptr_t)out % elem) return fail(c, XFOLD_ERR_ARG, "relative bias: alignment of the result");
  const bool vec = a.pitch % wide == 0 && (uintptr_t)out % 16 == 0;
  if (form == XFOLD_BIAS_F32) vec ? launch_rel_fwd<float, 4>(c, a, st) : launch_rel_fwd<float, 1>(c, a, st);
  else if (form == XFOLD_BIAS_BF16) vec ? launch_rel_fwd<bf16, 8>(c, a, st) : launch_rel_fwd<bf16, 1>(c, a, st);
  else vec ? launch_rel_fwd<__half, 8>(c, a, st) : launch_rel_fwd<__half, 1>(c, a, st);
  return check_launch(c, "rel_bias_kernel");
}

size_t xfold_relative_bias_bwd_workspace_bytes(xfold_ctx* cx, int num_buckets, int H, int Sq, int Sk) {
  if (!cx || num_buckets < 1 || H < 1 || Sq < 1 || Sk < 1) return 0;
  const Ctx* c = reinterpret_cast<const Ctx*>(cx);
  return (size_t)rel_bwd_slices(num_buckets, H, Sq, true, c->sm_count) * H * num_buckets * sizeof(float);
}

int xfold_relative_bias_bwd(xfold_ctx* cx, const void* grad, int is_f32, long long head_stride, long long query_stride, int num_buckets,
                            int H, const int* buckets, int reach, const int* q_pos, const int* k_pos, const int* q_group,
                            const int* k_group, int Sq, int Sk, float* dtable, void* ws, size_t ws_bytes, void* stream) {
  if (!cx) return XFOLD_ERR_ARG;
  Ctx* c = reinterpret_cast<Ctx*>(cx);
  CallLock call(c);
  if (int rc = rel_check(c, num_buckets, H, reach, Sq, Sk, buckets, q_pos, k_pos, q_group, k_group)) return rc;
  if (is_f32 != 0 && is_f32 != 1) return fail(c, XFOLD_ERR_ARG, "relative bias gradient: type");
  if (!dtable) return fail(c, XFOLD_ERR_ARG, "relative bias gradient: null argument");
  DeviceGuard dev(c);
  cudaStream_t st = (cudaStream_t)stream;
  if (!Sq || !Sk) {
    if (cudaMemsetAsync(dtable, 0, sizeof(float) * H * num_buckets, st) != cudaSuccess) return check_launch(c, "relative bias gradient");
    return XFOLD_OK;
  }
  if (!grad || (uintptr_t)grad % (is_f32 ? 4 : 2)) return fail(c, XFOLD_ERR_ARG, "relative bias gradient: the gradient's address");
  const int V = is_f32 ? 4 : 8;
  const bool vec = (uintptr_t)grad % 16 == 0 && head_stride % V == 0 && query_stride % V == 0 && Sk % V == 0;
  const RelBwdPlan p = rel_bwd_plan(num_buckets, H, Sq, Sk, reach, V, vec, c->sm_count);
  if (!ws || (uintptr_t)ws % 4 || ws_bytes < sizeof(float) * (size_t)H * p.slices * num_buckets)
    return fail(c, XFOLD_ERR_ARG, "relative bias gradient: workspace too small");
  RelBwdArgs a{};
  a.s = RelShared{buckets, q_pos, k_pos, q_group, k_group, reach, num_buckets, H, Sq, Sk};
  a.grad = grad;
  a.sh = head_stride;
  a.sq = query_stride;
  a.partial = (float*)ws;
  a.slices = p.slices;
  a.cblocks = p.cblocks;
  a.row_sets = p.row_sets;
  int rc = is_f32 ? (vec ? launch_rel_bwd<float, 4, true>(c, a, p, st) : launch_rel_bwd<float, 4, false>(c, a, p, st))
                  : (vec ? launch_rel_bwd<bf16, 8, true>(c, a, p, st) : launch_rel_bwd<bf16, 8, false>(c, a, p, st));
  if (rc) return rc;
  ProfScope ps(c, XFOLD_K_MASK_BIAS, st);
  launch_pdl(rel_bias_grad_sum_kernel, dim3((num_buckets * H + 7) / 8), 256, 0, st, (const float*)a.partial, dtable, num_buckets, H, p.slices);
  return check_launch(c, "rel_bias_grad_sum_kernel");
}

int xfold_qk_norm_rotate_fwd(xfold_ctx* cx, const xfold_qk_norm* n, void* stream) {
  if (!cx) return XFOLD_ERR_ARG;
  Ctx* c = reinterpret_cast<Ctx*>(cx);
  CallLock call(c);
  QkArgs a;
  if (int rc = qk_fill(c, n, a, false, "qk norm")) return rc;
  if (!a.B || !a.S || !(n->Hq + n->Hk)) return XFOLD_OK;
  DeviceGuard dev(c);
  return launch_qk<false>(c, a, n->is_f32, n->neighbours, (cudaStream_t)stream);
}

size_t xfold_qk_norm_rotate_bwd_workspace_bytes(xfold_ctx* cx, int D) {
  return cx && D > 0 ? (size_t)qk_ctas(reinterpret_cast<const Ctx*>(cx)) * 2 * D * sizeof(float) : 0;
}

int xfold_qk_norm_rotate_bwd(xfold_ctx* cx, const xfold_qk_norm* n, float* dq_weight, float* dk_weight, void* ws, size_t ws_bytes, void* stream) {
  if (!cx) return XFOLD_ERR_ARG;
  Ctx* c = reinterpret_cast<Ctx*>(cx);
  CallLock call(c);
  QkArgs a;
  if (int rc = qk_fill(c, n, a, true, "qk norm gradient")) return rc;
  DeviceGuard dev(c);
  cudaStream_t st = (cudaStream_t)stream;
  if (!a.B || !a.S || !(n->Hq + n->Hk)) {
    for (float* w : {dq_weight, dk_weight})
      if (w && cudaMemsetAsync(w, 0, sizeof(float) * a.D, st) != cudaSuccess) return check_launch(c, "qk norm gradient");
    return XFOLD_OK;
  }
  if (!ws || (uintptr_t)ws % 4 || ws_bytes < xfold_qk_norm_rotate_bwd_workspace_bytes(cx, a.D))
    return fail(c, XFOLD_ERR_ARG, "qk norm gradient: workspace too small");
  a.partial = (float*)ws;
  return launch_qk<true>(c, a, n->is_f32, n->neighbours, st, dq_weight, dk_weight);
}

}  // extern "C"
