// Positions in attention: a learned bias of the logits by buckets of relative position, with the gradient of its table, and
// the norms of queries and keys for each head together with the rotation by position, with their gradients.  All of them are
// bound by what they read and write; the compiler's fast approximations stay off here (see build.py).
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

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
// the CTA.  Where the V columns share a bucket (beyond the reach, or in another group), and those of the warp's other lanes do
// too, a head's value is fetched once.  Bound by the result's bytes, in the order that CTAs come by them: 16 heads x 2048^2
// float32 44 us (a fill with zeros 37), 16 bits 24, prepared 16 x 1999 x 2000 24.  Rows of odd lengths as plain numbers are
// written element by element (16 x 1999^2 float32 67, 16 bits 47).
template <typename E, int V>
__global__ void __launch_bounds__(256, V == 1 ? 4 : 0) rel_bias_kernel(const RelFwdArgs a) {
  extern __shared__ uint8_t smem_raw[];
  const RelShared& s = a.s;
  const int rows_tab = s.nb + 2, h0 = blockIdx.z * a.hg, hn = min(a.hg, s.H - h0);
  E* tab = reinterpret_cast<E*>(smem_raw);  // [hg][nb + 2]: row nb is zero, row nb + 1 not a number
  uint16_t* lut = reinterpret_cast<uint16_t*>(smem_raw + (((size_t)a.hg * rows_tab * sizeof(E) + 15) & ~size_t(15)));
  const int cx = 1 << a.log_cx, ry = 256 >> a.log_cx;
  const long long col = ((long long)blockIdx.x * cx + (threadIdx.x & (cx - 1))) * V;
  pdl_wait();
  pdl_launch();
  // the columns' positions are on their way while the table is made
  int kp[V], kg[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const bool in = col + v < s.Sk;
    kp[v] = in ? s.k_pos[col + v] : 0;
    kg[v] = in && s.k_grp ? s.k_grp[col + v] : 0;
  }
  stage_lut(s, lut);
#pragma unroll 4
  for (int i = threadIdx.x; i < hn * rows_tab; i += 256) {
    const int b = i / hn, h = i - b * hn;
    rel_value(b < s.nb ? a.table[(long long)b * s.H + h0 + h] : b == s.nb ? 0.f : __int_as_float(0x7fffffff), tab[h * rows_tab + b]);
  }
  __syncthreads();
  if (col >= a.cols) return;
  int pmin = 0x7fffffff, pmax = -0x7fffffff - 1;
  bool whole = true;  // one group, no padding
#pragma unroll
  for (int v = 0; v < V; ++v) {
    whole = whole && col + v < s.Sk && kg[v] == kg[0];
    pmin = min(pmin, kp[v]);
    pmax = max(pmax, kp[v]);
  }
  for (int i = blockIdx.y * ry + (threadIdx.x >> a.log_cx); i < s.Sq; i += gridDim.y * ry) {
    const int qp = s.q_pos[i], qg = s.q_grp ? s.q_grp[i] : 0;
    E* dst = static_cast<E*>(a.out) + ((long long)h0 * s.Sq + i) * a.pitch + col;
    const long long plane = (long long)s.Sq * a.pitch;
    const int lo = offset_in_lut(pmin, qp, s.reach), hi = offset_in_lut(pmax, qp, s.reach);
    const bool other = whole && kg[0] != qg;
    const bool alike = other || (whole && lo == hi);
    if (__all_sync(__activemask(), alike)) {  // (whichever lanes are together: a warp goes one way, not both)
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
#pragma unroll(V == 8 ? 1 : 4)  // (eight reads of the table are enough on their way, and 64 registers let four CTAs on an SM)
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
  // heads of a CTA: as many as 32 KB of table hold (less where the buckets of the longest reach leave less of 48 KB), fewer where
  // the SMs would otherwise have nothing to do
  const size_t lut = (2 * a.s.reach + 1) * 2, room = std::min<size_t>(32768, (48 * 1024 - lut) & ~size_t(15));
  a.hg = std::max(1, std::min(a.s.H, int(room / ((a.s.nb + 2) * sizeof(E)))));
  while (a.hg > 1 && (long long)gx * gy_most * ((a.s.H + a.hg - 1) / a.hg) < c->sm_count) a.hg = (a.hg + 1) / 2;
  const int gz = (a.s.H + a.hg - 1) / a.hg;
  const int gy = (int)std::max(1ll, std::min({(long long)gy_most, 8ll * c->sm_count / std::max(1ll, (long long)gx * gz), 65535ll}));
  const size_t smem = (((size_t)a.hg * (a.s.nb + 2) * sizeof(E) + 15) & ~size_t(15)) + lut;
  ProfScope ps(c, XFOLD_K_MASK_BIAS, st);
  launch_pdl(rel_bias_kernel<E, V>, dim3(gx, gy, gz), 256, smem, st, a);
}

// ---------------------------------------------------------------------------------------------
// Gradient of the table: dtable[b][h] = sum over (i, j) with b(i, j) = b of grad[h][i][j].
//
// A warp keeps 32 V columns of one head, V neighbours to a lane, and goes down its rows, eight at a time.  Of each 32 columns (a
// group of lanes) the eight rows' entries lie before the reach, behind it or in another group of tokens, all of them: then a
// lane adds its V to one of three sums in registers.  Or they do not: a band along the diagonal.  Its rows are put into shared
// memory and taken a column to a lane, into sums [nb + 2][32 lanes] of the warp's (a lane's bank is its own: no conflicts, no
// atomics, and the order of the sum is always the same).
// The eights of a CTA lie `slices` apart, so that every warp has its share of the band.  CTAs leave their sums in the workspace;
// a second kernel adds them.
// 16 heads x 2048^2 in 16 bits, buckets up to 128 apart: 33.6 us for both (4.0 TB/s; without a band 24.3, the bytes 20.5), float32
// 47.5 (5.6 TB/s).  Row by row instead of by eights 45: two dozen instructions for each row and block of columns to find out
// where it lies.  Bound by the band's reads and writes of shared memory, then by bytes; small ones by the two launches.
// ---------------------------------------------------------------------------------------------
struct RelBwdArgs {
  RelShared s;
  const void* grad;
  long long sh, sq;       // strides of heads and queries, in elements
  float* partial;         // [H][slices][nb]
  int slices;             // CTAs for each head: eights of rows slice, slice + slices, ...
  int cblocks, row_sets;  // blocks of 32 V columns; sets of eights that warps take such a block in
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }

constexpr int REL_ROWS = 8, REL_HALF = 4;  // rows that are on their way together; that lie in shared memory
template <int V>
__host__ __device__ constexpr size_t rel_bwd_warp_bytes() { return REL_HALF * 512 + REL_ROWS * 16 + 32 * V * 8; }  // rows; what is known of them; columns' positions, groups

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
  E* srow = reinterpret_cast<E*>(own);                        // [REL_HALF][W]
  int4* sinfo = reinterpret_cast<int4*>(own + REL_HALF * 512);  // of a row: where its buckets end, what makes a place in the lut, group
  int* skp = reinterpret_cast<int*>(sinfo + REL_ROWS);
  int* skg = skp + W;
  float* sums = reinterpret_cast<float*>(smem_raw + warps * rel_bwd_warp_bytes<V>());
  uint16_t* lut = reinterpret_cast<uint16_t*>(sums + (size_t)warps * hrows * 32);
  float* acc = sums + (size_t)warp * hrows * 32 + lane;
  pdl_wait();
  pdl_launch();
  const int h = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  const int eights = ((s.Sq + REL_ROWS - 1) / REL_ROWS - slice + a.slices - 1) / a.slices;  // of this CTA
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
    const bool mine = c1 < s.Sk;
    RelPiece<E, V> x[REL_ROWS];
    int qp = 0, qg = 0;  // lane u: of row u of the eight
    auto first = [&](int n) { return (n * a.slices + slice) * REL_ROWS; };
    auto load_row = [&](int u, int i) {  // row i; zeros where there is none
      const E* row = g0 + (long long)i * a.sq;
      if constexpr (VEC) {
        x[u] = RelPiece<E, V>{};
        if (i < s.Sq && mine) x[u] = *reinterpret_cast<const RelPiece<E, V>*>(row + c1);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int j = c0 + v * 32 + lane;
          x[u].e[v] = E(0.f);
          if (i < s.Sq && j < s.Sk) x[u].e[v] = row[j];
        }
      }
    };
    auto load_positions = [&](int i0) {  // (behind the last row: the last one's)
      const int i = min(i0 + (lane & (REL_ROWS - 1)), s.Sq - 1);
      qp = s.q_pos[i];
      if (GROUPS) qg = s.q_grp[i];
    };
    if (set < eights) {
#pragma unroll
      for (int u = 0; u < REL_ROWS; ++u) load_row(u, first(set) + u);
      load_positions(first(set));
    }
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
    const bool same = grp == gmax && fits;
    for (int n = set; n < eights; n += a.row_sets) {
      const int pmin = __reduce_min_sync(0xffffffffu, qp), pmax = __reduce_max_sync(0xffffffffu, qp);
      // (all lanes take part in these: none of them behind a condition)
      const int g = GROUPS ? __reduce_min_sync(0xffffffffu, qg) : 0, g_most = GROUPS ? __reduce_max_sync(0xffffffffu, qg) : 0;
      const bool one = same && g == g_most, other = GROUPS && one && grp != g;
      const bool beh = one && !other && until >= pmax, bef = one && !other && !beh && after <= pmin;
      uint32_t band = __ballot_sync(0xffffffffu, mine && !other && !beh && !bef);
      if (band) {
        if (lane < REL_ROWS) sinfo[lane] = make_int4(low_end(qp, s.reach), high_end(qp, s.reach), int(unsigned(s.reach) - unsigned(qp)), qg);
      }
      const int i0 = n + a.row_sets < eights ? first(n + a.row_sets) : s.Sq;  // the next rows
      load_positions(i0);
      float t = 0.f;
#pragma unroll
      for (int half = 0; half < REL_ROWS; half += REL_HALF) {
#pragma unroll
        for (int u = half; u < half + REL_HALF; ++u) {
          E* row = srow + (u - half) * W;
          if constexpr (!VEC) {  // a lane's columns lie apart: everything passes through shared memory
#pragma unroll
            for (int v = 0; v < V; ++v) row[v * 32 + lane] = x[u].e[v];
            __syncwarp();
            t += piece_sum(*reinterpret_cast<const RelPiece<E, V>*>(row + lane * V));
          } else {
            if (band) *reinterpret_cast<RelPiece<E, V>*>(row + lane * V) = x[u];
            t += piece_sum(x[u]);
          }
          load_row(u, i0 + u);
        }
        if (band) {
          __syncwarp();
          uint32_t left = band;
          do {
            const int at = (__ffs(left) - 1) / SHARE * 32 + lane;  // this lane's of the first 32 columns left
            left &= ~(((1u << SHARE) - 1) << (at / 32 * SHARE));
            const int kp = skp[at], kg = GROUPS ? skg[at] : 0;
            int k[REL_HALF];
            float v[REL_HALF];
#pragma unroll
            for (int u = 0; u < REL_HALF; ++u) {
              const int4 r = sinfo[half + u];
              k[u] = lut[unsigned(min(max(kp, r.x), r.y)) + unsigned(r.z)];
              if (GROUPS && kg != r.w) k[u] = (s.nb - 1) * 32;
              v[u] = to_float(srow[u * W + at]);
            }
#pragma unroll
            for (int u = 0; u < REL_HALF; ++u) acc[k[u]] += v[u];
          } while (left);
        }
        __syncwarp();
      }
      before += bef ? t : 0.f;
      behind += beh ? t : 0.f;
      if (GROUPS) others += other ? t : 0.f;
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
  return std::max(1, std::min(per_sm * sms / H, (Sq + REL_ROWS - 1) / REL_ROWS));
}
static RelBwdPlan rel_bwd_plan(int nb, int H, int Sq, int Sk, int reach, int V, bool vec, int sms) {
  RelBwdPlan p;
  const size_t per_warp = (size_t)(nb + 2) * 128 + (V == 8 ? rel_bwd_warp_bytes<8>() : rel_bwd_warp_bytes<4>()), rest = (2 * reach + 1) * 2;
  p.warps = 8;
  while (p.warps > 1 && p.warps * per_warp + rest > 113 * 1024) p.warps /= 2;
  p.smem = p.warps * per_warp + rest;
  p.slices = rel_bwd_slices(nb, H, Sq, vec, sms);
  p.cblocks = (Sk + 32 * V - 1) / (32 * V);
  // sets of rows: the warps' rounds over the units are to come out even, but a unit costs about as much as half an eight to begin
  const int eights = ((Sq + REL_ROWS - 1) / REL_ROWS + p.slices - 1) / p.slices;
  double best = 1e30;
  for (int n = 1; n <= 8; n *= 2) {
    const double cost = double((p.cblocks * n + p.warps - 1) / p.warps) * ((eights + n - 1) / n + 0.5);
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
  static std::atomic<bool> attr_done[8];
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
  // rows are counted in 32 bits, all CTAs' at a time (eight for each SM, of up to 256 rows)
  if (std::max(Sq, Sk) > 0x7fffffff - (1 << 20)) return fail(c, XFOLD_ERR_ARG, "relative bias: too many queries or keys");
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
// (beyond `rot`: 2 V neighbours that do not rotate).  Its place in the head is the same for all heads of a token, and so an
// element of the result is own * A + partner * B (and r, the reciprocal root), with A and B made of weights, cosines and sines
// once for a token: in registers, at three instructions for two elements.  Angles are made once for a token and warp, as 64-bit
// fractions of a turn: 32-bit floats would lose far positions.
// Pieces are 16 bytes where sizes allow it: of 8, sums over twice as many lanes and addresses for half as much work cost more than
// the fewer registers give back (4 x 4096 tokens, 32 + 8 heads of 128 in 16 bits: 79 and, backward, 137 us).  Warps take ranges of
// passes that begin and end anywhere in a token, so that none has a token more than another.
// Now 61 us (5.5 TB/s), backward 99 (5.1); 2 x 2048 tokens, 32 heads of 64, half rotated: 9.6 and 18.8.  Bound by bytes and the
// chain of a pass (sums over the lanes, root); where a head's width is no power of two some lanes idle (80 of 128: 5 of 8 lanes; groups of any
// size were slower, by their sums).
// ---------------------------------------------------------------------------------------------
struct QkTensor {
  const void *x, *d;  // d: gradient of the result (backward)
  void* y;
  long long xb, xt, xh, db, dt, dh, yb, yt, yh;  // strides of batch, token and head, in elements
  const float* w;
  float scale;
  int H, passes, wide_w;   // passes: of a token, as many heads each as a warp has groups of lanes; wide_w: the weights lie at a 16-byte boundary
  int ctas, share, more;   // a warp takes `share` passes, the first `more` one more
};
struct QkArgs {
  QkTensor t[2];
  const double* freqs;
  const int* pos;
  long long pos_b;
  int B, S, D, rot, log_g;
  float eps;
  int early;            // the next kernel may start while this one runs
  float* partial;       // backward: [CTAs][D], those of the queries in front
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
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (sizeof(T) == 4 || V == 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = to_float(reinterpret_cast<const T*>(&raw)[v]);
    } else {
#pragma unroll
      for (int v = 0; v < V; v += 2) {
        const uint32_t u = reinterpret_cast<const uint32_t*>(&raw)[v / 2];
        f[v] = bf16_lo(u);
        f[v + 1] = bf16_hi(u);
      }
    }
  }
  __device__ __forceinline__ void set(const float* f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int v = 0; v < V; ++v) reinterpret_cast<float*>(&raw)[v] = f[v];
    } else if constexpr (V == 1) {
      *reinterpret_cast<bf16*>(&raw) = __float2bfloat16(f[0]);
    } else {
#pragma unroll
      for (int v = 0; v < V; v += 2) reinterpret_cast<uint32_t*>(&raw)[v / 2] = pack_bf16x2(f[v], f[v + 1]);
    }
  }
};

// slots (pairs of pieces) of a lane: heads are at most 256 wide, so 32 lanes with pieces of 4 hold one
template <int V>
__host__ __device__ constexpr int qk_slots() { return V >= 4 ? 1 : 4 / V; }

// where a lane's pieces of a head lie (pa < 0: behind the head's end), and their angles (< 0: not rotated).  Neighbouring lanes'
// pieces lie next to each other, those of neighbours that rotate too: their pairs lie within a piece.
struct QkPlace {
  int pa, pb, angle, angle_b;
};
template <int V, bool NEIGH>
__device__ __forceinline__ QkPlace qk_place(const QkArgs& a, int sl) {
  const int turning = a.rot / (2 * V);
  QkPlace p;
  if (sl < turning) {
    if (NEIGH && V == 1) {
      p = {2 * sl, 2 * sl + 1, sl, sl};
    } else {
      p.pa = V * sl;
      p.pb = p.pa + a.rot / 2;
      p.angle = NEIGH ? p.pa / 2 : p.pa;
      p.angle_b = NEIGH ? p.pb / 2 : p.pa;
    }
  } else {
    p.pa = a.rot + V * (sl - turning);
    p.pb = p.pa + (a.D - a.rot) / 2;
    p.angle = p.angle_b = -1;
    if (p.pb >= a.D) p.pa = -1;
  }
  return p;
}

// An angle's whole turns are of no interest, so turns for each position are kept as a fraction of 64 bits (once for a CTA), and
// their product with the position as one that wraps around, without another rounding.  The fraction is as good as the frequency's
// 53 bits and their product with 1 / (2 pi) (2^-55 of a turn at about one radian), and off by that times the position.  The lowest
// of them stands for a frequency that is not finite (of half a turn the next is as good).
constexpr unsigned long long NO_ANGLE = 1ull << 63;
__device__ __forceinline__ void qk_turns_of_a_position(const QkArgs& a, unsigned long long* turns) {
  for (int i = threadIdx.x; i < a.rot / 2; i += blockDim.x) {
    const double f = a.freqs[i] * 0.15915494309189533577;  // 1 / (2 pi)
    const long long part = __double2ll_rn((f - rint(f)) * 18446744073709551616.0);
    turns[i] = !isfinite(f) ? NO_ANGLE : (unsigned long long)part == NO_ANGLE ? NO_ANGLE + 1 : (unsigned long long)part;
  }
}
// cosines and sines of a position's angles, by a warp
__device__ __forceinline__ void qk_angles(const QkArgs& a, const unsigned long long* turns, int pos, float2* sm) {
  __syncwarp();
  for (int i = threadIdx.x & 31; i < a.rot / 2; i += 32) {
    const unsigned long long turn = turns[i];
    const int part = int((turn * (unsigned long long)(long long)pos) >> 32);  // of 2^32
    float c, s;
    sincospif(float(part) * 0x1p-31f, &s, &c);
    if (turn == NO_ANGLE) c = s = __int_as_float(0x7fffffff);
    sm[i] = make_float2(c, s);
  }
  __syncwarp();
}

// Of a part of the head that does not rotate: its elements have no partners, whose infinities would become theirs (0 * inf).
__device__ __forceinline__ bool qk_alone(const QkPlace& pl) { return pl.angle < 0 && pl.pa >= 0; }

// The lane's 2 V elements are V pairs of neighbouring registers.  An element's partner is V elements on (halves), or the other
// of its pair.
template <int V, bool NEIGH>
__device__ __forceinline__ float2 qk_partner(const float2 (&z)[V], int j) {
  if constexpr (NEIGH || V == 1) return make_float2(z[j].y, z[j].x);
  else return z[(j + V / 2) % V];
}

// own * A + partner * B: cosines, and sines with the sign of a turn by the angle (SIGN 1) or back (-1), times f
template <int V, bool NEIGH, int SIGN>
__device__ __forceinline__ void qk_factors(const float2* sm, const QkPlace& pl, float f, float2 (&A)[V], float2 (&B)[V]) {
  const float2 none = make_float2(1.f, 0.f);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float2 x, y;  // of elements 2 j and 2 j + 1
    if constexpr (V == 1) {
      x = y = pl.angle >= 0 ? sm[pl.angle] : none;
    } else if constexpr (NEIGH) {
      x = y = pl.angle >= 0 ? (j < V / 2 ? sm[pl.angle + j] : sm[pl.angle_b + j - V / 2]) : none;
    } else {
      x = pl.angle >= 0 ? sm[pl.angle + 2 * j % V] : none;
      y = pl.angle >= 0 ? sm[pl.angle + (2 * j + 1) % V] : none;
    }
    // the first of two partners gets minus the sine in a turn by the angle
    const float sx = NEIGH || V == 1 || j < V / 2 ? -SIGN : SIGN, sy = NEIGH || V == 1 ? SIGN : j < V / 2 ? -SIGN : SIGN;
    A[j] = make_float2(x.x * f, y.x * f);
    B[j] = make_float2(x.y * sx * f, y.y * sy * f);
  }
}

// the lane's weights
template <int V>
__device__ __forceinline__ void qk_weights(const QkTensor& q, const QkPlace& pl, float2 (&w)[V]) {
  float* f = reinterpret_cast<float*>(w);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int at = half ? pl.pb : pl.pa;
    if (!q.w || pl.pa < 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) f[half * V + v] = 1.f;
    } else if (V >= 4 && q.wide_w) {
#pragma unroll
      for (int v = 0; v + 3 < V; v += 4) {
        const float4 u = *reinterpret_cast<const float4*>(q.w + at + v);
        f[half * V + v] = u.x; f[half * V + v + 1] = u.y; f[half * V + v + 2] = u.z; f[half * V + v + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) f[half * V + v] = q.w[at + v];
    }
  }
}

constexpr int QK_WARPS = 4;

// a warp's passes: those of its range, which begins and ends anywhere in a token
struct QkRange {
  int p, t, b, left;
  __device__ __forceinline__ QkRange(const QkArgs& a, const QkTensor& q, int warp) {
    const int first = warp * q.share + min(warp, q.more), token = first / q.passes;
    p = first - token * q.passes;
    b = token / a.S;
    t = token - b * a.S;
    left = q.share + (warp < q.more);
  }
  // whether the next pass is another token's
  __device__ __forceinline__ bool next(const QkArgs& a, const QkTensor& q) {
    --left;
    if (++p < q.passes) return false;
    p = 0;
    if (++t == a.S) {
      t = 0;
      ++b;
    }
    return true;
  }
};

// The passes' pieces on their way through shared memory: a lane copies those that it will use itself, so that nothing but its
// own copies is waited for.  (In registers a pass or two ahead is all that fits beside the factors; 16 warps of that keep 16 to
// 32 KB on their way to an SM, and the chain of a pass was exposed.)
// Pieces of two bytes cannot be copied so and are loaded where they are used.
template <typename T, int V, bool GRAD>
struct QkStream {
  static constexpr int NS = qk_slots<V>(), BYTES = sizeof(T) * V, PIECES = (GRAD ? 4 : 2) * NS;
  static constexpr bool ASYNC = BYTES >= 4;
  static constexpr int STAGES = !ASYNC ? 1 : PIECES * BYTES * 32 * 6 <= 8192 ? 6 : 4;
  static constexpr int SMEM = ASYNC ? STAGES * PIECES * BYTES * 32 : 16;  // of a warp
  const QkArgs& a;
  const QkTensor& q;
  const QkPlace (&at)[NS];
  uint8_t* ring;
  QkRange to;
  int slot = 0, per_pass, sub;
  const T *src, *grd;

  __device__ __forceinline__ QkStream(const QkArgs& a_, const QkTensor& q_, const QkPlace (&at_)[NS], uint8_t* ring_, const QkRange& range)
      : a(a_), q(q_), at(at_), ring(ring_ + (threadIdx.x & 31) * BYTES), to(range), per_pass(32 >> a_.log_g), sub((threadIdx.x & 31) >> a_.log_g) {
    seek();
#pragma unroll 1
    for (int s = 0; s < STAGES - 1; ++s) ahead();
  }
  __device__ __forceinline__ void seek() {
    const long long h = to.p * per_pass + sub;
    src = static_cast<const T*>(q.x) + to.b * q.xb + to.t * q.xt + h * q.xh;
    if (GRAD) grd = static_cast<const T*>(q.d) + to.b * q.db + to.t * q.dt + h * q.dh;
  }
  __device__ __forceinline__ void step() {
    src += per_pass * q.xh;
    if (GRAD) grd += per_pass * q.dh;
    if (to.next(a, q)) seek();
  }
  __device__ __forceinline__ void copy(const T* from, int piece) {
    const uint32_t dst = smem_u32(ring + (slot * PIECES + piece) * BYTES * 32);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
    else if constexpr (ASYNC) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(from), "n"(BYTES >= 4 ? BYTES : 4) : "memory");
  }
  // starts the next pass' copies (an empty group behind the last)
  __device__ __forceinline__ void ahead() {
    if constexpr (ASYNC) {
      if (to.left > 0) {
        if (to.p * per_pass + sub < q.H) {
#pragma unroll
          for (int n = 0; n < NS; ++n)
            if (at[n].pa >= 0) {
              copy(src + at[n].pa, 2 * n);
              copy(src + at[n].pb, 2 * n + 1);
              if (GRAD) {
                copy(grd + at[n].pa, 2 * NS + 2 * n);
                copy(grd + at[n].pb, 2 * NS + 2 * n + 1);
              }
            }
        }
        step();
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      slot = slot + 1 == STAGES ? 0 : slot + 1;
    }
  }
  // this pass' pieces (`in`: the lane has a head there)
  __device__ __forceinline__ void take(bool in, float2 (&x)[NS][V], float2 (&g)[NS][V]) {
    if constexpr (ASYNC) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES >= 2 ? STAGES - 2 : 0) : "memory");
    const int oldest = slot + 1 >= STAGES ? slot + 1 - STAGES : slot + 1;
    auto get = [&](int piece, const T* from, bool is, float* f) {
      Piece<T, V> c;
      c.clear();
      if (is) {
        if constexpr (ASYNC) c.load(reinterpret_cast<const T*>(ring + (oldest * PIECES + piece) * BYTES * 32));
        else c.load(from);
      }
      c.get(f);
    };
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const bool is = in && at[n].pa >= 0;
      float* f = reinterpret_cast<float*>(x[n]);
      get(2 * n, src + at[n].pa, is, f);
      get(2 * n + 1, src + at[n].pb, is, f + V);
      if (GRAD) {
        f = reinterpret_cast<float*>(g[n]);
        get(2 * NS + 2 * n, grd + at[n].pa, is, f);
        get(2 * NS + 2 * n + 1, grd + at[n].pb, is, f + V);
      }
    }
    if constexpr (ASYNC) ahead();
    else step();
  }
};

template <typename T, int V>
__device__ __forceinline__ void qk_store(const float2 (&z)[V], const QkPlace& pl, T* dst) {
  Piece<T, V> a, b;
  a.set(reinterpret_cast<const float*>(z));
  b.set(reinterpret_cast<const float*>(z) + V);
  a.store(dst + pl.pa);
  b.store(dst + pl.pb);
}

// position of a token; where there is no such token, that of one that is
__device__ __forceinline__ int qk_position(const QkArgs& a, int b, int t) {
  return a.pos ? a.pos[min(b, a.B - 1) * a.pos_b + t] : t;
}

// The first CTAs take the queries, the others the keys.
template <typename T, int V, bool NEIGH>
__global__ void __launch_bounds__(QK_WARPS * 32) qk_norm_rotate_kernel(const QkArgs a) {
  typedef QkStream<T, V, false> Stream;
  constexpr int NS = qk_slots<V>();
  __shared__ float2 sm[QK_WARPS][128];
  __shared__ unsigned long long turns[128];
  __shared__ __align__(16) uint8_t ring[QK_WARPS][Stream::SMEM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  if (a.early) pdl_launch();
  const int which = int(blockIdx.x) >= a.t[0].ctas;
  const QkTensor& q = a.t[which];
  QkPlace at[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) at[n] = qk_place<V, NEIGH>(a, (lane & ((1 << a.log_g) - 1)) + n * 32);
  QkRange now(a, q, (blockIdx.x - (which ? a.t[0].ctas : 0)) * QK_WARPS + warp);
  int pos = qk_position(a, now.b, now.t);
  Stream in(a, q, at, ring[warp], now);
  qk_turns_of_a_position(a, turns);
  float2 w[NS][V];
#pragma unroll
  for (int n = 0; n < NS; ++n) qk_weights<V>(q, at[n], w[n]);
  __syncthreads();
  const int per_pass = 32 >> a.log_g, sub = lane >> a.log_g;
  const float inv_d = 1.f / a.D;
  while (now.left > 0) {
    qk_angles(a, turns, pos, sm[warp]);
    float2 A[NS][V], B[NS][V];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      qk_factors<V, NEIGH, 1>(sm[warp], at[n], q.scale, A[n], B[n]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        A[n][j] = fmul2(A[n][j], w[n][j]);
        B[n][j] = fmul2(B[n][j], qk_partner<V, NEIGH>(w[n], j));
      }
    }
    T* dst = static_cast<T*>(q.y) + now.b * q.yb + now.t * q.yt + (long long)(now.p * per_pass + sub) * q.yh;
    pos = now.t + 1 < a.S ? qk_position(a, now.b, now.t + 1) : qk_position(a, now.b + 1, 0);  // the next token's
    bool over;
    do {
      const bool mine = now.p * per_pass + sub < q.H;
      float2 x[NS][V], ss = make_float2(0.f, 0.f);
      in.take(mine, x, x);
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int j = 0; j < V; ++j) ss = ffma2(x[n][j], x[n][j], ss);
      float s = ss.x + ss.y;
#pragma unroll
      for (int i = 0; i < 5; ++i)
        if (i < a.log_g) s += __shfl_xor_sync(0xffffffffu, s, 1 << i);
      const float r = rsqrtf(s * inv_d + a.eps);
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        float2 y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) x[n][j] = fmul2(x[n][j], make_float2(r, r));  // (first: large elements and weights could overflow)
        if (qk_alone(at[n])) {
#pragma unroll
          for (int j = 0; j < V; ++j) y[j] = fmul2(x[n][j], A[n][j]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) y[j] = ffma2(qk_partner<V, NEIGH>(x[n], j), B[n][j], fmul2(x[n][j], A[n][j]));
        }
        if (mine && at[n].pa >= 0) qk_store<T, V>(y, at[n], dst);
      }
      dst += per_pass * q.yh;
      over = now.next(a, q);
    } while (!over && now.left > 0);
  }
}

// Backward, with g = the gradient turned back, times the scale, and r = rsqrt(mean(x^2) + eps):
//   dw_i = sum over tokens and heads of g_i x_i r;  dx = r (g w - x r^2 mean(g w x)).
// A lane's place in the head is always the same: the weights' gradients are sums in its registers until the end.
// PART: some elements do not rotate.  (A kernel of its own: 4 x 4096 tokens, 40 heads of 128, neighbours 90.4 us, and 93.3 where
// partners of no use are looked for.  Two ways through, as in the forward, which loses nothing by them: 100.9.)
template <typename T, int V, bool NEIGH, bool PART>
__global__ void __launch_bounds__(QK_WARPS * 32) qk_norm_rotate_grad_kernel(const QkArgs a) {
  typedef QkStream<T, V, true> Stream;
  constexpr int NS = qk_slots<V>();
  __shared__ float2 sm[QK_WARPS][128];
  __shared__ unsigned long long turns[128];
  __shared__ float red[256];
  __shared__ __align__(16) uint8_t ring[QK_WARPS][Stream::SMEM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  if (a.early) pdl_launch();
  const int which = int(blockIdx.x) >= a.t[0].ctas;
  const QkTensor& q = a.t[which];
  QkPlace at[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) at[n] = qk_place<V, NEIGH>(a, (lane & ((1 << a.log_g) - 1)) + n * 32);
  QkRange now(a, q, (blockIdx.x - (which ? a.t[0].ctas : 0)) * QK_WARPS + warp);
  int pos = qk_position(a, now.b, now.t);
  Stream in(a, q, at, ring[warp], now);
  qk_turns_of_a_position(a, turns);
  float2 w[NS][V], dw[NS][V];
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    qk_weights<V>(q, at[n], w[n]);
#pragma unroll
    for (int j = 0; j < V; ++j) dw[n][j] = make_float2(0.f, 0.f);
  }
  __syncthreads();
  const int per_pass = 32 >> a.log_g, sub = lane >> a.log_g;
  const float inv_d = 1.f / a.D;
  while (now.left > 0) {
    qk_angles(a, turns, pos, sm[warp]);
    float2 A[NS][V], B[NS][V];
#pragma unroll
    for (int n = 0; n < NS; ++n) qk_factors<V, NEIGH, -1>(sm[warp], at[n], q.scale, A[n], B[n]);
    T* dst = static_cast<T*>(q.y) + now.b * q.yb + now.t * q.yt + (long long)(now.p * per_pass + sub) * q.yh;
    pos = now.t + 1 < a.S ? qk_position(a, now.b, now.t + 1) : qk_position(a, now.b + 1, 0);  // the next token's
    bool over;
    do {
      const bool mine = now.p * per_pass + sub < q.H;
      float2 x[NS][V], g[NS][V], ss = make_float2(0.f, 0.f), sg = ss;
      in.take(mine, x, g);
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        float2 e[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float2 partner = qk_partner<V, NEIGH>(g[n], j);
          if (PART && qk_alone(at[n])) partner = make_float2(0.f, 0.f);
          e[j] = ffma2(partner, B[n][j], fmul2(g[n][j], A[n][j]));
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          g[n][j] = e[j];
          ss = ffma2(x[n][j], x[n][j], ss);
          sg = ffma2(fmul2(e[j], w[n][j]), x[n][j], sg);
        }
      }
      float s0 = ss.x + ss.y, s1 = sg.x + sg.y;
#pragma unroll
      for (int i = 0; i < 5; ++i)
        if (i < a.log_g) {
          s0 += __shfl_xor_sync(0xffffffffu, s0, 1 << i);
          s1 += __shfl_xor_sync(0xffffffffu, s1, 1 << i);
        }
      const float r = rsqrtf(s0 * inv_d + a.eps), m = -(s1 * inv_d) * r * r;
      const float2 r2 = make_float2(r, r), m2 = make_float2(m, m);
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        float2 y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (mine) dw[n][j] = ffma2(g[n][j], fmul2(x[n][j], r2), dw[n][j]);  // (no head: zeros, and with eps = 0 infinitely many of them)
          y[j] = fmul2(ffma2(x[n][j], m2, fmul2(g[n][j], w[n][j])), r2);
        }
        if (mine && at[n].pa >= 0) qk_store<T, V>(y, at[n], dst);
      }
      dst += per_pass * q.yh;
      over = now.next(a, q);
    } while (!over && now.left > 0);
  }
  // lanes with the same place in other heads, then the warps one after the other
  for (int o = 1 << a.log_g; o < 32; o <<= 1)
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        dw[n][j].x += __shfl_xor_sync(0xffffffffu, dw[n][j].x, o);
        dw[n][j].y += __shfl_xor_sync(0xffffffffu, dw[n][j].y, o);
      }
  for (int turn = 0; turn < QK_WARPS; ++turn) {
    if (warp == turn && sub == 0) {
#pragma unroll
      for (int n = 0; n < NS; ++n)
        if (at[n].pa >= 0) {
          const float* f = reinterpret_cast<const float*>(dw[n]);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            red[at[n].pa + v] = (turn ? red[at[n].pa + v] : 0.f) + f[v];
            red[at[n].pb + v] = (turn ? red[at[n].pb + v] : 0.f) + f[V + v];
          }
        }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < a.D; i += QK_WARPS * 32) a.partial[(long long)blockIdx.x * a.D + i] = red[i];
}

// the weights' gradients: the sums of the CTAs' parts, 32 elements of one weight to a CTA, a lane for each
__global__ void __launch_bounds__(1024) qk_weight_grad_kernel(const float* partial, float* dqw, float* dkw, int D, int q_ctas, int k_ctas) {
  __shared__ float part[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, i = blockIdx.x * 32 + lane, ctas = blockIdx.y ? k_ctas : q_ctas;
  float* const dst = blockIdx.y ? dkw : dqw;
  pdl_wait();
  pdl_launch();
  if (!dst) return;
  const float* src = partial + (blockIdx.y ? (long long)q_ctas * D : 0) + min(i, D - 1);
  float t = 0.f;
#pragma unroll 8
  for (int c = warp; c < ctas; c += 32) t += src[(long long)c * D];
  part[warp][lane] = t;
  __syncthreads();
  t = warp_total(part[lane][warp]);  // element `warp` of the 32
  if (lane == 0 && blockIdx.x * 32 + warp < D) dst[blockIdx.x * 32 + warp] = t;
}

constexpr int QK_MOST = 8;  // CTAs of an SM
static int qk_ctas(const Ctx* c) { return QK_MOST * c->sm_count; }

// the widest pieces, up to 16 bytes, that sizes, strides and addresses allow
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

// Whether a result has a cache line in common with what the call reads.  Pieces of less than 16 bytes are read through L1 (cp.async
// past it takes 16), where a line's copy does not learn of what other SMs write to it.  A next kernel on the same SM that started
// before those writes would read the old numbers: it starts behind the last of them then.
static bool qk_over_its_inputs(const QkArgs& a, int elem, bool grad) {
  auto meet = [&](const QkTensor& p, const void* x, long long xb, long long xt, long long xh, const QkTensor& q, const void* y, long long yb, long long yt,
                  long long yh) {
    auto lines = [&](const void* at, long long b, long long t, long long h, int H, bool last) {
      long long off = last ? a.D : 0;
      const long long reach[3] = {(a.B - 1) * b, (a.S - 1) * t, (H - 1) * h};
      for (long long r : reach) off += last ? std::max(r, 0ll) : std::min(r, 0ll);
      return ((long long)(uintptr_t)at + off * elem - (last ? 1 : 0)) >> 7;
    };
    return p.H && q.H && lines(x, xb, xt, xh, p.H, false) <= lines(y, yb, yt, yh, q.H, true) && lines(y, yb, yt, yh, q.H, false) <= lines(x, xb, xt, xh, p.H, true);
  };
  for (const QkTensor& p : a.t)
    for (const QkTensor& q : a.t)
      if (meet(p, p.x, p.xb, p.xt, p.xh, q, q.y, q.yb, q.yt, q.yh) || (grad && meet(p, p.d, p.db, p.dt, p.dh, q, q.y, q.yb, q.yt, q.yh))) return true;
  return false;
}

// queries and keys get CTAs by their heads and what a token costs besides (about two passes)
static int qk_divide(Ctx* c, QkArgs& a, int per_sm, int& grid) {
  const long long tokens = (long long)a.B * a.S;
  const int all = per_sm * c->sm_count, weigh[2] = {a.t[0].H ? a.t[0].passes + 2 : 0, a.t[1].H ? a.t[1].passes + 2 : 0};
  grid = 0;
  for (int i = 0; i < 2; ++i) {
    QkTensor& q = a.t[i];
    const int share = q.H ? std::max(1, (int)((long long)(all - 1) * weigh[i] / (weigh[0] + weigh[1]))) : 0;
    const long long total = tokens * q.passes;
    if (total > 0x7fffffffll) return fail(c, XFOLD_ERR_ARG, "qk norm: too many tokens");
    q.ctas = (int)std::min<long long>(share, (total + QK_WARPS - 1) / QK_WARPS);
    if (q.ctas) {
      q.share = (int)(total / (q.ctas * QK_WARPS));
      q.more = (int)(total % (q.ctas * QK_WARPS));
    }
    grid += q.ctas;
  }
  return XFOLD_OK;
}

template <typename T, int V, bool GRAD>
static int launch_qk_one(Ctx* c, QkArgs& a, int neighbours, cudaStream_t st) {
  auto kern = [&] {
    if constexpr (GRAD) {
      if (a.rot < a.D) return neighbours ? qk_norm_rotate_grad_kernel<T, V, true, true> : qk_norm_rotate_grad_kernel<T, V, false, true>;
      return neighbours ? qk_norm_rotate_grad_kernel<T, V, true, false> : qk_norm_rotate_grad_kernel<T, V, false, false>;
    } else {
      return neighbours ? qk_norm_rotate_kernel<T, V, true> : qk_norm_rotate_kernel<T, V, false>;
    }
  }();
  // resident CTAs; contexts in other threads may find them at the same time
  static std::atomic<int> per_sm[4];
  std::atomic<int>& known = per_sm[(neighbours ? 1 : 0) + (a.rot < a.D ? 2 : 0)];
  int n = known.load(std::memory_order_relaxed);
  if (!n) {
    int got = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&got, kern, QK_WARPS * 32, 0) != cudaSuccess || got < 1)
      return fail(c, XFOLD_ERR_LAUNCH, "qk norm: occupancy");
    known.store(n = std::min(got, QK_MOST), std::memory_order_relaxed);
  }
  int grid = 0;
  if (int rc = qk_divide(c, a, n, grid)) return rc;
  ProfScope ps(c, XFOLD_K_LAYERNORM, st);
  launch_pdl(kern, dim3(grid), QK_WARPS * 32, 0, st, a);
  return check_launch(c, "qk_norm_rotate");
}

template <bool GRAD>
static int launch_qk(Ctx* c, QkArgs a, int f32, int neighbours, cudaStream_t st, float* dqw = nullptr, float* dkw = nullptr) {
  const int elem = f32 ? 4 : 2, V = qk_piece(a, elem, GRAD), slots = (a.D / 2 + V - 1) / V;
  a.early = V * elem == 16 || !qk_over_its_inputs(a, elem, GRAD);
  a.log_g = 0;
  while ((1 << a.log_g) < slots && a.log_g < 5) ++a.log_g;
  for (QkTensor& q : a.t) q.passes = (q.H + (32 >> a.log_g) - 1) / (32 >> a.log_g);
  int rc;
  if (f32) {
    rc = V == 4 ? launch_qk_one<float, 4, GRAD>(c, a, neighbours, st) : V == 2 ? launch_qk_one<float, 2, GRAD>(c, a, neighbours, st)
                                                                              : launch_qk_one<float, 1, GRAD>(c, a, neighbours, st);
  } else {
    rc = V == 8   ? launch_qk_one<bf16, 8, GRAD>(c, a, neighbours, st)
         : V == 4 ? launch_qk_one<bf16, 4, GRAD>(c, a, neighbours, st)
         : V == 2 ? launch_qk_one<bf16, 2, GRAD>(c, a, neighbours, st)
                  : launch_qk_one<bf16, 1, GRAD>(c, a, neighbours, st);
  }
  if (rc || (!dqw && !dkw)) return rc;
  ProfScope ps(c, XFOLD_K_LAYERNORM, st);
  launch_pdl(qk_weight_grad_kernel, dim3((a.D + 31) / 32, 2), 1024, 0, st, (const float*)a.partial, dqw, dkw, a.D, a.t[0].ctas, a.t[1].ctas);
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
    t.wide_w = (uintptr_t)t.w % 16 == 0;
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
  return cx && D > 0 ? (size_t)qk_ctas(reinterpret_cast<const Ctx*>(cx)) * D * sizeof(float) : 0;
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
