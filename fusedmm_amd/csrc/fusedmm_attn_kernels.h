// Kernels of attention over a planned pattern: forward, delta, the two backward passes, and the joins of split blocks.
//
// A plan (fusedmm_attn_plan.hip) lists, for every block of 64 rows, the columns that any of them names, with one bit per
// row.  A unit is a run of such columns of one block; a block whose rows are long is several units, whose partial sums
// the join kernels add in order.  A workgroup does one unit for one head: 4 waves of 16 resident rows share the tiles of
// 32 gathered rows.  What the block size gives: a gathered row is loaded once for 64 rows instead of once for each that
// names it, and one 16 x 16 product serves 16 rows; a tile that no row of a wave names is skipped by that wave.
#pragma once
#include "fusedmm_attn_core.h"

namespace fmm_attn {

struct Unit {
   int32_t block;     // rows 64 * block ...
   int32_t part;      // slot of its partial sums, -1: the block's only unit
   int32_t tile0;     // first tile of its columns
   int32_t tiles;
};
struct Join {         // a block of several units: partial sums part0 .. part0 + parts - 1
   int32_t block, part0, parts, pad;
};

struct PlanView {
   const int32_t *cols;    // [tiles * 32], -1: no column
   const uint16_t *masks;  // [tiles][4 waves][32]: bit r is row 16 * wave + r of the block
   const Unit *units;
   const Join *joins;
   int32_t n_units, n_joins;
   int64_t rows, cols_n;
};

struct Params {
   PlanView plan;
   int64_t m, n;                      // query rows, key rows
   int32_t heads, kv_heads, group, d, dv;
   float scale;
   int64_t ldq, hdq, ldk, hdk, ldv, hdv, ldo, hdo;
   int32_t vec;                       // every row of every tensor is 16-byte aligned and d, dv are multiples of a 16-byte chunk
   const void *q, *k, *v, *o, *o2, *dout;
   const float *lambda;
   const float *lse_in;
   void *out, *out2;                  // forward
   float *lse;                        // may be null
   void *dq, *dk, *dvv;
   float *dlambda;
   float *delta;                      // [m][heads][maps]
   float *dlam_rows;                  // [m][heads]: sum_j P_2 dP
   float *part;                       // partial sums of split blocks
};

template <int T, int DC, int MAPS> struct Geo {
   typedef Num<T> N;
   typedef typename N::E E;
   static constexpr int W = DC * MAPS;                // padded width of a gathered row: all maps of q or k; v and do
   static constexpr int LD = W + N::EPL;              // of a tile row in LDS: 16 bytes more, so that rows start in other banks
   static constexpr int CR = W / N::EPL;              // 16-byte chunks of a row
   static constexpr int NCH = (kTile * CR + 255) / 256;   // chunks a thread stages
   static constexpr int CQ = DC / N::KC;              // chunks of a product over one map's features
   static constexpr int CV = W / N::KC;
   static constexpr int NT = W / 16, NTQ = DC / 16;   // 16-feature tiles of v's and of one map's accumulators
   static constexpr bool kWide = W * sizeof(E) >= 512;
   static constexpr bool kIdle = kTile * CR < 256;    // the tile has fewer chunks than the workgroup threads
};

// ---- staging: 32 gathered rows of two tensors, global -> registers -> LDS ----------------------------------------------------

template <class G> struct Stage {
   u4 a[G::NCH], b[G::NCH];
};

template <class G> __device__ inline void stage_cols(int32_t (&c)[G::NCH], const int32_t *cols, int tid)
{
#pragma unroll
   for (int j = 0; j < G::NCH; j++)
   {
      const int q = tid + 256 * j;
      c[j] = (!G::kIdle || q < kTile * G::CR) ? cols[q / G::CR] : -1;
   }
}

// a: rows of `maps` pieces of d features each; b: rows of dv features
template <class G, int T, int DC>
__device__ inline void stage_load(Stage<G> &s, const int32_t (&c)[G::NCH], const typename G::E *a, int64_t lda, int d,
                                  const typename G::E *b, int64_t ldb, int dv, bool vec, int tid)
{
#pragma unroll
   for (int j = 0; j < G::NCH; j++)
   {
      const int e = ((tid + 256 * j) % G::CR) * G::N::EPL;
      const int mp = e / DC, f = e - mp * DC;
      const bool live = c[j] >= 0;
      const int64_t row = live ? c[j] : 0;
      s.a[j] = load_chunk<T>(a + row * lda + mp * d + f, live ? (d - f < G::N::EPL ? d - f : G::N::EPL) : 0, vec);
      s.b[j] = load_chunk<T>(b + row * ldb + e, live ? (dv - e < G::N::EPL ? dv - e : G::N::EPL) : 0, vec);
   }
}

// returns bit 0 / 1: an infinity or NaN among this thread's chunks of a / b
template <class G, int T>
__device__ inline int stage_store(const Stage<G> &s, typename G::E *a, typename G::E *b, int tid, bool look_a, bool look_b)
{
   int odd = 0;
#pragma unroll
   for (int j = 0; j < G::NCH; j++)
   {
      const int q = tid + 256 * j;
      if (G::kIdle && q >= kTile * G::CR) break;
      const int off = (q / G::CR) * G::LD + (q % G::CR) * G::N::EPL;
      *reinterpret_cast<u4 *>(a + off) = s.a[j];
      *reinterpret_cast<u4 *>(b + off) = s.b[j];
      if (look_a && odd_chunk<T>(s.a[j])) odd |= 1;
      if (look_b && odd_chunk<T>(s.b[j])) odd |= 2;
   }
   return odd;
}

// the resident rows of a wave as the second operand: lane i holds its 16 bytes of every chunk of row i
template <int T, int CQ> __device__ inline void load_resident(u4 (&r)[CQ], const typename Num<T>::E *row, bool live, int d, int g, bool vec)
{
#pragma unroll
   for (int c = 0; c < CQ; c++)
   {
      const int f = c * Num<T>::KC + g * Num<T>::EPL;
      r[c] = load_chunk<T>(row + f, live ? (d - f < Num<T>::EPL ? d - f : Num<T>::EPL) : 0, vec);
   }
}

// scores of the tile's 32 rows against the resident rows: s[a] rows 16a + 4g + r
template <int T, int CQ>
__device__ inline void tile_scores(f4 (&s)[2], const typename Num<T>::E *tile, int ld, const u4 (&res)[CQ], int g, int i)
{
   s[0] = f4{0, 0, 0, 0};
   s[1] = f4{0, 0, 0, 0};
#pragma unroll
   for (int c = 0; c < CQ; c++)
   {
      const int f = c * Num<T>::KC + g * Num<T>::EPL;
      s[0] = Num<T>::mma(*reinterpret_cast<const u4 *>(tile + i * ld + f), res[c], s[0]);
      s[1] = Num<T>::mma(*reinterpret_cast<const u4 *>(tile + (16 + i) * ld + f), res[c], s[1]);
   }
}

// this lane's bits of a tile's masks: bit 4a + r for gathered row 16a + 4g + r and resident row i
__device__ inline unsigned my_bits(uint64_t m0, uint64_t m1, int i)
{
   unsigned b = 0;
#pragma unroll
   for (int r = 0; r < 4; r++)
   {
      b |= (unsigned)((m0 >> (16 * r + i)) & 1) << r;
      b |= (unsigned)((m1 >> (16 * r + i)) & 1) << (4 + r);
   }
   return b;
}

// ---- forward ----------------------------------------------------------------------------------------------------------------------
// One pass over a unit's columns with a running maximum and sum of every row and map.  Scores are kept times log2(e).
template <int T, int DC, int MAPS>
__global__ __launch_bounds__(256, (Geo<T, DC, MAPS>::kWide && (T == kF32 || MAPS == 2) ? 1 : 2)) void attn_forward(Params p)
{
   typedef Geo<T, DC, MAPS> G;
   typedef typename G::E E;
   __shared__ __align__(16) E ks[2][kTile * G::LD];
   __shared__ __align__(16) E vs[2][kTile * G::LD];
   __shared__ int odd[2];
   const int64_t item = xcd_item(blockIdx.x, (int64_t)p.plan.n_units * p.heads);
   if (item >= (int64_t)p.plan.n_units * p.heads) return;
   const int head = (int)(item / p.plan.n_units);
   const Unit u = p.plan.units[item % p.plan.n_units];
   const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, i = lane & 15;
   const int kvh = head / p.group;
   const E *k = (const E *)p.k + kvh * p.hdk, *v = (const E *)p.v + kvh * p.hdv;
   const int64_t row = (int64_t)u.block * kBlockRows + 16 * wave + i;
   const bool live = row < p.m;
   if (tid < 2) odd[tid] = 0;

   u4 qr[MAPS][G::CQ];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
      load_resident<T, G::CQ>(qr[mp], (const E *)p.q + (live ? row : 0) * p.ldq + head * p.hdq + mp * p.d, live, p.d, g, p.vec);

   f4 acc[MAPS][G::NT];
   float top[MAPS], sum[MAPS];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
   {
      top[mp] = -INFINITY;
      sum[mp] = 0;
#pragma unroll
      for (int t = 0; t < G::NT; t++) acc[mp][t] = f4{0, 0, 0, 0};
   }
   const float c2 = p.scale * kLog2e;

   const int32_t *cols = p.plan.cols + (int64_t)u.tile0 * kTile;
   const uint16_t *masks = p.plan.masks + (int64_t)u.tile0 * (4 * kTile) + wave * kTile + 4 * g;
   int32_t cn[G::NCH];
   Stage<G> st;
   uint64_t m0 = 0, m1 = 0;
   if (u.tiles > 0)
   {
      stage_cols<G>(cn, cols, tid);
      stage_load<G, T, DC>(st, cn, k, p.ldk, p.d, v, p.ldv, p.dv, p.vec, tid);
      m0 = *(const uint64_t *)masks;
      m1 = *(const uint64_t *)(masks + 16);
      if (u.tiles > 1) stage_cols<G>(cn, cols + kTile, tid);
      __syncthreads();   // the flags are clear
      if (stage_store<G, T>(st, ks[0], vs[0], tid, false, true)) odd[0] = 1;
   }
   __syncthreads();
   for (int t = 0; t < u.tiles; t++)
   {
      const int b = t & 1;
      const uint64_t n0 = m0, n1 = m1;
      if (t + 1 < u.tiles)
      {
         stage_load<G, T, DC>(st, cn, k, p.ldk, p.d, v, p.ldv, p.dv, p.vec, tid);
         m0 = *(const uint64_t *)(masks + (int64_t)(t + 1) * (4 * kTile));
         m1 = *(const uint64_t *)(masks + (int64_t)(t + 1) * (4 * kTile) + 16);
         if (t + 2 < u.tiles) stage_cols<G>(cn, cols + (int64_t)(t + 2) * kTile, tid);
      }
      if (__any((n0 | n1) != 0))
      {
         const unsigned mine = my_bits(n0, n1, i);
         float w[MAPS][2][4];
#pragma unroll
         for (int mp = 0; mp < MAPS; mp++)
         {
            f4 s[2];
            tile_scores<T, G::CQ>(s, ks[b] + mp * DC, G::LD, qr[mp], g, i);
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; j++)
            {
               w[mp][j / 4][j % 4] = ((mine >> j) & 1) ? s[j / 4][j % 4] * c2 : -INFINITY;
               mx = fmaxf(mx, w[mp][j / 4][j % 4]);
            }
            mx = fmaxf(top[mp], group_max(mx));
            const float base = mx == -INFINITY ? 0.0f : mx;   // nothing named so far: every weight below is exp2(-inf)
            const float keep = exp2_fast(top[mp] - base);
            float add = 0;
#pragma unroll
            for (int j = 0; j < 8; j++)
            {
               w[mp][j / 4][j % 4] = exp2_fast(w[mp][j / 4][j % 4] - base);
               add += w[mp][j / 4][j % 4];
            }
            if (__any(mx != top[mp]))
            {
#pragma unroll
               for (int x = 0; x < G::NT; x++) acc[mp][x] *= keep;
            }
            sum[mp] = sum[mp] * keep + add;   // of this lane's columns: the four groups are added at the end
            top[mp] = mx;
         }
         if (__builtin_expect(odd[b] == t + 1, 0))
         {
#pragma unroll
            for (int mp = 0; mp < MAPS; mp++) add_weighted<T, G::NT>(acc[mp], w[mp], mine, vs[b], G::LD, g, i, true);
         }
         else
         {
            typename G::N::TFrag wf[MAPS];
#pragma unroll
            for (int mp = 0; mp < MAPS; mp++) wf[mp] = pack_scores<T>(w[mp]);
#pragma unroll
            for (int x = 0; x < G::NT; x++)
            {
               const typename G::N::TFrag vt = load_t<T>(vs[b], G::LD, x, g, i);
#pragma unroll
               for (int mp = 0; mp < MAPS; mp++) acc[mp][x] = G::N::mma_t(vt, wf[mp], acc[mp][x]);
            }
         }
      }
      if (t + 1 < u.tiles)
      {
         if (stage_store<G, T>(st, ks[b ^ 1], vs[b ^ 1], tid, false, true)) odd[b ^ 1] = t + 2;
      }
      __syncthreads();
   }

#pragma unroll
   for (int mp = 0; mp < MAPS; mp++) sum[mp] = group_sum(sum[mp]);
   if (u.part >= 0)
   {
      // [part][head][map][64 rows][W + 2]: sums, then the running maximum and sum
      float *to = p.part + (((int64_t)u.part * p.heads + head) * MAPS * kBlockRows + 16 * wave + i) * (G::W + 2);
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
      {
         float *r = to + (int64_t)mp * kBlockRows * (G::W + 2);
#pragma unroll
         for (int x = 0; x < G::NT; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) r[16 * x + 4 * g + e] = acc[mp][x][e];
         if (g == 0)
         {
            r[G::W] = top[mp];
            r[G::W + 1] = sum[mp];
         }
      }
      return;
   }
   if (!live) return;
   const float lam = MAPS == 2 ? p.lambda[head] : 0.0f;
   float inv[MAPS];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
   {
      inv[mp] = sum[mp] == 0.0f ? 0.0f : 1.0f / sum[mp];   // a row without edges is zero
      if (p.lse && g == 0) p.lse[(row * p.heads + head) * MAPS + mp] = sum[mp] == 0.0f ? -INFINITY : (top[mp] + log2f(sum[mp])) * kLn2;
   }
   E *out = (E *)p.out + row * p.ldo + head * p.hdo;
   E *out2 = MAPS == 2 && p.out2 ? (E *)p.out2 + row * p.ldo + head * p.hdo : nullptr;
#pragma unroll
   for (int x = 0; x < G::NT; x++)
   {
      f4 r = acc[0][x] * inv[0];
      if constexpr (MAPS == 2)
      {
         const f4 r2 = acc[1][x] * inv[1];
         if (out2) store4<T>(out2, 16 * x + 4 * g, p.dv, r2, p.vec);
         r -= lam * r2;
      }
      store4<T>(out, 16 * x + 4 * g, p.dv, r, p.vec);
   }
}

// Blocks of several units: one wave per (block, head, row).
template <int T, int DC, int MAPS> __global__ __launch_bounds__(256) void attn_forward_join(Params p)
{
   typedef Geo<T, DC, MAPS> G;
   typedef typename G::E E;
   const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
   const int lane = threadIdx.x & 63;
   const int r = (int)(id % kBlockRows);
   const int head = (int)((id / kBlockRows) % p.heads);
   const int64_t jn = id / kBlockRows / p.heads;
   if (jn >= p.plan.n_joins) return;
   const Join j = p.plan.joins[jn];
   const int64_t row = (int64_t)j.block * kBlockRows + r;
   if (row >= p.m) return;
   const float lam = MAPS == 2 ? p.lambda[head] : 0.0f;
   constexpr int PER = (G::W + 63) / 64;
   float o[MAPS][PER];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
   {
      const int64_t step = (int64_t)p.heads * MAPS * kBlockRows * (G::W + 2);
      const float *from = p.part + (((int64_t)j.part0 * p.heads + head) * MAPS + mp) * kBlockRows * (G::W + 2) + (int64_t)r * (G::W + 2);
      float top = -INFINITY;
      for (int u = 0; u < j.parts; u++) top = fmaxf(top, from[u * step + G::W]);
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0;
#pragma unroll
      for (int x = 0; x < PER; x++) o[mp][x] = 0;
      for (int u = 0; u < j.parts; u++)
      {
         const float *s = from + u * step;
         const float keep = exp2_fast(s[G::W] - base);
         sum += s[G::W + 1] * keep;
#pragma unroll
         for (int x = 0; x < PER; x++)
            if (lane + 64 * x < G::W) o[mp][x] += s[lane + 64 * x] * keep;
      }
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int x = 0; x < PER; x++) o[mp][x] *= inv;
      if (p.lse && lane == 0) p.lse[(row * p.heads + head) * MAPS + mp] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
   }
   E *out = (E *)p.out + row * p.ldo + head * p.hdo;
#pragma unroll
   for (int x = 0; x < PER; x++)
   {
      const int f = lane + 64 * x;
      if (f >= p.dv) continue;
      float res = o[0][x];
      if constexpr (MAPS == 2)
      {
         if (p.out2) ((E *)p.out2)[row * p.ldo + head * p.hdo + f] = (E)Num<T>::from(o[1][x]);
         res -= lam * o[1][x];
      }
      out[f] = (E)Num<T>::from(res);
   }
}

// ---- backward ---------------------------------------------------------------------------------------------------------------------
// delta_p = <do, O_p>: 16 lanes per (row, head).  With O_2 at hand, <do, O_1> = <do, o> + lambda <do, O_2>.
template <int T, int MAPS> __global__ __launch_bounds__(256) void attn_delta(Params p)
{
   typedef typename Num<T>::E E;
   const int64_t id = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
   const int lane = threadIdx.x & 15;
   const bool live = id < p.m * p.heads;
   const int64_t row = live ? id / p.heads : 0;
   const int head = live ? (int)(id % p.heads) : 0;
   const E *g = (const E *)p.dout + row * p.ldo + head * p.hdo;
   const E *o = (const E *)p.o + row * p.ldo + head * p.hdo;
   const E *o2 = MAPS == 2 ? (const E *)p.o2 + row * p.ldo + head * p.hdo : nullptr;
   float s = 0, s2 = 0;
   for (int f = lane; f < p.dv; f += 16)
   {
      const float x = Num<T>::to(g[f]);
      s = fmaf(x, Num<T>::to(o[f]), s);
      if constexpr (MAPS == 2) s2 = fmaf(x, Num<T>::to(o2[f]), s2);
   }
#pragma unroll
   for (int k = 8; k; k >>= 1)
   {
      s += __shfl_xor(s, k);
      if constexpr (MAPS == 2) s2 += __shfl_xor(s2, k);
   }
   if (!live || lane) return;
   float *to = p.delta + id * MAPS;
   if constexpr (MAPS == 2)
   {
      to[0] = s + p.lambda[head] * s2;
      to[1] = s2;
   }
   else to[0] = s;
}

// dq: resident q and do of 16 rows per wave, gathered k and v; both maps share the gathered v and dP.
template <int T, int DC, int MAPS>
__global__ __launch_bounds__(256, (Geo<T, DC, MAPS>::kWide ? 1 : 2)) void attn_dq(Params p)
{
   typedef Geo<T, DC, MAPS> G;
   typedef typename G::E E;
   __shared__ __align__(16) E ks[2][kTile * G::LD];
   __shared__ __align__(16) E vs[2][kTile * G::LD];
   __shared__ int odd[2];
   const int64_t item = xcd_item(blockIdx.x, (int64_t)p.plan.n_units * p.heads);
   if (item >= (int64_t)p.plan.n_units * p.heads) return;
   const int head = (int)(item / p.plan.n_units);
   const Unit u = p.plan.units[item % p.plan.n_units];
   const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, i = lane & 15;
   const int kvh = head / p.group;
   const E *k = (const E *)p.k + kvh * p.hdk, *v = (const E *)p.v + kvh * p.hdv;
   const int64_t row = (int64_t)u.block * kBlockRows + 16 * wave + i;
   const bool live = row < p.m;
   const int64_t srow = live ? row : 0;
   if (tid < 2) odd[tid] = 0;

   u4 qr[MAPS][G::CQ], gr[G::CV];
   float lse2[MAPS], delta[MAPS], sign[MAPS];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
   {
      load_resident<T, G::CQ>(qr[mp], (const E *)p.q + srow * p.ldq + head * p.hdq + mp * p.d, live, p.d, g, p.vec);
      lse2[mp] = p.lse_in[(srow * p.heads + head) * MAPS + mp] * kLog2e;
      delta[mp] = p.delta[(srow * p.heads + head) * MAPS + mp];
      sign[mp] = mp == 0 ? 1.0f : -p.lambda[head];
   }
   load_resident<T, G::CV>(gr, (const E *)p.dout + srow * p.ldo + head * p.hdo, live, p.dv, g, p.vec);

   f4 acc[MAPS][G::NTQ];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
      for (int t = 0; t < G::NTQ; t++) acc[mp][t] = f4{0, 0, 0, 0};
   float mean2 = 0;
   const float c2 = p.scale * kLog2e;

   const int32_t *cols = p.plan.cols + (int64_t)u.tile0 * kTile;
   const uint16_t *masks = p.plan.masks + (int64_t)u.tile0 * (4 * kTile) + wave * kTile + 4 * g;
   int32_t cn[G::NCH];
   Stage<G> st;
   uint64_t m0 = 0, m1 = 0;
   if (u.tiles > 0)
   {
      stage_cols<G>(cn, cols, tid);
      stage_load<G, T, DC>(st, cn, k, p.ldk, p.d, v, p.ldv, p.dv, p.vec, tid);
      m0 = *(const uint64_t *)masks;
      m1 = *(const uint64_t *)(masks + 16);
      if (u.tiles > 1) stage_cols<G>(cn, cols + kTile, tid);
      __syncthreads();
      if (stage_store<G, T>(st, ks[0], vs[0], tid, true, false)) odd[0] = 1;
   }
   __syncthreads();
   for (int t = 0; t < u.tiles; t++)
   {
      const int b = t & 1;
      const uint64_t n0 = m0, n1 = m1;
      if (t + 1 < u.tiles)
      {
         stage_load<G, T, DC>(st, cn, k, p.ldk, p.d, v, p.ldv, p.dv, p.vec, tid);
         m0 = *(const uint64_t *)(masks + (int64_t)(t + 1) * (4 * kTile));
         m1 = *(const uint64_t *)(masks + (int64_t)(t + 1) * (4 * kTile) + 16);
         if (t + 2 < u.tiles) stage_cols<G>(cn, cols + (int64_t)(t + 2) * kTile, tid);
      }
      if (__any((n0 | n1) != 0))
      {
         const unsigned mine = my_bits(n0, n1, i);
         const bool bad = odd[b] == t + 1;
         f4 dp[2];
         tile_scores<T, G::CV>(dp, vs[b], G::LD, gr, g, i);
#pragma unroll
         for (int mp = 0; mp < MAPS; mp++)
         {
            f4 s[2];
            tile_scores<T, G::CQ>(s, ks[b] + mp * DC, G::LD, qr[mp], g, i);
            float w[2][4];
#pragma unroll
            for (int j = 0; j < 8; j++)
            {
               const bool named = (mine >> j) & 1;
               const float pr = named ? exp2_fast(s[j / 4][j % 4] * c2 - lse2[mp]) : 0.0f;
               const float x = named ? dp[j / 4][j % 4] : 0.0f;
               w[j / 4][j % 4] = pr * sign[mp] * (x - delta[mp]);
               if (mp == 1) mean2 = fmaf(pr, x, mean2);
            }
            add_weighted<T, G::NTQ>(acc[mp], w, mine, ks[b] + mp * DC, G::LD, g, i, bad);
         }
      }
      if (t + 1 < u.tiles)
      {
         if (stage_store<G, T>(st, ks[b ^ 1], vs[b ^ 1], tid, true, false)) odd[b ^ 1] = t + 2;
      }
      __syncthreads();
   }

   if (MAPS == 2) mean2 = group_sum(mean2);
   if (u.part >= 0)
   {
      // [part][head][64 rows][W + 1]
      float *r = p.part + (((int64_t)u.part * p.heads + head) * kBlockRows + 16 * wave + i) * (G::W + 1);
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
         for (int x = 0; x < G::NTQ; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) r[mp * DC + 16 * x + 4 * g + e] = acc[mp][x][e];
      if (g == 0) r[G::W] = mean2;
      return;
   }
   if (!live) return;
   if (MAPS == 2 && g == 0) p.dlam_rows[row * p.heads + head] = mean2;
   E *out = (E *)p.dq + row * p.ldq + head * p.hdq;
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
      for (int x = 0; x < G::NTQ; x++) store4<T>(out + mp * p.d, 16 * x + 4 * g, p.d, acc[mp][x] * p.scale, p.vec);
}

template <int T, int DC, int MAPS> __global__ __launch_bounds__(256) void attn_dq_join(Params p)
{
   typedef Geo<T, DC, MAPS> G;
   typedef typename G::E E;
   const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
   const int lane = threadIdx.x & 63;
   const int r = (int)(id % kBlockRows);
   const int head = (int)((id / kBlockRows) % p.heads);
   const int64_t jn = id / kBlockRows / p.heads;
   if (jn >= p.plan.n_joins) return;
   const Join j = p.plan.joins[jn];
   const int64_t row = (int64_t)j.block * kBlockRows + r;
   if (row >= p.m) return;
   const int64_t step = (int64_t)p.heads * kBlockRows * (G::W + 1);
   const float *from = p.part + (((int64_t)j.part0 * p.heads + head) * kBlockRows + r) * (G::W + 1);
   for (int f = lane; f <= G::W; f += 64)
   {
      float s = 0;
      for (int u = 0; u < j.parts; u++) s += from[u * step + f];
      if (f == G::W)
      {
         if (MAPS == 2) p.dlam_rows[row * p.heads + head] = s;
         continue;
      }
      const int mp = f / DC, e = f - mp * DC;
      if (e < p.d) ((E *)p.dq)[row * p.ldq + head * p.hdq + mp * p.d + e] = (E)Num<T>::from(s * p.scale);
   }
}

// dlambda_h = - sum of dlam_rows: one workgroup per head, in 64 bits, every thread's rows and then the threads in order
template <int T> __global__ __launch_bounds__(256) void attn_dlambda(Params p)
{
   __shared__ double s[256];
   const int head = blockIdx.x;
   double x = 0;
   for (int64_t r = threadIdx.x; r < p.m; r += 256) x += (double)p.dlam_rows[r * p.heads + head];
   s[threadIdx.x] = x;
   __syncthreads();
   for (int k = 128; k; k >>= 1)
   {
      if ((int)threadIdx.x < k) s[threadIdx.x] += s[threadIdx.x + k];
      __syncthreads();
   }
   if (threadIdx.x == 0) p.dlambda[head] = (float)-s[0];
}

// dk, dv: resident k and v of 16 key rows per wave, gathered q and do of the query rows that name them, for every query
// head of the key head in turn.  p.plan is the plan of the transposed pattern.
template <int T, int DC, int MAPS>
__global__ __launch_bounds__(256, (Geo<T, DC, MAPS>::kWide ? 1 : 2)) void attn_dkv(Params p)
{
   typedef Geo<T, DC, MAPS> G;
   typedef typename G::E E;
   __shared__ __align__(16) E qs[2][kTile * G::LD];
   __shared__ __align__(16) E gs[2][kTile * G::LD];
   __shared__ __align__(16) float stat[2][2 * MAPS][kTile];   // lse * log2(e), delta of the gathered rows
   __shared__ int odd[2];
   const int64_t item = xcd_item(blockIdx.x, (int64_t)p.plan.n_units * p.kv_heads);
   if (item >= (int64_t)p.plan.n_units * p.kv_heads) return;
   const int kvh = (int)(item / p.plan.n_units);
   const Unit u = p.plan.units[item % p.plan.n_units];
   const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, i = lane & 15;
   const int64_t row = (int64_t)u.block * kBlockRows + 16 * wave + i;
   const bool live = row < p.n;
   const int64_t srow = live ? row : 0;
   if (tid < 2) odd[tid] = 0;

   u4 kr[MAPS][G::CQ], vr[G::CV];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
      load_resident<T, G::CQ>(kr[mp], (const E *)p.k + srow * p.ldk + kvh * p.hdk + mp * p.d, live, p.d, g, p.vec);
   load_resident<T, G::CV>(vr, (const E *)p.v + srow * p.ldv + kvh * p.hdv, live, p.dv, g, p.vec);

   f4 dk[MAPS][G::NTQ], dv[G::NT];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
      for (int t = 0; t < G::NTQ; t++) dk[mp][t] = f4{0, 0, 0, 0};
#pragma unroll
   for (int t = 0; t < G::NT; t++) dv[t] = f4{0, 0, 0, 0};
   const float c2 = p.scale * kLog2e;

   const int32_t *cols = p.plan.cols + (int64_t)u.tile0 * kTile;
   const uint16_t *masks = p.plan.masks + (int64_t)u.tile0 * (4 * kTile) + wave * kTile + 4 * g;
   const int steps = u.tiles * p.group;   // tile by tile, the heads of the group within a tile
   int32_t cn[G::NCH];
   Stage<G> st;
   float sv = 0;
   // thread tid < 64 * MAPS also carries one statistic of the tile's rows: number tid / 32 of row tid % 32
   const int sk = tid >> 5;
   auto load_stat = [&](int tile, int head) {
      float x = 0;
      if (sk < 2 * MAPS)
      {
         const int32_t c = cols[(int64_t)tile * kTile + (tid & 31)];
         if (c >= 0)
         {
            const int64_t at = ((int64_t)c * p.heads + head) * MAPS + (sk % MAPS);
            x = sk < MAPS ? p.lse_in[at] * kLog2e : p.delta[at];
         }
      }
      return x;
   };
   auto load_step = [&](int s) {
      const int tile = s / p.group, head = kvh * p.group + s % p.group;
      stage_cols<G>(cn, cols + (int64_t)tile * kTile, tid);
      stage_load<G, T, DC>(st, cn, (const E *)p.q + head * p.hdq, p.ldq, p.d, (const E *)p.dout + head * p.hdo, p.ldo, p.dv, p.vec, tid);
      sv = load_stat(tile, head);
   };
   auto store_step = [&](int b, int mark) {
      if (stage_store<G, T>(st, qs[b], gs[b], tid, true, true)) odd[b] = mark;
      if (sk < 2 * MAPS) stat[b][sk][tid & 31] = sv;
   };
   if (steps > 0)
   {
      load_step(0);
      __syncthreads();
      store_step(0, 1);
   }
   __syncthreads();
   uint64_t m0 = 0, m1 = 0;
   unsigned mine = 0;
   for (int s = 0; s < steps; s++)
   {
      const int b = s & 1, hh = s % p.group;
      if (s + 1 < steps) load_step(s + 1);
      if (hh == 0)
      {
         const int64_t off = (int64_t)(s / p.group) * (4 * kTile);
         m0 = *(const uint64_t *)(masks + off);
         m1 = *(const uint64_t *)(masks + off + 16);
         mine = my_bits(m0, m1, i);
      }
      if (__any((m0 | m1) != 0))
      {
         const bool bad = odd[b] == s + 1;
         const float lam = MAPS == 2 ? p.lambda[kvh * p.group + hh] : 0.0f;
         f4 dp[2];
         tile_scores<T, G::CV>(dp, gs[b], G::LD, vr, g, i);
         float wv[2][4];
#pragma unroll
         for (int mp = 0; mp < MAPS; mp++)
         {
            f4 sc[2];
            tile_scores<T, G::CQ>(sc, qs[b] + mp * DC, G::LD, kr[mp], g, i);
            const float sign = mp == 0 ? 1.0f : -lam;
            float w[2][4];
#pragma unroll
            for (int a = 0; a < 2; a++)
            {
               const f4 l = *(const f4 *)&stat[b][mp][16 * a + 4 * g], dl = *(const f4 *)&stat[b][MAPS + mp][16 * a + 4 * g];
#pragma unroll
               for (int r = 0; r < 4; r++)
               {
                  const bool named = (mine >> (4 * a + r)) & 1;
                  const float pr = named ? sign * exp2_fast(sc[a][r] * c2 - l[r]) : 0.0f;
                  w[a][r] = named ? pr * (dp[a][r] - dl[r]) : 0.0f;
                  wv[a][r] = mp == 0 ? pr : wv[a][r] + pr;
               }
            }
            add_weighted<T, G::NTQ>(dk[mp], w, mine, qs[b] + mp * DC, G::LD, g, i, bad);
         }
#pragma unroll
         for (int j = 0; j < 8; j++) wv[j / 4][j % 4] *= G::N::kPScale;
         add_weighted<T, G::NT>(dv, wv, mine, gs[b], G::LD, g, i, bad);
      }
      if (s + 1 < steps) store_step(b ^ 1, s + 2);
      __syncthreads();
   }

   constexpr float unscale = 1.0f / G::N::kPScale;
   if (u.part >= 0)
   {
      // [part][kv head][64 rows][2 W]
      float *r = p.part + (((int64_t)u.part * p.kv_heads + kvh) * kBlockRows + 16 * wave + i) * (2 * G::W);
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
         for (int x = 0; x < G::NTQ; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) r[mp * DC + 16 * x + 4 * g + e] = dk[mp][x][e];
#pragma unroll
      for (int x = 0; x < G::NT; x++)
#pragma unroll
         for (int e = 0; e < 4; e++) r[G::W + 16 * x + 4 * g + e] = dv[x][e] * unscale;
      return;
   }
   if (!live) return;
   E *outk = (E *)p.dk + row * p.ldk + kvh * p.hdk;
   E *outv = (E *)p.dvv + row * p.ldv + kvh * p.hdv;
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
      for (int x = 0; x < G::NTQ; x++) store4<T>(outk + mp * p.d, 16 * x + 4 * g, p.d, dk[mp][x] * p.scale, p.vec);
#pragma unroll
   for (int x = 0; x < G::NT; x++) store4<T>(outv, 16 * x + 4 * g, p.dv, dv[x] * unscale, p.vec);
}

template <int T, int DC, int MAPS> __global__ __launch_bounds__(256) void attn_dkv_join(Params p)
{
   typedef Geo<T, DC, MAPS> G;
   typedef typename G::E E;
   const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
   const int lane = threadIdx.x & 63;
   const int r = (int)(id % kBlockRows);
   const int kvh = (int)((id / kBlockRows) % p.kv_heads);
   const int64_t jn = id / kBlockRows / p.kv_heads;
   if (jn >= p.plan.n_joins) return;
   const Join j = p.plan.joins[jn];
   const int64_t row = (int64_t)j.block * kBlockRows + r;
   if (row >= p.n) return;
   const int64_t step = (int64_t)p.kv_heads * kBlockRows * (2 * G::W);
   const float *from = p.part + (((int64_t)j.part0 * p.kv_heads + kvh) * kBlockRows + r) * (2 * G::W);
   for (int f = lane; f < 2 * G::W; f += 64)
   {
      float s = 0;
      for (int u = 0; u < j.parts; u++) s += from[u * step + f];
      if (f < G::W)
      {
         const int mp = f / DC, e = f - mp * DC;
         if (e < p.d) ((E *)p.dk)[row * p.ldk + kvh * p.hdk + mp * p.d + e] = (E)Num<T>::from(s * p.scale);
      }
      else if (f - G::W < p.dv) ((E *)p.dvv)[row * p.ldv + kvh * p.hdv + f - G::W] = (E)Num<T>::from(s);
   }
}

}  // namespace fmm_attn
