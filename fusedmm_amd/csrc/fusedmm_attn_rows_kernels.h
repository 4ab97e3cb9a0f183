// Serving form of attention over a CSR pattern: few query rows, each over its own list of cache slots, with keys and
// values in the tensors' own type or in 4 bits.
//
// The 16 resident columns of the products are the query heads that share a key head (twice, with two maps), so that a
// cached row is read once for all of them; the call is bound by those reads.  A row's list is cut into pieces of `piece`
// slots, one workgroup each: its 4 waves take tiles of 32 slots in turn, each on its own - the keys go from memory
// straight into the operand layout, the values through the wave's own part of LDS, where they are read transposed - and
// join their sums at the end.  Rows of several pieces are joined by attn_rows_join.
#pragma once
#include "fusedmm_attn_core.h"

namespace fmm_attn {

struct RowsParams {
   int64_t m, n;
   int32_t heads, kv_heads, group, d, dv;
   int32_t passes;                    // runs of 16 / maps query heads within a group
   float scale;
   int32_t index_bytes;
   const void *indx, *pntrb, *pntre;
   const void *q, *k, *v;
   int64_t ldq, hdq, ldk, hdk, ldv, hdv, ldo, hdo;
   int32_t vec_q, vec_kv;
   const uint8_t *cache;              // 4-bit records, instead of k and v
   int64_t ldc, hdc;
   const float *lambda;
   void *out;
   int32_t out_type;                  // 4-bit cache: element type of q and out
   int64_t piece;                     // slots of a piece; doubled on the device while the pieces are more than cap
   int64_t cap;                       // pieces that the workspace has room for; 0: rows are not cut
   float *part;                       // [piece][kv head][pass][16 columns][W + kPartExtra]: W features, base, sum of weights
   int64_t *table;                    // m > kTableRows: [0] slots of a piece, [1 + r] pieces of the rows before r
};
constexpr int kPartExtra = 4;         // (two are used: columns stay on 16 bytes)
constexpr int kTableRows = 256;       // up to this many rows, every wave finds its piece from the row pointers itself

struct Kv4Params {
   int64_t tokens, n;
   int32_t kv_heads, k_width, v_width;   // maps * d, dv
   int32_t index_bytes;
   const void *slots;
   const void *k, *v;
   void *to_k, *to_v;
   int64_t ldk, hdk, ldv, hdv;
   int32_t vec;
   uint8_t *cache;
   int64_t ldc, hdc;
   int32_t per_group;                    // tokens of a workgroup (writing)
};

typedef float f2 __attribute__((ext_vector_type(2)));

__device__ inline int64_t index_of(const void *a, int64_t i, int bytes)
{
   return bytes == 4 ? (int64_t)((const int32_t *)a)[i] : ((const int64_t *)a)[i];
}

__device__ inline int64_t row_length(const RowsParams &p, int64_t row)
{
   const int64_t len = index_of(p.pntre, row, p.index_bytes) - index_of(p.pntrb, row, p.index_bytes);
   return len < 0 ? 0 : len;
}

__device__ inline int64_t pieces_of(int64_t len, int64_t piece)
{
   return len <= piece ? 1 : (len + piece - 1) / piece;
}

struct Spot {
   int64_t row, first, count;   // first piece of the row, number of its pieces
   int64_t piece;               // slots of a piece
   int64_t begin, len;          // the row's slots
};

__device__ inline void row_slots(const RowsParams &p, Spot &s)
{
   s.begin = index_of(p.pntrb, s.row, p.index_bytes);
   s.len = row_length(p, s.row);
}

// The row that piece `id` belongs to (id < 0: row `want` is asked for).  Called by whole waves; the result is uniform.
__device__ inline Spot find_piece(const RowsParams &p, int64_t id, int64_t want)
{
   Spot s;
   s.row = -1;
   if (p.cap == 0)   // one piece per row
   {
      s.row = id < 0 ? want : id < p.m ? id : -1;
      s.first = s.row;
      s.count = 1;
      s.piece = INT64_MAX;
      if (s.row >= 0) row_slots(p, s);
      return s;
   }
   if (p.m > kTableRows)
   {
      const int64_t *t = p.table + 1;
      s.piece = p.table[0];
      int64_t lo = 0;
      if (id < 0) lo = want;
      else
      {
         if (id >= t[p.m]) return s;
         int64_t hi = p.m;   // t[lo] <= id < t[hi]
         while (hi - lo > 1)
         {
            const int64_t mid = (lo + hi) / 2;
            if (t[mid] <= id) lo = mid;
            else hi = mid;
         }
      }
      s.row = lo;
      s.first = t[lo];
      s.count = t[lo + 1] - t[lo];
      row_slots(p, s);
      return s;
   }
   const int lane = threadIdx.x & 63;
   constexpr int kBatches = kTableRows / 64;
   int64_t begin[kBatches], len[kBatches];
#pragma unroll
   for (int b = 0; b < kBatches; b++)
   {
      len[b] = -1;
      begin[b] = 0;
      if (64 * b + lane < p.m)
      {
         begin[b] = index_of(p.pntrb, 64 * b + lane, p.index_bytes);
         len[b] = index_of(p.pntre, 64 * b + lane, p.index_bytes) - begin[b];
         if (len[b] < 0) len[b] = 0;
      }
   }
   int64_t piece = p.piece;
   for (;;)   // ends at the latest where every row is one piece: m <= cap
   {
      int64_t total = 0;
#pragma unroll
      for (int b = 0; b < kBatches; b++)
      {
         if (64 * b >= p.m) break;
         // (pieces in all are at most nnz / piece + m of the call's arguments, or more for wrong ones: kept within 32 bits)
         const int64_t most = len[b] < 0 ? 0 : pieces_of(len[b], piece);
         const int own = (int)(most < (1 << 24) ? most : 1 << 24);
         int x = own;
#pragma unroll
         for (int k = 1; k < 64; k <<= 1)
         {
            const int y = __shfl_up(x, k);
            if (lane >= k) x += y;
         }
         const bool here = id < 0 ? 64 * b + lane == want : len[b] >= 0 && total + x - own <= id && id < total + x;
         const unsigned long long hit = __ballot(here);
         if (hit)
         {
            const int src = __ffsll(hit) - 1;
            s.row = 64 * b + src;
            s.count = __shfl(own, src);
            s.first = total + __shfl(x, src) - s.count;
            s.begin = __shfl((long long)begin[b], src);
            s.len = __shfl((long long)len[b], src);
         }
         total += __shfl(x, 63);
      }
      s.piece = piece;
      if (total <= p.cap) return s;
      piece *= 2;
      s.row = -1;
   }
}

// m > kTableRows: one workgroup of 1024 threads
template <int UNIT> __global__ __launch_bounds__(1024) void attn_rows_table(RowsParams p)
{
   __shared__ int64_t sums[1024];
   const int tid = threadIdx.x;
   const int64_t per = (p.m + 1023) / 1024, lo = tid * per, hi = lo + per < p.m ? lo + per : p.m;
   int64_t piece = p.piece;
   for (;;)
   {
      int64_t x = 0;
      for (int64_t r = lo; r < hi; r++) x += pieces_of(row_length(p, r), piece);
      sums[tid] = x;
      __syncthreads();
      for (int s = 1; s < 1024; s <<= 1)
      {
         const int64_t y = tid >= s ? sums[tid - s] : 0;
         __syncthreads();
         sums[tid] += y;
         __syncthreads();
      }
      const int64_t total = sums[1023];
      if (total <= p.cap)
      {
         int64_t at = sums[tid] - x;
         for (int64_t r = lo; r < hi; r++)
         {
            p.table[1 + r] = at;
            at += pieces_of(row_length(p, r), piece);
         }
         if (tid == 0)
         {
            p.table[0] = piece;
            p.table[1 + p.m] = total;
         }
         return;
      }
      piece *= 2;
      __syncthreads();
   }
}

template <int T, int DC, int MAPS> struct RowGeo {
   typedef Num<T> N;
   typedef typename N::E E;
   static constexpr int W = DC * MAPS, CR = W / N::EPL;
   typedef TileView<T, W> V;
   static constexpr int CQ = DC / N::KC, NT = W / 16;
   static constexpr int HP = 16 / MAPS;               // query heads of a pass
   static constexpr int NV = kTile * CR / 64;         // 16-byte chunks of the values that a lane carries
};

__device__ inline void wave_lds_order()   // this wave's LDS writes before its later LDS reads
{
   __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
   __builtin_amdgcn_wave_barrier();
}

// products of 32 slots with the columns -> weights, and the weighted values
template <class G, int T, bool CAREFUL, bool TWICE>
__device__ inline void row_step(Softmax<G::NT, G::N::kLift> &r, f4 (&sc)[2], float c2, unsigned mine, bool all, const unsigned char *vs, int g, int i)
{
   if (!all)
   {
      keep_branch();
#pragma unroll
      for (int j = 0; j < 8; j++) sc[j / 4][j % 4] = masked(sc[j / 4][j % 4], mine, j, -INFINITY);
   }
   float w[2][4];
   r.weights(w, sc, c2);
   add_weighted<T, G::W, CAREFUL, TWICE>(r.acc, w, mine, vs, 0, g, i, G::V::lane(g, i));
}

// The four waves' sums -> the row's output, or its piece of the partial sums.  O: element type of the output.
template <class G, int MAPS, int O>
__device__ inline void rows_finish(const RowsParams &p, Softmax<G::NT, G::N::kLift> &r, unsigned char *vs_all, float (*stat)[16][2], const Spot &s, int64_t id, int kvh, int pass)
{
   const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, i = lane & 15;
   r.sum = group_sum(r.sum);
   float *mine = reinterpret_cast<float *>(vs_all + wave * G::V::kBytes) + i * G::W;   // 16 columns x W floats fit 32 rows of values
   wave_lds_order();
#pragma unroll
   for (int x = 0; x < G::NT; x++) *reinterpret_cast<f4 *>(mine + 16 * x + 4 * g) = r.acc[x];
   if (g == 0)
   {
      stat[wave][i][0] = r.base;
      stat[wave][i][1] = r.sum;
   }
   __syncthreads();
   // four features of a column, and the column's base and sum of weights
   auto column = [&](int c, int f, float &top, float &sum) {
      top = fmaxf(fmaxf(stat[0][c][0], stat[1][c][0]), fmaxf(stat[2][c][0], stat[3][c][0]));
      const float base = top == -INFINITY ? 0.0f : top;
      sum = 0;
      f4 x = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 4; w++)
      {
         const float keep = exp2_fast(stat[w][c][0] - base);
         sum += stat[w][c][1] * keep;
         x += *reinterpret_cast<const f4 *>(vs_all + w * G::V::kBytes + (c * G::W + f) * 4) * keep;
      }
      return x;
   };
   const int left = p.group - pass * G::HP, heads = left < G::HP ? left : G::HP;
   constexpr int C4 = G::W / 4;
   if (s.count > 1)
   {
      float *to = p.part + ((id * p.kv_heads + kvh) * p.passes + pass) * 16 * (G::W + kPartExtra);
      for (int e = tid; e < 16 * C4; e += 256)
      {
         const int c = e / C4, f = e % C4 * 4;
         if (c % G::HP >= heads) continue;
         float top, sum;
         *reinterpret_cast<f4 *>(to + c * (G::W + kPartExtra) + f) = column(c, f, top, sum);
         if (f == 0)
         {
            to[c * (G::W + kPartExtra) + G::W] = top;
            to[c * (G::W + kPartExtra) + G::W + 1] = sum;
         }
      }
      return;
   }
   typedef typename Num<O>::E EO;
   for (int e = tid; e < heads * C4; e += 256)
   {
      const int hh = e / C4, f = e % C4 * 4;
      if (f >= p.dv) continue;
      const int head = kvh * p.group + pass * G::HP + hh;
      float top, sum;
      f4 x = column(hh, f, top, sum);
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = sum == 0.0f ? 0.0f : x[j] / sum;
      if constexpr (MAPS == 2)
      {
         const f4 y = column(hh + 8, f, top, sum);
         const float lambda = p.lambda[head];
#pragma unroll
         for (int j = 0; j < 4; j++) x[j] -= lambda * (sum == 0.0f ? 0.0f : y[j] / sum);
      }
      store4<O>((EO *)p.out + s.row * p.ldo + head * p.hdo, f, p.dv, x, false);
   }
}

// Rows of several pieces: a workgroup per (row, head).  W / 4 lanes take a piece, batches of 8 without conditions so that
// their loads are under way together (places behind the last piece read the last one); the base follows the batches.
// Bound by the latency of a few dependent loads.  LDS: waves x MAPS x (W + 2) floats.  (UNIT: the object it is compiled into)
template <int UNIT, int O, int DC, int MAPS> __global__ __launch_bounds__(1024) void attn_rows_join(RowsParams p)
{
   constexpr int W = DC * MAPS, HP = 16 / MAPS, LANES = W / 4, B = 8, kMine = W + 2;
   typedef typename Num<O>::E EO;
   extern __shared__ float part[];
   const int64_t row = blockIdx.x / p.heads;
   const int head = (int)(blockIdx.x % p.heads), kvh = head / p.group, hh = head % p.group, pass = hh / HP;
   const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
   const int f0 = lane % LANES * 4, workers = waves * (64 / LANES), worker = wave * (64 / LANES) + lane / LANES;
   const Spot s = find_piece(p, -1, row);
   if (s.count <= 1) return;
   const int64_t step = (int64_t)p.kv_heads * p.passes * 16 * (W + kPartExtra);
   const float *from = p.part + ((s.first * p.kv_heads + kvh) * p.passes + pass) * 16 * (W + kPartExtra) + hh % HP * (W + kPartExtra);
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++, from += HP * (W + kPartExtra))
   {
      float base = -INFINITY, sum = 0;
      f4 o = {0, 0, 0, 0};
      auto follow = [&](float to) {   // the base becomes `to`, which is no lower
         const float keep = to == base ? 1.0f : exp2_fast(base - to);
         sum *= keep;
         o *= keep;
         base = to;
         return to == -INFINITY ? 0.0f : to;
      };
      for (int64_t u0 = 0; u0 < s.count; u0 += B * workers)
      {
         float top = base;
         f4 x[B];
         f2 n[B];
#pragma unroll
         for (int b = 0; b < B; b++)
         {
            const int64_t u = u0 + worker + b * workers;
            const float *f = from + (u < s.count ? u : s.count - 1) * step;
            n[b] = *reinterpret_cast<const f2 *>(f + W);
            x[b] = *reinterpret_cast<const f4 *>(f + f0);
         }
#pragma unroll
         for (int b = 0; b < B; b++) top = fmaxf(top, n[b][0]);
         const float at = follow(top);
#pragma unroll
         for (int b = 0; b < B; b++)
         {
            if (u0 + worker + b * workers >= s.count) break;
            const float keep = exp2_fast(n[b][0] - at);
            sum += n[b][1] * keep;
            o += x[b] * keep;
         }
      }
#pragma unroll
      for (int k = LANES; k < 64; k <<= 1)   // the pieces of a wave
      {
         follow(fmaxf(base, __shfl_xor(base, k)));
         sum += __shfl_xor(sum, k);
#pragma unroll
         for (int j = 0; j < 4; j++) o[j] += __shfl_xor(o[j], k);
      }
      float *mine = part + (wave * MAPS + mp) * kMine;
      if (lane < LANES)
      {
#pragma unroll
         for (int j = 0; j < 4; j++) mine[f0 + j] = o[j];
      }
      if (lane == 0)
      {
         mine[W] = base;
         mine[W + 1] = sum;
      }
   }
   __syncthreads();
   EO *out = (EO *)p.out + row * p.ldo + head * p.hdo;
   for (int f = threadIdx.x; f < p.dv; f += blockDim.x)
   {
      float r[MAPS];
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
      {
         float top = -INFINITY, sum = 0, x = 0;
         for (int w = 0; w < waves; w++) top = fmaxf(top, part[(w * MAPS + mp) * kMine + W]);
         const float at = top == -INFINITY ? 0.0f : top;
         for (int w = 0; w < waves; w++)
         {
            const float *of = part + (w * MAPS + mp) * kMine;
            const float keep = exp2_fast(of[W] - at);
            sum += of[W + 1] * keep;
            x += of[f] * keep;
         }
         r[mp] = sum == 0.0f ? 0.0f : x / sum;
      }
      if constexpr (MAPS == 2) r[0] -= p.lambda[head] * r[1];
      out[f] = (EO)Num<O>::from(r[0]);
   }
}

// workgroup b of a launch -> (piece, key head, pass): the key heads of a piece run next to each other on one XCD
struct RowsItem {
   int64_t id;
   int kvh, pass;
};
__device__ inline RowsItem rows_item(const RowsParams &p)
{
   const int64_t b = blockIdx.x, j = b >> 3;
   const int y = p.kv_heads * p.passes;
   RowsItem r;
   r.id = (j / y) * 8 + (b & 7);
   r.kvh = (int)(j % y) / p.passes;
   r.pass = (int)(j % y) % p.passes;
   return r;
}

// Slot of the tile's row lane % 32, -1 where there is none.  No branches: a load under a condition leaves the compiler
// without a count of the loads under way, and it then waits for all of them, the next tile's among them.  So the place is
// kept within the piece, and the two halves of a 64-bit id are read as such (of a 32-bit id, the same one twice).
__device__ inline int32_t tile_slot(const RowsParams &p, int64_t at, int64_t end, int lane)
{
   const int64_t e = at + (lane & 31), last = end - 1;
   const unsigned char *from = (const unsigned char *)p.indx + (e < end ? e : last) * p.index_bytes;
   const int32_t lo = *(const int32_t *)from, hi = *(const int32_t *)(from + p.index_bytes - 4);
   const bool wide = hi != (p.index_bytes == 8 ? 0 : lo);
   return e < end && !wide && lo >= 0 && lo < p.n ? lo : -1;
}

// the same with branches, where the loads are conditional anyhow
__device__ inline int32_t tile_slot_any(const RowsParams &p, int64_t at, int64_t end, int lane)
{
   const int64_t e = at + (lane & 31);
   if (e >= end) return -1;
   const int64_t c = index_of(p.indx, e, p.index_bytes);
   return c >= 0 && c < p.n ? (int32_t)c : -1;
}

__device__ inline unsigned tile_bits(int32_t slot, int g, bool *all)
{
   const uint32_t live = (uint32_t)__ballot(slot >= 0);
   *all = live == 0xffffffffu;
   return ((live >> (4 * g)) & 15) | (((live >> (16 + 4 * g)) & 15) << 4);
}

// ---- keys and values in their own type ------------------------------------------------------------------------------------------
// FULL: d and dv fill the width and every chunk is 16-byte aligned.  All loads are then unconditional: a place without a
// slot reads slot 0, whose scores are masked, and whose values have weight zero (or, if they are not finite, are seen by
// the pass that takes care of those).
template <int T, int DC, int MAPS, bool FULL>
__global__ __launch_bounds__(256, (sizeof(typename Num<T>::E) * DC * MAPS >= 512 ? 1 : 2)) void attn_rows(RowsParams p)
{
   typedef RowGeo<T, DC, MAPS> G;
   typedef typename G::E E;
   __shared__ __align__(16) unsigned char vs_all[4 * G::V::kBytes];
   __shared__ float stat[4][16][2];
   const RowsItem it = rows_item(p);
   const Spot s = find_piece(p, it.id, 0);
   if (s.row < 0) return;
   const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, i = lane & 15;
   unsigned char *vs = vs_all + wave * G::V::kBytes;
   const int64_t begin = s.begin, len = s.len;
   // (a cache without slots: nothing is read)
   const int64_t lo = s.count > 1 ? (it.id - s.first) * s.piece : 0, hi = p.n == 0 ? lo : s.count > 1 && lo + s.piece < len ? lo + s.piece : len;
   const E *k = (const E *)p.k + it.kvh * p.hdk, *v = (const E *)p.v + it.kvh * p.hdv;

   const int mp_i = i / G::HP, hh = it.pass * G::HP + i % G::HP;
   const bool col = hh < p.group;
   u4 q[G::CQ];
   auto query = [&](auto mode) __attribute__((always_inline)) {
      const E *from = (const E *)p.q + s.row * p.ldq + (col ? (it.kvh * p.group + hh) * p.hdq + mp_i * p.d : 0);
#pragma unroll
      for (int c = 0; c < G::CQ; c++) q[c] = load_part<T, decltype(mode)::value>(from, c * G::N::KC + g * G::N::EPL, p.d, col);
   };
   const int mode_q = part_mode<T>(p.vec_q, p.d);
   if (mode_q == kAligned) query(Mode<kAligned>());
   else if (mode_q == kShifted) query(Mode<kShifted>());
   else query(Mode<kElements>());
   if (p.scale < 0)
   {
#pragma unroll
      for (int c = 0; c < G::CQ; c++) q[c] = negated<T>(q[c]);
   }
   Softmax<G::NT, G::N::kLift> r;
   const float c2 = score_factor(p.scale);

   u4 kf[2][MAPS][G::CQ], vf[G::NV];
   auto load_as = [&](int32_t slot, auto mode) __attribute__((always_inline)) {
      constexpr int MODE = decltype(mode)::value;
#pragma unroll
      for (int a = 0; a < 2; a++)
      {
         const int32_t c = __shfl(slot, 16 * a + i);
         const E *row = k + (int64_t)(c < 0 ? 0 : c) * p.ldk;
#pragma unroll
         for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
            for (int x = 0; x < G::CQ; x++)
            {
               const int f = x * G::N::KC + g * G::N::EPL;
               if constexpr (FULL) kf[a][mp][x] = *reinterpret_cast<const u4 *>(row + mp * DC + f);
               else kf[a][mp][x] = load_part<T, MODE>(row + mp * p.d, f, p.d, c >= 0);
            }
      }
#pragma unroll
      for (int j = 0; j < G::NV; j++)
      {
         const int e = lane + 64 * j, f = (e % G::CR) * G::N::EPL;
         const int32_t c = __shfl(slot, e / G::CR);
         const E *at = v + (int64_t)(c < 0 ? 0 : c) * p.ldv;
         if constexpr (FULL) vf[j] = *reinterpret_cast<const u4 *>(at + f);
         else vf[j] = load_part<T, MODE>(at, f, p.dv, c >= 0);
      }
   };
   const int mode_kv = part_mode<T>(p.vec_kv, p.d < p.dv ? p.d : p.dv);
   auto load = [&](int32_t slot) __attribute__((always_inline)) {
      if (FULL || mode_kv == kAligned) load_as(slot, Mode<kAligned>());
      else if (mode_kv == kShifted) load_as(slot, Mode<kShifted>());
      else load_as(slot, Mode<kElements>());
   };
   constexpr int64_t kStride = 4 * kTile;
   const int64_t end = begin + hi;
   auto pass = [&](auto careful) {
      constexpr bool CAREFUL = decltype(careful)::value;
      r.clear();
      int64_t at = begin + lo + wave * kTile;
      int32_t slot = -1, next = -1;
      if (at < end)
      {
         slot = tile_slot(p, at, end, lane);
         next = tile_slot(p, at + kStride, end, lane);
         load(slot);
      }
      for (; at < end; at += kStride)
      {
         bool all;
         const unsigned mine = tile_bits(slot, g, &all);
#pragma unroll
         for (int j = 0; j < G::NV; j++)
         {
            const int e = lane + 64 * j;
            *reinterpret_cast<u4 *>(vs + (e / G::CR) * G::V::RB + ((e % G::CR) ^ G::V::twist(e / G::CR)) * 16) = vf[j];
         }
         f4 sc[MAPS][2];
#pragma unroll
         for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
            for (int a = 0; a < 2; a++)
            {
               sc[mp][a] = f4{0, 0, 0, 0};
#pragma unroll
               for (int x = 0; x < G::CQ; x++) sc[mp][a] = G::N::mma(kf[a][mp][x], q[x], sc[mp][a]);
            }
         slot = next;
         if (at + kStride < end)
         {
            load(slot);
            next = tile_slot(p, at + 2 * kStride, end, lane);
         }
         if constexpr (MAPS == 2)
         {
            sc[0][0] = mp_i ? sc[1][0] : sc[0][0];
            sc[0][1] = mp_i ? sc[1][1] : sc[0][1];
         }
         wave_lds_order();
         row_step<G, T, CAREFUL, T != kF32>(r, sc[0], c2, mine, all, vs, g, i);
         wave_lds_order();
      }
      return odd_sums(r.acc);
   };
   if (__any(pass(Flag<false>()))) (void)pass(Flag<true>());
   rows_finish<G, MAPS, T>(p, r, vs_all, stat, s, it.id, it.kvh, it.pass);
}

// ---- keys and values in 4 bits ----------------------------------------------------------------------------------------------------
// A record: codes of k (maps * d / 2 bytes), codes of v (dv / 2), one 16-bit word per 32 values of k and then of v.  The
// word is an fp16 scale with the zero point z in its low four mantissa bits; the value of code c is s (c - z).  s has at
// most 7 significant bits, c - z at most 4, so the value is exact in fp16 and the products run on fp16 operands.
// A code becomes 1024 + c with one and-or (0x6400 is fp16 1024; Kim et al., "Who Says Elephants Can't Run", 2022), c - z with
// one packed subtraction, the value with one packed product: 2 operations for 2 values, a third for the shift.
// The weights enter the second product as a rounded value and its rounded rest, as everywhere: with the value alone a row of
// 1500 slots was 2.5e-4 off in fp16, with both 2.1e-4, which is the output's own rounding.  It costs 64 rows up to
// 16384 slots 145.5 us instead of 144, two rows of 65k and 262k slots 37.4 instead of 36.
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
struct Scale4 {
   h2 scale, zero;
};
__device__ inline Scale4 scale_of(uint32_t word)
{
   const uint32_t s = word & 0xFFF0u, z = 0x6400u | (word & 15u);
   return Scale4{__builtin_bit_cast(h2, s | (s << 16)), __builtin_bit_cast(h2, z | (z << 16))};
}
__device__ inline u4 dequant8(uint32_t codes, Scale4 q)
{
   // (one of an and-or's two constants has to be a register: hidden from the compiler, which would split it in two)
   uint32_t bias = 0x64006400u;
   asm("" : "+v"(bias));
   u4 r;
#pragma unroll
   for (int j = 0; j < 4; j++)
   {
      const h2 x = __builtin_bit_cast(h2, ((codes >> (4 * j)) & 0x000F000Fu) | bias);
      const h2 y = (x - q.zero) * q.scale;
      r[j] = __builtin_bit_cast(uint32_t, y);
   }
   return r;
}

// FULL: d == DC and dv == DC * MAPS; a lane then reads a contiguous quarter of a row's codes, otherwise 4 bytes of every
// 32 codes.  Feature at which word j of lane group g starts:
template <bool FULL, int WORDS> __device__ inline int code_feature(int j, int g) { return FULL ? g * (WORDS * 8) + 8 * j : 32 * j + 8 * g; }

template <bool FULL, int WORDS> __device__ inline void load_codes(uint32_t (&to)[WORDS], const uint8_t *from, int width, int g)
{
   if constexpr (FULL && WORDS % 4 == 0)
   {
#pragma unroll
      for (int j = 0; j < WORDS / 4; j++)
      {
         const u4 x = *reinterpret_cast<const u4 *>(from + g * (WORDS * 4) + 16 * j);
#pragma unroll
         for (int e = 0; e < 4; e++) to[4 * j + e] = x[e];
      }
   }
   else if constexpr (FULL && WORDS == 2)
   {
      const u2 x = *reinterpret_cast<const u2 *>(from + g * 8);
      to[0] = x[0];
      to[1] = x[1];
   }
   else
   {
#pragma unroll
      for (int j = 0; j < WORDS; j++) to[j] = 32 * j < width ? *reinterpret_cast<const uint32_t *>(from + 16 * j + 4 * g) : 0;
   }
}

// The 16-bit words of a lane's codes: contiguous codes share one per 32
template <bool FULL, int WORDS> struct Words4 {
   static constexpr int N = FULL ? (WORDS + 3) / 4 : WORDS;
};
template <bool FULL, int WORDS, int N> __device__ inline void load_scales(uint32_t (&to)[N], const uint8_t *from, int width, int g)
{
#pragma unroll
   for (int j = 0; j < N; j++)
   {
      const int f = code_feature<FULL, WORDS>(FULL ? 4 * j : j, g);
      if constexpr (FULL) to[j] = *reinterpret_cast<const uint16_t *>(from + f / 32 * 2);
      else to[j] = f < width ? *reinterpret_cast<const uint16_t *>(from + f / 32 * 2) : 0;
   }
}

// one map's key and all of a value row of one slot, as a lane holds them
template <int DC, int MAPS, bool FULL> struct Record4 {
   static constexpr int WQ = DC / 32, WV = DC * MAPS / 32;
   uint32_t kc[MAPS][WQ], ks[MAPS][Words4<FULL, WQ>::N], vc[WV], vs[Words4<FULL, WV>::N];
};

template <int DC, int MAPS, bool FULL>
__global__ __launch_bounds__(256, (DC * MAPS >= 256 ? 1 : DC * MAPS == 128 && FULL ? 3 : 2)) void attn_rows_kv4(RowsParams p)
{
   typedef RowGeo<kF16, DC, MAPS> G;
   constexpr int WQ = DC / 32, WV = G::W / 32;   // 4-byte words of codes that a lane reads of one map's key, of a value row
   __shared__ __align__(16) unsigned char vs_all[4 * G::V::kBytes];
   __shared__ float stat[4][16][2];
   const RowsItem it = rows_item(p);
   const Spot s = find_piece(p, it.id, 0);
   if (s.row < 0) return;
   const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, i = lane & 15;
   unsigned char *vs = vs_all + wave * G::V::kBytes;
   const int64_t begin = s.begin, len = s.len;
   // (a cache without slots: nothing is read)
   const int64_t lo = s.count > 1 ? (it.id - s.first) * s.piece : 0, hi = p.n == 0 ? lo : s.count > 1 && lo + s.piece < len ? lo + s.piece : len;
   const uint8_t *cache = p.cache + it.kvh * p.hdc;
   const int kw = MAPS * p.d;
   const int off_v = kw / 2, off_kw = (kw + p.dv) / 2, off_vw = off_kw + kw / 16;   // bytes

   const int mp_i = i / G::HP, hh = it.pass * G::HP + i % G::HP;
   const bool col = hh < p.group;
   // The query as fp16, each head scaled by a power of two so that its largest feature is near 1: bf16's range does not
   // fit fp16's, its 8 bits of significand do.
   float qf[WQ][8];
   float top = 0;
#pragma unroll
   for (int j = 0; j < WQ; j++)
   {
      const int f = code_feature<FULL, WQ>(j, g);
      const uint16_t *from = (const uint16_t *)p.q + s.row * p.ldq + (col ? (it.kvh * p.group + hh) * p.hdq + mp_i * p.d + f : 0);
      u4 x = {0, 0, 0, 0};
      if (col && f < p.d) x = load_chunk<kF16>(from, p.vec_q);   // (d is a multiple of 32)
#pragma unroll
      for (int e = 0; e < 8; e++)
      {
         const uint16_t b = (uint16_t)(x[e / 2] >> (16 * (e & 1)));
         const float y = p.out_type == kF16 ? Num<kF16>::to(b) : Num<kBF16>::to(b);
         qf[j][e] = p.scale < 0 ? -y : y;
         top = fmaxf(top, fabsf(y));
      }
   }
   top = group_max(top);
   const int ex = top > 0 && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
   u4 q[WQ];
#pragma unroll
   for (int j = 0; j < WQ; j++)
   {
#pragma unroll
      for (int e = 0; e < 4; e++)
         q[j][e] = (uint32_t)Num<kF16>::from(ldexpf(qf[j][2 * e], -ex)) | (uint32_t)Num<kF16>::from(ldexpf(qf[j][2 * e + 1], -ex)) << 16;
   }
   const float c2 = score_factor(ldexpf(p.scale, ex));

   Softmax<G::NT, G::N::kLift> r;

   typedef Record4<DC, MAPS, FULL> Rec;
   auto load = [&](Rec (&to)[2], int32_t slot) __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < 2; a++)
      {
         // (a place without a slot reads record 0: see attn_rows)
         const int32_t c = __shfl(slot, 16 * a + i);
         const uint8_t *rec = cache + (int64_t)(c < 0 ? 0 : c) * p.ldc;
#pragma unroll
         for (int mp = 0; mp < MAPS; mp++)
         {
            load_codes<FULL>(to[a].kc[mp], rec + mp * p.d / 2, p.d, g);
            load_scales<FULL, WQ>(to[a].ks[mp], rec + off_kw + mp * p.d / 16, p.d, g);
         }
         load_codes<FULL>(to[a].vc, rec + off_v, p.dv, g);
         load_scales<FULL, WV>(to[a].vs, rec + off_vw, p.dv, g);
         if (!FULL && c < 0)
         {
#pragma unroll
            for (int j = 0; j < Words4<FULL, WV>::N; j++) to[a].vs[j] = 0;   // values of zero, whatever the record holds
         }
      }
   };
   constexpr int64_t kStride = 4 * kTile;
   const int64_t end = begin + hi;
   auto pass = [&](auto careful) {
      constexpr bool CAREFUL = decltype(careful)::value;
      r.clear();
      int64_t at = begin + lo + wave * kTile;
      auto use = [&](const Rec (&rec)[2], int32_t slot) __attribute__((always_inline)) {
         bool all;
         const unsigned mine = tile_bits(slot, g, &all);
         f4 sc[MAPS][2];
#pragma unroll
         for (int a = 0; a < 2; a++)
         {
#pragma unroll
            for (int mp = 0; mp < MAPS; mp++)
            {
               sc[mp][a] = f4{0, 0, 0, 0};
#pragma unroll
               for (int j = 0; j < WQ; j++) sc[mp][a] = G::N::mma(dequant8(rec[a].kc[mp][j], scale_of(rec[a].ks[mp][FULL ? j / 4 : j])), q[j], sc[mp][a]);
            }
#pragma unroll
            for (int j = 0; j < WV; j++)
               *reinterpret_cast<u4 *>(vs + (16 * a + i) * G::V::RB + ((code_feature<FULL, WV>(j, g) / 8) ^ G::V::twist(i)) * 16) =
                  dequant8(rec[a].vc[j], scale_of(rec[a].vs[FULL ? j / 4 : j]));
         }
         if constexpr (MAPS == 2)
         {
            sc[0][0] = mp_i ? sc[1][0] : sc[0][0];
            sc[0][1] = mp_i ? sc[1][1] : sc[0][1];
         }
         wave_lds_order();
         row_step<G, kF16, CAREFUL, true>(r, sc[0], c2, mine, all, vs, g, i);
         wave_lds_order();
      };
      // two tiles in turn, so that one is under way while the other is used
      Rec even[2], odd[2];
      int32_t slot = -1, next = -1;
      auto slot_of = [&](int64_t at) __attribute__((always_inline)) { return FULL ? tile_slot(p, at, end, lane) : tile_slot_any(p, at, end, lane); };
      if (at < end)
      {
         slot = slot_of(at);
         next = slot_of(at + kStride);
         load(even, slot);
      }
      while (at < end)
      {
         const int32_t after = slot_of(at + 2 * kStride);
         if (FULL || at + kStride < end) load(odd, next);   // (behind the end: slot 0, not used)
         use(even, slot);
         at += kStride;
         if (at >= end) break;
         slot = slot_of(at + 2 * kStride);
         if (FULL || at + kStride < end) load(even, after);
         use(odd, next);
         at += kStride;
         next = slot;
         slot = after;
      }
      return odd_sums(r.acc);
   };
   if (__any(pass(Flag<false>()))) (void)pass(Flag<true>());
   if (p.out_type == kF16) rows_finish<G, MAPS, kF16>(p, r, vs_all, stat, s, it.id, it.kvh, it.pass);
   else rows_finish<G, MAPS, kBF16>(p, r, vs_all, stat, s, it.id, it.kvh, it.pass);
}

// ---- into the 4-bit cache and back ---------------------------------------------------------------------------------------------------
// The step between codes is the group's range (with zero in it) over 15, rounded up to 7 significant bits and to a multiple
// of 2^-20; code and zero point are rounded to nearest, ties to even.  The borders between codes are decided by the
// correctly rounded quotient x / s, in 64 bits for 32-bit values.  For 16-bit values 32 bits decide alike: x has 11
// significant bits and a border 12, so a quotient that is not a border is further from it than 2^-24 of its size; and
// with the correctly rounded 1 / s, q + (x - q s) / s is the correctly rounded quotient (Markstein, 1990).
template <int T> __device__ inline float code_of(float x, float s, float inv)
{
   if constexpr (T == kF32) return (float)rint((double)x / (double)s);
   else
   {
      const float q = x * inv;
      return rintf(fmaf(fmaf(-q, s, x), inv, q));
   }
}

constexpr int kKv4Tokens = 8;   // most tokens of a workgroup: it compares their slots, in registers, with all later ones

// A lane per group of 32 values: the 64-bit arithmetic of the step, once per group, then costs less than the codes.
template <int T> __global__ __launch_bounds__(256) void kv4_write(Kv4Params p)
{
   typedef typename Num<T>::E E;
   constexpr int EPL = Num<T>::EPL;
   __shared__ int32_t slot[kKv4Tokens];
   __shared__ int later[kKv4Tokens];
   const int tid = threadIdx.x;
   const int64_t t0 = (int64_t)blockIdx.x * p.per_group;
   const int here = (int)(p.tokens - t0 < p.per_group ? p.tokens - t0 : p.per_group);
   auto slot_at = [&](int64_t t) {   // -1: the token goes nowhere
      const int64_t c = index_of(p.slots, t, p.index_bytes);
      return c >= 0 && c < p.n ? (int32_t)c : -1;
   };
   if (tid < kKv4Tokens)
   {
      later[tid] = 0;
      slot[tid] = tid < here ? slot_at(t0 + tid) : -1;
   }
   __syncthreads();
   // a slot that is named more than once takes the last token that names it
   int32_t mine[kKv4Tokens];
#pragma unroll
   for (int x = 0; x < kKv4Tokens; x++) mine[x] = slot[x];
   unsigned dup = 0;
#pragma unroll 4
   for (int64_t t = t0 + 1 + tid; t < p.tokens; t += 256)
   {
      const int32_t c = slot_at(t);
#pragma unroll
      for (int x = 0; x < kKv4Tokens; x++) dup |= (unsigned)(mine[x] == c && t0 + x < t) << x;
   }
#pragma unroll
   for (int x = 0; x < kKv4Tokens; x++)
      if (__any((dup >> x) & 1) && (tid & 63) == 0) later[x] = 1;
   __syncthreads();
   const int groups = (p.k_width + p.v_width) / 32, per_token = groups * p.kv_heads;
   for (int x = tid; x < here * per_token; x += 256)
   {
      const int tok = x / per_token, head = x % per_token / groups, grp = x % groups;
      const int64_t c = slot[tok];
      if (c < 0 || later[tok]) continue;
      const bool is_v = 32 * grp >= p.k_width;
      const int f = is_v ? 32 * grp - p.k_width : 32 * grp;
      const E *from = is_v ? (const E *)p.v + (t0 + tok) * p.ldv + head * p.hdv + f : (const E *)p.k + (t0 + tok) * p.ldk + head * p.hdk + f;
      float v[32];
#pragma unroll
      for (int j = 0; j < 32 / EPL; j++)
      {
         const u4 a = load_chunk<T>(from + j * EPL, p.vec);
#pragma unroll
         for (int e = 0; e < EPL; e++)
         {
            if constexpr (T == kF32) v[4 * j + e] = __uint_as_float(a[e]);
            else v[8 * j + e] = Num<T>::to((E)(a[e / 2] >> (16 * (e & 1))));
         }
      }
      float lo = 0, hi = 0;
      bool nan = false;   // makes its whole group NaN
#pragma unroll
      for (int e = 0; e < 32; e++)
      {
         nan |= v[e] != v[e];
         v[e] = fminf(fmaxf(v[e], -32768.0f), 32768.0f);   // what a step of fp16 reaches
         lo = fminf(lo, v[e]);
         hi = fmaxf(hi, v[e]);
      }
      const double step = ((double)hi - (double)lo) / 15.0;
      int e2;
      (void)frexp(step, &e2);   // step in [2^(e2 - 1), 2^e2)
      const int unit = step == 0 || e2 - 7 < -20 ? -20 : e2 - 7;
      const float s = (float)ldexp(ceil(ldexp(step, -unit)), unit);
      const float z = s > 0 ? (float)rint(-(double)lo / (double)s) : 0.0f, inv = s > 0 ? 1.0f / s : 0.0f;
      u4 codes = {0, 0, 0, 0};
      if (s > 0 && !nan)
      {
#pragma unroll
         for (int e = 0; e < 32; e++)
         {
            const float q = fminf(fmaxf(code_of<T>(v[e], s, inv) + z, 0.0f), 15.0f);
            codes[e / 8] |= (uint32_t)q << (4 * ((e % 2) * 4 + e % 8 / 2));
         }
      }
      uint8_t *rec = p.cache + c * p.ldc + head * p.hdc;
      *reinterpret_cast<u4 *>(rec + 16 * grp) = codes;
      const uint32_t word = nan ? 0x7E00u : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)s) | (uint32_t)z;
      *reinterpret_cast<uint16_t *>(rec + 16 * groups + 2 * grp) = (uint16_t)word;
   }
}

template <int T> __global__ __launch_bounds__(256) void kv4_read(Kv4Params p)
{
   typedef typename Num<T>::E E;
   const int words = (p.k_width + p.v_width) / 8;
   const int64_t total = p.tokens * p.kv_heads * words;
   for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < total; x += (int64_t)gridDim.x * 256)
   {
      const int64_t tok = x / (p.kv_heads * words);
      const int head = (int)(x / words % p.kv_heads), w = (int)(x % words);
      const int64_t c = index_of(p.slots, tok, p.index_bytes);
      uint32_t codes = 0, word = 0;
      if (c >= 0 && c < p.n)
      {
         const uint8_t *rec = p.cache + c * p.ldc + head * p.hdc;
         codes = *reinterpret_cast<const uint32_t *>(rec + 4 * w);
         word = *reinterpret_cast<const uint16_t *>(rec + 4 * words + w / 4 * 2);
      }
      const u4 h = dequant8(codes, scale_of(word));
      const bool is_v = 8 * w >= p.k_width;
      const int f = is_v ? 8 * w - p.k_width : 8 * w;
      E *to = is_v ? (E *)p.to_v + tok * p.ldv + head * p.hdv + f : (E *)p.to_k + tok * p.ldk + head * p.hdk + f;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = Num<kF16>::to((uint16_t)(h[e / 2] >> (16 * (e & 1))));
      store4<T>(to, 0, 8, f4{v[0], v[1], v[2], v[3]}, p.vec);
      store4<T>(to, 4, 8, f4{v[4], v[5], v[6], v[7]}, p.vec);
   }
}

}  // namespace fmm_attn
