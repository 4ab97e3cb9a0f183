// Kernels of attention over a planned pattern: forward, the two backward passes, the joins of split blocks, and the packing of
// rows that are not whole chunks.
//
// A plan (fusedmm_attn_plan.hip) lists, for every block of BR = 64 or 16 rows, the columns that any of them names, with
// one bit per row.  A unit is a run of such columns of one block; a block whose rows are long is several units, whose
// partial sums the join kernels add in order.  A workgroup does one unit for one head: BR / 16 waves of 16 resident rows
// share the tiles of 32 gathered rows, and one 16 x 16 product serves 16 rows.  With BR = 64 a gathered row is loaded once
// for 64 rows (a tile that no row of a wave names is skipped by that wave); with BR = 16 nothing is shared but nothing
// is multiplied for the rows of other waves either, which is what rows without common neighbours want.
//
// The tiles go from memory straight into LDS (no registers in between), with BR = 64 one ahead of the one in use.  Column
// ids and masks run ahead of them the same way, in groups of 8 tiles.
#pragma once
#include "fusedmm_attn_core.h"

namespace fmm_attn {

struct Unit {
   int32_t block;     // rows BR * block ...
   int32_t part;      // slot of its partial sums, -1: the block's only unit
   int32_t tile0;     // first tile of its columns
   int32_t tiles;
};
struct Join {         // a block of several units: partial sums part0 .. part0 + parts - 1
   int32_t block, part0, parts, pad;
};

constexpr int kAhead = 8;   // tiles of a group of column ids and masks; the arrays of a plan are padded by a group

struct PlanView {
   const int32_t *cols;    // [tiles][32]; behind a unit's last column that column again, named by no row
   const uint32_t *masks;  // [tiles][BR]: row r of the block; bit 8g + 4a + r is the tile's column 16a + 4g + r, as the lanes hold them
   const Unit *units;
   const Join *joins;
   int32_t n_units, n_joins;
   int32_t block_rows;     // BR
};

// The tensors whose rows are gathered: k and v (forward, dq), or q and do (dkv), as the caller has them or, where their rows
// are not whole 16-byte chunks, in rows of W elements that attn_pack has laid out: every row is then gathered once per
// block that names it by direct loads, instead of being shifted into place each time.
struct Gathered {
   const void *a, *b;                 // rows of maps pieces of d features, rows of dv features
   int64_t ha, hb;                    // elements from head to head
   int32_t lda_bytes, ldb_bytes;      // bytes from row to row
   int32_t d, dv;
   int32_t vec;                       // every row is 16-byte aligned and d, dv are multiples of a 16-byte chunk
   int32_t full;                      // vec, and d and dv fill the instance's width
};

struct Params {
   PlanView plan;
   Gathered gat;
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
   float *stats;                      // [m][heads][2 maps]: lse * log2(e) of every map, delta of every map
   float *dlam_units;                 // [unit][wave][heads]: sum over a wave's rows of sum_j P_2 dP
   int64_t dlam_count;                // units * waves
   float *part;                       // partial sums of split blocks
};

__device__ u4 zero_chunk;   // what lanes whose chunk is behind the features load

template <int T, int DC, int MAPS, int BR> struct Geo {
   typedef Num<T> N;
   typedef typename N::E E;
   static constexpr int W = DC * MAPS;                // padded width of a gathered row: all maps of q or k; v and do
   typedef TileView<T, W> V;
   static constexpr int CR = V::CR;
   static constexpr int THREADS = BR * 4, WAVES = BR / 16;
   static constexpr int NCH = (kTile * CR + THREADS - 1) / THREADS;   // chunks a thread loads of one tensor's tile
   static constexpr int CQ = DC / N::KC;              // chunk groups of a product over one map's features
   static constexpr int CV = W / N::KC;
   static constexpr int MC = DC / N::EPL;             // chunks of one map
   static constexpr int NT = W / 16, NTQ = DC / 16;   // 16-feature tiles of v's and of one map's accumulators
   // Tiles of a workgroup, in flight and being used.  A workgroup of one wave is better off with one tile and more company:
   // training over a graph with 16 neighbours, 4 heads of 128 bf16 (f32) features, 139 us (580) with one, 218 (1069) with
   // two.  Only where two tensors' tiles are 8 KB two are ahead, 92 us against 97 (64 bf16 features), 158 against 180 (32
   // f32).  Workgroups of four waves: two are 1 to 3 % ahead of one with 16-bit types and as good with f32; three or four cost
   // residency (a window of 512 at 128 bf16 features 55 us, 44 with two).
   static constexpr int kPair = 2 * V::kBytes;
   static constexpr int S = BR == 64 || kPair == 8192 ? 2 : 1;
   static constexpr int kMaskBytes = BR * 4;               // of a tile
   static constexpr int kStat = 2 * MAPS * kTile * 4;      // statistics of a tile's rows (dk, dv)
};

__device__ inline void wait_loads()   // all loads have arrived, LDS operations are done
{
   asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}
template <int BR> __device__ inline void tile_barrier()
{
   if constexpr (BR > 16) asm volatile("s_barrier" ::: "memory");
}

// 16 (4) bytes per lane, memory -> LDS at base + 16 (4) * lane.  The address registers are read when the load issues, it
// writes no register but m0, which is named so that the compiler keeps nothing in it across (it warns that it would not save
// a reserved register; none is wanted back).  The waits are wait_loads(): the compiler's own waits for its own loads
// count these as later or earlier ones and only get stricter.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ inline void load_lds16(uint32_t base, const void *from)
{
   asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(base)), "v"(from) : "memory", "m0");
}
__device__ inline void load_lds4(uint32_t base, const void *from)
{
   asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(base)), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ inline uint32_t lds_address(const void *p)
{
   return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p);
}

// ---- the stream of tiles ------------------------------------------------------------------------------------------------------------

template <class G, int T, int DC, int BR> struct Stream {
   typedef typename G::E E;
   typedef typename G::V V;
   const unsigned char *tiles;   // LDS: [S][a, b] tiles
   unsigned char *ids, *bits;    // LDS: two groups of column ids, of masks
   const int32_t *cols;          // of the unit
   const uint32_t *masks;
   int tid, wave;
   const unsigned char *a, *b;
   uint32_t lda, ldb;            // bytes from row to row
   int d, dv;
   bool vec;
   static constexpr int NB = BR == 64 ? G::NCH : 1;
   const unsigned char *pa[NB], *pb[NB];   // BR = 64: this thread's chunks of row 0 (more threads would be more registers)

   __device__ inline void set(const unsigned char *t, unsigned char *i, unsigned char *m, const Params &p, const Unit &u, int64_t head)
   {
      tiles = t;
      ids = i;
      bits = m;
      cols = p.plan.cols + (int64_t)u.tile0 * kTile;
      masks = p.plan.masks + (int64_t)u.tile0 * BR;
      tid = threadIdx.x;
      wave = __builtin_amdgcn_readfirstlane(tid >> 6);
      a = (const unsigned char *)((const E *)p.gat.a + head * p.gat.ha);
      b = (const unsigned char *)((const E *)p.gat.b + head * p.gat.hb);
      lda = p.gat.lda_bytes;
      ldb = p.gat.ldb_bytes;
      d = p.gat.d;
      dv = p.gat.dv;
      vec = p.gat.vec;
      if constexpr (BR == 64)
      {
#pragma unroll
         for (int j = 0; j < G::NCH; j++)
         {
            const int x = tid + G::THREADS * j, at = ((x % G::CR) ^ V::twist(x / G::CR)) * 16;
            pa[j] = a + at;
            pb[j] = b + at;
         }
      }
   }

   // column ids and masks of tiles 8 g .. 8 g + 7; waves 0 and 1 (the ones that always load tiles) do it
   __device__ __forceinline__ void load_ids(int g) const
   {
      const uint32_t to_ids = lds_address(ids + (g & 1) * (kAhead * kTile * 4)), to_bits = lds_address(bits + (g & 1) * (kAhead * G::kMaskBytes));
      const unsigned char *from = (const unsigned char *)masks + (int64_t)g * (kAhead * G::kMaskBytes);
      const int lane = tid & 63;
      if (wave == 0) load_lds16(to_ids, (const unsigned char *)cols + (int64_t)g * (kAhead * kTile * 4) + lane * 16);
      if constexpr (BR == 64)
      {
         if (wave < 2) load_lds16(to_bits + 1024 * wave, from + 1024 * wave + lane * 16);
      }
      else
      {
         if (lane < kAhead * G::kMaskBytes / 16) load_lds16(to_bits, from + lane * 16);
      }
   }

   __device__ inline const int32_t *tile_ids(int t) const
   {
      return (const int32_t *)(ids + ((t / kAhead) & 1) * (kAhead * kTile * 4) + (t % kAhead) * (kTile * 4));
   }
   // which of the tile's columns resident row i names
   __device__ inline uint32_t row_mask(int t, int i) const
   {
      return *(const uint32_t *)(bits + ((t / kAhead) & 1) * (kAhead * G::kMaskBytes) + (t % kAhead) * G::kMaskBytes + (wave * 16 + i) * 4);
   }

   // Tile t -> buffer; the rows start oa and ob bytes behind a and b (other heads).
   // d and dv fill the width and every chunk is 16-byte aligned: the shortest way.
   __device__ __forceinline__ void load_full(int t, int buf, int64_t oa, int64_t ob) const
   {
      const int32_t *c = tile_ids(t);
      const uint32_t la = lds_address(tiles + buf * G::kPair) + wave * 1024, lb = la + V::kBytes;
      int me = tid;
      if constexpr (BR != 64) asm volatile("" : "+v"(me));   // the places are formed again for every tile, not kept in registers
#pragma unroll
      for (int j = 0; j < G::NCH; j++)
      {
         const int x = me + G::THREADS * j, r = x / G::CR;
         if (kTile * G::CR < G::THREADS && x >= kTile * G::CR) break;
         const uint32_t col = (uint32_t)c[r];
         const unsigned char *fa, *fb;
         if constexpr (BR == 64)
         {
            fa = pa[j];
            fb = pb[j];
         }
         else
         {
            const int at = ((x % G::CR) ^ V::twist(r)) * 16;
            fa = a + at;
            fb = b + at;
         }
         load_lds16(la + j * (G::THREADS * 16), fa + oa + (uint64_t)col * lda);
         load_lds16(lb + j * (G::THREADS * 16), fb + ob + (uint64_t)col * ldb);
      }
   }

   // any sizes
   __device__ __forceinline__ void load_any(int t, int buf, int64_t oa, int64_t ob) const
   {
      const int32_t *c = tile_ids(t);
      unsigned char *ta = const_cast<unsigned char *>(tiles) + buf * G::kPair, *tb = ta + V::kBytes;
      const uint32_t la = lds_address(ta) + wave * 1024, lb = la + V::kBytes;
      int me = tid;
      asm volatile("" : "+v"(me));
#pragma unroll
      for (int j = 0; j < G::NCH; j++)
      {
         if (!vec) break;
         const int x = me + G::THREADS * j, r = x / G::CR;
         if (kTile * G::CR < G::THREADS && x >= kTile * G::CR) break;
         const uint32_t col = (uint32_t)c[r];
         const int e = ((x % G::CR) ^ V::twist(r)) * G::N::EPL, f = e % DC;   // this thread's chunk of a gathered row
         const E *fa = (const E *)(a + oa + (uint64_t)col * lda) + (e / DC * d + f);
         const E *fb = (const E *)(b + ob + (uint64_t)col * ldb) + e;
         load_lds16(la + j * (G::THREADS * 16), f < d ? (const void *)fa : (const void *)&zero_chunk);
         load_lds16(lb + j * (G::THREADS * 16), e < dv ? (const void *)fb : (const void *)&zero_chunk);
      }
      if (vec) return;
      // a tensor that begins off 16 bytes (other rows off them are packed): through registers, a few chunks at a time
      constexpr int B = G::NCH < 4 ? G::NCH : 4;
#pragma unroll
      for (int j0 = 0; j0 < G::NCH; j0 += B)
      {
         u4 ra[B], rb[B];
#pragma unroll
         for (int j = 0; j < B; j++)
         {
            const int x = me + G::THREADS * (j0 + j), r = x / G::CR;
            const bool live = kTile * G::CR >= G::THREADS || x < kTile * G::CR;
            const uint32_t col = (uint32_t)c[live ? r : 0];
            const int e = ((x % G::CR) ^ V::twist(r)) * G::N::EPL, f = e % DC;
            ra[j] = load_part<T, kShifted>((const E *)(a + oa + (uint64_t)col * lda) + e / DC * d, f, d, live);
            rb[j] = load_part<T, kShifted>((const E *)(b + ob + (uint64_t)col * ldb), e, dv, live);
         }
#pragma unroll
         for (int j = 0; j < B; j++)
         {
            const int x = me + G::THREADS * (j0 + j);
            if (kTile * G::CR < G::THREADS && x >= kTile * G::CR) break;
            *(u4 *)(ta + x * 16) = ra[j];
            *(u4 *)(tb + x * 16) = rb[j];
         }
      }
   }

   template <bool FULL> __device__ __forceinline__ void load_tile(int t, int buf, int64_t oa, int64_t ob) const
   {
      if constexpr (FULL) load_full(t, buf, oa, ob);
      else load_any(t, buf, oa, ob);
   }
};

// Rows at any place -> rows of w elements (maps pieces of w / maps, zeros behind their d features; zeros behind dv), head by
// head.  A thread per 16-byte chunk; bound by reading and writing the tensors once.
struct PackParams {
   const void *a, *b;
   void *to_a, *to_b;
   int64_t rows, lda, ha, ldb, hb;    // elements
   int32_t heads, d, dv, dc, chunks;  // chunks of a row of w
   int32_t per_head;                  // workgroups
};
template <int T> __global__ __launch_bounds__(256) void attn_pack(PackParams p)
{
   typedef typename Num<T>::E E;
   const unsigned z = blockIdx.x / p.per_head;   // heads of a, then of b
   const bool second = z >= (unsigned)p.heads;
   const int64_t head = second ? z - p.heads : z;
   const E *from = second ? (const E *)p.b + head * p.hb : (const E *)p.a + head * p.ha;
   const int64_t ld = second ? p.ldb : p.lda, total = p.rows * p.chunks;
   u4 *to = (u4 *)(second ? p.to_b : p.to_a) + head * total;
   const bool small = p.d < Num<T>::EPL || p.dv < Num<T>::EPL;
   for (int64_t x = (int64_t)(blockIdx.x % p.per_head) * 256 + threadIdx.x; x < total; x += (int64_t)p.per_head * 256)
   {
      const int e = (int)(x & (p.chunks - 1)) * Num<T>::EPL;   // (a power of two of chunks)
      const E *row = from + (x / p.chunks) * ld + (second ? 0 : e / p.dc * p.d);
      const int f = second ? e : e % p.dc, width = second ? p.dv : p.d;
      to[x] = small ? load_part<T, kElements>(row, f, width, true) : load_part<T, kShifted>(row, f, width, true);
   }
}

// the resident rows of a wave as the second operand: lane i holds its 16 bytes of every chunk of row i
template <int T, int MODE, int CQ> __device__ inline void load_resident_as(u4 (&r)[CQ], const typename Num<T>::E *row, bool live, int d, int g)
{
#pragma unroll
   for (int c = 0; c < CQ; c++) r[c] = load_part<T, MODE>(row, c * Num<T>::KC + g * Num<T>::EPL, d, live);
}

template <int T, int CQ> __device__ inline void load_resident(u4 (&r)[CQ], const typename Num<T>::E *row, bool live, int d, int g, bool vec)
{
   const int mode = part_mode<T>(vec, d);
   if (mode == kAligned) load_resident_as<T, kAligned>(r, row, live, d, g);
   else if (mode == kShifted) load_resident_as<T, kShifted>(r, row, live, d, g);
   else load_resident_as<T, kElements>(r, row, live, d, g);
}

// this lane's part of the product of two resident rows
template <int T, int CQ> __device__ inline float chunk_dot(const u4 (&a)[CQ], const u4 (&b)[CQ])
{
   float s = 0;
#pragma unroll
   for (int c = 0; c < CQ; c++)
#pragma unroll
      for (int e = 0; e < 4; e++)
      {
         if constexpr (T == kF32) s = fmaf(__uint_as_float(a[c][e]), __uint_as_float(b[c][e]), s);
         else
         {
            s = fmaf(Num<T>::to((uint16_t)a[c][e]), Num<T>::to((uint16_t)b[c][e]), s);
            s = fmaf(Num<T>::to((uint16_t)(a[c][e] >> 16)), Num<T>::to((uint16_t)(b[c][e] >> 16)), s);
         }
      }
   return s;
}

// scores of the tile's 32 rows, from chunk `chunk` on, against the resident rows: s[a] rows 16a + 4g + r
template <int T, int W, int CQ> __device__ inline void tile_scores(f4 (&s)[2], const unsigned char *tile, int chunk, const u4 (&res)[CQ], const typename TileView<T, W>::Lane &l)
{
   typedef TileView<T, W> V;
   s[0] = f4{0, 0, 0, 0};
   s[1] = f4{0, 0, 0, 0};
#pragma unroll
   for (int c = 0; c < CQ; c++)
   {
      s[0] = Num<T>::mma(V::direct(tile, chunk + 4 * c, 0, l), res[c], s[0]);
      s[1] = Num<T>::mma(V::direct(tile, chunk + 4 * c, 1, l), res[c], s[1]);
   }
}

template <int BR> __device__ inline bool any_odd(bool odd)
{
   if constexpr (BR == 16) return __any(odd);
   else return __syncthreads_or(odd);
}
// How a pass over a unit runs: full 16-byte chunks, any sizes, or any sizes with care for infinities and NaN.
enum : int { kFull, kAny, kCareful };
// The loop over a unit's tiles that all kernels share.  steps = tiles * per_tile; load(step, buffer), use(step, buffer).
// The ids of the next group are asked for a group ahead: the waits for the tiles in between include them.
template <class G, int BR, class S, class Load, class Use> __device__ __forceinline__ void for_tiles(const S &st, int steps, int per_tile, Load load, Use use)
{
   if (steps > 0)
   {
      st.load_ids(0);
      wait_loads();
      tile_barrier<BR>();
      if (G::S == 2) load(0, 0);
   }
   for (int s = 0; s < steps; s++)
   {
      const int group = s / (kAhead * per_tile) + 1;
      const bool ids = s % (kAhead * per_tile) == 0 && group * (kAhead * per_tile) < steps;
      if constexpr (G::S == 1)
      {
         if (ids) st.load_ids(group);
         load(s, 0);
         wait_loads();
         tile_barrier<BR>();
         use(s, 0);
         wait_loads();   // (LDS: this wave has read the tile)
         tile_barrier<BR>();
      }
      else
      {
         wait_loads();
         tile_barrier<BR>();
         if (ids) st.load_ids(group);
         if (s + 1 < steps) load(s + 1, (s + 1) & 1);
         use(s, s & 1);
      }
   }
   wait_loads();   // nothing is under way into LDS when it is used again
   tile_barrier<BR>();
}

// What a backward pass takes off the scores: lse in units of log2.  A row that weighs nothing (no edges, or all scores minus
// infinity) has minus infinity there; plus infinity makes all its weights zero, not NaN.
__device__ inline float row_offset(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }
// lse is off by up to |lse| 2^-24 and is turned between logarithms twice: all weights of a row are then off alike, by some 1e-7.
// Their sum tells by how much.  dq and the means are divided by it; the offset that dkv takes off is moved by its logarithm.
__device__ inline float row_share(float total) { return total == 0.0f ? 0.0f : 1.0f / total; }
__device__ inline float row_offset(float lse2, float total) { return total > 0.0f ? lse2 + log2f(total) : lse2; }

#define ATTN_LDS(EXTRA)                                                                                                                        \
   __shared__ __align__(1024) unsigned char lds[G::S * G::kPair + 2 * kAhead * kTile * 4 + 2 * kAhead * G::kMaskBytes + G::S * (EXTRA)];          \
   unsigned char *lds_ids = lds + G::S * G::kPair, *lds_bits = lds_ids + 2 * kAhead * kTile * 4;                                                   \
   [[maybe_unused]] unsigned char *lds_extra = lds_bits + 2 * kAhead * G::kMaskBytes;

// ---- forward ----------------------------------------------------------------------------------------------------------------------
// One pass over a unit's columns with a running maximum and sum of every row and map.  Scores are kept times log2(e).
template <int T, int DC, int MAPS, int BR> __global__ __launch_bounds__(BR * 4, (DC * MAPS >= 256 || (BR == 16 && T == kF32 && DC * MAPS >= 128) ? 1 : 2)) void attn_forward(Params p)
{
   typedef Geo<T, DC, MAPS, BR> G;
   typedef typename G::E E;
   ATTN_LDS(0)
   const int64_t item = xcd_item(blockIdx.x, (int64_t)p.plan.n_units * p.heads);
   if (item >= (int64_t)p.plan.n_units * p.heads) return;
   const int head = (int)(item / p.plan.n_units);
   const Unit u = p.plan.units[item % p.plan.n_units];
   const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, i = lane & 15;
   const int kvh = head / p.group;
   const int64_t row = (int64_t)u.block * BR + 16 * wave + i;
   const bool live = row < p.m;
   Stream<G, T, DC, BR> st;
   st.set(lds, lds_ids, lds_bits, p, u, kvh);

   u4 qr[MAPS][G::CQ];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
      load_resident<T, G::CQ>(qr[mp], (const E *)p.q + (live ? row : 0) * p.ldq + head * p.hdq + mp * p.d, live, p.d, g, p.vec);
   const float c2 = score_factor(p.scale);
   if (p.scale < 0)
   {
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
         for (int c = 0; c < G::CQ; c++) qr[mp][c] = negated<T>(qr[mp][c]);
   }
   Softmax<G::NT, G::N::kLift> soft[MAPS];
   auto pass = [&](auto mode) {
      constexpr bool CAREFUL = decltype(mode)::value == kCareful, FULL = decltype(mode)::value == kFull;
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++) soft[mp].clear();
      for_tiles<G, BR>(
         st, u.tiles, 1, [&](int t, int buf) __attribute__((always_inline)) { st.template load_tile<FULL>(t, buf, 0, 0); },
         [&](int t, int buf) __attribute__((always_inline)) {
            const uint32_t word = st.row_mask(t, i);
            if (!__any(word != 0)) return;
            const bool all = __all(word == 0xffffffffu);   // most tiles of a window: nothing to mask
            const unsigned mine = (word >> (8 * g)) & 255;
            const typename G::V::Lane l = G::V::lane(g, i);
            const unsigned char *ks = lds + buf * G::kPair, *vs = ks + G::V::kBytes;
            float w[MAPS][2][4];
#pragma unroll
            for (int mp = 0; mp < MAPS; mp++)
            {
               f4 s[2];
               tile_scores<T, G::W, G::CQ>(s, ks, mp * G::MC, qr[mp], l);
               if (!all)
               {
                  keep_branch();
#pragma unroll
                  for (int j = 0; j < 8; j++) s[j / 4][j % 4] = masked(s[j / 4][j % 4], mine, j, -INFINITY);
               }
               soft[mp].weights(w[mp], s, c2);
            }
            if constexpr (CAREFUL)
            {
#pragma unroll
               for (int mp = 0; mp < MAPS; mp++) add_weighted<T, G::W, true, T != kF32>(soft[mp].acc, w[mp], mine, vs, 0, g, i, l);
               return;
            }
            typename G::N::TFrag wf[MAPS], wr[MAPS];   // the weights, and (16-bit) what rounding took from them
#pragma unroll
            for (int mp = 0; mp < MAPS; mp++)
            {
               wf[mp] = pack_scores<T>(w[mp]);
               if constexpr (T != kF32) wr[mp] = pack_rest<T>(w[mp], wf[mp]);
            }
#pragma unroll
            for (int x = 0; x < G::NT; x++)
            {
               const typename G::N::TFrag vt = G::V::transposed(vs, x, l);
#pragma unroll
               for (int mp = 0; mp < MAPS; mp++)
               {
                  soft[mp].acc[x] = G::N::mma_t(vt, wf[mp], soft[mp].acc[x]);
                  if constexpr (T != kF32) soft[mp].acc[x] = G::N::mma_t(vt, wr[mp], soft[mp].acc[x]);
               }
            }
         });
      bool odd = odd_sums(soft[0].acc);
      if constexpr (MAPS == 2) odd |= odd_sums(soft[1].acc);
      return odd;
   };
   if (any_odd<BR>(p.gat.full ? pass(Mode<kFull>()) : pass(Mode<kAny>()))) (void)pass(Mode<kCareful>());

#pragma unroll
   for (int mp = 0; mp < MAPS; mp++) soft[mp].sum = group_sum(soft[mp].sum);
   if (u.part >= 0)
   {
      // [part][head][map][BR rows][W + 2]: sums, then what they are relative to and the sum of weights
      float *to = p.part + (((int64_t)u.part * p.heads + head) * MAPS * BR + 16 * wave + i) * (G::W + 2);
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
      {
         float *r = to + (int64_t)mp * BR * (G::W + 2);
#pragma unroll
         for (int x = 0; x < G::NT; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) r[16 * x + 4 * g + e] = soft[mp].acc[x][e];
         if (g == 0)
         {
            r[G::W] = soft[mp].base;
            r[G::W + 1] = soft[mp].sum;
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
      inv[mp] = soft[mp].sum == 0.0f ? 0.0f : 1.0f / soft[mp].sum;   // a row without edges is zero
      if (p.lse && g == 0) p.lse[(row * p.heads + head) * MAPS + mp] = soft[mp].sum == 0.0f ? -INFINITY : (soft[mp].base - G::N::kLift + log2f(soft[mp].sum)) * kLn2;
   }
   E *out = (E *)p.out + row * p.ldo + head * p.hdo;
   E *out2 = MAPS == 2 && p.out2 ? (E *)p.out2 + row * p.ldo + head * p.hdo : nullptr;
#pragma unroll
   for (int x = 0; x < G::NT; x++)
   {
      f4 r = soft[0].acc[x] * inv[0];
      if constexpr (MAPS == 2)
      {
         const f4 r2 = soft[1].acc[x] * inv[1];
         if (out2) store4<T>(out2, 16 * x + 4 * g, p.dv, r2, p.vec);
         r -= lam * r2;
      }
      store4<T>(out, 16 * x + 4 * g, p.dv, r, p.vec);
   }
}

// Blocks of several units: a wave for every 64 features of a (block, head, row); the units' sums in order.
#define JOIN_WHERE(HEADS, PIECES)                                                        \
   const int br = p.plan.block_rows, lane = threadIdx.x & 63;                             \
   const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);                       \
   const int piece = (int)(id % (PIECES)), r = (int)(id / (PIECES) % br);                 \
   const int head = (int)(id / (PIECES) / br % (HEADS));                                  \
   if (id / (PIECES) / br / (HEADS) >= p.plan.n_joins) return;                            \
   const Join j = p.plan.joins[id / (PIECES) / br / (HEADS)];

template <int T, int DC, int MAPS> __global__ __launch_bounds__(256) void attn_forward_join(Params p)
{
   constexpr int W = DC * MAPS;
   typedef typename Num<T>::E E;
   JOIN_WHERE(p.heads, (W + 63) / 64)
   const int64_t row = (int64_t)j.block * br + r;
   if (row >= p.m) return;
   const int f = 64 * piece + lane;
   const bool live = f < W;
   float o[MAPS];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
   {
      const int64_t step = (int64_t)p.heads * MAPS * br * (W + 2);
      const float *from = p.part + (((int64_t)j.part0 * p.heads + head) * MAPS + mp) * br * (W + 2) + (int64_t)r * (W + 2);
      float top = -INFINITY;
#pragma unroll 8
      for (int u = 0; u < j.parts; u++) top = fmaxf(top, from[u * step + W]);
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0, x = 0;
#pragma unroll 8
      for (int u = 0; u < j.parts; u++)
      {
         const float *s = from + u * step;
         const float keep = exp2_fast(s[W] - base);
         sum += s[W + 1] * keep;
         if (live) x += s[f] * keep;
      }
      o[mp] = sum == 0.0f ? 0.0f : x / sum;
      if (p.lse && lane == 0 && piece == 0) p.lse[(row * p.heads + head) * MAPS + mp] = sum == 0.0f ? -INFINITY : (top - Num<T>::kLift + log2f(sum)) * kLn2;
   }
   if (f >= p.dv) return;
   const int64_t at = row * p.ldo + head * p.hdo + f;
   if constexpr (MAPS == 2)
   {
      if (p.out2) ((E *)p.out2)[at] = (E)Num<T>::from(o[1]);
      o[0] -= p.lambda[head] * o[1];
   }
   ((E *)p.out)[at] = (E)Num<T>::from(o[0]);
}

// ---- backward ---------------------------------------------------------------------------------------------------------------------
// dq: resident q and do of 16 rows per wave, gathered k and v; both maps share the gathered v and dP.
//
// delta_p = <do, O_p>: with O_2 at hand, <do, O_1> = <do, o> + lambda <do, O_2>; the rows are resident, so the unit forms it.
// It comes from o as it was rounded to 16 bits, which a row of few edges feels: with mean = sum_j P dP, formed here in
// fp32, dq = sum_j P (dP - delta) k + (delta - mean) sum_j P k.  The second sum is small where it counts, so its own rounding
// does not matter; the exact mean replaces delta for dk.  fp32 needs none of it: there delta is off by what o's own
// rounding is.
//
// The 16-bit weights and scores' gradients enter dq, dk and dv as a rounded value and its rounded rest, as the forward pass's
// do: rounded once they left bf16 gradients 0.0024 off in two norms, where their own rounding is 0.0017.  A window of 256
// and 16 first columns, 16384 rows, 8 heads, two maps of 64 x 128: 316 us a training pass instead of 286; in fp16, with
// Range, 351 instead of 293.  The weights' sum takes another 1 %.
template <int T, int DC, int MAPS, int BR> __global__ __launch_bounds__(BR * 4, (DC * MAPS >= 256 || T == kF32 ? 1 : 2)) void attn_dq(Params p)
{
   typedef Geo<T, DC, MAPS, BR> G;
   typedef typename G::E E;
   constexpr bool kMend = T != kF32;
   ATTN_LDS(0)
   const int64_t item = xcd_item(blockIdx.x, (int64_t)p.plan.n_units * p.heads);
   if (item >= (int64_t)p.plan.n_units * p.heads) return;
   const int head = (int)(item / p.plan.n_units);
   const Unit u = p.plan.units[item % p.plan.n_units];
   const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, i = lane & 15;
   const int kvh = head / p.group;
   const int64_t row = (int64_t)u.block * BR + 16 * wave + i;
   const bool live = row < p.m;
   const int64_t srow = live ? row : 0;
   Stream<G, T, DC, BR> st;
   st.set(lds, lds_ids, lds_bits, p, u, kvh);

   u4 qr[MAPS][G::CQ], gr[G::CV];
   float lse2[MAPS], delta[MAPS], sign[MAPS], mean[MAPS], total[MAPS];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
   {
      load_resident<T, G::CQ>(qr[mp], (const E *)p.q + srow * p.ldq + head * p.hdq + mp * p.d, live, p.d, g, p.vec);
      lse2[mp] = row_offset(p.lse_in[(srow * p.heads + head) * MAPS + mp]);
      sign[mp] = mp == 0 ? 1.0f : -p.lambda[head];
   }
   load_resident<T, G::CV>(gr, (const E *)p.dout + srow * p.ldo + head * p.hdo, live, p.dv, g, p.vec);
   {
      u4 orow[G::CV];
      load_resident<T, G::CV>(orow, (const E *)p.o + srow * p.ldo + head * p.hdo, live, p.dv, g, p.vec);
      delta[0] = group_sum(chunk_dot<T>(gr, orow));
      if constexpr (MAPS == 2)
      {
         load_resident<T, G::CV>(orow, (const E *)p.o2 + srow * p.ldo + head * p.hdo, live, p.dv, g, p.vec);
         delta[1] = group_sum(chunk_dot<T>(gr, orow));
         delta[0] -= sign[1] * delta[1];
      }
   }

   const float c2 = p.scale * kLog2e;
   f4 acc[MAPS][G::NTQ], pk[kMend ? MAPS : 1][kMend ? G::NTQ : 1];
   Range<T> range[MAPS];
   auto pass = [&](auto mode) {
      constexpr bool CAREFUL = decltype(mode)::value == kCareful, FULL = decltype(mode)::value == kFull;
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
      {
         mean[mp] = total[mp] = 0;
         range[mp] = Range<T>();
#pragma unroll
         for (int t = 0; t < G::NTQ; t++)
         {
            acc[mp][t] = f4{0, 0, 0, 0};
            if constexpr (kMend) pk[mp][t] = f4{0, 0, 0, 0};
         }
      }
      for_tiles<G, BR>(
         st, u.tiles, 1, [&](int t, int buf) __attribute__((always_inline)) { st.template load_tile<FULL>(t, buf, 0, 0); },
         [&](int t, int buf) __attribute__((always_inline)) {
            const uint32_t word = st.row_mask(t, i);
            if (!__any(word != 0)) return;
            const bool all = __all(word == 0xffffffffu);   // most tiles of a window: nothing to mask
            const unsigned mine = (word >> (8 * g)) & 255;
            const typename G::V::Lane l = G::V::lane(g, i);
            const unsigned char *ks = lds + buf * G::kPair, *vs = ks + G::V::kBytes;
            f4 dp[2];
            tile_scores<T, G::W, G::CV>(dp, vs, 0, gr, l);
            if (!all)   // (zero times what is masked has to be zero)
            {
               keep_branch();
#pragma unroll
               for (int j = 0; j < 8; j++) dp[j / 4][j % 4] = masked(dp[j / 4][j % 4], mine, j, 0.0f);
            }
#pragma unroll
            for (int mp = 0; mp < MAPS; mp++)
            {
               f4 s[2];
               tile_scores<T, G::W, G::CQ>(s, ks, mp * G::MC, qr[mp], l);
               float w[2][4], pr[2][4];
#pragma unroll
               for (int j = 0; j < 8; j++) pr[j / 4][j % 4] = exp2_fast(fmaf(s[j / 4][j % 4], c2, -lse2[mp]));
               if (!all)
               {
                  keep_branch();
#pragma unroll
                  for (int j = 0; j < 8; j++) pr[j / 4][j % 4] = masked(pr[j / 4][j % 4], mine, j, 0.0f);
               }
#pragma unroll
               for (int j = 0; j < 8; j++)
               {
                  w[j / 4][j % 4] = pr[j / 4][j % 4] * (dp[j / 4][j % 4] - delta[mp]);   // sign: at the end
                  mean[mp] = fmaf(pr[j / 4][j % 4], dp[j / 4][j % 4], mean[mp]);
                  total[mp] += pr[j / 4][j % 4];
                  if constexpr (G::N::kPScale != 1.0f) pr[j / 4][j % 4] *= G::N::kPScale;
               }
               range[mp].fit(w, acc[mp]);
               if constexpr (CAREFUL)
               {
                  add_weighted<T, G::W, true, kMend>(acc[mp], w, mine, ks, mp * DC, g, i, l);
                  if constexpr (kMend) add_weighted<T, G::W, true>(pk[mp], pr, mine, ks, mp * DC, g, i, l);
                  continue;
               }
               const typename G::N::TFrag wf = pack_scores<T>(w);
               typename G::N::TFrag wr, pf;
               if constexpr (kMend)
               {
                  wr = pack_rest<T>(w, wf);
                  pf = pack_scores<T>(pr);
               }
#pragma unroll
               for (int x = 0; x < G::NTQ; x++)
               {
                  const typename G::N::TFrag kt = G::V::transposed(ks, mp * G::NTQ + x, l);
                  acc[mp][x] = G::N::mma_t(kt, wf, acc[mp][x]);
                  if constexpr (kMend)
                  {
                     acc[mp][x] = G::N::mma_t(kt, wr, acc[mp][x]);
                     pk[mp][x] = G::N::mma_t(kt, pf, pk[mp][x]);
                  }
               }
            }
         });
      bool odd = false;
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
      {
         odd |= odd_sums(acc[mp]);
         if constexpr (kMend) odd |= odd_sums(pk[mp]);
      }
      return odd;
   };
   if (any_odd<BR>(p.gat.full ? pass(Mode<kFull>()) : pass(Mode<kAny>()))) (void)pass(Mode<kCareful>());

#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
   {
      mean[mp] = group_sum(mean[mp]);
      total[mp] = group_sum(total[mp]);
      if (u.part < 0) mean[mp] *= row_share(total[mp]);
      range[mp].undo(acc[mp]);
      if constexpr (G::N::kPScale != 1.0f)
      {
#pragma unroll
         for (int t = 0; t < G::NTQ; t++) pk[mp][t] *= 1.0f / G::N::kPScale;
      }
   }
   if constexpr (MAPS == 2)
   {
      // (a row behind the last one names nothing: its mean is zero; the units of a split block add up, without the share)
      float x = mean[1];
#pragma unroll
      for (int k = 8; k; k >>= 1) x += __shfl_xor(x, k);
      if (lane == 0) p.dlam_units[((item % p.plan.n_units) * G::WAVES + wave) * p.heads + head] = x;
   }
   if (u.part >= 0)
   {
      // [part][head][BR rows][W + W + 6]: the two sums, the means, the deltas, the weights
      float *r = p.part + (((int64_t)u.part * p.heads + head) * BR + 16 * wave + i) * (2 * G::W + 6);
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
      {
#pragma unroll
         for (int x = 0; x < G::NTQ; x++)
#pragma unroll
            for (int e = 0; e < 4; e++)
            {
               r[mp * DC + 16 * x + 4 * g + e] = acc[mp][x][e];
               if constexpr (kMend) r[G::W + mp * DC + 16 * x + 4 * g + e] = pk[mp][x][e];
            }
         if (g == 0)
         {
            r[2 * G::W + mp] = mean[mp];
            r[2 * G::W + 2 + mp] = delta[mp];
            r[2 * G::W + 4 + mp] = total[mp];
         }
      }
      return;
   }
   if (!live) return;
   if (g == 0)
   {
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
      {
         p.stats[(row * p.heads + head) * (2 * MAPS) + mp] = row_offset(lse2[mp], total[mp]);
         p.stats[(row * p.heads + head) * (2 * MAPS) + MAPS + mp] = kMend ? mean[mp] : delta[mp];
      }
   }
   E *out = (E *)p.dq + row * p.ldq + head * p.hdq;
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
      for (int x = 0; x < G::NTQ; x++)
      {
         f4 r = acc[mp][x];
         if constexpr (kMend) r += (delta[mp] - mean[mp]) * pk[mp][x];
         store4<T>(out + mp * p.d, 16 * x + 4 * g, p.d, r * (sign[mp] * p.scale * row_share(total[mp])), p.vec);
      }
}

template <int T, int DC, int MAPS> __global__ __launch_bounds__(256) void attn_dq_join(Params p)
{
   constexpr int W = DC * MAPS;
   constexpr bool kMend = T != kF32;
   typedef typename Num<T>::E E;
   JOIN_WHERE(p.heads, (W + 63) / 64)
   const int64_t row = (int64_t)j.block * br + r;
   if (row >= p.m) return;
   const int64_t step = (int64_t)p.heads * br * (2 * W + 6);
   const float *from = p.part + (((int64_t)j.part0 * p.heads + head) * br + r) * (2 * W + 6);
   float mend[MAPS], share[MAPS];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
   {
      float mean = 0, total = 0;
#pragma unroll 8
      for (int u = 0; u < j.parts; u++)
      {
         mean += from[u * step + 2 * W + mp];
         total += from[u * step + 2 * W + 4 + mp];
      }
      share[mp] = row_share(total);
      mean *= share[mp];
      const float delta = from[2 * W + 2 + mp];
      mend[mp] = delta - mean;
      if (lane == 0 && piece == 0)
      {
         p.stats[(row * p.heads + head) * (2 * MAPS) + mp] = row_offset(row_offset(p.lse_in[(row * p.heads + head) * MAPS + mp]), total);
         p.stats[(row * p.heads + head) * (2 * MAPS) + MAPS + mp] = kMend ? mean : delta;
      }
   }
   const int f = 64 * piece + lane;
   if (f >= W) return;
   float s = 0, s2 = 0;
#pragma unroll 8
   for (int u = 0; u < j.parts; u++)
   {
      s += from[u * step + f];
      if (kMend) s2 += from[u * step + W + f];
   }
   const int mp = f / DC, e = f - mp * DC;
   if (kMend) s += (mp == 0 ? mend[0] : mend[MAPS - 1]) * s2;
   if (e < p.d) ((E *)p.dq)[row * p.ldq + head * p.hdq + mp * p.d + e] = (E)Num<T>::from(s * ((mp == 0 ? share[0] : -p.lambda[head] * share[MAPS - 1]) * p.scale));
}

// dlambda_h = - sum of dlam_units, in 64 bits: every thread's entries and then the threads in order.  The last `heads`
// workgroups of the dk, dv launch do it: its input is there, and a launch of its own would take longer than the sum.
template <int THREADS> __device__ inline void dlambda_of(const Params &p, int head, double *s)
{
   double x = 0;
#pragma unroll 4
   for (int64_t u = threadIdx.x; u < p.dlam_count; u += THREADS) x += (double)p.dlam_units[u * p.heads + head];
   s[threadIdx.x] = x;
   __syncthreads();
   for (int k = THREADS / 2; k; k >>= 1)
   {
      if ((int)threadIdx.x < k) s[threadIdx.x] += s[threadIdx.x + k];
      __syncthreads();
   }
   if (threadIdx.x == 0) p.dlambda[head] = (float)-s[0];
}

// dk, dv: resident k and v of 16 key rows per wave, gathered q and do of the query rows that name them, for every query
// head of the key head in turn.  p.plan is the plan of the transposed pattern.
template <int T, int DC, int MAPS, int BR> __global__ __launch_bounds__(BR * 4, (DC * MAPS >= 256 || T == kF32 ? 1 : 2)) void attn_dkv(Params p)
{
   typedef Geo<T, DC, MAPS, BR> G;
   typedef typename G::E E;
   ATTN_LDS(G::kStat)
   const int64_t work_groups = ((int64_t)p.plan.n_units * p.kv_heads + 7) / 8 * 8;
   if (MAPS == 2 && blockIdx.x >= work_groups)
   {
      dlambda_of<G::THREADS>(p, (int)(blockIdx.x - work_groups), (double *)lds);
      return;
   }
   const int64_t item = xcd_item(blockIdx.x, (int64_t)p.plan.n_units * p.kv_heads);
   if (item >= (int64_t)p.plan.n_units * p.kv_heads) return;
   const int kvh = (int)(item / p.plan.n_units);
   const Unit u = p.plan.units[item % p.plan.n_units];
   const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, i = lane & 15;
   const int64_t row = (int64_t)u.block * BR + 16 * wave + i;
   const bool live = row < p.n;
   const int64_t srow = live ? row : 0;
   Stream<G, T, DC, BR> st;
   st.set(lds, lds_ids, lds_bits, p, u, 0);

   u4 kr[MAPS][G::CQ], vr[G::CV];
#pragma unroll
   for (int mp = 0; mp < MAPS; mp++)
      load_resident<T, G::CQ>(kr[mp], (const E *)p.k + srow * p.ldk + kvh * p.hdk + mp * p.d, live, p.d, g, p.vec);
   load_resident<T, G::CV>(vr, (const E *)p.v + srow * p.ldv + kvh * p.hdv, live, p.dv, g, p.vec);
   const float c2 = p.scale * kLog2e;
   f4 dk[MAPS][G::NTQ], dv[G::NT];
   Range<T> range_k[MAPS], range_v;

   auto load = [&](int s, int buf, auto full) __attribute__((always_inline)) {
      const int t = s / p.group, head = kvh * p.group + s % p.group;
      st.template load_tile<decltype(full)::value>(t, buf, head * p.gat.ha * (int64_t)sizeof(E), head * p.gat.hb * (int64_t)sizeof(E));
      // the statistics of the tile's rows: [32 rows][2 maps], 8 or 16 bytes of a row each
      if (tid < (MAPS == 2 ? 32 : 64))
      {
         const int32_t c = st.tile_ids(t)[MAPS == 2 ? tid : tid >> 1];
         const float *from = p.stats + ((int64_t)c * p.heads + head) * (2 * MAPS);
         if constexpr (MAPS == 2) load_lds16(lds_address(lds_extra + buf * G::kStat), from);
         else load_lds4(lds_address(lds_extra + buf * G::kStat), from + (tid & 1));
      }
   };
   auto use = [&](int s, int buf, auto careful) __attribute__((always_inline)) {
      constexpr bool CAREFUL = decltype(careful)::value;
      const uint32_t word = st.row_mask(s / p.group, i);
      if (!__any(word != 0)) return;
      const bool all = __all(word == 0xffffffffu);
      const unsigned mine = (word >> (8 * g)) & 255;
      const typename G::V::Lane l = G::V::lane(g, i);
      const unsigned char *qs = lds + buf * G::kPair, *gs = qs + G::V::kBytes;
      const float *stat = (const float *)(lds_extra + buf * G::kStat);
      const float lam = MAPS == 2 ? p.lambda[kvh * p.group + s % p.group] : 0.0f;
      f4 dp[2];
      tile_scores<T, G::W, G::CV>(dp, gs, 0, vr, l);
      float rs[8][2 * MAPS];   // statistics of this lane's gathered rows
#pragma unroll
      for (int j = 0; j < 8; j++)
#pragma unroll
         for (int k = 0; k < 2 * MAPS; k++) rs[j][k] = stat[(16 * (j / 4) + 4 * g + j % 4) * (2 * MAPS) + k];
      float wv[2][4];
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
      {
         f4 sc[2];
         tile_scores<T, G::W, G::CQ>(sc, qs, mp * G::MC, kr[mp], l);
         float w[2][4];
#pragma unroll
         for (int j = 0; j < 8; j++) w[j / 4][j % 4] = exp2_fast(fmaf(sc[j / 4][j % 4], c2, -rs[j][mp]));
         if (!all)
         {
            keep_branch();
#pragma unroll
            for (int j = 0; j < 8; j++) w[j / 4][j % 4] = masked(w[j / 4][j % 4], mine, j, 0.0f);
         }
#pragma unroll
         for (int j = 0; j < 8; j++)
         {
            float pr = w[j / 4][j % 4];
            if (mp == 1) pr *= -lam;
            w[j / 4][j % 4] = pr * (dp[j / 4][j % 4] - rs[j][MAPS + mp]);
            wv[j / 4][j % 4] = mp == 0 ? pr : wv[j / 4][j % 4] + pr;
         }
         if (!all)   // (zero times the products and statistics of a row that is masked has to be zero)
         {
            keep_branch();
#pragma unroll
            for (int j = 0; j < 8; j++) w[j / 4][j % 4] = masked(w[j / 4][j % 4], mine, j, 0.0f);
         }
         range_k[mp].fit(w, dk[mp]);
         add_weighted<T, G::W, CAREFUL, T != kF32>(dk[mp], w, mine, qs, mp * DC, g, i, l);
      }
      range_v.fit(wv, dv);
      add_weighted<T, G::W, CAREFUL, T != kF32>(dv, wv, mine, gs, 0, g, i, l);
   };
   auto pass = [&](auto mode) {
      constexpr bool CAREFUL = decltype(mode)::value == kCareful, FULL = decltype(mode)::value == kFull;
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
         for (int t = 0; t < G::NTQ; t++) dk[mp][t] = f4{0, 0, 0, 0};
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++) range_k[mp] = Range<T>();
      range_v = Range<T>();
#pragma unroll
      for (int t = 0; t < G::NT; t++) dv[t] = f4{0, 0, 0, 0};
      // (steps of one tile, the heads of the group, follow each other: tiles * group < 2^31 is checked by the host)
      for_tiles<G, BR>(st, u.tiles * p.group, p.group,
         [&](int s, int buf) __attribute__((always_inline)) { load(s, buf, Flag<FULL>()); },
         [&](int s, int buf) __attribute__((always_inline)) { use(s, buf, Flag<CAREFUL>()); });
      bool odd = odd_sums(dv);
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++) odd |= odd_sums(dk[mp]);
      return odd;
   };
   if (any_odd<BR>(p.gat.full ? pass(Mode<kFull>()) : pass(Mode<kAny>()))) (void)pass(Mode<kCareful>());

#pragma unroll
   for (int mp = 0; mp < MAPS; mp++) range_k[mp].undo(dk[mp]);
   range_v.undo(dv);
   if (u.part >= 0)
   {
      // [part][kv head][BR rows][2 W]
      float *r = p.part + (((int64_t)u.part * p.kv_heads + kvh) * BR + 16 * wave + i) * (2 * G::W);
#pragma unroll
      for (int mp = 0; mp < MAPS; mp++)
#pragma unroll
         for (int x = 0; x < G::NTQ; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) r[mp * DC + 16 * x + 4 * g + e] = dk[mp][x][e];
#pragma unroll
      for (int x = 0; x < G::NT; x++)
#pragma unroll
         for (int e = 0; e < 4; e++) r[G::W + 16 * x + 4 * g + e] = dv[x][e];
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
   for (int x = 0; x < G::NT; x++) store4<T>(outv, 16 * x + 4 * g, p.dv, dv[x], p.vec);
}

template <int T, int DC, int MAPS> __global__ __launch_bounds__(256) void attn_dkv_join(Params p)
{
   constexpr int W = DC * MAPS;
   typedef typename Num<T>::E E;
   JOIN_WHERE(p.kv_heads, (2 * W + 63) / 64)
   const int64_t row = (int64_t)j.block * br + r;
   if (row >= p.n) return;
   const int64_t step = (int64_t)p.kv_heads * br * (2 * W);
   const float *from = p.part + (((int64_t)j.part0 * p.kv_heads + head) * br + r) * (2 * W);
   const int f = 64 * piece + lane;
   if (f >= 2 * W) return;
   float s = 0;
#pragma unroll 8
   for (int u = 0; u < j.parts; u++) s += from[u * step + f];
   if (f < W)
   {
      const int mp = f / DC, e = f - mp * DC;
      if (e < p.d) ((E *)p.dk)[row * p.ldk + head * p.hdk + mp * p.d + e] = (E)Num<T>::from(s * p.scale);
   }
   else if (f - W < p.dv) ((E *)p.dvv)[row * p.ldv + head * p.hdv + f - W] = (E)Num<T>::from(s);
}

}  // namespace fmm_attn
