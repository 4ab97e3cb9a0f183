// Attention over a CSR pattern: what the kernels of this family share.
//
// For row i, head h and map p:  s_j = scale * <q_p[i], k_p[c_j]>,  P_p = softmax of s over the row's edges,
// o[i] = sum_j (P_1 - lambda_h P_2)_j v[c_j]  (one map: P_1 alone).  Backward, with dP_j = <do[i], v[c_j]> and
// delta_p = <do[i], O_p[i]>:  dS_p = sign_p P_p (dP - delta_p),  dq_p = scale sum_j dS_p k_p[c_j],
// dk_p[c] = scale sum_i dS_p q_p[i],  dv[c] = sum_i (P_1 - lambda P_2) do[i],  dlambda_h = - sum_i sum_j P_2 dP.
//
// All of it is small dense products between rows that stay in registers ("resident": 16 per wave) and tiles of 32
// gathered rows in LDS, on the matrix cores.  Every product is formed transposed, gathered x resident: a lane then
// holds, for ONE resident row (lane % 16), the scores of gathered rows 4g..4g+3 and 16+4g..16+4g+3 (g = lane / 16),
// which is - up to an order of the contraction index that both operands share - the register layout in which the
// scores enter the second product.  Scores, weights and their gradients therefore never leave the registers, and the
// row statistics are one value per lane.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fmm_attn {

enum : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kTile = 32;         // gathered rows of a tile

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 16-bit and 32-bit element types.  A "chunk" is KC features of a row, of which a lane holds EPL (16 bytes).
template <int T> struct Num;

template <> struct Num<kBF16> {
   typedef uint16_t E;
   static constexpr int KC = 32, EPL = 8;
   typedef s8 TFrag;
   static constexpr float kPScale = 1.0f;
   static constexpr int kLift = 0;
   static __device__ inline f4 mma(u4 a, u4 b, f4 c)
   {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
   }
   static __device__ inline f4 mma_t(s8 a, s8 b, f4 c)
   {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
   }
   static __device__ inline E from(float x) { return __builtin_bit_cast(E, (__bf16)x); }   // to nearest even
   static __device__ inline float to(E x) { return __builtin_bit_cast(float, (uint32_t)x << 16); }
   static __device__ inline bool odd_word(uint32_t w)   // an infinity or a NaN in either half
   {
      return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
   }
};

template <> struct Num<kF16> {
   typedef uint16_t E;
   static constexpr int KC = 32, EPL = 8;
   typedef s8 TFrag;
   // softmax weights of long rows are small: 2^14 keeps them clear of fp16's subnormals (they are at most 1)
   static constexpr float kPScale = 16384.0f;
   static constexpr int kLift = 7;
   static __device__ inline f4 mma(u4 a, u4 b, f4 c)
   {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
   }
   static __device__ inline f4 mma_t(s8 a, s8 b, f4 c)
   {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
   }
   static __device__ inline E from(float x) { return __builtin_bit_cast(E, (_Float16)x); }
   static __device__ inline float to(E x) { return (float)__builtin_bit_cast(_Float16, x); }
   static __device__ inline bool odd_word(uint32_t w)
   {
      return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
   }
};

template <> struct Num<kF32> {
   typedef float E;
   static constexpr int KC = 16, EPL = 4;
   typedef f8 TFrag;
   static constexpr float kPScale = 1.0f;
   static constexpr int kLift = 0;
   static __device__ inline f4 mma(u4 a, u4 b, f4 c)
   {
      const f4 x = __builtin_bit_cast(f4, a), y = __builtin_bit_cast(f4, b);
#pragma unroll
      for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
      return c;
   }
   static __device__ inline f4 mma_t(f8 a, f8 b, f4 c)
   {
#pragma unroll
      for (int j = 0; j < 8; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
      return c;
   }
   static __device__ inline E from(float x) { return x; }
   static __device__ inline float to(E x) { return x; }
   static __device__ inline bool odd_word(uint32_t w) { return (w & 0x7F800000u) == 0x7F800000u; }
};

// EPL elements at p (aligned: on 16 bytes; the hardware takes any other address as well)
template <int T> __device__ inline u4 load_chunk(const typename Num<T>::E *p, bool aligned)
{
   typedef u4 u4_anywhere __attribute__((aligned(2)));
   return aligned ? *reinterpret_cast<const u4 *>(p) : *reinterpret_cast<const u4_anywhere *>(p);
}

// How chunks of rows are read: the row is 16-byte aligned and its width a multiple of EPL; at any place and width from EPL
// on; a row shorter than a chunk.  The same for all rows of a call, so that callers choose once, outside their loops.
enum : int { kAligned, kShifted, kElements };
template <int M> struct Mode {
   static constexpr int value = M;
};
template <int T> __device__ inline int part_mode(bool vec, int width) { return vec ? kAligned : width >= Num<T>::EPL ? kShifted : kElements; }

// Elements f .. f + EPL - 1 of a row of `width`; behind its end, and without a live row, zeros.  `row` can be read, live or
// not, so that the load has no condition.  kShifted reads the row's last whole chunk where the row ends and shifts it down:
// a chunk read element by element cost as many trips to memory as it had elements (forward and backward of a graph with 176 rows,
// 12 heads of 93 and 115 bf16 features: 123 us, shifted 77).
template <int T, int MODE> __device__ inline u4 load_part(const typename Num<T>::E *row, int f, int width, bool live)
{
   constexpr int EPL = Num<T>::EPL;
   u4 r = {0, 0, 0, 0};
   if constexpr (MODE == kAligned)
   {
      const bool here = live && f < width;
      r = load_chunk<T>(row + (f < width ? f : 0), true);
#pragma unroll
      for (int k = 0; k < 4; k++) r[k] = here ? r[k] : 0;
   }
   else if constexpr (MODE == kElements)
   {
#pragma unroll
      for (int k = 0; k < EPL; k++)   // (the other tensor may be the one with the short rows)
      {
         if (!live || f + k >= width) continue;
         if constexpr (T == kF32) r[k] = __float_as_uint(row[f + k]);
         else r[k / 2] |= (uint32_t)row[f + k] << (16 * (k & 1));
      }
   }
   else
   {
      const int at = f < width - EPL ? f : width - EPL, less = live && f - at < EPL ? f - at : EPL;
      r = load_chunk<T>(row + at, false);
      const int bytes = less * (int)sizeof(typename Num<T>::E);
      if constexpr (T != kF32)
      {
         const bool half = bytes & 2;
#pragma unroll
         for (int k = 0; k < 4; k++) r[k] = half ? __builtin_amdgcn_alignbit(k < 3 ? r[k < 3 ? k + 1 : 3] : 0, r[k], 16) : r[k];
      }
      const bool one = bytes & 4, two = bytes & 8, all = bytes & 16;
#pragma unroll
      for (int k = 0; k < 4; k++) r[k] = !one ? r[k] : k < 3 ? r[k < 3 ? k + 1 : 3] : 0;
#pragma unroll
      for (int k = 0; k < 4; k++) r[k] = all ? 0 : !two ? r[k] : k < 2 ? r[k < 2 ? k + 2 : 3] : 0;
   }
   return r;
}

// scores of 32 gathered rows for one resident row, in the layout of the second product
template <int T> __device__ inline typename Num<T>::TFrag pack_scores(const float (&p)[2][4])
{
   typename Num<T>::TFrag r;
#pragma unroll
   for (int j = 0; j < 8; j++)
   {
      if constexpr (T == kF32) r[j] = p[j / 4][j % 4];
      else r[j] = (short)Num<T>::from(p[j / 4][j % 4]);
   }
   return r;
}

// what rounding took from them, rounded in turn
template <int T> __device__ inline typename Num<T>::TFrag pack_rest(const float (&p)[2][4], typename Num<T>::TFrag b)
{
   float r[2][4];
#pragma unroll
   for (int j = 0; j < 8; j++) r[j / 4][j % 4] = T == kF32 ? 0.0f : p[j / 4][j % 4] - Num<T>::to((typename Num<T>::E)b[j]);
   return pack_scores<T>(r);
}

// A tile in LDS: 32 rows of W elements.  A row's 16-byte chunks are stored in an order that depends on the row (chunk ^
// twist(row)): the 16 rows that a matrix operand reads at one chunk, and the 16 that a transposing read touches, then
// lie in different banks, without padding - loads that go straight to LDS leave no room for any.
template <int T, int W> struct TileView {
   typedef typename Num<T>::E E;
   static constexpr int EPL = Num<T>::EPL;
   static constexpr int RB = W * (int)sizeof(E);       // bytes of a row
   static constexpr int CR = RB / 16;                  // chunks of a row
   static constexpr int kBytes = kTile * RB;
   static constexpr int kTwistRows = CR >= 16 ? 1 : 16 / CR;
   static constexpr int kTwistMask = CR >= 16 ? 15 : CR - 1;
   static __device__ inline int twist(int row) { return (row / kTwistRows) & kTwistMask; }

   // Where this lane's reads of a tile start.  The chunk number enters by exclusive or, which leaves one address for every
   // chunk; the compiler would keep them all in registers over the loop, so the starts are hidden from it for each tile
   // and the addresses are formed again, one operation each.
   struct Lane {
      int direct;
      int transposed[T == kF32 ? 4 : 1];
   };
   static __device__ inline Lane lane(int g, int i)
   {
      Lane l;
      l.direct = i * RB + (g ^ twist(i)) * 16;
      if constexpr (T == kF32)
      {
#pragma unroll
         for (int r = 0; r < 4; r++) l.transposed[r] = (4 * g + r) * RB + (((i / 4) ^ twist(4 * g + r)) * 16) + (i % 4) * 4;
      }
      else l.transposed[0] = (4 * g + i / 4) * RB + ((((i % 4) / 2) ^ twist(4 * g + i / 4)) * 16) + (i % 2) * 8;
      asm volatile("" : "+v"(l.direct));
#pragma unroll
      for (int r = 0; r < (T == kF32 ? 4 : 1); r++) asm volatile("" : "+v"(l.transposed[r]));
      return l;
   }

   // chunk (a multiple of 4) + g of row i: the 16 bytes of a first operand; a is 0 or 1: rows 16a + i
   static __device__ inline u4 direct(const unsigned char *tile, int chunk, int a, const Lane &l)
   {
      return *reinterpret_cast<const u4 *>(tile + (l.direct ^ (chunk * 16)) + 16 * a * RB);
   }

   // features 16t .. 16t+15 of the 32 rows, transposed: lane i of group g gets feature 16t + i of rows 4g..4g+3 and
   // 16+4g..16+4g+3 (which have the same twist).  16-bit: two transposing LDS reads, in which lane i of a group of 16 names
   // the address of four elements of row i / 4 and receives element i of the four rows.  32-bit: eight plain reads.
   static __device__ inline typename Num<T>::TFrag transposed(const unsigned char *tile, int t, const Lane &l)
   {
      typename Num<T>::TFrag r;
      if constexpr (T == kF32)
      {
#pragma unroll
         for (int j = 0; j < 8; j++) r[j] = *reinterpret_cast<const float *>(tile + (l.transposed[j % 4] ^ (4 * t * 16)) + 16 * (j / 4) * RB);
      }
      else
      {
         typedef __attribute__((address_space(3))) s4 lds_s4;
         const unsigned char *p = tile + (l.transposed[0] ^ (2 * t * 16));
         const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)p);
         const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + 16 * RB));
         r = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
      }
      return r;
   }

   static __device__ inline E element(const unsigned char *tile, int row, int f)
   {
      return *reinterpret_cast<const E *>(tile + row * RB + (((f / EPL) ^ twist(row)) * 16) + (f % EPL) * (int)sizeof(E));
   }
};

// an infinity or a NaN
template <int T> __device__ inline bool odd_element(typename Num<T>::E x)
{
   if constexpr (T == kF32) return Num<T>::odd_word(__float_as_uint(x));
   else return Num<T>::odd_word(x);
}

template <int T> __device__ inline typename Num<T>::TFrag without_odd(typename Num<T>::TFrag v)
{
#pragma unroll
   for (int j = 0; j < 8; j++)
   {
      if constexpr (T == kF32) v[j] = odd_element<T>(v[j]) ? 0.0f : v[j];
      else v[j] = odd_element<T>((uint16_t)v[j]) ? (short)0 : v[j];
   }
   return v;
}

// No load moves over this: the rare path below would otherwise load ahead into registers that set the kernels' occupancy.
__device__ inline void keep_order() { asm volatile("" ::: "memory"); }

// What the tile's infinities and NaN add: a matrix instruction would multiply them by the zero weights of rows that do not
// name them, so it runs without them (without_odd) and every row adds those of the gathered rows that it does name.
// Rows that name none keep the bits they have without them.
// mine: bit 4a + r says that gathered row 16a + 4g + r is named by this lane's resident row.
template <int T, int W, int NT>
__device__ inline void add_odd(f4 (&acc)[NT], const float (&p)[2][4], unsigned mine, const unsigned char *tile, int f0, int g, int i)
{
   for (int key = 0; key < kTile; key++)
   {
      const int src = ((key & 15) >> 2) * 16 + i, a = key >> 4, r = key & 3;
      float x = 0;
#pragma unroll
      for (int j = 0; j < 8; j++)
         if (j == 4 * a + r) x = p[j / 4][j % 4];
      const float w = __shfl(x, src);
      const bool named = (__shfl((int)mine, src) >> (4 * a + r)) & 1;
      if (!named) continue;
#pragma unroll
      for (int t = 0; t < NT; t++)
      {
#pragma unroll
         for (int k = 0; k < 4; k++)
         {
            const typename Num<T>::E e = TileView<T, W>::element(tile, key, f0 + 16 * t + 4 * g + k);
            if (odd_element<T>(e)) acc[t][k] = fmaf(w, Num<T>::to(e), acc[t][k]);
         }
         keep_order();
      }
   }
}

// acc += (weights of the tile's 32 rows) x (their features f0 .. f0 + 16 NT - 1); CAREFUL: the tile may hold infinities or
// NaN; TWICE: 16-bit weights enter as a rounded value and its rounded rest.  One rounding of the weights errs by as much
// as the rounding of the output does; with the rest, outputs are as exact as their own rounding.  (Once is enough for the
// sum in dq that only multiplies what a rounded delta is off by.)
template <int T, int W, bool CAREFUL, bool TWICE = false, int NT>
__device__ inline void add_weighted(f4 (&acc)[NT], const float (&p)[2][4], unsigned mine, const unsigned char *tile, int f0, int g, int i, const typename TileView<T, W>::Lane &l)
{
   typedef TileView<T, W> V;
   const typename Num<T>::TFrag b = pack_scores<T>(p);
   typename Num<T>::TFrag low;
   if constexpr (TWICE) low = pack_rest<T>(p, b);
   if constexpr (CAREFUL)
   {
#pragma unroll
      for (int t = 0; t < NT; t++)
      {
         const typename Num<T>::TFrag v = without_odd<T>(V::transposed(tile, f0 / 16 + t, l));
         acc[t] = Num<T>::mma_t(v, b, acc[t]);
         if constexpr (TWICE) acc[t] = Num<T>::mma_t(v, low, acc[t]);
         keep_order();
      }
      add_odd<T, W, NT>(acc, p, mine, tile, f0, g, i);
   }
   else
   {
#pragma unroll
      for (int t = 0; t < NT; t++)
      {
         const typename Num<T>::TFrag v = V::transposed(tile, f0 / 16 + t, l);
         acc[t] = Num<T>::mma_t(v, b, acc[t]);
         if constexpr (TWICE) acc[t] = Num<T>::mma_t(v, low, acc[t]);
      }
   }
}

// Sums that are not finite may be the matrix instructions' zero times infinity: the work is then done again with CAREFUL.
// Finite sums cannot be wrong in that way.
template <int NT> __device__ inline bool odd_sums(const f4 (&acc)[NT])
{
   bool odd = false;
#pragma unroll
   for (int t = 0; t < NT; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) odd |= !(fabsf(acc[t][e]) < INFINITY);
   return odd;
}
template <bool X> struct Flag {
   static constexpr bool value = X;
};

// four consecutive features of an output row, f .. f+3 of `width`
template <int T> __device__ inline void store4(typename Num<T>::E *row, int f, int width, f4 v, bool vec)
{
   typedef typename Num<T>::E E;
   if (f >= width) return;
   if (vec && f + 4 <= width)
   {
      if constexpr (T == kF32) *reinterpret_cast<f4 *>(row + f) = v;
      else
      {
         s4 s;
#pragma unroll
         for (int k = 0; k < 4; k++) s[k] = (short)Num<T>::from(v[k]);
         *reinterpret_cast<s4 *>(row + f) = s;
      }
      return;
   }
#pragma unroll
   for (int k = 0; k < 4; k++)
      if (f + k < width) row[f + k] = (E)Num<T>::from(v[k]);
}

// over the four lane groups: the lanes of one resident row
typedef unsigned int u2 __attribute__((ext_vector_type(2)));
__device__ inline float group_max(float x)
{
   const u2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
   x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
   const u2 b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
   return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float group_sum(float x)
{
   const u2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
   x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
   const u2 b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
   return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// what stands behind this in a branch is not done without it (the compiler would rather select than branch)
__device__ inline void keep_branch() { asm volatile(""); }

// Sums of weights that have no bound of their own, P1 - lambda P2 or the scores' gradients P (dP - delta): in fp16 they enter the
// product times 2^up, which follows the largest one of the resident row so far down, 2^14 at most after each step: none of
// them overflows, and what fp16's smallest step takes is 2^-38 of the largest.  Other types have fp32's range.
template <int T> struct Range {
   int up = 100;
   template <int NT> __device__ inline void fit(float (&w)[2][4], f4 (&acc)[NT])
   {
      if constexpr (T == kF16)
      {
         float top = 0;
#pragma unroll
         for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(w[j / 4][j % 4]));
         top = group_max(top);
         const bool over = ldexpf(top, up) > 32768.0f && top < INFINITY;   // (an infinite weight stays one)
         if (__any(over))
         {
            const int to = over ? 14 - __builtin_amdgcn_frexp_expf(top) : up;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
               for (int e = 0; e < 4; e++) acc[t][e] = ldexpf(acc[t][e], to - up);
            up = to;
         }
#pragma unroll
         for (int j = 0; j < 8; j++) w[j / 4][j % 4] = ldexpf(w[j / 4][j % 4], up);
      }
   }
   template <int NT> __device__ inline void undo(f4 (&acc)[NT]) const
   {
      if constexpr (T == kF16)
      {
#pragma unroll
         for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[t][e] = ldexpf(acc[t][e], -up);
      }
   }
};

// scores whose bit of `mine` is clear -> `other`
__device__ inline float masked(float x, unsigned mine, int j, float other)
{
   const unsigned m = (unsigned)((int)(mine << (31 - j)) >> 31);
   return __uint_as_float((__float_as_uint(x) & m) | (__float_as_uint(other) & ~m));
}

// The score factor, times log2(e) and made positive (a negative one changes the sign of the resident queries instead, so
// that the largest product is the largest score) and not zero (a masked score of minus infinity stays one).
__device__ inline float score_factor(float scale) { return fmaxf(fabsf(scale) * kLog2e, 1.17549435e-38f); }
template <int T> __device__ inline u4 negated(u4 v)
{
   const uint32_t m = T == kF32 ? 0x80000000u : 0x80008000u;
   return u4{v[0] ^ m, v[1] ^ m, v[2] ^ m, v[3] ^ m};
}

// Running softmax of one resident row per lane.  The sums are relative to 2^(base - LIFT); base follows the largest score only
// when that runs ahead by more than 2^8, so that most tiles rescale nothing: weights are then at most 2^(8 + LIFT), and one of
// them was 2^LIFT when base was set.  LIFT is 7 where the weights become fp16: they use its range up to 2^15, and vanish below
// 2^-32 of the largest instead of 2^-25 - 2^18 slots at 2^-25 of a dominant one are 0.8 % of the row, which their sum has.
template <int NT, int LIFT> struct Softmax {
   f4 acc[NT];
   float base, sum;
   __device__ inline void clear()
   {
      base = -INFINITY;
      sum = 0;
#pragma unroll
      for (int t = 0; t < NT; t++) acc[t] = f4{0, 0, 0, 0};
   }
   // products s (masked ones -infinity) -> weights
   __device__ inline void weights(float (&w)[2][4], const f4 (&s)[2], float c2)
   {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; j++) mx = fmaxf(mx, s[j / 4][j % 4]);
      mx = group_max(mx) * c2;
      if (__any(mx > base + 8.0f))
      {
         const float to = mx > base + 8.0f ? mx : base, keep = to == base ? 1.0f : exp2_fast(base - to);
#pragma unroll
         for (int t = 0; t < NT; t++) acc[t] *= keep;
         sum *= keep;
         base = to;
      }
      const float from = base == -INFINITY ? 0.0f : base - LIFT;   // nothing named so far: every weight is exp2(-infinity)
#pragma unroll
      for (int j = 0; j < 8; j++)
      {
         w[j / 4][j % 4] = exp2_fast(fmaf(s[j / 4][j % 4], c2, -from));
         sum += w[j / 4][j % 4];   // of this lane's columns: the four groups are added at the end
      }
   }
};

// Workgroups go round-robin to the 8 XCDs.  Work item of workgroup b of n items: every XCD takes a contiguous eighth, so
// that the items of one head (whose gathered rows overlap) meet in one L2.  Items at or past n have no work.
__device__ inline int64_t xcd_item(int64_t b, int64_t n)
{
   const int64_t per = (n + 7) / 8;
   return (b & 7) * per + (b >> 3);
}

}  // namespace fmm_attn
