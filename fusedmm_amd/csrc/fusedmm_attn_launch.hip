// Instances of the attention kernels, one object per (element type, kernel): -DFMM_ATTN_UNIT=3 * kernel + type, kernels in
// the order forward, dq, dkv, rows; unit 12 is the 4-bit cache.
#include <algorithm>

#include "fusedmm_attn.hpp"

#ifndef FMM_ATTN_UNIT
#error "compile with -DFMM_ATTN_UNIT=0..12"
#endif
#define KERNEL (FMM_ATTN_UNIT / 3)
#define TYPE (FMM_ATTN_UNIT % 3)
#if TYPE == 0
#define NAMED(f) f##_f32
#elif TYPE == 1
#define NAMED(f) f##_f16
#else
#define NAMED(f) f##_bf16
#endif

namespace fmm_attn {

namespace {

[[maybe_unused]] unsigned unit_groups(const Params &p, int heads) { return (unsigned)eighths((Wide)p.plan.n_units * heads); }
[[maybe_unused]] dim3 join_grid(const Params &p, int heads, int width) { return dim3((unsigned)join_groups({p.plan.n_units, p.plan.n_joins, 0, p.plan.block_rows}, heads, width)); }

// F<DC, MAPS>()(args) for the instance of (dc, maps)
template <template <int, int> class F, class... A> int choose(int dc, int maps, A... a)
{
   if (maps == 1)
      switch (dc)
      {
         case 32: return F<32, 1>()(a...);
         case 64: return F<64, 1>()(a...);
         case 128: return F<128, 1>()(a...);
         case 256: return F<256, 1>()(a...);
      }
   else
      switch (dc)
      {
         case 32: return F<32, 2>()(a...);
         case 64: return F<64, 2>()(a...);
         case 128: return F<128, 2>()(a...);
      }
   return kNoImpl;
}

#if KERNEL == 0
template <int DC, int MAPS> struct Forward {
   int operator()(const Params &p, hipStream_t s)
   {
      const dim3 grid(unit_groups(p, p.heads));
      if (p.plan.block_rows == 64) hipLaunchKernelGGL((attn_forward<TYPE, DC, MAPS, 64>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((attn_forward<TYPE, DC, MAPS, 16>), grid, dim3(64), 0, s, p);
      ATTN_HIP(hipGetLastError());
      if (p.plan.n_joins)
      {
         hipLaunchKernelGGL((attn_forward_join<TYPE, DC, MAPS>), join_grid(p, p.heads, DC * MAPS), dim3(256), 0, s, p);
         ATTN_HIP(hipGetLastError());
      }
      return kOk;
   }
};
#elif KERNEL == 1
template <int DC, int MAPS> struct Dq {
   int operator()(const Params &p, hipStream_t s)
   {
      const dim3 grid(unit_groups(p, p.heads));
      if (p.plan.block_rows == 64) hipLaunchKernelGGL((attn_dq<TYPE, DC, MAPS, 64>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((attn_dq<TYPE, DC, MAPS, 16>), grid, dim3(64), 0, s, p);
      ATTN_HIP(hipGetLastError());
      if (p.plan.n_joins)
      {
         hipLaunchKernelGGL((attn_dq_join<TYPE, DC, MAPS>), join_grid(p, p.heads, DC * MAPS), dim3(256), 0, s, p);
         ATTN_HIP(hipGetLastError());
      }
      return kOk;
   }
};
#elif KERNEL == 2
template <int DC, int MAPS> struct Dkv {
   int operator()(const Params &p, hipStream_t s)
   {
      const dim3 grid(unit_groups(p, p.kv_heads) + (p.dlambda ? (unsigned)p.heads : 0u));
      if (p.plan.block_rows == 64) hipLaunchKernelGGL((attn_dkv<TYPE, DC, MAPS, 64>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((attn_dkv<TYPE, DC, MAPS, 16>), grid, dim3(64), 0, s, p);
      ATTN_HIP(hipGetLastError());
      if (p.plan.n_joins)
      {
         hipLaunchKernelGGL((attn_dkv_join<TYPE, DC, MAPS>), join_grid(p, p.kv_heads, 2 * DC * MAPS), dim3(256), 0, s, p);
         ATTN_HIP(hipGetLastError());
      }
      return kOk;
   }
};
#endif

#if KERNEL >= 3
int make_table(const RowsParams &p, hipStream_t s)
{
   if (!p.cap || p.m <= kTableRows) return kOk;
   hipLaunchKernelGGL((attn_rows_table<FMM_ATTN_UNIT>), dim3(1), dim3(1024), 0, s, p);
   ATTN_HIP(hipGetLastError());
   return kOk;
}

template <int O, int DC, int MAPS> int join(const RowsParams &p, hipStream_t s)
{
   if (!p.cap) return kOk;
   const int waves = join_waves(p.cap, p.m, p.heads, DC * MAPS);
   const size_t lds = (size_t)waves * MAPS * (DC * MAPS + 2) * sizeof(float);
   hipLaunchKernelGGL((attn_rows_join<FMM_ATTN_UNIT, O, DC, MAPS>), dim3((unsigned)(p.m * p.heads)), dim3(64 * waves), lds, s, p);
   ATTN_HIP(hipGetLastError());
   return kOk;
}

unsigned rows_grid(const RowsParams &p) { return (unsigned)rows_groups(p.cap ? p.cap : p.m, p.kv_heads * p.passes); }
#endif

#if KERNEL == 3
template <int DC, int MAPS> struct Rows {
   int operator()(const RowsParams &p, hipStream_t s)
   {
      int st = make_table(p, s);
      if (st) return st;
      if (p.vec_kv && p.d == DC && p.dv == DC * MAPS) hipLaunchKernelGGL((attn_rows<TYPE, DC, MAPS, true>), dim3(rows_grid(p)), dim3(256), 0, s, p);
      else hipLaunchKernelGGL((attn_rows<TYPE, DC, MAPS, false>), dim3(rows_grid(p)), dim3(256), 0, s, p);
      ATTN_HIP(hipGetLastError());
      return join<TYPE, DC, MAPS>(p, s);
   }
};
#elif KERNEL == 4
template <int DC, int MAPS> struct Rows4 {
   int operator()(const RowsParams &p, hipStream_t s)
   {
      int st = make_table(p, s);
      if (st) return st;
      if (p.d == DC && p.dv == DC * MAPS) hipLaunchKernelGGL((attn_rows_kv4<DC, MAPS, true>), dim3(rows_grid(p)), dim3(256), 0, s, p);
      else if constexpr (DC * MAPS < 256) hipLaunchKernelGGL((attn_rows_kv4<DC, MAPS, false>), dim3(rows_grid(p)), dim3(256), 0, s, p);
      else return kNoImpl;   // refused by the entry point
      ATTN_HIP(hipGetLastError());
      return p.out_type == kF16 ? join<kF16, DC, MAPS>(p, s) : join<kBF16, DC, MAPS>(p, s);
   }
};
#endif

}  // namespace

#if KERNEL == 0
int NAMED(launch_forward)(const Params &p, int dc, int maps, hipStream_t s) { return choose<Forward>(dc, maps, p, s); }

int NAMED(launch_pack)(const PackParams &p, hipStream_t s)
{
   hipLaunchKernelGGL((attn_pack<TYPE>), dim3((unsigned)(2 * (int64_t)p.heads * p.per_head)), dim3(256), 0, s, p);
   ATTN_HIP(hipGetLastError());
   return kOk;
}
#elif KERNEL == 1
int NAMED(launch_dq)(const Params &p, int dc, int maps, hipStream_t s) { return choose<Dq>(dc, maps, p, s); }
#elif KERNEL == 2
int NAMED(launch_dkv)(const Params &p, int dc, int maps, hipStream_t s) { return choose<Dkv>(dc, maps, p, s); }
#elif KERNEL == 3
int NAMED(launch_rows)(const RowsParams &p, int dc, int maps, hipStream_t s) { return choose<Rows>(dc, maps, p, s); }
#else
int launch_rows_kv4(const RowsParams &p, int dc, int maps, hipStream_t s) { return choose<Rows4>(dc, maps, p, s); }

// Slices of tokens one behind the other: a workgroup compares its slots with all later ones of its slice, and a later slice
// overwrites what an earlier one wrote, so that the work grows with the tokens, not with their square.  8 key heads of 128 + 128
// bf16: 131072 tokens 302 us in slices of 8192, 355 of 4096, 319 of 16384, 1167 us at once; 2^20 tokens 2.4 ms.
constexpr int64_t kKv4Slice = 8192;

int launch_kv4_write(const Kv4Params &all, int type, hipStream_t s)
{
   const int64_t bytes = type == kF32 ? 4 : 2;
   for (int64_t first = 0; first < all.tokens; first += kKv4Slice)
   {
      Kv4Params p = all;
      p.tokens = std::min(kKv4Slice, all.tokens - first);
      p.slots = (const unsigned char *)all.slots + first * all.index_bytes;
      p.k = (const unsigned char *)all.k + first * all.ldk * bytes;
      p.v = (const unsigned char *)all.v + first * all.ldv * bytes;
      // Tokens of a workgroup share its walk as soon as there are enough of them: 8192 tokens in 1024 workgroups 16.3 us, in
      // 2048 20.3, in 8192 53; 2048 tokens in 1024 6.9, in 2048 9.0.
      p.per_group = (int)std::min<int64_t>(kKv4Tokens, std::max<int64_t>(1, p.tokens / 1024));
      const dim3 grid((unsigned)((p.tokens + p.per_group - 1) / p.per_group));
      if (type == kF32) hipLaunchKernelGGL((kv4_write<kF32>), grid, dim3(256), 0, s, p);
      else if (type == kF16) hipLaunchKernelGGL((kv4_write<kF16>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((kv4_write<kBF16>), grid, dim3(256), 0, s, p);
      ATTN_HIP(hipGetLastError());
   }
   return kOk;
}

int launch_kv4_read(const Kv4Params &p, int type, hipStream_t s)
{
   const int64_t words = p.tokens * p.kv_heads * ((p.k_width + p.v_width) / 8);
   const dim3 grid((unsigned)std::min<int64_t>((words + 255) / 256, 1 << 16));
   if (type == kF32) hipLaunchKernelGGL((kv4_read<kF32>), grid, dim3(256), 0, s, p);
   else if (type == kF16) hipLaunchKernelGGL((kv4_read<kF16>), grid, dim3(256), 0, s, p);
   else hipLaunchKernelGGL((kv4_read<kBF16>), grid, dim3(256), 0, s, p);
   ATTN_HIP(hipGetLastError());
   return kOk;
}
#endif

}  // namespace fmm_attn
