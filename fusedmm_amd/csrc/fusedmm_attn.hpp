// Host side of the attention family: plan object, launch units, and what the entry points check.
//
//   fusedmm_attn_exports.hip   the entry points (extern "C"), built once per (INDEXTYPE, VALUETYPE) as the others are
//   fusedmm_attn_plan.hip      the plan of a pattern, built on the GPU
//   fusedmm_attn_launch.hip    the kernels' instances, one object per (element type, kernel) (-DFMM_ATTN_UNIT=n)
//
// The kernels read 32-bit or 64-bit index arrays by a run-time flag and take the element type as an argument, so the
// plan and launch objects do not depend on INDEXTYPE or VALUETYPE: they are compiled once and linked into every library.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <vector>

#include "fusedmm_attn_kernels.h"
#include "fusedmm_attn_rows_kernels.h"
#include "fusedmm_attn_sizes.h"

namespace fmm_attn {

// status codes of include/fusedMM.h
enum : int { kOk = 0, kFail = 1, kNoMem = -1, kNoImpl = 128 };

#define ATTN_LOG(...)                                  \
   do {                                                \
      fprintf(stderr, "fusedmm_amd: " __VA_ARGS__);    \
      fprintf(stderr, "\n");                           \
   } while (0)

inline int hip_code(hipError_t e, const char *what)
{
   if (e == hipSuccess) return kOk;
   ATTN_LOG("%s failed: %s", what, hipGetErrorString(e));
   (void)hipGetLastError();
   return e == hipErrorOutOfMemory ? kNoMem : kFail;
}
#define ATTN_HIP(call)                                 \
   do {                                                \
      int st_ = ::fmm_attn::hip_code((call), #call);   \
      if (st_ != ::fmm_attn::kOk) return st_;          \
   } while (0)

constexpr uint32_t kPlanMagic = 0x504c414eu;
constexpr int64_t kMaxPlanCols = (1 << 26) - 1;   // (column, row of the block) is one 32-bit sort key
constexpr int64_t kMaxPlanRows = (int64_t)1 << 31;

struct Plan {
   uint32_t magic = kPlanMagic;
   int device = 0;
   int64_t rows = 0, cols = 0;
   int64_t tiles = 0, parts = 0;
   PlanView view{};
   void *memory = nullptr;
};

int plan_create(Plan *p, int64_t m, int64_t n, int64_t nnz, const void *indx, const void *pntrb, const void *pntre, int index_bytes,
                hipStream_t stream);
void plan_release(Plan *p);

// padded width of a map's features that the instances come in: the smallest with d <= it and dv <= maps * it
inline int width_class(int d, int dv, int maps)
{
   for (int c = 32; c <= (maps == 2 ? 128 : 256); c *= 2)
      if (d <= c && dv <= maps * c) return c;
   return 0;
}

// floats of partial sums that one split unit of one head leaves
inline int64_t forward_part(int dc, int maps, int br) { return (int64_t)maps * br * (dc * maps + 2); }
inline int64_t dq_part(int dc, int maps, int br) { return (int64_t)br * (2 * dc * maps + 6); }
inline int64_t dkv_part(int dc, int maps, int br) { return (int64_t)br * (2 * dc * maps); }

// one function per (type, kernel) object; dc and maps choose the instance
int launch_forward_f32(const Params &p, int dc, int maps, hipStream_t s);
int launch_forward_f16(const Params &p, int dc, int maps, hipStream_t s);
int launch_forward_bf16(const Params &p, int dc, int maps, hipStream_t s);
int launch_pack_f32(const PackParams &p, hipStream_t s);
int launch_pack_f16(const PackParams &p, hipStream_t s);
int launch_pack_bf16(const PackParams &p, hipStream_t s);
int launch_dq_f32(const Params &p, int dc, int maps, hipStream_t s);      // dq, and the statistics and sums that dkv reads
int launch_dq_f16(const Params &p, int dc, int maps, hipStream_t s);
int launch_dq_bf16(const Params &p, int dc, int maps, hipStream_t s);
int launch_dkv_f32(const Params &p, int dc, int maps, hipStream_t s);
int launch_dkv_f16(const Params &p, int dc, int maps, hipStream_t s);
int launch_dkv_bf16(const Params &p, int dc, int maps, hipStream_t s);
int launch_rows_f32(const RowsParams &p, int dc, int maps, hipStream_t s);
int launch_rows_f16(const RowsParams &p, int dc, int maps, hipStream_t s);
int launch_rows_bf16(const RowsParams &p, int dc, int maps, hipStream_t s);
int launch_rows_kv4(const RowsParams &p, int dc, int maps, hipStream_t s);
int launch_kv4_write(const Kv4Params &p, int type, hipStream_t s);
int launch_kv4_read(const Kv4Params &p, int type, hipStream_t s);

}  // namespace fmm_attn
