// Sizes of the attention family's launches: what the launch units ask for and what the entry points refuse beforehand, so that
// no call ends with some of its kernels enqueued.  Plain C++ (a test compiles it without a GPU).
#pragma once
#include <stdint.h>

namespace fmm_attn {

typedef __int128 Wide;   // products of sizes that each fit 64 bits

// A dispatch counts the threads of its grid in 32 bits.
constexpr bool launch_fits(Wide groups, int threads) { return groups * threads < ((Wide)1 << 32); }

constexpr Wide eighths(Wide n) { return (n + 7) / 8 * 8; }   // workgroups of n items in eighths (xcd_item)

// ---- over a plan ----
struct PlanSizes {
   int64_t units, joins, tiles;
   int block_rows;
};
constexpr int unit_threads(int block_rows) { return 4 * block_rows; }
// (a wave of the join for every 64 of a row's sums, four to a workgroup)
constexpr Wide join_groups(const PlanSizes &p, int64_t heads, int width) { return (Wide)p.joins * heads * (p.block_rows / 4) * ((width + 63) / 64); }

constexpr bool over_plan_fits(const PlanSizes &p, int64_t heads, int width, int64_t more)   // forward, dq; dk and dv
{
   return launch_fits(eighths((Wide)p.units * heads) + more, unit_threads(p.block_rows)) && launch_fits(join_groups(p, heads, width), 256);
}
constexpr bool forward_fits(const PlanSizes &p, int64_t heads, int width) { return over_plan_fits(p, heads, width, 0); }
constexpr bool backward_fits(const PlanSizes &p, const PlanSizes &t, int64_t heads, int64_t kv_heads, int width)
{
   // (dk, dv: sums of both, a workgroup per head for dlambda, and tiles times the group's heads are steps of one loop)
   return over_plan_fits(p, heads, width, 0) && over_plan_fits(t, kv_heads, 2 * width, heads) && (Wide)t.tiles * (heads / kv_heads) <= INT32_MAX;
}

// ---- packing: two tensors, per_head workgroups for each head of each ----
constexpr int64_t pack_per_head(int64_t rows, int64_t heads, int chunks)
{
   // enough workgroups to fill the GPU, each of a few chunks per thread where there is more
   const Wide want = ((Wide)rows * chunks + 255) / 256;
   const int64_t most = 16384 / (2 * heads) > 1 ? 16384 / (2 * heads) : 1;
   return want < most ? (int64_t)want : most;
}
constexpr bool pack_fits(int64_t heads) { return launch_fits((Wide)2 * heads * pack_per_head(INT64_MAX / 1024, heads, 1), 256); }

// ---- serving rows ----
constexpr Wide rows_groups(int64_t pieces, int64_t columns) { return eighths(pieces) * columns; }
// Waves of a join: 4 where they take a row in one batch of 8 pieces per worker, else 16, if the launch has room for them.  48 rows
// up to 16384 slots take 124 us with 4 waves, 133 with 16 (64 rows over a 4-bit cache 146 and 159), two rows of 65k and 262k
// slots 47 and 37, one row of 500k slots 233 and 212.
constexpr int join_waves(int64_t cap, int64_t m, int64_t heads, int width)
{
   return (Wide)cap > (Wide)8 * 4 * (256 / width) * m && launch_fits((Wide)m * heads, 1024) ? 16 : 4;
}
constexpr bool rows_fit(int64_t pieces, int64_t m, int64_t columns, int64_t heads) { return launch_fits(rows_groups(pieces, columns), 256) && launch_fits((Wide)m * heads, 256); }

// ---- making a plan: so many chunks (of up to 1024 threads each) to a launch ----
constexpr int64_t kPlanSlice = (int64_t)1 << 16;

}  // namespace fmm_attn
