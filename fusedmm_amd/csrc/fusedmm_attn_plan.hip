// The plan of a pattern: for every block of 64 rows, the columns that any of them names, ascending, with one bit per row.
// Where rows have few neighbours in common - the four runs of 16 rows of a block together name less than kShare times as
// many columns as the block does - blocks of 16 rows take their place: a gathered row is then loaded once for each run, but
// multiplied only for the run that names it.
//
// The rows' lists are cut into chunks of 512 slots each (at most 32768 edges); a workgroup sorts a chunk's (column, row)
// keys in LDS and keeps one entry for each column.  Columns that are in ascending order within the rows, as loaders leave
// them, put the same stretch of columns into one chunk; any other order is as right and only shares less.  A column that a
// row names twice gets a second entry, so that it counts twice, as it does in every sum over edges.  Sorting costs
// log2(E)^2 / 2 passes over LDS, once per pattern.
#include <algorithm>

#include "fusedmm_attn.hpp"

namespace fmm_attn {

namespace {

constexpr int kMostRows = 64;
// Training over windows, so many runs per column (32k rows, 4 heads of 128 bf16 features; 32 f32 features), blocks of 64 and of
// 16 rows: 1.6 runs 117 and 105 us (91 and 73), 1.8 runs 120 and 126 us (97 and 101), 2.3 runs 134 and 147 us (119 and 131).
// A random graph of 16 neighbours has 1.
constexpr double kShare = 1.7;
constexpr int kChunkSlots = 512;
constexpr uint32_t kNoKey = 0xffffffffu;

struct Chunk {
   int32_t block, number;
   int64_t at;        // first entry in the unpacked arrays
   int32_t edges;     // of its rows' slots: an upper bound of its entries
   int32_t pad;
};

struct Piece {        // a chunk's entries, in their place in the plan
   int64_t from, to;
   int32_t count, end;   // entries at to + count .. to + end - 1 fill the unit's last tile
};

__device__ inline int64_t index_at(const void *a, int64_t i, int bytes)
{
   return bytes == 4 ? (int64_t)((const int32_t *)a)[i] : ((const int64_t *)a)[i];
}

// one wave per block: its longest row and all its edges
__global__ __launch_bounds__(256) void plan_count(int64_t m, int br, int64_t blocks, const void *pb, const void *pe, int ib, int64_t *longest, int64_t *edges, int *bad)
{
   const int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
   if (b >= blocks) return;
   const int lane = threadIdx.x & 63;
   const int64_t row = b * br + lane;
   int64_t len = 0;
   if (lane < br && row < m)
   {
      const int64_t lo = index_at(pb, row, ib), hi = index_at(pe, row, ib);
      if (lo > hi || lo < 0) *bad = 1;
      else len = hi - lo;
   }
   int64_t top = len, all = len;
   for (int k = 1; k < 64; k <<= 1)
   {
      top = max(top, (int64_t)__shfl_xor((long long)top, k));
      all += __shfl_xor((long long)all, k);
   }
   if ((threadIdx.x & 63) == 0)
   {
      longest[b] = top;
      edges[b] = all;
   }
}

__device__ inline int64_t chunk_length(int64_t len, int number)
{
   const int64_t left = len - (int64_t)number * kChunkSlots;
   return left < 0 ? 0 : left > kChunkSlots ? kChunkSlots : left;
}

// one wave per chunk: its edges
__global__ __launch_bounds__(256) void plan_chunk_edges(Chunk *chunks, int64_t n_chunks, int64_t m, int br, const void *pb, const void *pe, int ib)
{
   const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
   if (c >= n_chunks) return;
   const int lane = threadIdx.x & 63;
   const int64_t row = (int64_t)chunks[c].block * br + lane;
   int x = lane < br && row < m ? (int)chunk_length(index_at(pe, row, ib) - index_at(pb, row, ib), chunks[c].number) : 0;
   for (int k = 1; k < 64; k <<= 1) x += __shfl_xor(x, k);
   if ((threadIdx.x & 63) == 0) chunks[c].edges = x;
}

// SIZE: keys that fit; chunks of at most that many edges
template <int SIZE, int THREADS>
__global__ __launch_bounds__(THREADS) void plan_fill(const Chunk *chunks, int64_t n_chunks, int64_t m, int br, int64_t n, const void *indx, const void *pb,
                                                      const void *pe, int ib, int32_t *cols, uint64_t *masks, int2 *counts)
{
   __shared__ uint32_t key[SIZE];
   __shared__ int32_t start[kMostRows + 1];
   __shared__ int32_t runs;
   __shared__ int32_t sums[THREADS];
   const int tid = threadIdx.x;
   if ((int64_t)blockIdx.x >= n_chunks) return;
   const Chunk c = chunks[blockIdx.x];
   const bool mine = SIZE == 4096 ? c.edges <= 4096 : c.edges > 4096;
   if (!mine) return;   // the other instance's chunk
   if (tid < kMostRows)
   {
      const int64_t row = (int64_t)c.block * br + tid;
      int64_t len = 0;
      if (tid < br && row < m) len = chunk_length(index_at(pe, row, ib) - index_at(pb, row, ib), c.number);
      start[tid + 1] = (int32_t)len;
      if (tid == 0) start[0] = runs = 0;
   }
   __syncthreads();
   if (tid == 0)
      for (int r = 0; r < kMostRows; r++) start[r + 1] += start[r];
   __syncthreads();
   const int total = start[kMostRows] < SIZE ? start[kMostRows] : SIZE;
   int size = 64;
   while (size < total) size <<= 1;
   for (int e = tid; e < size; e += THREADS)
   {
      uint32_t k = kNoKey;
      if (e < total)
      {
         int r = 0;   // the row of edge e
#pragma unroll
         for (int s = 32; s; s >>= 1)
            if (start[r + s] <= e) r += s;
         const int64_t row = (int64_t)c.block * br + r;
         const int64_t col = index_at(indx, index_at(pb, row, ib) + (int64_t)c.number * kChunkSlots + (e - start[r]), ib);
         if (col >= 0 && col < n) k = ((uint32_t)col << 6) | (uint32_t)r;   // any other id names no column
      }
      key[e] = k;
   }
   __syncthreads();
   for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j; j >>= 1)
      {
         for (int t = tid; t < size / 2; t += THREADS)
         {
            const int a = 2 * t - (t & (j - 1)), b = a + j;
            const uint32_t x = key[a], y = key[b];
            if ((x > y) == ((a & k) == 0))
            {
               key[a] = y;
               key[b] = x;
            }
         }
         __syncthreads();
      }
   // an entry starts where the column changes, and at every repetition of one (column, row)
   const int per = (size + THREADS - 1) / THREADS, lo = tid * per, hi = min(lo + per, size);
   auto starts = [&](int e) {
      const uint32_t k = key[e];
      if (k == kNoKey) return false;
      return e == 0 || (key[e - 1] >> 6) != (k >> 6) || key[e - 1] == k;
   };
   int count = 0;
   for (int e = lo; e < hi; e++) count += starts(e);
   sums[tid] = count;
   __syncthreads();
   for (int s = 1; s < THREADS; s <<= 1)
   {
      const int x = tid >= s ? sums[tid - s] : 0;
      __syncthreads();
      sums[tid] += x;
      __syncthreads();
   }
   int64_t to = c.at + sums[tid] - count;
   int in_runs = 0;   // columns, counted once for every run of 16 rows that names them
   for (int e = lo; e < hi; e++)
      if (starts(e))
      {
         const uint32_t k = key[e];
         uint64_t bits = (uint64_t)1 << (k & 63);
         for (int f = e + 1; f < size && key[f] != kNoKey && !starts(f); f++) bits |= (uint64_t)1 << (key[f] & 63);
         cols[to] = (int32_t)(k >> 6);
         masks[to] = bits;
         to++;
         for (int w = 0; w < 4; w++) in_runs += ((bits >> (16 * w)) & 0xffff) != 0;
      }
   atomicAdd(&runs, in_runs);   // (whole numbers: the order does not matter)
   __syncthreads();
   if (tid == THREADS - 1) counts[blockIdx.x] = make_int2(sums[tid], runs);
}

__global__ __launch_bounds__(256) void plan_pack(const Piece *pieces, const int32_t *cols, const uint64_t *masks, int32_t *to_cols, uint64_t *to_masks)
{
   const Piece p = pieces[blockIdx.x];
   for (int e = threadIdx.x; e < p.end; e += 256)
   {
      // behind the last column: that column again, named by no row
      to_cols[p.to + e] = cols[p.from + (e < p.count ? e : p.count - 1)];
      to_masks[p.to + e] = e < p.count ? masks[p.from + e] : 0;
   }
}

// per column a bit for each row -> per row a bit for each of the tile's 32 columns, in the order in which lanes hold scores
__global__ __launch_bounds__(256) void plan_masks(const uint64_t *masks, int64_t tiles, int br, uint32_t *to)
{
   for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < tiles * br; x += (int64_t)gridDim.x * 256)
   {
      const int64_t tile = x / br;
      const int row = (int)(x % br);
      uint32_t word = 0;
      for (int c = 0; c < kTile; c++) word |= (uint32_t)((masks[tile * kTile + c] >> row) & 1) << (8 * (c % 16 / 4) + 4 * (c / 16) + c % 4);
      to[x] = word;
   }
}

struct Memory {   // freed when the building ends, however it does
   void *p = nullptr;
   ~Memory() { if (p) (void)hipFree(p); }
   int get(size_t bytes) { return hip_code(hipMalloc(&p, bytes ? bytes : 16), "hipMalloc (attention plan)"); }
};

// launch(first, count) for n items, kPlanSlice at a time
template <class F> int in_slices(int64_t n, F launch)
{
   for (int64_t first = 0; first < n; first += kPlanSlice)
   {
      launch(first, std::min(kPlanSlice, n - first));
      ATTN_HIP(hipGetLastError());
   }
   return kOk;
}

template <class X> int upload(Memory &to, const std::vector<X> &v)
{
   const int st = to.get(v.size() * sizeof(X));
   if (st) return st;
   if (!v.empty()) ATTN_HIP(hipMemcpy(to.p, v.data(), v.size() * sizeof(X), hipMemcpyHostToDevice));
   return kOk;
}

// with blocks of br rows; *shared: false where blocks of 64 rows share too little (nothing is built then)
int build(Plan *plan, int br, bool *shared, int64_t m, int64_t n, int64_t nnz, const void *indx, const void *pb, const void *pe, int ib, hipStream_t stream)
{
   *shared = true;
   ATTN_HIP(hipGetDevice(&plan->device));
   plan->rows = m;
   plan->cols = n;
   const int64_t blocks = (m + br - 1) / br;
   std::vector<int64_t> longest((size_t)blocks), edges((size_t)blocks);
   if (blocks)
   {
      Memory scratch;
      int st = scratch.get((size_t)blocks * 16 + 16);
      if (st) return st;
      int64_t *d = (int64_t *)scratch.p;
      int *bad = (int *)(d + 2 * blocks);
      ATTN_HIP(hipMemsetAsync(bad, 0, 16, stream));
      hipLaunchKernelGGL(plan_count, dim3((unsigned)((blocks + 3) / 4)), dim3(256), 0, stream, m, br, blocks, pb, pe, ib, d, d + blocks, bad);
      ATTN_HIP(hipGetLastError());
      int is_bad = 0;
      ATTN_HIP(hipMemcpyAsync(longest.data(), d, (size_t)blocks * 8, hipMemcpyDeviceToHost, stream));
      ATTN_HIP(hipMemcpyAsync(edges.data(), d + blocks, (size_t)blocks * 8, hipMemcpyDeviceToHost, stream));
      ATTN_HIP(hipMemcpyAsync(&is_bad, bad, 4, hipMemcpyDeviceToHost, stream));
      ATTN_HIP(hipStreamSynchronize(stream));
      int64_t sum = 0;
      for (int64_t b = 0; b < blocks && sum <= nnz; b++) sum += edges[b];
      if (is_bad || sum > nnz)
      {
         ATTN_LOG("attention plan: %s", is_bad ? "a row has pntre < pntrb or a negative pntrb" : "the rows have more than nnz slots");
         return kFail;
      }
   }

   // chunks, with room for every edge of theirs
   std::vector<Chunk> chunks;
   for (int64_t b = 0; b < blocks; b++)
      for (int64_t number = 0; number * kChunkSlots < longest[b]; number++)
      {
         if (chunks.size() >= (size_t)INT32_MAX)
         {
            ATTN_LOG("attention plan: too many edges");
            return kFail;
         }
         chunks.push_back(Chunk{(int32_t)b, (int32_t)number, 0, 0, 0});
      }
   int64_t at = 0;
   bool small = false, large = false;
   std::vector<int2> counts(chunks.size());
   Memory d_chunks, d_cols, d_masks, d_counts;
   if (!chunks.empty())
   {
      int st = upload(d_chunks, chunks);
      if (st) return st;
      st = in_slices((int64_t)chunks.size(), [&](int64_t first, int64_t count) {
         hipLaunchKernelGGL(plan_chunk_edges, dim3((unsigned)((count + 3) / 4)), dim3(256), 0, stream, (Chunk *)d_chunks.p + first, count, m, br, pb, pe, ib);
      });
      if (st) return st;
      ATTN_HIP(hipMemcpyAsync(chunks.data(), d_chunks.p, chunks.size() * sizeof(Chunk), hipMemcpyDeviceToHost, stream));
      ATTN_HIP(hipStreamSynchronize(stream));
      for (Chunk &c : chunks)
      {
         c.at = at;
         at += c.edges;
         (c.edges <= 4096 ? small : large) = true;
      }
      ATTN_HIP(hipMemcpy(d_chunks.p, chunks.data(), chunks.size() * sizeof(Chunk), hipMemcpyHostToDevice));
      st = d_cols.get((size_t)at * 4);
      if (!st) st = d_masks.get((size_t)at * 8);
      if (!st) st = d_counts.get(chunks.size() * sizeof(int2));
      if (st) return st;
      st = in_slices((int64_t)chunks.size(), [&](int64_t first, int64_t count) {
         const Chunk *of = (const Chunk *)d_chunks.p + first;
         int2 *to = (int2 *)d_counts.p + first;
         if (small)
            hipLaunchKernelGGL((plan_fill<4096, 256>), dim3((unsigned)count), dim3(256), 0, stream, of, count, m, br, n, indx, pb, pe, ib, (int32_t *)d_cols.p,
                               (uint64_t *)d_masks.p, to);
         if (large)
            hipLaunchKernelGGL((plan_fill<kMostRows * kChunkSlots, 1024>), dim3((unsigned)count), dim3(1024), 0, stream, of, count, m, br, n, indx, pb, pe, ib,
                               (int32_t *)d_cols.p, (uint64_t *)d_masks.p, to);
      });
      if (st) return st;
      ATTN_HIP(hipMemcpyAsync(counts.data(), d_counts.p, chunks.size() * sizeof(int2), hipMemcpyDeviceToHost, stream));
      ATTN_HIP(hipStreamSynchronize(stream));
      if (br == 64)
      {
         double columns = 0, runs = 0;
         for (const int2 &c : counts)
         {
            columns += c.x;
            runs += c.y;
         }
         *shared = runs >= kShare * columns;
         if (!*shared) return kOk;
      }
   }

   // Units.  A unit of many chunks has little to join, one of few leaves more workgroups: a chunk of full rows is 16
   // tiles, and 2048 units keep 256 compute units of two to four workgroups each busy for a few turns.  Training, causal, 64
   // bf16 features, chunks per unit 1 / 2 / 4 / 8: 512 chunks and one head 85 / 101 / 164 / 286 us, 2048 and one head 151 / 155 /
   // 208 / 304, 2048 and 8 heads 845 / 744 / 744 / 799 (a plan does not know the heads), 8192 and 2 heads 803 / 702 / 709 / 779.
   const int64_t per_unit = std::max<int64_t>(1, std::min<int64_t>(8, (int64_t)chunks.size() / 2048));
   std::vector<Unit> units;
   std::vector<Join> joins;
   std::vector<Piece> pieces;
   int64_t to = 0, parts = 0;
   size_t c = 0;
   for (int64_t b = 0; b < blocks; b++)
   {
      const size_t first = c;
      while (c < chunks.size() && chunks[c].block == b) c++;
      const int64_t n_units = std::max<int64_t>(1, ((int64_t)(c - first) + per_unit - 1) / per_unit);
      for (int64_t k = 0; k < n_units; k++)
      {
         const size_t lo = first + (size_t)(k * per_unit), hi = std::min(c, lo + (size_t)per_unit);
         const int64_t begin = to;
         for (size_t x = lo; x < hi; x++)
         {
            if (!counts[x].x) continue;
            pieces.push_back(Piece{chunks[x].at, to, counts[x].x, counts[x].x});
            to += counts[x].x;
         }
         const int64_t padded = begin + (to - begin + kTile - 1) / kTile * kTile;
         if (padded != to) pieces.back().end += (int32_t)(padded - to);
         to = padded;
         units.push_back(Unit{(int32_t)b, n_units > 1 ? (int32_t)(parts + k) : -1, (int32_t)(begin / kTile), (int32_t)((to - begin) / kTile)});
      }
      if (n_units > 1)
      {
         joins.push_back(Join{(int32_t)b, (int32_t)parts, (int32_t)n_units, 0});
         parts += n_units;
      }
   }
   if (to / kTile > INT32_MAX || units.size() > (size_t)INT32_MAX || parts > INT32_MAX)
   {
      ATTN_LOG("attention plan: too many edges");
      return kFail;
   }
   plan->tiles = to / kTile;
   plan->parts = parts;
   auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
   // (a group of column ids and masks is read ahead as a whole: room for one behind the last tile)
   const size_t off_masks = up((size_t)(to + kAhead * kTile) * 4), off_units = off_masks + up((size_t)(to / kTile + kAhead) * br * 4), off_joins = off_units + up(units.size() * sizeof(Unit));
   const size_t bytes = off_joins + up(joins.size() * sizeof(Join)) + 256;
   ATTN_HIP(hipMalloc(&plan->memory, bytes));
   unsigned char *base = (unsigned char *)plan->memory;
   if (!units.empty()) ATTN_HIP(hipMemcpy(base + off_units, units.data(), units.size() * sizeof(Unit), hipMemcpyHostToDevice));
   if (!joins.empty()) ATTN_HIP(hipMemcpy(base + off_joins, joins.data(), joins.size() * sizeof(Join), hipMemcpyHostToDevice));
   Memory d_pieces;
   if (!pieces.empty())
   {
      int st = upload(d_pieces, pieces);
      if (st) return st;
      Memory by_column;
      st = by_column.get((size_t)to * 8);
      if (st) return st;
      st = in_slices((int64_t)pieces.size(), [&](int64_t first, int64_t count) {
         hipLaunchKernelGGL(plan_pack, dim3((unsigned)count), dim3(256), 0, stream, (const Piece *)d_pieces.p + first, (const int32_t *)d_cols.p,
                            (const uint64_t *)d_masks.p, (int32_t *)base, (uint64_t *)by_column.p);
      });
      if (st) return st;
      hipLaunchKernelGGL(plan_masks, dim3((unsigned)std::min<int64_t>((to / kTile * br + 255) / 256, 1 << 16)), dim3(256), 0, stream,
                         (const uint64_t *)by_column.p, to / kTile, br, (uint32_t *)(base + off_masks));
      ATTN_HIP(hipGetLastError());
      ATTN_HIP(hipStreamSynchronize(stream));
   }
   ATTN_HIP(hipStreamSynchronize(stream));
   plan->view = PlanView{(const int32_t *)base, (const uint32_t *)(base + off_masks), (const Unit *)(base + off_units),
                         (const Join *)(base + off_joins), (int32_t)units.size(), (int32_t)joins.size(), br};
   return kOk;
}

}  // namespace

int plan_create(Plan *plan, int64_t m, int64_t n, int64_t nnz, const void *indx, const void *pb, const void *pe, int ib, hipStream_t stream)
{
   bool shared;
   const int st = build(plan, 64, &shared, m, n, nnz, indx, pb, pe, ib, stream);
   return st || shared ? st : build(plan, 16, &shared, m, n, nnz, indx, pb, pe, ib, stream);
}

void plan_release(Plan *p)
{
   if (p->memory) (void)hipFree(p->memory);
   p->memory = nullptr;
   p->magic = 0;
}

}  // namespace fmm_attn
